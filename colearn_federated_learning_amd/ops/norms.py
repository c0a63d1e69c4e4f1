"""BatchNorm2d and LayerNorm with fused HIP kernels on the GPU path.

SURVEY.md §2b N6 (BatchNorm, ResNet path) and N7 (LayerNorm, BERT path).
Both are memory-bound: the HIP kernels (csrc/norms.hip) do one fused sweep
per pass with vectorized bf16 loads (G13) and wave-level reductions; stats
accumulate in fp32.  CPU path = stock PyTorch math (oracle).

Autocast note: like PyTorch's own norms, statistics are computed in fp32;
inputs may be bf16, parameters stay fp32.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn

from . import is_vmapped, native_enabled, require_ext


def _native(x: torch.Tensor) -> bool:
    return (x.is_cuda and native_enabled() and not is_vmapped(x)
            and x.dtype == torch.bfloat16)


class _BatchNormFn(torch.autograd.Function):
    """BatchNorm with optional fused residual-add + ReLU (the ResNet block
    epilogue runs inside the BN sweeps on gfx950 — see csrc/norms.hip)."""

    generate_vmap_rule = True

    @staticmethod
    def forward(x, weight, bias, running_mean, running_var, residual,
                training: bool, momentum: float, eps: float, relu: bool,
                groups: int = 1, gslot_w=None, gslot_b=None):
        # gslot_w/gslot_b: flat-grad views; when set, the backward writes
        # the param grads straight into them and returns None for w/b, so
        # no AccumulateGrad add kernels run (stacked engine fast path).
        if _native(x):
            m = require_ext()
            y, save_mean, save_invstd = m.batchnorm_fwd(
                x, weight, bias, running_mean, running_var,
                residual if residual is not None
                else torch.empty(0, device=x.device, dtype=x.dtype),
                training, momentum, eps, relu, groups,
            )
            return y, save_mean, save_invstd
        assert groups == 1, "stacked BN has no CPU fast path here"

        if training:
            dims = (0, 2, 3)
            xf = x.float()
            mean = xf.mean(dim=dims)
            var = xf.var(dim=dims, unbiased=False)
            n = x.numel() / x.shape[1]
            with torch.no_grad():
                running_mean.mul_(1 - momentum).add_(mean, alpha=momentum)
                running_var.mul_(1 - momentum).add_(
                    var * n / max(n - 1, 1), alpha=momentum
                )
            invstd = (var + eps).rsqrt()
        else:
            # clone: an input returned as an output may not be saved for
            # backward under the setup_context protocol
            mean = running_mean.clone()
            invstd = (running_var + eps).rsqrt()
            xf = x.float()
        y = (xf - mean[None, :, None, None]) * invstd[None, :, None, None] \
            * weight[None, :, None, None] + bias[None, :, None, None]
        if residual is not None:
            y = y + residual.float()
        if relu:
            y = y.relu()
        return y.to(x.dtype), mean, invstd

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, weight = inputs[0], inputs[1]
        y, save_mean, save_invstd = output
        ctx.save_for_backward(x, weight, save_mean, save_invstd, y)
        ctx.training = inputs[6]
        ctx.relu = inputs[9]
        ctx.groups = inputs[10] if len(inputs) > 10 else 1
        ctx.gslot_w = inputs[11] if len(inputs) > 11 else None
        ctx.gslot_b = inputs[12] if len(inputs) > 12 else None
        ctx.n_inputs = len(inputs)
        ctx.has_res = inputs[5] is not None
        ctx.mark_non_differentiable(output[1], output[2])
        # without this the engine materializes ZERO tensors for the two
        # non-differentiable outputs' grads — 2 fills per BN per step
        # (40/step on ResNet-18, measured: the FillFunctor tail)
        ctx.set_materialize_grads(False)

    @staticmethod
    def backward(ctx, gy, _gmean, _ginvstd):
        x, weight, mean, invstd, y = ctx.saved_tensors
        direct = ctx.gslot_w is not None and _native(x)
        if _native(x):
            e = torch.empty(0, device=x.device, dtype=torch.float32)
            gx, gw, gb, gres = require_ext().batchnorm_bwd(
                gy, y, x, weight, mean, invstd, ctx.training, ctx.relu,
                ctx.groups,
                ctx.gslot_w if direct else e,
                ctx.gslot_b if direct else e,
            )
        else:
            gyf = gy.float()
            if ctx.relu:
                gyf = gyf * (y > 0).float()
            gres = gyf.to(x.dtype)
            xf = x.float()
            xhat = (xf - mean[None, :, None, None]) * invstd[None, :, None, None]
            n = x.numel() / x.shape[1]
            gb = gyf.sum(dim=(0, 2, 3))
            gw = (gyf * xhat).sum(dim=(0, 2, 3))
            if ctx.training:
                gx = (weight * invstd)[None, :, None, None] * (
                    gyf - gb[None, :, None, None] / n
                    - xhat * gw[None, :, None, None] / n
                )
            else:
                gx = (weight * invstd)[None, :, None, None] * gyf
            gx = gx.to(x.dtype)
        out = [gx, None if direct else gw, None if direct else gb,
               None, None, gres if ctx.has_res else None,
               None, None, None, None, None, None, None]
        return tuple(out[: ctx.n_inputs])


class ColearnBatchNorm2d(nn.Module):
    """BatchNorm2d with an optional fused ``+ residual`` / ReLU epilogue."""

    def __init__(self, num_features: int, eps: float = 1e-5,
                 momentum: float = 0.1, relu: bool = False) -> None:
        super().__init__()
        self.num_features = num_features
        self.eps = eps
        self.momentum = momentum
        self.relu = relu
        self.weight = nn.Parameter(torch.ones(num_features))
        self.bias = nn.Parameter(torch.zeros(num_features))
        self.register_buffer("running_mean", torch.zeros(num_features))
        self.register_buffer("running_var", torch.ones(num_features))
        self.register_buffer("num_batches_tracked",
                             torch.tensor(0, dtype=torch.long))

    def forward(self, x: torch.Tensor, residual=None) -> torch.Tensor:
        # num_batches_tracked is kept for state-dict compatibility but NOT
        # incremented: torch only consults it when momentum is None (ours
        # is fixed), and the on-device `+= 1` cost one extra launch per BN
        # layer per captured step (20/step on ResNet-18 — measured in
        # profiles/final_resnet18_kernel_stats.txt as the 1980-launch
        # CUDAFunctorOnSelf_add<long> row).
        y, _, _ = _BatchNormFn.apply(
            x, self.weight, self.bias, self.running_mean, self.running_var,
            residual, self.training, self.momentum, self.eps, self.relu, 1,
        )
        return y


class _LayerNormFn(torch.autograd.Function):
    """LayerNorm over the last dim; ``groups`` > 1 = stacked-client LN
    (weight/bias [G, H], client-major rows — the BERT stacking path)."""

    generate_vmap_rule = True

    @staticmethod
    def forward(x, weight, bias, eps: float, groups: int = 1,
                gslot_w=None, gslot_b=None):
        if _native(x):
            y, mean, invstd = require_ext().layernorm_fwd(
                x.contiguous(), weight.view(-1), bias.view(-1), eps,
                groups,
            )
            return y, mean, invstd
        if groups > 1:
            # CPU oracle: per-client loop
            G = groups
            rows = x.numel() // x.shape[-1]
            x3 = x.reshape(G, rows // G, x.shape[-1])
            w2, b2 = weight.view(G, -1), bias.view(G, -1)
            xf = x3.float()
            mean = xf.mean(dim=-1)
            var = xf.var(dim=-1, unbiased=False)
            invstd = (var + eps).rsqrt()
            y = ((xf - mean[..., None]) * invstd[..., None]
                 * w2[:, None, :] + b2[:, None, :])
            return (y.to(x.dtype).reshape(x.shape),
                    mean.reshape(x.shape[:-1]),
                    invstd.reshape(x.shape[:-1]))
        xf = x.float()
        mean = xf.mean(dim=-1)
        var = xf.var(dim=-1, unbiased=False)
        invstd = (var + eps).rsqrt()
        y = ((xf - mean[..., None]) * invstd[..., None] * weight
             + bias).to(x.dtype)
        return y, mean, invstd

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, weight = inputs[0], inputs[1]
        _, mean, invstd = output
        ctx.save_for_backward(x, weight, mean, invstd)
        ctx.groups = inputs[4] if len(inputs) > 4 else 1
        ctx.gslot_w = inputs[5] if len(inputs) > 5 else None
        ctx.gslot_b = inputs[6] if len(inputs) > 6 else None
        ctx.n_inputs = len(inputs)
        ctx.mark_non_differentiable(output[1], output[2])
        ctx.set_materialize_grads(False)  # see _BatchNormFn

    @staticmethod
    def backward(ctx, gy, _gmean, _ginvstd):
        x, weight, mean, invstd = ctx.saved_tensors
        G = ctx.groups
        gy = gy.contiguous()
        if _native(x) and ctx.gslot_w is not None:
            # direct-slot path: gw/gb land straight in the flat-grad
            # views (no clones, no AccumulateGrad adds)
            gx = require_ext().layernorm_bwd_slots(
                gy, x.contiguous(), weight.view(-1), mean, invstd, G,
                ctx.gslot_w.view(-1), ctx.gslot_b.view(-1),
            )
            gw = gb = None
        elif _native(x):
            gx, gw, gb = require_ext().layernorm_bwd(
                gy, x.contiguous(), weight.view(-1), mean, invstd, G
            )
            # weight.shape covers both plain [H] and stacked [G, H] —
            # including the G==1 stack ([1, H]), whose grad must keep the
            # leading slot dim (8-rank runs stack ONE client per rank)
            gw = gw.view(weight.shape)
            gb = gb.view(weight.shape)
        elif G > 1:
            h = x.shape[-1]
            rows = x.numel() // h
            x3 = x.reshape(G, rows // G, h).float()
            gy3 = gy.reshape(G, rows // G, h).float()
            m3 = mean.reshape(G, rows // G)
            i3 = invstd.reshape(G, rows // G)
            w2 = weight.view(G, h)
            xhat = (x3 - m3[..., None]) * i3[..., None]
            gw = (gy3 * xhat).sum(dim=1).view(weight.shape)
            gb = gy3.sum(dim=1).view(weight.shape)
            wg = gy3 * w2[:, None, :]
            gx = (i3[..., None] * (
                wg - wg.mean(dim=-1, keepdim=True)
                - xhat * (wg * xhat).mean(dim=-1, keepdim=True)
            )).to(x.dtype).reshape(x.shape)
        else:
            xf, gyf = x.float(), gy.float()
            xhat = (xf - mean[..., None]) * invstd[..., None]
            h = x.shape[-1]
            gw = (gyf * xhat).reshape(-1, h).sum(dim=0).view(weight.shape)
            gb = gyf.reshape(-1, h).sum(dim=0).view(weight.shape)
            wg = gyf * weight
            gx = invstd[..., None] * (
                wg - wg.mean(dim=-1, keepdim=True)
                - xhat * (wg * xhat).mean(dim=-1, keepdim=True)
            )
            gx = gx.to(x.dtype)
        out = [gx, gw, gb, None, None, None, None]
        return tuple(out[: ctx.n_inputs])


class ColearnLayerNorm(nn.Module):
    def __init__(self, hidden: int, eps: float = 1e-12) -> None:
        super().__init__()
        self.weight = nn.Parameter(torch.ones(hidden))
        self.bias = nn.Parameter(torch.zeros(hidden))
        self.eps = eps

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        y, _, _ = _LayerNormFn.apply(x, self.weight, self.bias, self.eps)
        return y


def _add_layer_norm_ref(x, residual, weight, bias, eps, groups):
    """The same formulas in torch (differentiable): CPU tensors, float64,
    functorch transforms; the kernel's oracle."""
    wide = torch.promote_types(x.dtype, torch.float32)
    # gradients of both outputs meet in the wide sum and are rounded once;
    # what is normalised has the rounded sum's value
    t = x.to(wide)
    if residual is not None:
        t = t + residual.to(wide)
    s = t.to(x.dtype)
    h = (t + (s.to(wide) - t).detach()).reshape(groups, -1, x.shape[-1])
    mean = h.mean(dim=-1, keepdim=True)
    c = h - mean
    inv = (c.square().mean(dim=-1, keepdim=True) + eps).rsqrt()
    y = (c * inv * weight.reshape(groups, 1, -1)
         + bias.reshape(groups, 1, -1))
    return y.to(x.dtype).reshape(x.shape), s


def colearn_add_layer_norm(
    x: torch.Tensor, residual: Optional[torch.Tensor],
    weight: torch.Tensor, bias: torch.Tensor, eps: float = 1e-12,
    groups: int = 1, gslot_w: Optional[torch.Tensor] = None,
    gslot_b: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(LayerNorm(s), s)`` with ``s = x + residual`` (``x`` itself without a
    residual), over the last dimension: the join of a transformer block and
    its norm in one pass.  ``s`` has x's type, and what is normalised is the
    rounded ``s``; both outputs take gradients.

    ``groups`` > 1: stacked clients, rows client-major, ``weight`` and ``bias``
    [groups, H].  ``gslot_w`` / ``gslot_b`` (both or none, float32, weight's
    size, contiguous, apart from each other and from the parameters): the
    backward writes the parameters' gradients there (overwriting them) and
    returns none, as the stacked engine's norms do.

    float32, bfloat16 and float16 on the GPU, rows up to 16384, run the HIP
    kernels (csrc/add_norm.hip; up to 2^26 rows of 1024, 2^24 of 4096, 2^22 of
    more elements); the parameters are float32.  Other operands
    run the same formulas in torch (without gslots).  A residual of another
    type is joined in the wider of the two.
    """
    h = x.shape[-1] if x.dim() else 0
    if h < 1 or weight.numel() != groups * h or bias.numel() != groups * h:
        raise ValueError(
            f"weight and bias must have {groups} x {h} elements, got "
            f"{tuple(weight.shape)} and {tuple(bias.shape)}")
    if groups < 1 or (x.numel() // h) % groups:
        raise ValueError(f"{x.numel() // h} rows do not divide into {groups} "
                         f"groups")
    if not x.is_floating_point():
        raise TypeError(f"x must be floating, got {x.dtype}")
    if (gslot_w is None) != (gslot_b is None):
        raise ValueError("gslot_w and gslot_b go together")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"the residual's shape {tuple(residual.shape)} "
                             f"is not x's {tuple(x.shape)}")
        if residual.dtype != x.dtype:
            dt = torch.promote_types(x.dtype, residual.dtype)
            x, residual = x.to(dt), residual.to(dt)
    for t in (residual, weight, bias):
        if t is not None and t.device != x.device:
            raise ValueError(f"operands on {x.device} and {t.device}")
    native = (x.is_cuda and native_enabled() and not is_vmapped(x, weight)
              and x.dtype in (torch.float32, torch.bfloat16, torch.float16)
              and h <= 16384)
    if not native:
        if gslot_w is not None:
            raise ValueError("gslots need the native kernel")
        return _add_layer_norm_ref(x, residual, weight, bias, eps, groups)
    if weight.dtype != torch.float32 or bias.dtype != torch.float32:
        raise TypeError("weight and bias must be float32")
    return require_ext().add_layer_norm(
        x.contiguous(),
        None if residual is None else residual.contiguous(),
        weight.contiguous(), bias.contiguous(), eps, groups, gslot_w,
        gslot_b)
