"""Fused SGD / Adam / AdamW optimizers (multi-tensor-apply style).

SURVEY.md §2b N8: on gfx950 the whole optimizer step for all parameters runs
as a single HIP kernel over a flat view of the parameter/grad/momentum
buffers — pure HBM bandwidth, fused with the FedProx proximal term
(N14: g += mu * (w - w_global)) so the proximal pass costs no extra memory
sweep.  CPU tensors use an equivalent torch._foreach_* implementation which
doubles as the numerics oracle for tests/test_kernels_gpu.py.

Flat-buffer layout: parameters are trained out of ONE contiguous fp32 buffer
(see parallel.flat.FlatParams), so the fused kernels take single tensors,
not tensor lists — simpler, and the same flat buffer feeds the bucketed
RCCL all-reduce aggregator with zero repacking.
"""

from __future__ import annotations

from typing import List, Optional, Sequence, Tuple, Union

import torch

from . import native_enabled, require_ext


class FlatSGD:
    """SGD(momentum, weight-decay, FedProx mu) over one flat parameter buffer.

    update: g = grad + wd * w + mu * (w - w_ref)
            m = momentum * m + g
            w = w - lr * m
    """

    def __init__(
        self,
        flat_params: torch.Tensor,
        flat_grads: torch.Tensor,
        lr: float,
        momentum: float = 0.0,
        weight_decay: float = 0.0,
        fedprox_mu: float = 0.0,
        flat_ref: Optional[torch.Tensor] = None,
    ) -> None:
        assert flat_params.shape == flat_grads.shape
        self.w = flat_params
        self.g = flat_grads
        self.lr = lr
        self.momentum = momentum
        self.weight_decay = weight_decay
        self.fedprox_mu = fedprox_mu
        self.ref = flat_ref
        self.m = (
            torch.zeros_like(flat_params) if momentum != 0.0 else None
        )

    def reset(self) -> None:
        if self.m is not None:
            self.m.zero_()

    def host_prepare(self) -> None:
        pass  # SGD's update is stateless on the host: graph-safe as-is

    @torch.no_grad()
    def device_step(self) -> None:
        mu = self.fedprox_mu
        require_ext().fused_sgd(
            self.w, self.g,
            self.m if self.m is not None
            else torch.empty(0, device=self.w.device),
            self.ref if (mu != 0.0 and self.ref is not None)
            else torch.empty(0, device=self.w.device),
            self.lr, self.momentum, self.weight_decay, mu,
        )

    @torch.no_grad()
    def step(self) -> None:
        mu = self.fedprox_mu
        if self.w.is_cuda and native_enabled():
            self.device_step()
            return
        g = self.g
        if self.weight_decay != 0.0:
            g = g.add(self.w, alpha=self.weight_decay)
        if mu != 0.0 and self.ref is not None:
            g = g.add(self.w - self.ref, alpha=mu)
        if self.m is not None:
            self.m.mul_(self.momentum).add_(g)
            g = self.m
        self.w.add_(g, alpha=-self.lr)

    def zero_grad(self) -> None:
        self.g.zero_()


class FlatAdam:
    """Adam(W) over one flat parameter buffer, with optional FedProx term."""

    def __init__(
        self,
        flat_params: torch.Tensor,
        flat_grads: torch.Tensor,
        lr: float,
        betas=(0.9, 0.999),
        eps: float = 1e-8,
        weight_decay: float = 0.0,
        fedprox_mu: float = 0.0,
        flat_ref: Optional[torch.Tensor] = None,
    ) -> None:
        self.w = flat_params
        self.g = flat_grads
        self.lr = lr
        self.beta1, self.beta2 = betas
        self.eps = eps
        self.weight_decay = weight_decay
        self.fedprox_mu = fedprox_mu
        self.ref = flat_ref
        self.m = torch.zeros_like(flat_params)
        self.v = torch.zeros_like(flat_params)
        self.t = 0
        # live bias-correction buffer: under hipGraph replay the kernel's
        # scalar args are frozen, so [bc1, bc2] travels through device
        # memory, refreshed by host_prepare() before each step/replay.
        self._bc = (
            torch.ones(2, device=flat_params.device)
            if flat_params.is_cuda else None
        )

    def reset(self) -> None:
        self.m.zero_()
        self.v.zero_()
        self.t = 0

    def host_prepare(self) -> None:
        """Host-side half of step(): advance t, refresh the device bc
        buffer.  Must run OUTSIDE any graph capture/replay."""
        self.t += 1
        if self._bc is not None:
            bc = torch.tensor(
                [1.0 - self.beta1 ** self.t, 1.0 - self.beta2 ** self.t],
                dtype=torch.float32,
            )
            self._bc.copy_(bc, non_blocking=True)

    @torch.no_grad()
    def device_step(self) -> None:
        """Device-side half (graph-capturable)."""
        mu = self.fedprox_mu
        require_ext().fused_adam(
            self.w, self.g, self.m, self.v,
            self.ref if (mu != 0.0 and self.ref is not None)
            else torch.empty(0, device=self.w.device),
            self._bc,
            self.lr, self.beta1, self.beta2, self.eps,
            self.weight_decay, mu, 1.0, 1.0,
        )

    @torch.no_grad()
    def step(self) -> None:
        if self.w.is_cuda and native_enabled():
            self.host_prepare()
            self.device_step()
            return
        self.t += 1
        bc1 = 1.0 - self.beta1 ** self.t
        bc2 = 1.0 - self.beta2 ** self.t
        mu = self.fedprox_mu
        g = self.g
        if self.weight_decay != 0.0:
            g = g.add(self.w, alpha=self.weight_decay)
        if mu != 0.0 and self.ref is not None:
            g = g.add(self.w - self.ref, alpha=mu)
        self.m.mul_(self.beta1).add_(g, alpha=1 - self.beta1)
        self.v.mul_(self.beta2).addcmul_(g, g, value=1 - self.beta2)
        denom = (self.v / bc2).sqrt_().add_(self.eps)
        self.w.addcdiv_(self.m, denom, value=-self.lr / bc1)

    def zero_grad(self) -> None:
        self.g.zero_()


STATE_BLOCK = 256   # elements of a tensor that share one 8-bit scale
_E4M3_MAX = 448.0
_E4M3_MIN = 2.0 ** -9
_TINY = 1e-30


def adamw_state(
    params: Sequence[torch.Tensor], state_bits: int = 32,
) -> Tuple[List[torch.Tensor], List[torch.Tensor],
           Optional[List[torch.Tensor]], Optional[List[torch.Tensor]]]:
    """Zero states for ``adamw_step``: (exp_avg, exp_avg_sq, their scales).

    32 bits: float32 moments, no scales.  8 bits: float8_e4m3fn codes, one
    float32 scale a block of 256 elements of a tensor; ``code * scale`` is the
    first moment and the ROOT of the second."""
    if state_bits not in (8, 32):
        raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
    if state_bits == 32:
        m, v = ([torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                 for p in params] for _ in range(2))
        return m, v, None, None
    m, v = ([torch.zeros(p.shape, dtype=torch.uint8, device=p.device)
             .view(torch.float8_e4m3fn) for p in params] for _ in range(2))
    ms, vs = ([torch.zeros(-(-p.numel() // STATE_BLOCK), dtype=torch.float32,
                           device=p.device) for p in params]
              for _ in range(2))
    return m, v, ms, vs


def _sqrt(x: torch.Tensor) -> torch.Tensor:
    """To nearest, as the kernel's; torch's fp32 root on the CPU is not."""
    return torch.sqrt(x.double()).float()


def _blocks(x: torch.Tensor) -> torch.Tensor:
    return torch.nn.functional.pad(
        x, (0, -x.numel() % STATE_BLOCK)).view(-1, STATE_BLOCK)


def _dequantise(code: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    x = _blocks(code.reshape(-1).float()) * scale[:, None]
    return x.view(-1)[: code.numel()]


def _quantise_(x: torch.Tensor, code: torch.Tensor, scale: torch.Tensor,
               positive: bool) -> None:
    blocks = _blocks(x)
    top = blocks.abs().nan_to_num(nan=0.0, posinf=float("inf")).amax(dim=1)
    live = top > _TINY
    # products with reciprocals, as the kernel's: a division by a number is one
    # on the GPU, and none on the CPU
    inv = top.reciprocal() * _E4M3_MAX
    u = blocks * torch.where(live, inv, 0.0)[:, None]
    if positive:
        u = torch.where(u > 0, u.clamp_min(_E4M3_MIN), u)
    scale.copy_(torch.where(live, top * (1.0 / _E4M3_MAX), 0.0))
    code.view(-1).copy_(u.view(-1)[: x.numel()].to(code.dtype))


@torch.no_grad()
def adamw_step(
    params: Sequence[torch.Tensor], grads: Sequence[Optional[torch.Tensor]],
    exp_avg: Sequence[torch.Tensor], exp_avg_sq: Sequence[torch.Tensor], *,
    exp_avg_scales: Optional[Sequence[torch.Tensor]] = None,
    exp_avg_sq_scales: Optional[Sequence[torch.Tensor]] = None,
    step: int, lr: float, betas: Tuple[float, float] = (0.9, 0.999),
    eps: float = 1e-8, weight_decay: Union[float, Sequence[float]] = 0.01,
    fedprox_mu: float = 0.0, refs: Optional[Sequence[torch.Tensor]] = None,
    live: Optional[torch.Tensor] = None,
) -> None:
    """One AdamW step of every tensor, in place (csrc/adamw.hip).

        g = grad + mu * (w - ref)                 (FedProx, with ``refs``)
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        w = (1 - lr * wd) * w - lr / bc1 * m / (sqrt(v / bc2) + eps)

    ``step`` counts from 1 (``bc = 1 - beta ** step``).  ``weight_decay``: one
    value, or one a tensor.  States are ``adamw_state``'s; with scales they are
    held in 8 bits, and the step uses the moments before they are rounded.  A
    non-finite gradient makes its whole 256-element block of 8-bit states
    non-finite, an infinite one, or its own entry, a NaN.  Tensors whose
    gradient is None are left out.

    Parameters are all float32 or all bfloat16 (rounded to nearest), and so
    are gradients; gradients, moments and references have their parameter's
    shape; everything is contiguous and on one device, and no tensor
    that is written may overlap another operand.  ``live``: float32 ``[lr / bc1,
    1 / bc2]`` on the device, read by the kernel in place of what ``step`` and
    ``lr`` give (a captured graph's arguments are frozen).
    """
    b1, b2 = betas
    if step < 1 and live is None:
        raise ValueError(f"step counts from 1, got {step}")
    # eps is added in float32: one below its smallest value would be lost, and
    # a weight without gradients divided by zero
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and eps >= 2.0 ** -149):
        raise ValueError(f"betas must be in [0, 1) and eps positive in "
                         f"float32, got {betas}, {eps}")
    if (exp_avg_scales is None) != (exp_avg_sq_scales is None):
        raise ValueError("scales of both moments, or of none")
    if (refs is None) != (fedprox_mu == 0.0):
        raise ValueError("fedprox_mu and refs go together")
    count = len(params)
    wd = ([float(weight_decay)] * count
          if isinstance(weight_decay, (int, float)) else list(weight_decay))
    lists = [list(params), list(grads), list(exp_avg), list(exp_avg_sq),
             None if exp_avg_scales is None else list(exp_avg_scales),
             None if exp_avg_sq_scales is None else list(exp_avg_sq_scales),
             None if refs is None else list(refs), wd]
    if any(x is not None and len(x) != count for x in lists):
        raise ValueError("every list must have one entry a parameter")
    if any(g is None for g in lists[1]):
        keep = [i for i, g in enumerate(lists[1]) if g is not None]
        lists = [x if x is None else [x[i] for i in keep] for x in lists]
    ps, gs, ms, vs, msc, vsc, rs, wd = lists
    if not ps:
        return
    bc1, bc2 = 1.0 - b1 ** max(step, 1), 1.0 - b2 ** max(step, 1)
    scale = [1.0 - lr * x for x in wd]
    if ps[0].is_cuda and native_enabled():
        require_ext().adamw_step(
            ps, gs, ms, vs, msc or [], vsc or [], rs or [], scale, b1, b2,
            eps, fedprox_mu, lr / bc1, 1.0 / bc2, live)
        return
    up, inv_bc2 = lr / bc1, 1.0 / bc2
    if live is not None:
        up, inv_bc2 = live.unbind()  # not read by the host: may be captured
    if any(t.dtype not in (torch.float32, torch.bfloat16) for t in ps + gs):
        raise TypeError("parameters and gradients must be float32 or "
                        "bfloat16")
    for ts in (gs, ms, vs, rs or ps):
        for p, t in zip(ps, ts):
            if t.shape != p.shape:
                raise ValueError(f"{tuple(t.shape)} beside a parameter "
                                 f"{tuple(p.shape)}")
    for i, (p, g) in enumerate(zip(ps, gs)):
        w, gw = p.float().reshape(-1), g.float().reshape(-1)
        if rs is not None:
            gw = gw + (w - rs[i].reshape(-1)) * fedprox_mu
        if msc is None:
            m, v = ms[i].reshape(-1), vs[i].reshape(-1)
        else:
            m = _dequantise(ms[i], msc[i])
            v = _dequantise(vs[i], vsc[i])
            v = v * v
        # every operation rounded by itself, as the kernel does
        m = m * b1 + gw * (1 - b1)
        v = v * b2 + (gw * gw) * (1 - b2)
        w = w * scale[i] - (m / (_sqrt(v * inv_bc2) + eps)) * up
        p.copy_(w.view(p.shape))
        if msc is None:
            ms[i].copy_(m.view(p.shape))
            vs[i].copy_(v.view(p.shape))
        else:
            _quantise_(m, ms[i], msc[i], False)
            _quantise_(_sqrt(v), vs[i], vsc[i], True)


class FlatAdamW:
    """AdamW over flat parameter and gradient buffers that hold many tensors.

    ``segments``: (elements, decays) of each tensor in the buffers' order;
    those that do not decay (biases, norms) are stepped without weight decay,
    and 8-bit blocks never straddle two tensors.  Without it the buffer is one
    tensor that decays.  ``state_bits`` 8 holds the moments in 2 bytes a
    parameter instead of 8.
    """

    def __init__(
        self,
        flat_params: torch.Tensor,
        flat_grads: torch.Tensor,
        lr: float,
        betas=(0.9, 0.999),
        eps: float = 1e-8,
        weight_decay: float = 0.01,
        fedprox_mu: float = 0.0,
        flat_ref: Optional[torch.Tensor] = None,
        state_bits: int = 32,
        segments: Optional[Sequence[Tuple[int, bool]]] = None,
    ) -> None:
        n = flat_params.numel()
        if segments is None:
            segments = [(n, True)]
        if sum(k for k, _ in segments) != n or flat_grads.numel() != n:
            raise ValueError(
                f"segments of {sum(k for k, _ in segments)} elements and "
                f"gradients of {flat_grads.numel()} for {n} parameters")
        if state_bits == 32:  # nothing but the decay tells tensors apart
            joined: List[Tuple[int, bool]] = []
            for k, decays in segments:
                if joined and joined[-1][1] == decays:
                    joined[-1] = (joined[-1][0] + k, decays)
                else:
                    joined.append((k, decays))
            segments = joined
        sizes = [k for k, _ in segments]
        self.w = flat_params
        self.g = flat_grads
        self.lr = lr
        self.beta1, self.beta2 = betas
        self.eps = eps
        self.weight_decay = [weight_decay if d else 0.0 for _, d in segments]
        self.fedprox_mu = fedprox_mu
        self._p = list(flat_params.split(sizes))
        self._g = list(flat_grads.split(sizes))
        self.m, self.v, self.ms, self.vs = adamw_state(self._p, state_bits)
        self._ref = None
        if fedprox_mu != 0.0 and flat_ref is not None:
            if flat_ref.numel() != n:
                raise ValueError(f"a reference of {flat_ref.numel()} elements "
                                 f"for {n} parameters")
            self._ref = list(flat_ref.split(sizes))
        self.t = 0
        # what a graph replay reads in place of its frozen arguments
        self._live = (torch.ones(2, device=flat_params.device)
                      if flat_params.is_cuda else None)

    def reset(self) -> None:
        for ts in (self.m, self.v, self.ms, self.vs):
            for t in ts or ():
                (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn
                 else t).zero_()
        self.t = 0

    def _update(self, live) -> None:
        adamw_step(
            self._p, self._g, self.m, self.v, exp_avg_scales=self.ms,
            exp_avg_sq_scales=self.vs, step=self.t, lr=self.lr,
            betas=(self.beta1, self.beta2), eps=self.eps,
            weight_decay=self.weight_decay,
            fedprox_mu=self.fedprox_mu if self._ref is not None else 0.0,
            refs=self._ref, live=live,
        )

    def host_prepare(self) -> None:
        """Host-side half of step(): advance t, refresh the live scalars.
        Must run OUTSIDE any graph capture/replay."""
        self.t += 1
        if self._live is not None:
            # fills, whose values travel in their launches: no host memory has
            # to outlive this call
            self._live[0].fill_(self.lr / (1.0 - self.beta1 ** self.t))
            self._live[1].fill_(1.0 / (1.0 - self.beta2 ** self.t))

    @torch.no_grad()
    def device_step(self) -> None:
        """Device-side half (graph-capturable)."""
        self._update(self._live)

    @torch.no_grad()
    def step(self) -> None:
        self.t += 1
        self._update(None)

    def zero_grad(self) -> None:
        self.g.zero_()


def make_flat_optimizer(kind: str, flat_params, flat_grads, train_cfg,
                        flat_ref=None, segments=None):
    """``segments``: (elements, decays) of each tensor of the buffers, for
    the optimizers that tell them apart."""
    if kind == "sgd":
        return FlatSGD(
            flat_params, flat_grads, lr=train_cfg.lr,
            momentum=train_cfg.momentum,
            weight_decay=train_cfg.weight_decay,
            fedprox_mu=train_cfg.fedprox_mu, flat_ref=flat_ref,
        )
    if kind == "adam":
        return FlatAdam(
            flat_params, flat_grads, lr=train_cfg.lr,
            weight_decay=train_cfg.weight_decay,
            fedprox_mu=train_cfg.fedprox_mu, flat_ref=flat_ref,
        )
    if kind in ("adamw", "adamw8"):
        return FlatAdamW(
            flat_params, flat_grads, lr=train_cfg.lr,
            weight_decay=train_cfg.weight_decay,
            fedprox_mu=train_cfg.fedprox_mu, flat_ref=flat_ref,
            state_bits=8 if kind == "adamw8" else 32, segments=segments,
        )
    raise ValueError(f"unknown optimizer {kind!r}")
