"""Multi-head self-attention.

``colearn_attention`` / ``colearn_attention_qkv``: any length, with document
masks and padding, causal and prefix masks, capped scores, linear distance
biases and shared key heads (csrc/masked_attn.h, masked_attn_fwd.hip,
masked_attn_bwd.hip).

``fused_attention``: unmasked, with dropout (BERT shapes: seq 128, dh = 64).

One forward + two backward HIP launches per (batch of heads) replace the
~12-kernel torch chain per attention layer (score bmm, scale, fp32
softmax, dropout, context bmm, reshape copies — fwd and bwd).  Dropout
is philox-keyed on (seed, head-block, element): deterministic,
layout-independent, and regenerated in the backward (csrc/attn.hip).
"""

from __future__ import annotations

from typing import Optional

import torch

from . import is_vmapped, native_enabled, require_ext


class _FusedAttnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, heads, scale, p, seed):
        out, P, mask = require_ext().attn_fwd(qkv, heads, scale, p, seed)
        ctx.save_for_backward(qkv, P, mask)
        ctx.args = (heads, scale, p, seed)
        return out

    @staticmethod
    def backward(ctx, dctx):
        qkv, P, mask = ctx.saved_tensors
        heads, scale, p, seed = ctx.args
        dqkv = require_ext().attn_bwd(dctx.contiguous(), qkv, P, mask,
                                      heads, scale, p, seed)
        return dqkv, None, None, None, None


def fused_attention_applicable(qkv: torch.Tensor) -> bool:
    """qkv [N, S, 3, H, dh]: native path needs bf16 CUDA, dh 64 and
    S == 128 exactly — the kernel's fragment layout is specialized to
    the BERT-base MLM config (8 key-fragments per wave); other shapes
    fall back to the batched-GEMM composition."""
    return (qkv.is_cuda and native_enabled()
            and qkv.dtype == torch.bfloat16 and qkv.shape[-1] == 64
            and qkv.shape[1] == 128)


def fused_attention(qkv: torch.Tensor, heads: int, scale: float,
                    p: float, seed: int) -> torch.Tensor:
    """Returns ctx [N, S, H*dh]."""
    return _FusedAttnFn.apply(qkv.contiguous(), heads, scale, p, seed)


# ---------------------------------------------------------------------------
# masked attention
# ---------------------------------------------------------------------------
def _masked_attention_ref(q, k, v, scale, causal, softcap, prefix, doc,
                          slopes):
    """The same formulas in torch (differentiable): CPU tensors, float32 and
    float64 operands, functorch transforms; the kernels' oracle."""
    wide = torch.promote_types(q.dtype, torch.float32)
    s, h, hkv = q.shape[1], q.shape[2], k.shape[2]
    qw, kw, vw = (t.to(wide).transpose(1, 2) for t in (q, k, v))
    real = None
    if doc is not None:  # whatever a padded token holds reaches no result
        real = (doc >= 0)[:, None, :, None]
        qw, kw, vw = (torch.where(real, t, 0.0) for t in (qw, kw, vw))
    if hkv != h:
        kw = kw.repeat_interleave(h // hkv, dim=1)
        vw = vw.repeat_interleave(h // hkv, dim=1)
    z = qw @ kw.transpose(-1, -2) * scale
    if softcap:
        z = torch.tanh(z / softcap) * softcap
    i = torch.arange(s, device=q.device)
    if slopes is not None:
        z = z - slopes.to(wide)[:, None, None] * (
            i[:, None] - i[None, :]).abs().to(wide)
    ok = None
    if causal:
        ok = (i[None, :] <= i[:, None])[None]
        if prefix is not None:
            ok = ok | (i[None, None, :] < prefix[:, None, None])
    if doc is not None:
        same = (doc[:, :, None] == doc[:, None, :]) & (doc >= 0)[:, :, None]
        ok = same if ok is None else ok & same
    if ok is not None:
        # the lowest finite value: a row without any pair stays free of NaN
        # (and its probabilities are cleared below)
        z = z.masked_fill(~ok[:, None], torch.finfo(wide).min)
    p = torch.softmax(z, dim=-1)
    if real is None:
        return (p @ vw).transpose(1, 2).to(q.dtype)
    # cleared twice: the outputs' gradients of padded rows are not read either
    out = torch.where(real, torch.where(real, p, 0.0) @ vw, 0.0)
    return out.transpose(1, 2).to(q.dtype)


def _check_masked(q, k, v, scale, causal, softcap, prefix, doc, slopes):
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or (
            q.shape[0] != k.shape[0] or q.shape[1] != k.shape[1]
            or q.shape[3] != k.shape[3]):
        raise ValueError(
            f"attention takes q [N, S, H, D] and k, v [N, S, Hkv, D], got "
            f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    n, s, h, _ = q.shape
    if k.shape[2] < 1 or h % k.shape[2]:
        raise ValueError(f"{h} heads do not divide over {k.shape[2]} key "
                         f"heads")
    if not (q.dtype == k.dtype == v.dtype) or not q.is_floating_point():
        raise TypeError(f"q, k and v must have one floating type, got "
                        f"{q.dtype}, {k.dtype}, {v.dtype}")
    if not 1e-18 <= scale <= 1e18:
        raise ValueError(f"the scale must be within 1e-18 and 1e18, got "
                         f"{scale}")
    if softcap != 0.0 and not 1e-18 <= softcap <= 1e18:
        raise ValueError(f"softcap must be 0 or within 1e-18 and 1e18, got "
                         f"{softcap}")
    if prefix is not None:
        if not causal:
            raise ValueError("a prefix widens a causal mask: causal=True")
        if prefix.dtype != torch.int32 or prefix.shape != (n,):
            raise ValueError(f"prefix must be int32 [{n}]")
    if doc is not None and (doc.dtype != torch.int32
                            or doc.shape != (n, s)):
        raise ValueError(f"doc must be int32 [{n}, {s}]")
    if slopes is not None:
        if slopes.dtype != torch.float32 or slopes.shape != (h,):
            raise ValueError(f"slopes must be float32 [{h}]")
        if slopes.requires_grad:
            raise ValueError("slopes are constants: they get no gradient")
    for name, t in (("k", k), ("v", v), ("prefix", prefix), ("doc", doc),
                    ("slopes", slopes)):
        if t is not None and t.device != q.device:
            raise ValueError(f"{name} is on {t.device}, q on {q.device}")


def _masked_native(q, *rest) -> bool:
    return (q.is_cuda and native_enabled()
            and q.dtype in (torch.bfloat16, torch.float16) and q.dim() >= 4
            and q.shape[-1] % 8 == 0 and 8 <= q.shape[-1] <= 128
            and not is_vmapped(q, *rest))


def colearn_attention(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
    scale: Optional[float] = None, causal: bool = False,
    prefix: Optional[torch.Tensor] = None,
    doc: Optional[torch.Tensor] = None, softcap: float = 0.0,
    slopes: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Self-attention of q [N, S, H, D] over k, v [N, S, Hkv, D]; returns
    [N, S, H, D].  Key head ``h // (H // Hkv)`` serves head ``h``.

    - ``scale``: of the scores, 1e-18 to 1e18 (default ``D ** -0.5``)
    - ``softcap``: scores become ``softcap * tanh(score / softcap)`` (0: not;
      else within the same bounds)
    - ``slopes`` float32 [H]: ``slopes[h] * |i - j|`` is taken off the score
      of query i and key j (after the cap); constants, without gradient
    - ``causal``: a query attends to keys up to its own position; with
      ``prefix`` int32 [N] also to every key before ``prefix[n]``
    - ``doc`` int32 [N, S]: a query attends to keys of its own document only;
      negative marks padding, whose outputs and gradients are zeros and whose
      values (NaN and infinities included) reach no other token.  Ids need not
      be sorted; packed rows (each document in one piece) cost least.  A NaN or
      an infinity in a token that is not padding may reach every token of its
      sequence, masked or not (0 times it is NaN).

    Gradients of q, k and v are bitwise the same from run to run.  bfloat16 and
    float16 operands on the GPU with D a multiple of 8 up to 128 run the HIP
    kernels (up to 2^25 elements a token over all heads; rows may be strided; a
    last dimension that is not contiguous, or rows that do not start at 16
    bytes, are copied first); other operands run the same formulas in torch.
    Under autocast operands are cast first.
    """
    if torch.is_autocast_enabled("cuda") and q.is_cuda:
        dt = torch.get_autocast_dtype("cuda")
        q, k, v = q.to(dt), k.to(dt), v.to(dt)
    if scale is None:
        scale = q.shape[-1] ** -0.5 if q.dim() and q.shape[-1] else 1.0
    if _masked_native(q, k, v):  # checks its operands itself
        return require_ext().masked_attention(q, k, v, scale, causal, softcap,
                                              prefix, doc, slopes)
    _check_masked(q, k, v, scale, causal, softcap, prefix, doc, slopes)
    return _masked_attention_ref(q, k, v, scale, causal, softcap, prefix, doc,
                                 slopes)


def colearn_attention_qkv(
    qkv: torch.Tensor, *, scale: Optional[float] = None,
    causal: bool = False, prefix: Optional[torch.Tensor] = None,
    doc: Optional[torch.Tensor] = None, softcap: float = 0.0,
    slopes: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``colearn_attention`` of the fused projection's output
    [N, S, 3, H, D]; returns [N, S, H * D]."""
    if qkv.dim() != 5 or qkv.shape[2] != 3:
        raise ValueError(f"qkv must be [N, S, 3, H, D], got "
                         f"{tuple(qkv.shape)}")
    if torch.is_autocast_enabled("cuda") and qkv.is_cuda:
        qkv = qkv.to(torch.get_autocast_dtype("cuda"))
    if scale is None:
        scale = qkv.shape[-1] ** -0.5 if qkv.shape[-1] else 1.0
    if _masked_native(qkv):  # checks its operands itself
        return require_ext().masked_attention_qkv(qkv, scale, causal, softcap,
                                                  prefix, doc, slopes)
    q, k, v = qkv.unbind(2)
    _check_masked(q, k, v, scale, causal, softcap, prefix, doc, slopes)
    return _masked_attention_ref(q, k, v, scale, causal, softcap, prefix, doc,
                                 slopes).flatten(2)


def distance_slopes(heads: int, device=None) -> torch.Tensor:
    """float32 [heads]: a geometric row of slopes from ``2 ** (-8 / heads)``
    down to 1/256, for ``colearn_attention``'s distance bias."""
    i = torch.arange(1, heads + 1, dtype=torch.float32, device=device)
    return torch.pow(2.0, -8.0 * i / heads)
