"""colearn_add_layer_norm against its definition in 64 bits.

Tolerances, per element: u (half a step of the type) of each 16-bit output;
f = 2^-18 relative of every summed magnitude for the fp32 statistics (a row's
sums run over at most 16384 terms in trees of depth below 32 plus 16 in line:
2^-24 * 48 < 2^-18); a column's sum over R rows adds its terms one after
another in parts of at most R / 4 and joins 64 of them: 2^-24 (R / 4 + 64).
"""

import math

import pytest
import torch

from colearn_federated_learning_amd.ops.norms import (
    ColearnLayerNorm, colearn_add_layer_norm)

GPU = pytest.param("cuda", marks=pytest.mark.gpu)
DEVICES = ["cpu", GPU]
F = 2.0 ** -18


def _unit(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def _check(dev, rows, h, dtype, groups=1, residual=True, use="y", eps=1e-12,
           seed=0, shift=0.0):
    g = torch.Generator().manual_seed(seed)

    def rand(*shape, dt=dtype):
        return torch.randn(*shape, generator=g).to(dt)

    x = (rand(rows, h) + shift).to(dtype)
    r = rand(rows, h) if residual else None
    w, b = rand(groups, h, dt=torch.float32), rand(groups, h,
                                                   dt=torch.float32)
    gy, gs = rand(rows, h), rand(rows, h)
    leaves = [t.to(dev).requires_grad_() for t in (x, w, b)]
    rd = None if r is None else r.to(dev).requires_grad_()
    y, s = colearn_add_layer_norm(leaves[0], rd, leaves[1], leaves[2],
                                  eps=eps, groups=groups)
    outs = {"y": [y], "sum": [s], "both": [y, s]}[use]
    gos = {"y": [gy], "sum": [gs], "both": [gy, gs]}[use]
    wrt = leaves + ([rd] if residual else [])
    grads = torch.autograd.grad(outs, wrt, [t.to(dev) for t in gos],
                                allow_unused=True)
    assert y.dtype == s.dtype == dtype

    u = _unit(dtype)
    want_s = x.double() if r is None else (x.double() + r.double()).to(
        dtype).double()
    assert torch.equal(s.detach().cpu().double(), want_s)
    a = want_s.view(groups, -1, h)
    mean = a.mean(2, keepdim=True)
    var = (a - mean).square().mean(2, keepdim=True)
    inv = 1 / torch.sqrt(var + eps)
    xh = (a - mean) * inv
    # the mean's error, relative to the row's spread
    em = F * (a.abs().mean(2, keepdim=True) * inv + 1)
    w2, b2 = w.double()[:, None], b.double()[:, None]
    want = xh * w2 + b2
    tol = u * want.abs() + w2.abs() * (em + F * xh.abs()) + F * b2.abs()

    def near(name, got, want, tol):
        off = (got.detach().cpu().double().reshape(want.shape) - want).abs()
        assert not off.isnan().any(), name
        worst = (off / (tol + 1e-30)).max().item() if off.numel() else 0.0
        assert worst <= 1.0, f"{name}: {worst:.2f} times its tolerance"

    near("y", y, want, tol)
    gx = torch.zeros_like(a)
    tx = torch.zeros_like(a)
    if use != "sum":
        gyd = gy.double().view(groups, -1, h)
        n = a.shape[1]
        col = 2.0 ** -24 * (n / 4 + 64) + F
        near("dw", grads[1], (gyd * xh).sum(1),
             col * (gyd * xh).abs().sum(1) + (gyd.abs() * em).sum(1))
        near("db", grads[2], gyd.sum(1), col * gyd.abs().sum(1))
        t = gyd * w2
        m1, m2 = t.mean(2, keepdim=True), (t * xh).mean(2, keepdim=True)
        gx = inv * (t - m1 - xh * m2)
        size = t.abs() + t.abs().mean(2, keepdim=True) + (
            xh.abs() + em) * (t * xh).abs().mean(2, keepdim=True)
        tx = inv * (F * size + em * (t.abs().mean(2, keepdim=True)
                                     * xh.abs() + m2.abs())) * 2
    if use != "y":
        gx = gx + gs.double().view(groups, -1, h)
        tx = tx + F * gx.abs()
    tx = tx + u * gx.abs()
    near("dx", grads[0], gx, tx)
    if residual:
        assert torch.equal(grads[0], grads[3])
    if use == "sum":
        assert grads[1] is None or not grads[1].any()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16,
                                   torch.float16])
@pytest.mark.parametrize("rows,h", [
    (1, 1), (3, 2), (5, 63), (7, 64), (9, 65), (6, 256), (5, 260), (33, 768),
    (4, 1023), (70, 1024), (5, 1025), (6, 1100), (5, 2052), (3, 4096),
    (3, 4097), (5, 5000), (2, 16383), (2, 16384)])
def test_shapes(dev, dtype, rows, h):
    _check(dev, rows, h, dtype, seed=rows + h)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("use", ["y", "sum", "both"])
@pytest.mark.parametrize("residual", [True, False])
def test_what_is_used(dev, use, residual):
    _check(dev, 21, 96, torch.bfloat16, residual=residual, use=use)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("groups,rows,h", [(2, 2, 64), (3, 51, 100),
                                           (8, 800, 768), (5, 10, 2048)])
def test_groups(dev, groups, rows, h):
    _check(dev, rows, h, torch.bfloat16, groups=groups)
    _check(dev, rows, h, torch.float32, groups=groups, use="both")


@pytest.mark.gpu
def test_many_rows():
    _check("cuda", 20000, 64, torch.bfloat16)
    _check("cuda", 9001, 1536, torch.float16, use="both")


@pytest.mark.parametrize("dev", DEVICES)
def test_far_from_zero(dev):
    """A mean a hundred times the spread: the variance is of distances from
    the mean, not a difference of large squares."""
    _check(dev, 17, 768, torch.float32, shift=100.0)


@pytest.mark.parametrize("dev", DEVICES)
def test_constant_row(dev):
    x = torch.full((3, 64), 2.5, dtype=torch.bfloat16, device=dev)
    w, b = (torch.full((64,), f, device=dev) for f in (3.0, 0.5))
    y, _ = colearn_add_layer_norm(x, None, w, b, eps=1e-5)
    assert (y == 0.5).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_nan_stays_in_its_row(dev):
    x = torch.randn(5, 300).to(torch.bfloat16)
    x[2, 7] = math.nan
    y, _ = colearn_add_layer_norm(x.to(dev), None, torch.ones(300).to(dev),
                                  torch.zeros(300).to(dev))
    bad = y.isnan().any(1).cpu()
    assert bad.tolist() == [False, False, True, False, False]


@pytest.mark.parametrize("dev", DEVICES)
def test_mixed_types_join_in_the_wider(dev):
    x = torch.randn(4, 32).to(torch.bfloat16).to(dev)
    r = torch.randn(4, 32).to(dev).requires_grad_()
    y, s = colearn_add_layer_norm(x, r, torch.ones(32).to(dev),
                                  torch.zeros(32).to(dev))
    assert y.dtype == s.dtype == torch.float32
    assert torch.equal(s, x.float() + r)
    y.square().sum().backward()
    assert r.grad.dtype == torch.float32


@pytest.mark.parametrize("dev", DEVICES)
def test_same_norm_as_the_module(dev):
    """Within the two roundings of what ColearnLayerNorm gives of the sum."""
    x, r = (torch.randn(40, 768).to(torch.bfloat16).to(dev) for _ in range(2))
    ln = ColearnLayerNorm(768).to(dev)
    y, s = colearn_add_layer_norm(x, r, ln.weight, ln.bias)
    want = ln(x + r)
    assert torch.equal(s, x + r)
    assert ((y.float() - want.float()).abs()
            <= 2 ** -7 * want.float().abs() + 2 ** -10).all()


@pytest.mark.gpu
def test_slots_are_zeros_where_only_the_sum_is_used():
    x, w = (torch.ones(6, 8, device="cuda", requires_grad=True)
            for _ in range(2))
    slots = [torch.full((6, 8), math.nan, device="cuda") for _ in range(2)]
    _, s = colearn_add_layer_norm(x, x.detach(), w, w, groups=6,
                                  gslot_w=slots[0], gslot_b=slots[1])
    s.sum().backward()
    assert (x.grad == 1).all() and all((t == 0).all() for t in slots)


@pytest.mark.gpu
def test_more_than_32_bits_of_elements():
    rows, h = 2 ** 21 + 5, 1024
    g = torch.Generator("cuda").manual_seed(0)
    x = torch.empty(rows, h, dtype=torch.bfloat16, device="cuda")
    x.normal_(generator=g)
    gy = torch.zeros_like(x)
    ends = torch.cat([torch.arange(8), torch.arange(rows - 8, rows)]).cuda()
    gy[ends] = torch.randn(16, h, generator=g, device="cuda").to(x.dtype)
    w, b = (torch.randn(h, generator=g, device="cuda").requires_grad_()
            for _ in range(2))

    def run(x, gy):
        x = x.requires_grad_()
        y, s = colearn_add_layer_norm(x, x.detach(), w, b)
        return [y, s, *torch.autograd.grad(y, (x, w, b), gy)]

    few = run(x[ends], gy[ends])
    all_ = run(x, gy)
    for a, c in zip(all_[:3], few[:3]):
        assert torch.equal(a[ends], c)
    # sums of the same 16 terms in another order: 15 roundings each, of 2^-24
    # of what the terms add up to; a normalised element is at most 32
    most = gy[ends].float().abs().sum(0) * 32
    for a, c in zip(all_[3:], few[3:]):
        assert ((a - c).abs() <= 2 * 15 * 2.0 ** -24 * most).all()


@pytest.mark.gpu
def test_slots_order_streams_and_replay():
    g = torch.Generator().manual_seed(0)
    x, r, gy = (torch.randn(64, 96, generator=g).to(torch.bfloat16).cuda()
                for _ in range(3))
    w, b = (torch.randn(4, 96, generator=g).cuda().requires_grad_()
            for _ in range(2))
    slots = [torch.full((4, 96), math.nan, device="cuda") for _ in range(2)]

    def run(x, **kw):
        x = x.detach().requires_grad_()
        y, s = colearn_add_layer_norm(x, r, w, b, groups=4, **kw)
        wrt = (x,) if kw else (x, w, b)
        return [y.detach(), s.detach(),
                *torch.autograd.grad(y, wrt, gy)]

    want = run(x)
    got = run(x, gslot_w=slots[0], gslot_b=slots[1])
    assert all(torch.equal(a, c) for a, c in zip(got + slots, want))
    # operands that are not contiguous
    assert all(torch.equal(a, c) for a, c in zip(
        run(x.t().contiguous().t()), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x)
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    graphs = []
    buf = x.clone()
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = run(buf)
        graphs.append((gr, out))
    other = (x.float() * 2 + 1).to(torch.bfloat16)
    want2 = run(other)
    for src, ref in ((x, want), (other, want2), (x, want)):
        buf.copy_(src)
        for gr, _ in graphs:
            gr.replay()
        run(other)
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, c) for a, c in zip(out, ref))


def test_gradients_by_differences():
    g = torch.Generator().manual_seed(0)
    x, r = (torch.randn(6, 5, generator=g, dtype=torch.float64,
                        requires_grad=True) for _ in range(2))
    w, b = (torch.randn(2, 5, generator=g, dtype=torch.float64,
                        requires_grad=True) for _ in range(2))
    assert torch.autograd.gradcheck(
        lambda *a: colearn_add_layer_norm(*a, eps=1e-3, groups=2),
        (x, r, w, b))


@pytest.mark.gpu
def test_gradients_by_differences_gpu():
    """fp32: the quotient of a sum of 12 x 40 outputs over a step of 2^-7 is
    off by its roundings, F of every term over the step, and by the third
    derivative's share, measured by doubling the step."""
    g = torch.Generator().manual_seed(0)
    x, way, go = (torch.randn(12, 40, generator=g).cuda() for _ in range(3))
    w, b = (torch.randn(40, generator=g).cuda() for _ in range(2))
    y = x.clone().requires_grad_()
    out, _ = colearn_add_layer_norm(y, None, w, b)
    (gr,) = torch.autograd.grad(out, y, go)

    def at(h):
        o, _ = colearn_add_layer_norm(x + h * way, None, w, b)
        return (o.double() * go.double()).sum().item()

    h = 2.0 ** -7
    q1 = (at(h) - at(-h)) / (2 * h)
    q2 = (at(2 * h) - at(-2 * h)) / (4 * h)
    slope = (gr.double() * way.double()).sum().item()
    noise = F * (out.double() * go.double()).abs().sum().item() / h
    assert abs(q1 - slope) <= abs(q2 - q1) + noise


@pytest.mark.parametrize("dev", DEVICES)
def test_refusals(dev):
    x = torch.zeros(6, 8, device=dev)
    w = torch.ones(8, device=dev)

    def refuse(kind, *a, **kw):
        with pytest.raises(kind):
            colearn_add_layer_norm(*a, **kw)

    refuse(ValueError, x, None, w[:7], w)
    refuse(ValueError, x, None, w, w, groups=2)
    refuse(ValueError, x[:5], None, torch.ones(2, 8, device=dev),
           torch.ones(2, 8, device=dev), groups=2)
    refuse(ValueError, x, None, w, w, groups=0)
    refuse(ValueError, x, x[:5], w, w)
    refuse(TypeError, x.int(), None, w, w)
    refuse(ValueError, x, None, w, w, gslot_w=w)
    if dev == "cuda":
        for bad in (w[:7], w.half(), w.cpu(), torch.ones(16, device=dev)[::2]):
            refuse(RuntimeError, x, None, w, w, gslot_w=w.clone(), gslot_b=bad)
        many = torch.zeros(2 ** 26, 1, dtype=torch.bfloat16, device=dev)
        refuse(RuntimeError, many, None, w[:1], w[:1])
        refuse(ValueError, x, None, w.cpu(), w)
        refuse(TypeError, x, None, w.half(), w.half())
        y, _ = colearn_add_layer_norm(x.requires_grad_(), None, w, w)
        (gx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            gx.sum().backward()
    else:
        refuse(ValueError, x, None, w, w, gslot_w=w, gslot_b=w)


@pytest.mark.parametrize("dev", DEVICES)
def test_empty(dev):
    x = torch.zeros(0, 8, device=dev, requires_grad=True)
    w = torch.ones(8, device=dev, requires_grad=True)
    y, s = colearn_add_layer_norm(x, None, w, w.detach())
    y.sum().backward()
    assert y.shape == s.shape == x.grad.shape == (0, 8)
    assert (w.grad == 0).all()


@pytest.mark.gpu
def test_slots_that_overlap_are_refused():
    x = torch.zeros(6, 8, device="cuda", requires_grad=True)
    flat = torch.ones(40, device="cuda")
    w, b, slot = flat[:8], flat[8:16], flat[16:24]
    for bad in (slot, flat[20:28], flat[12:20], w, b, flat[4:12]):
        for pair in ((slot, bad), (bad, slot)):
            with pytest.raises(RuntimeError, match="overlap"):
                colearn_add_layer_norm(x, None, w, b, gslot_w=pair[0],
                                       gslot_b=pair[1])
    y, _ = colearn_add_layer_norm(x, None, w, b, gslot_w=slot,
                                  gslot_b=flat[24:32])
    y.sum().backward()
    assert (flat[24:32] == 6).all() and (flat[16:24] == 0).all()
    assert (flat[:16] == 1).all() and (flat[32:] == 1).all()
