"""Timed cases for the encoder-training operators: attention with masks,
caps and distance biases, residual add + layer norm, and the AdamW step over
many tensors with 32-bit or 8-bit states.

``run`` computes each operator in its plain form (elementary torch operations
in 32 bits) or, with ``own`` set, through the package's entry points.
``exact`` evaluates the definition in 64 bits.
"""

import math
import random

import numpy as np
import torch
import torch.nn.functional as F

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
BLOCK = 256          # elements that share one scale of an 8-bit state
E4M3_MAX = 448.0     # largest value of the 8-bit float
E4M3_MIN = 2.0 ** -9  # its smallest positive value
TINY = 1e-30         # a block whose largest entry is below this is held as 0


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def _attn(name, n, s, h, hkv, d, dtype, train, packed=False, doc=0, pad=False,
          causal=False, prefix=0, softcap=0.0, slopes=False):
    return {"name": name, "op": "attention", "n": n, "s": s, "h": h,
            "hkv": hkv, "d": d, "dtype": dtype, "train": train,
            "packed": packed, "doc": doc, "pad": pad, "causal": causal,
            "prefix": prefix, "softcap": softcap, "slopes": slopes}


def _norm(name, rows, h, groups, dtype, train, both=False):
    return {"name": name, "op": "norm", "rows": rows, "h": h,
            "groups": groups, "dtype": dtype, "train": train, "both": both}


def _adamw(name, model, hidden, layers, vocab, bits, dtype):
    return {"name": name, "op": "adamw", "model": model, "hidden": hidden,
            "layers": layers, "vocab": vocab, "bits": bits, "dtype": dtype}


def listed():
    return [
        # evaluating a handful of short texts on a small encoder: latency
        _attn("attention_eval_short", 2, 47, 4, 4, 64, "bf16", False,
              packed=True, doc=0, pad=True),
        # BERT-base training on rows packed with several documents each, at
        # the full length of its position table
        _attn("attention_train_packed", 32, 512, 12, 12, 64, "bf16", True,
              packed=True, doc=150, pad=True),
        # an encoder-decoder style text: a bidirectional prefix, the rest
        # causal, capped scores, shared key heads, an odd length
        _attn("attention_train_prefix_cap", 2, 1999, 16, 4, 128, "fp16", True,
              causal=True, prefix=301, softcap=30.0),
        # distance-biased training without position table, padded rows
        _attn("attention_train_distance", 1, 4096, 12, 12, 64, "bf16", True,
              packed=True, pad=True, slopes=True),
        # scoring long texts beyond the trained length
        _attn("attention_eval_long", 1, 8192, 12, 12, 64, "bf16", False,
              packed=True, slopes=True),
        # one short text through the norm: latency
        _norm("norm_eval_short", 47, 768, 1, "bf16", False),
        # one client's batch, post-norm layer
        _norm("norm_train_client", 32 * 128, 768, 1, "bf16", True),
        # eight clients stacked, each with its own weight, at full length
        _norm("norm_train_stacked", 8 * 16 * 512, 768, 8, "bf16", True),
        # a wider pre-norm stream, odd width, full precision
        _norm("norm_train_odd", 4099, 1023, 1, "fp32", True, both=True),
        # the small image model of a constrained client: latency
        _adamw("adamw_cnn_8bit", "cnn", 0, 0, 0, 8, "fp32"),
        # BERT-base, every tensor of the model in one step
        _adamw("adamw_bert_32bit", "bert", 768, 12, 30522, 32, "fp32"),
        _adamw("adamw_bert_8bit", "bert", 768, 12, 30522, 8, "fp32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "norm", "adamw"])
    if op == "attention":
        s = _log_int(rng, 1, 4096)
        d = rng.choice([32, 40, 64, 64, 128])
        hkv = rng.choice([1, 2, 4, 6, 12])
        h = hkv * rng.choice([1, 1, 2, 4]) if hkv < 12 else 12
        # scores of one pass stay under those of the largest listed case
        most = max(1, min(64, 12 * 4096 * 4096 * 64 // (h * s * s * d)))
        n = _log_int(rng, 1, most)
        causal = rng.random() < 0.4
        doc = rng.choice([0, 0, 40, 150, 700])
        return _attn("", n, s, h, hkv, d, rng.choice(["bf16", "bf16", "fp16"]),
                     rng.random() < 0.6,
                     packed=h == hkv and rng.random() < 0.7, doc=doc,
                     pad=rng.random() < 0.5, causal=causal,
                     prefix=(rng.randint(0, s)
                             if causal and doc == 0 and rng.random() < 0.5
                             else 0),
                     softcap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                     slopes=rng.random() < 0.4)
    if op == "norm":
        h = _log_int(rng, 64, 4096)
        if rng.random() < 0.6:
            h = (h + 7) // 8 * 8
        groups = rng.choice([1, 1, 2, 8])
        most = 8 * 16 * 512 * 768 // h // 3
        rows = max(1, _log_int(rng, 1, most) // groups) * groups
        return _norm("", rows, h, groups, rng.choice(["bf16", "fp16", "fp32"]),
                     rng.random() < 0.7, both=rng.random() < 0.4)
    if rng.random() < 0.25:
        return _adamw("", "cnn", 0, 0, 0, rng.choice([8, 32]), "fp32")
    return _adamw("", "bert", 12 * _log_int(rng, 5, 60), rng.randint(1, 11),
                  _log_int(rng, 500, 30000), rng.choice([8, 32]),
                  rng.choice(["fp32", "fp32", "bf16"]))


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _doc_ids(case, seed):
    """int32 [n, s]: each row holds documents one after another, then
    (``pad``) padding marked -1.  The lengths go by the case alone, so every
    seed has the same number of attended pairs; their order goes by the
    seed."""
    if not case["doc"] and not case["pad"]:
        return None
    n, s, mean = case["n"], case["s"], case["doc"]
    rng = random.Random(n * 1000003 + s * 101 + mean)
    order = random.Random(seed)
    ids = np.full((n, s), -1, dtype=np.int32)
    for row in range(n):
        fill = s - rng.randint(0, s // 4) if case["pad"] else s
        lens = []
        while sum(lens) < fill:
            want = rng.randint(max(1, mean // 4), 2 * mean) if mean else fill
            lens.append(min(want, fill - sum(lens)))
        order.shuffle(lens)
        ids[row, :fill] = np.repeat(np.arange(len(lens), dtype=np.int32), lens)
    return ids


def _pairs(case):
    """Attended (query, key) pairs of one head, over the batch."""
    n, s = case["n"], case["s"]
    ids = _doc_ids(case, 0)
    total = 0
    for row in range(n):
        if ids is None:
            lens = np.array([s], dtype=np.int64)
        else:
            r = ids[row]
            lens = np.bincount(r[r >= 0]).astype(np.int64)
        if not case["causal"]:
            total += int((lens * lens).sum())
        elif case["prefix"]:
            fill, p = int(lens.sum()), min(case["prefix"], int(lens.sum()))
            total += p * p + (fill * (fill + 1) - p * (p + 1)) // 2
        else:
            total += int((lens * (lens + 1) // 2).sum())
    return total


def _shapes(case):
    """Parameter shapes of the model whose step is taken."""
    if case["model"] == "cnn":  # the image model at 28 x 28, one channel
        return [(32, 1, 3, 3), (32,), (64, 32, 3, 3), (64,),
                (128, 64 * 14 * 14), (128,), (10, 128), (10,)]
    d, v = case["hidden"], case["vocab"]
    shapes = [(v, d), (512, d), (d,), (d,)]
    for _ in range(case["layers"]):
        shapes += [(3 * d, d), (3 * d,), (d, d), (d,), (d,), (d,),
                   (4 * d, d), (4 * d,), (d, 4 * d), (d,), (d,), (d,)]
    return shapes + [(d, d), (d,), (d,), (d,), (v,)]


def _e4m3(x):
    return x.to(torch.float8_e4m3fn)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 17)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device=dev) * std).to(dtype)

    st = {"case": dict(case)}
    if case["op"] == "attention":
        n, s, h, hkv, d = (case[k] for k in ("n", "s", "h", "hkv", "d"))
        if case["packed"]:  # the fused projection's layout
            st["qkv"] = normal(n, s, 3, h, d)
        else:
            st["q"] = normal(n, s, h, d)
            st["k"] = normal(n, s, hkv, d)
            st["v"] = normal(n, s, hkv, d)
        ids = _doc_ids(case, seed)
        st["doc"] = None if ids is None else torch.from_numpy(ids).to(dev)
        st["prefix"] = (torch.full((n,), case["prefix"], dtype=torch.int32,
                                   device=dev) if case["prefix"] else None)
        st["slopes"] = (torch.pow(2.0, -8.0 * (torch.arange(
            h, device=dev, dtype=torch.float32) + 1) / h)
            if case["slopes"] else None)
        if case["train"]:
            st["grad"] = normal(n, s, h, d, std=0.02)
    elif case["op"] == "norm":
        rows, h, g = case["rows"], case["h"], case["groups"]
        st["x"] = normal(rows, h) + normal(1, h, std=0.3)
        st["r"] = normal(rows, h)
        st["w"] = 1 + normal(g, h, std=0.1, dtype=torch.float32)
        st["b"] = normal(g, h, std=0.1, dtype=torch.float32)
        if case["train"]:
            st["gy"] = normal(rows, h, std=0.02)
            st["gh"] = normal(rows, h, std=0.02) if case["both"] else None
    else:
        shapes = _shapes(case)
        sizes = [math.prod(sh) for sh in shapes]

        def views(flat):  # the model trains out of flat buffers
            return [f.view(sh) for f, sh in zip(flat.split(sizes), shapes)]

        n = sum(sizes)
        st["t"] = 3
        st["sizes"] = sizes
        st["flat_p"], st["flat_g"] = normal(n, std=0.02), normal(n, std=0.01)
        # states after a few steps: first moments of the gradients' size,
        # second moments of their squares'
        m = normal(n, std=0.003, dtype=torch.float32)
        v = normal(n, std=0.003, dtype=torch.float32).square() + 1e-10
        st["wd"] = [0.01 if len(sh) > 1 else 0.0 for sh in shapes]
        if case["bits"] == 8:
            mq = [_quantise(x, False) for x in m.split(sizes)]
            vq = [_quantise(x.sqrt(), True) for x in v.split(sizes)]
            m, v = (torch.cat([c.view(torch.uint8) for c, _ in x])
                    .view(torch.float8_e4m3fn) for x in (mq, vq))
            blocks = [-(-k // BLOCK) for k in sizes]
            st["flat_ms"] = torch.cat([sc for _, sc in mq])
            st["flat_vs"] = torch.cat([sc for _, sc in vq])
            st["ms"] = list(st["flat_ms"].split(blocks))
            st["vs"] = list(st["flat_vs"].split(blocks))
        st["flat_m"], st["flat_v"] = m, v
        st["p"], st["g"] = views(st["flat_p"]), views(st["flat_g"])
        st["m"], st["v"] = views(m), views(v)
    return st


# --------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------
def _split_qkv(st):
    if st["case"]["packed"]:
        return st["qkv"].unbind(2)
    return st["q"], st["k"], st["v"]


def _allowed(case, doc, prefix, device):
    """bool [n or 1, s, s]; None if every pair is attended."""
    s = case["s"]
    i = torch.arange(s, device=device)
    ok = None
    if case["causal"]:
        ok = (i[None, :] <= i[:, None])[None]
        if prefix is not None:
            ok = ok | (i[None, None, :] < prefix[:, None, None])
    if doc is not None:
        same = (doc[:, :, None] == doc[:, None, :]) & (doc >= 0)[:, :, None]
        ok = same if ok is None else ok & same
    return ok


def _plain_attention(st):
    case = st["case"]
    n, s, h, hkv, d = (case[k] for k in ("n", "s", "h", "hkv", "d"))
    q, k, v = (t.float().transpose(1, 2) for t in _split_qkv(st))
    k, v = k.contiguous(), v.contiguous()
    if hkv != h:
        k = k.repeat_interleave(h // hkv, dim=1)
        v = v.repeat_interleave(h // hkv, dim=1)
    dt = DTYPES[case["dtype"]]
    if st["doc"] is not None:  # padded tokens take no part, whatever they hold
        real = (st["doc"] >= 0)[:, None, :, None]
        q, k, v = (torch.where(real, t, 0.0) for t in (q, k, v))
    scale = 1.0 / math.sqrt(d)
    sc = torch.matmul(q, k.transpose(-1, -2)) * scale
    cap = case["softcap"]
    if cap:
        th = torch.tanh(sc / cap)
        sc = th * cap
    if st["slopes"] is not None:
        i = torch.arange(s, device=q.device, dtype=torch.float32)
        sc = sc - st["slopes"][None, :, None, None] * (
            i[:, None] - i[None, :]).abs()
    ok = _allowed(case, st["doc"], st["prefix"], q.device)
    if ok is not None:
        sc = sc.masked_fill(~ok[:, None], -math.inf)
    top = sc.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(sc - top)
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    del sc
    out = torch.matmul(p, v)
    res = {"out": out.transpose(1, 2).to(dt).contiguous()}
    if not case["train"]:
        return res
    go = st["grad"].float().transpose(1, 2)
    if st["doc"] is not None:
        go = torch.where(real, go, 0.0)
    dv = torch.matmul(p.transpose(-1, -2), go)
    dp = torch.matmul(go, v.transpose(-1, -2))
    ds = p * (dp - (dp * p).sum(dim=-1, keepdim=True))
    del dp, p
    if cap:
        ds = ds * (1 - th * th)
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(-1, -2), q) * scale
    if hkv != h:
        dk = dk.view(n, hkv, h // hkv, s, d).sum(2)
        dv = dv.view(n, hkv, h // hkv, s, d).sum(2)
    dq, dk, dv = (t.transpose(1, 2).to(dt) for t in (dq, dk, dv))
    if case["packed"]:
        res["dqkv"] = torch.stack([dq, dk, dv], dim=2)
    else:
        res["dq"], res["dk"], res["dv"] = (t.contiguous()
                                           for t in (dq, dk, dv))
    return res


def _own_attention(st):
    from colearn_federated_learning_amd.ops.attention import (
        colearn_attention, colearn_attention_qkv)

    case = st["case"]
    kw = dict(causal=case["causal"], prefix=st["prefix"], doc=st["doc"],
              softcap=case["softcap"], slopes=st["slopes"])
    n, s, h, d = (case[k] for k in ("n", "s", "h", "d"))
    if not case["train"]:
        with torch.no_grad():
            if case["packed"]:
                out = colearn_attention_qkv(st["qkv"], **kw)
            else:
                out = colearn_attention(st["q"], st["k"], st["v"], **kw)
        return {"out": out.view(n, s, h, d)}
    if case["packed"]:
        qkv = st["qkv"].detach().requires_grad_()
        out = colearn_attention_qkv(qkv, **kw).view(n, s, h, d)
        (dqkv,) = torch.autograd.grad(out, (qkv,), st["grad"])
        return {"out": out.detach(), "dqkv": dqkv}
    q, k, v = (st[x].detach().requires_grad_() for x in "qkv")
    out = colearn_attention(q, k, v, **kw)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), st["grad"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}


def _plain_norm(st):
    case = st["case"]
    rows, h, g = case["rows"], case["h"], case["groups"]
    dt = DTYPES[case["dtype"]]
    # the sum is a tensor of the model's own type, and what is normalised
    s = (st["x"].float() + st["r"].float()).to(dt)
    x = s.float().view(g, rows // g, h)
    mean = x.mean(dim=-1, keepdim=True)
    c = x - mean
    inv = (c.square().mean(dim=-1, keepdim=True) + 1e-12).rsqrt()
    xh = c * inv
    w, b = st["w"][:, None], st["b"][:, None]
    res = {"y": (xh * w + b).to(dt).view(rows, h), "sum": s}
    if not case["train"]:
        return res
    gy = st["gy"].float().view(g, rows // g, h)
    res["gw"], res["gb"] = (gy * xh).sum(dim=1), gy.sum(dim=1)
    gx = gy * w
    gx = inv * (gx - gx.mean(dim=-1, keepdim=True)
                - xh * (gx * xh).mean(dim=-1, keepdim=True))
    gx = gx.view(rows, h)
    if st["gh"] is not None:
        gx = gx + st["gh"].float()
    res["gx"] = gx.to(dt)
    return res


def _own_norm(st):
    from colearn_federated_learning_amd.ops.norms import colearn_add_layer_norm

    case = st["case"]
    if not case["train"]:
        with torch.no_grad():
            y, s = colearn_add_layer_norm(st["x"], st["r"], st["w"], st["b"],
                                          eps=1e-12, groups=case["groups"])
        return {"y": y, "sum": s}
    x, w, b = (st[k].detach().requires_grad_() for k in "xwb")
    y, s = colearn_add_layer_norm(x, st["r"], w, b, eps=1e-12,
                                  groups=case["groups"])
    outs, grads = ((y, s), (st["gy"], st["gh"])) if case["both"] else (
        (y,), (st["gy"],))
    gx, gw, gb = torch.autograd.grad(outs, (x, w, b), grads)
    return {"y": y.detach(), "sum": s.detach(), "gx": gx, "gw": gw, "gb": gb}


HYPER = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8)


def _quantise(x, positive):
    """fp32 [n] -> (e4m3 [n], fp32 scales, one a block of 256).  A positive
    entry of a second moment's root never becomes 0."""
    n = x.numel()
    blocks = F.pad(x, (0, -n % BLOCK)).view(-1, BLOCK)
    top = blocks.abs().amax(dim=1)
    live = top > TINY
    inv = torch.where(live, E4M3_MAX / top, 0.0)
    scale = torch.where(live, top / E4M3_MAX, 0.0)
    u = blocks * inv[:, None]
    if positive:
        u = torch.where(u > 0, u.clamp_min(E4M3_MIN), u)
    return _e4m3(u).view(-1)[:n].contiguous(), scale


def _blocked(flat, sizes):
    """The tensors of a flat buffer end to end, each padded to whole blocks."""
    return torch.cat([F.pad(t, (0, -t.numel() % BLOCK))
                      for t in flat.split(sizes)])


def _spread(blocked, flat, sizes):
    """The other way round, into the flat buffer."""
    padded = [k + (-k % BLOCK) for k in sizes]
    torch.cat([t[:k] for t, k in zip(blocked.split(padded), sizes)], out=flat)


def _plain_adamw(st):
    case, sizes = st["case"], st["sizes"]
    t, (b1, b2) = st["t"], HYPER["betas"]
    bc1, bc2 = 1 - b1 ** t, 1 - b2 ** t
    lr, eps = HYPER["lr"], HYPER["eps"]
    w, g = st["flat_p"].float(), st["flat_g"].float()
    keep = torch.tensor([1 - lr * wd for wd in st["wd"]],
                        dtype=torch.float32).to(w.device)
    count = torch.tensor(sizes).to(w.device)
    if case["bits"] == 32:
        m, v = st["flat_m"], st["flat_v"]
    else:  # every tensor in whole blocks
        w, g = _blocked(w, sizes), _blocked(g, sizes)
        count = (count + BLOCK - 1) // BLOCK * BLOCK
        m, v = ((_blocked(st[c].view(torch.uint8), sizes)
                 .view(torch.float8_e4m3fn).float().view(-1, BLOCK)
                 * st[sc][:, None]).view(-1)
                for c, sc in (("flat_m", "flat_ms"), ("flat_v", "flat_vs")))
        v = v * v
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    w = w * keep.repeat_interleave(count, output_size=w.numel())
    w = w - (m / (torch.sqrt(v * (1 / bc2)) + eps)) * (lr / bc1)
    if case["bits"] == 32:
        st["flat_p"].copy_(w)
        st["flat_m"].copy_(m)
        st["flat_v"].copy_(v)
        return
    _spread(w.to(DTYPES[case["dtype"]]), st["flat_p"], sizes)
    for x, c, sc, pos in ((m, "flat_m", "flat_ms", False),
                          (torch.sqrt(v), "flat_v", "flat_vs", True)):
        codes, scales = _quantise(x, pos)
        _spread(codes.view(torch.uint8), st[c].view(torch.uint8), sizes)
        st[sc].copy_(scales)


def _own_adamw(st):
    from colearn_federated_learning_amd.ops.fused_optim import adamw_step

    adamw_step(st["p"], st["g"], st["m"], st["v"],
               exp_avg_scales=st.get("ms"), exp_avg_sq_scales=st.get("vs"),
               step=st["t"], weight_decay=st["wd"], **HYPER)


def _adamw_outputs(st):
    """Every updated tensor, in the flat buffers that they are views of."""
    return {k: st[k] for k in ("flat_p", "flat_m", "flat_v", "flat_ms",
                               "flat_vs") if k in st}


def run(st):
    op = st["case"]["op"]
    if op == "attention":
        return _own_attention(st) if own else _plain_attention(st)
    if op == "norm":
        return _own_norm(st) if own else _plain_norm(st)
    _own_adamw(st) if own else _plain_adamw(st)
    st["t"] += 1
    return _adamw_outputs(st)


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    if case["op"] == "attention":
        n, s, h, hkv, d = (case[k] for k in ("n", "s", "h", "hkv", "d"))
        e = SIZE[case["dtype"]]
        q, kv = n * s * h * d * e, 2 * n * s * hkv * d * e
        pairs = _pairs(case) * h
        if not case["train"]:
            return {"bytes": 2 * q + kv, "flops": 4 * d * pairs}
        # forward: q k^T and p v; backward: dv, dp, dq, dk
        return {"bytes": 4 * q + 2 * kv, "flops": 12 * d * pairs}
    if case["op"] == "norm":
        e = SIZE[case["dtype"]] * case["rows"] * case["h"]
        if not case["train"]:
            return {"bytes": 4 * e, "flops": 9 * case["rows"] * case["h"]}
        return {"bytes": (7 if case["both"] else 6) * e,
                "flops": 24 * case["rows"] * case["h"]}
    n = sum(math.prod(s) for s in _shapes(case))
    e = SIZE[case["dtype"]]
    state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": (3 * e + state) * n, "flops": 15 * n}


# --------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, st)
    if case["op"] == "norm":
        return _exact_norm(case, st)
    return _exact_adamw(case, st)


def _exact_attention(case, st):
    """Row by row of the batch and head by head; attended pairs only."""
    n, s, h, hkv, d = (case[k] for k in ("n", "s", "h", "hkv", "d"))
    if 12 * d * h * n * s * s > 4e13 or n * h > 4000:
        return None
    if case["packed"]:
        q, k, v = (st["qkv"][:, :, i].double() for i in range(3))
    else:
        q, k, v = st["q"].double(), st["k"].double(), st["v"].double()
    dev = q.device
    out = torch.zeros(n, s, h, d, dtype=torch.float64, device=dev)
    dq = torch.zeros_like(out)
    dk = torch.zeros(n, s, hkv, d, dtype=torch.float64, device=dev)
    dv = torch.zeros_like(dk)
    pos = torch.arange(s, device=dev)
    for b in range(n):
        keep = torch.ones(s, s, dtype=torch.bool, device=dev)
        if case["causal"]:
            keep = pos[:, None] >= pos[None, :]
            if case["prefix"]:
                keep = keep | (pos < case["prefix"])[None, :]
        live = torch.ones(s, dtype=torch.bool, device=dev)
        if st["doc"] is not None:
            ids = st["doc"][b]
            live = ids >= 0
            keep = keep & (ids[:, None] == ids[None, :]) & live[None, :]
        for a in range(h):
            c = a // (h // hkv)
            qa, ka, va = q[b, :, a], k[b, :, c], v[b, :, c]
            z = qa @ ka.T / math.sqrt(d)
            slope = torch.ones((), dtype=torch.float64, device=dev)
            if case["softcap"]:
                u = torch.tanh(z / case["softcap"])
                z, slope = u * case["softcap"], 1 - u * u
            if st["slopes"] is not None:
                z = z - st["slopes"][a].double() * (
                    pos[:, None] - pos[None, :]).abs()
            z = torch.where(keep, z, -math.inf)
            p = torch.where(live[:, None], torch.softmax(z, dim=1), 0.0)
            out[b, :, a] = p @ va
            if case["train"]:
                go = st["grad"][b, :, a].double()
                dv[b, :, c] += p.T @ go
                dp = go @ va.T
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) * slope
                dq[b, :, a] = ds @ ka / math.sqrt(d)
                dk[b, :, c] += ds.T @ qa / math.sqrt(d)
    if not case["train"]:
        return {"out": out}
    if case["packed"]:
        return {"out": out, "dqkv": torch.stack([dq, dk, dv], dim=2)}
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _exact_norm(case, st):
    g, h = case["groups"], case["h"]
    # the sum is rounded to the model's type: that is part of the definition
    s = (st["x"].double() + st["r"].double()).to(DTYPES[case["dtype"]])
    x = s.double().view(g, -1, h)
    var, mean = torch.var_mean(x, dim=2, keepdim=True, correction=0)
    sd = torch.sqrt(var + 1e-12)
    z = (x - mean) / sd
    w, b = st["w"].double()[:, None], st["b"].double()[:, None]
    res = {"y": (z * w + b).view(-1, h), "sum": s.double()}
    if case["train"]:
        gy = st["gy"].double().view(g, -1, h)
        gz = gy * w
        gx = (gz - gz.mean(2, keepdim=True)
              - z * (gz * z).mean(2, keepdim=True)) / sd
        gx = gx.view(-1, h)
        if st["gh"] is not None:
            gx = gx + st["gh"].double()
        res.update(gx=gx, gw=(gy * z).sum(1), gb=gy.sum(1))
    return res


def _exact_adamw(case, st):
    (b1, b2), lr, eps, t = HYPER["betas"], HYPER["lr"], HYPER["eps"], st["t"]
    eight = case["bits"] == 8
    res = {k: [] for k in ("flat_p", "flat_m", "flat_v")}
    if eight:
        res.update(flat_ms=[], flat_vs=[])

    def widen(code, scale):
        flat = code.double().reshape(-1)
        return (flat * scale.double().repeat_interleave(BLOCK)[:flat.numel()])

    def narrow(flat, positive):
        n = flat.numel()
        rows = torch.zeros((n + BLOCK - 1) // BLOCK * BLOCK,
                           dtype=torch.float64, device=flat.device)
        rows[:n] = flat.abs()
        top = rows.view(-1, BLOCK).max(dim=1).values
        top = torch.where(top > TINY, top, 0.0)
        unit = (top / E4M3_MAX).repeat_interleave(BLOCK)[:n]
        u = torch.where(unit > 0, flat / unit, 0.0)
        if positive:
            u = torch.where((u > 0) & (u < E4M3_MIN), E4M3_MIN, u)
        # nearest of the 8-bit values, ties to the even one
        step = torch.pow(2.0, torch.floor(torch.log2(
            u.abs().clamp_min(2.0 ** -6))) - 3)
        return torch.round(u / step) * step, top / E4M3_MAX

    for i in range(len(st["p"])):
        g = st["g"][i].reshape(-1).double()
        p = st["p"][i].reshape(-1).double()
        if eight:
            m = widen(st["m"][i], st["ms"][i])
            v = widen(st["v"][i], st["vs"][i]).square()
        else:
            m = st["m"][i].reshape(-1).double()
            v = st["v"][i].reshape(-1).double()
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        up = m / (1 - b1 ** t) / (torch.sqrt(v / (1 - b2 ** t)) + eps)
        res["flat_p"].append(p - lr * (up + st["wd"][i] * p))
        if eight:
            m, sm = narrow(m, False)
            v, sv = narrow(v.sqrt(), True)
            res["flat_ms"].append(sm)
            res["flat_vs"].append(sv)
        res["flat_m"].append(m)
        res["flat_v"].append(v)
    return {k: torch.cat(v) for k, v in res.items()}
