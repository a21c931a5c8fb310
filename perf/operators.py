"""The workloads by which the block operators are measured: group norm with an
activation, keyed dropout with a residual, and the 8-bit integer product.

`own = False`: the operators in plain torch operations; `own = True`: the
framework's kernels through `ldsgnn.ops`.  Sizes are those of the framework's
workloads (Cora 2708 x 1433 -> 16, the 20 000-node synthetic graph, the 16
evaluation samples) and generic widths around them.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    gn, dr, i8 = dict(op="group_norm"), dict(op="dropout"), dict(op="int8")
    return [
        # one node embedded on its own (an inductive query): latency
        dict(gn, name="gn_node", s=1, n=1, groups=32, cg=8, dtype="bf16", act="silu", p=0.0, train=False),
        # the hidden layer of the Cora classifier in training: norm, silu, dropout 0.5, and back.  (No case takes
        # relu's gradient: it jumps at zero, so that a last bit of z there decides over a whole gradient entry.)
        dict(gn, name="gn_cora_train", s=1, n=2708, groups=4, cg=4, dtype="fp32", act="silu", p=0.5, train=True),
        # the 16 evaluation graphs as one batch, odd group width (12 groups of 5)
        dict(gn, name="gn_eval16_odd", s=16, n=2708, groups=12, cg=5, dtype="fp16", act="relu", p=0.0, train=False),
        # 8 graph samples of the 20 000-node problem, a wide hidden layer: forward
        dict(gn, name="gn_wide_fwd", s=8, n=20000, groups=32, cg=8, dtype="bf16", act="silu", p=0.0, train=False),
        # ... and one training pass of it
        dict(gn, name="gn_wide_train", s=8, n=20000, groups=32, cg=8, dtype="bf16", act="silu", p=0.1, train=True),
        # dropout of the raw Cora features (odd row length)
        dict(dr, name="drop_features", rows=2708, cols=1433, dtype="fp32", p=0.5, residual=False, train=False),
        # a residual block's dropout in training, odd width, fp16
        dict(dr, name="drop_res_train", rows=20000, cols=257, dtype="fp16", p=0.1, residual=True, train=True),
        # the largest: 8 samples x 20 000 nodes x 512 channels, residual added
        dict(dr, name="drop_res_wide", rows=160000, cols=512, dtype="bf16", p=0.1, residual=True, train=False),
        # one node through a wide layer: the weights' bytes
        dict(i8, name="i8_node", m=1, k=4096, n=4096, dtype="bf16", dynamic=True, features=False),
        # X W of the Cora classifier's first layer in evaluation (sparse features, some rows empty)
        dict(i8, name="i8_cora", m=2708, k=1433, n=16, dtype="fp32", dynamic=True, features=True),
        # a mini-batch of nodes, odd sizes, quantised by the caller
        dict(i8, name="i8_batch_odd", m=333, k=1031, n=1000, dtype="fp16", dynamic=False, features=False),
        # every node of the 20 000-node problem through a wide layer
        dict(i8, name="i8_wide", m=20000, k=4096, n=4096, dtype="bf16", dynamic=True, features=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["group_norm", "dropout", "int8"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    p = rng.choice([0.0, 0.1, 0.5, round(rng.uniform(0.05, 0.95), 3)])
    if op == "group_norm":
        cg, groups = rng.choice([1, 2, 3, 4, 5, 7, 8, 8, 12, 16, 16, 32, 64]), rng.randint(1, 32)
        s = rng.randint(1, 16)
        cap = 40960000 // SIZE[dtype] * 2 // (s * cg * groups)
        train = rng.random() < 0.5
        return dict(op=op, s=s, n=_log(rng, 1, max(1, min(20000, cap))), groups=groups, cg=cg, dtype=dtype,
                    act=rng.choice(["none", "silu"] if train else ["none", "relu", "silu"]), p=p, train=train)
    if op == "dropout":
        cols = _log(rng, 1, 2048)
        rows = _log(rng, 1, max(1, min(160000, 81920000 // SIZE[dtype] * 2 // cols // 3)))
        return dict(op=op, rows=rows, cols=cols, dtype=dtype, p=p, residual=rng.random() < 0.6,
                    train=rng.random() < 0.5)
    return dict(op=op, m=_log(rng, 1, 20000), k=_log(rng, 16, 4096), n=_log(rng, 7, 4096), dtype=dtype,
                dynamic=rng.random() < 0.6, features=rng.random() < 0.3)


def work(case):
    b = SIZE[case["dtype"]]
    if case["op"] == "group_norm":
        c = case["groups"] * case["cg"]
        e = case["s"] * case["n"] * c
        passes = 4 if case["train"] else 2  # x, y (and dy, dx)
        return {"bytes": passes * e * b + (4 if case["train"] else 2) * c * 4,
                "flops": e * (24 if case["train"] else 10)}
    if case["op"] == "dropout":
        e = case["rows"] * case["cols"]
        passes = 2 + int(case["residual"]) + (2 if case["train"] else 0)  # x, residual, y (and dy, dx)
        return {"bytes": passes * e * b, "flops": e * (4 if case["train"] else 2)}
    m, k, n = case["m"], case["k"], case["n"]
    x = m * k * b if case["dynamic"] else m * k + 4 * m
    return {"bytes": x + n * k + 4 * n + 4 * n + m * n * b, "flops": 2 * m * n * k}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lds-gnn_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from ldsgnn import ops
    return ops


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, dtype=torch.float32, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).add_(shift).to(dtype)

    dt = DTYPES[case["dtype"]]
    key = (0x9E3779B97F4A7C15 ^ (seed * 2654435761 & 0xFFFFFFFF), (3 << 24) | (seed & 0xFFFF), seed % 1000)
    if case["op"] == "group_norm":
        s, n, c = case["s"], case["n"], case["groups"] * case["cg"]
        st = dict(x=randn(s, n, c, dtype=dt, scale=1.5, shift=0.3), w=randn(c, scale=0.3, shift=1.0),
                  b=randn(c, scale=0.3), key=key)
        if case["train"]:
            st["dy"] = randn(s, n, c, dtype=dt)
        return st
    if case["op"] == "dropout":
        r, c = case["rows"], case["cols"]
        st = dict(x=randn(r, c, dtype=dt), key=key)
        if case["residual"]:
            st["res"] = randn(r, c, dtype=dt)
        if case["train"]:
            st["dy"] = randn(r, c, dtype=dt)
        return st
    m, k, n = case["m"], case["k"], case["n"]
    if case["features"]:  # bag of words, rows divided by their sums; some rows empty
        x = (torch.rand(m, k, generator=g, device="cuda") < 0.0127).float()
        x = (x / x.sum(1, keepdim=True).clamp(min=1.0)).to(dt)
    else:
        x = randn(m, k, dtype=dt)
    wq, ws = _quantize(randn(n, k, scale=1.0 / math.sqrt(k)))
    st = dict(x=x, wq=wq.to(torch.int8), ws=ws, b=randn(n, scale=0.1))
    if not case["dynamic"]:
        q, sx = _quantize(x)
        st.update(x=None, xq=q.to(torch.int8), sx=sx)
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    if own:
        st["ops"] = _ops()
        if case["op"] == "int8":
            # the weights laid out once; activations are new at every call, which lays them out itself
            st["wq"] = st["ops"].int8_rows(st["wq"])
        elif case["train"]:
            for name in ("x", "w", "b", "res"):
                if name in st:
                    st[name].requires_grad_(True)
    return st


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------


def _mask(key, rows, cols, p):
    """keep / (1 - p) of a rows x cols block: Philox4x32-10 with the key's two
    halves and the counter (column, row >> 2, tag, counter); u = the top 24 bits
    of word row & 3; kept where u < 1 - p, in fp32."""
    seed, tag, counter = key
    low = 0xFFFFFFFF
    quads = (rows + 3) // 4
    dev = "cuda"
    c0 = torch.arange(cols, device=dev, dtype=torch.int64).expand(quads, cols)
    c1 = torch.arange(quads, device=dev, dtype=torch.int64)[:, None].expand(quads, cols)
    c2 = torch.full((1, 1), tag & low, device=dev, dtype=torch.int64)
    c3 = torch.full((1, 1), counter & low, device=dev, dtype=torch.int64)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # low 64 bits; the shift below is masked to the high word
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([w.expand(quads, cols) for w in (c0, c1, c2, c3)], 1).reshape(4 * quads, cols)[:rows]
    keep = np.float32(1.0) - np.float32(p)
    u = (words >> 8).float() * (1.0 / 16777216.0)
    return (u < float(keep)), float(np.float32(1.0) / keep)


def _drop(v, mask):
    return v if mask is None else torch.where(mask[0].view(v.shape), v * mask[1], torch.zeros_like(v))


def _group_norm(st, eps=1e-5):
    case, x0 = st["case"], st["x"]
    s, n, g, cg = case["s"], case["n"], case["groups"], case["cg"]
    dt = x0.dtype
    x = x0.float().view(s, n, g, cg)
    w, b = st["w"].view(g, cg), st["b"].view(g, cg)
    mu = x.mean((1, 3), keepdim=True)
    d = x - mu
    r = 1.0 / ((d * d).mean((1, 3), keepdim=True) + eps).sqrt()
    xh = d * r
    z = xh * w + b
    mask = None if case["p"] == 0.0 else _mask(st["key"], s * n, g * cg, case["p"])
    act = case["act"]  # relu in forward cases only
    sig = 1.0 / (1.0 + torch.exp(-z)) if act == "silu" else None
    y = {"none": lambda: z, "relu": lambda: torch.where(z > 0, z, torch.zeros_like(z)),
         "silu": lambda: z * sig}[act]()
    y = _drop(y, mask).to(dt).view(s, n, g * cg)
    if not case["train"]:
        return y
    h = _drop(st["dy"].float().view(s, n, g, cg), mask)
    if act == "silu":
        h = h * (sig * (1.0 + z * (1.0 - sig)))
    db = h.sum((0, 1)).view(-1)
    dw = (h * xh).sum((0, 1)).view(-1)
    v = h * w
    dx = r * (v - v.mean((1, 3), keepdim=True) - xh * (v * xh).mean((1, 3), keepdim=True))
    return y, dx.to(dt).view(s, n, g * cg), dw, db


def _dropout(st):
    case, x = st["case"], st["x"]
    mask = None if case["p"] == 0.0 else _mask(st["key"], case["rows"], case["cols"], case["p"])
    y = _drop(x.float(), mask)
    if case["residual"]:
        y = y + st["res"].float()
    y = y.to(x.dtype)
    if not case["train"]:
        return y
    dx = _drop(st["dy"].float(), mask).to(x.dtype)
    return (y, dx, st["dy"]) if case["residual"] else (y, dx)


def _quantize(x):
    """Rows to 8 bits: scale = max|x| / 127 in fp32, q = x / scale rounded to
    even.  In 64 bits, so that quotients next to a half fall on the right side."""
    amax = x.float().abs().amax(1)
    scale = (amax.double() / 127.0).float()
    q = torch.round(x.double() / scale.double().clamp(min=1e-300)[:, None])
    return torch.where(scale[:, None] > 0, q, torch.zeros_like(q)), scale


def _int8(st):
    case = st["case"]
    if case["dynamic"]:
        q, sx = _quantize(st["x"])
    else:
        q, sx = st["xq"].double(), st["sx"]
    acc = q @ st["wq"].double().t()  # whole numbers past 2^24: 64 bits hold them
    y = acc.float() * sx[:, None] * st["ws"][None, :] + st["b"][None, :]
    return y.to(DTYPES[case["dtype"]])


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(state):
    case = state["case"]
    if not own:
        return {"group_norm": _group_norm, "dropout": _dropout, "int8": _int8}[case["op"]](state)
    ops = state["ops"]
    if case["op"] == "group_norm":
        x, w, b = state["x"], state["w"], state["b"]
        y = ops.group_norm_act(x, case["groups"], w, b, act=case["act"], p=case["p"],
                               key=state["key"] if case["p"] > 0.0 else None)
        if not case["train"]:
            return y
        return (y,) + torch.autograd.grad(y, (x, w, b), state["dy"])
    if case["op"] == "dropout":
        x, res = state["x"], state.get("res")
        y = ops.keyed_dropout(x, case["p"], state["key"], residual=res)
        if not case["train"]:
            return y
        return (y,) + torch.autograd.grad(y, (x,) if res is None else (x, res), state["dy"])
    if case["dynamic"]:
        return ops.int8_linear(state["x"], state["wq"], state["ws"], state["b"])
    return ops.int8_matmul(state["xq"], state["sx"], state["wq"], state["ws"], state["b"],
                           out_dtype=DTYPES[case["dtype"]])


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------


def _keep64(key, rows, cols, p):
    """The kept elements, on the host in unsigned 64-bit arithmetic, one column
    block at a time."""
    seed, tag, counter = key
    m32 = np.uint64(0xFFFFFFFF)
    quads = (rows + 3) // 4
    out = np.empty((quads, 4, cols), dtype=bool)
    limit = np.uint64(math.ceil(float(np.float32(1.0) - np.float32(p)) * (1 << 24)))  # u < keep, in 2^-24 steps
    step = max(1, (1 << 22) // max(cols, 1))
    for q0 in range(0, quads, step):
        q1 = min(quads, q0 + step)
        c = [np.broadcast_to(np.arange(cols, dtype=np.uint64), (q1 - q0, cols)),
             np.broadcast_to(np.arange(q0, q1, dtype=np.uint64)[:, None], (q1 - q0, cols)),
             np.full((q1 - q0, cols), tag, dtype=np.uint64), np.full((q1 - q0, cols), counter, dtype=np.uint64)]
        k = [np.uint64(seed & 0xFFFFFFFF), np.uint64(seed >> 32 & 0xFFFFFFFF)]
        for _ in range(10):
            pa, pb = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
            c = [(pb >> np.uint64(32)) ^ c[1] ^ k[0], pb & m32, (pa >> np.uint64(32)) ^ c[3] ^ k[1], pa & m32]
            k = [(k[0] + np.uint64(0x9E3779B9)) & m32, (k[1] + np.uint64(0xBB67AE85)) & m32]
        for i in range(4):
            out[q0:q1, i] = (c[i] >> np.uint64(8)) < limit
    return torch.from_numpy(out.reshape(4 * quads, cols)[:rows]).cuda()


def _scaled64(v, keep, p):
    return v if keep is None else torch.where(keep, v * float(np.float32(1.0) / (np.float32(1.0) - np.float32(p))), 0.0)


def exact(case, seed):
    st = _inputs(case, seed)
    if case["op"] == "int8":
        if case["dynamic"]:
            x = st["x"].double()
            sx = (x.abs().max(dim=1).values / 127.0).float().double()
            t = x / torch.where(sx > 0, sx, torch.ones_like(sx))[:, None]
            f = t.floor()
            up = (t - f > 0.5) | ((t - f == 0.5) & (f % 2 != 0))
            q = torch.where(sx[:, None] > 0, f + up, torch.zeros_like(t))
        else:
            q, sx = st["xq"].double(), st["sx"].double()
        out = torch.empty(case["m"], case["n"], dtype=torch.float64, device="cuda")
        wt = st["wq"].double() * st["ws"].double()[:, None]
        for i in range(0, case["m"], 4096):
            out[i:i + 4096] = torch.addmm(st["b"].double(), q[i:i + 4096] * sx[i:i + 4096, None], wt.t())
        return out
    rows, cols = (case["rows"], case["cols"]) if case["op"] == "dropout" else \
        (case["s"] * case["n"], case["groups"] * case["cg"])
    keep = _keep64(st["key"], rows, cols, case["p"]) if case["p"] > 0.0 else None
    if case["op"] == "dropout":
        y = _scaled64(st["x"].double(), keep, case["p"])
        if case["residual"]:
            y = y + st["res"].double()
        if not case["train"]:
            return y
        dy = st["dy"].double()
        dx = _scaled64(dy, keep, case["p"])
        return (y, dx, dy) if case["residual"] else (y, dx)
    s, n, g, cg = case["s"], case["n"], case["groups"], case["cg"]
    c = g * cg
    y = torch.empty(s, n, c, dtype=torch.float64, device="cuda")
    dx = torch.empty_like(y) if case["train"] else None
    dw, db = torch.zeros(c, dtype=torch.float64, device="cuda"), torch.zeros(c, dtype=torch.float64, device="cuda")
    for i in range(s):  # one sample at a time; the gradient by differentiation
        x = st["x"][i].double().requires_grad_(case["train"])
        w, b = (t.double().requires_grad_(case["train"]) for t in (st["w"], st["b"]))
        v, m = torch.var_mean(x.reshape(n, g, cg).transpose(0, 1).reshape(g, -1), dim=1, unbiased=False)
        z = (x - m.repeat_interleave(cg)) * (v + 1e-5).rsqrt().repeat_interleave(cg) * w + b
        a = {"none": lambda t: t, "relu": torch.relu, "silu": lambda t: t * torch.sigmoid(t)}[case["act"]](z)
        out = _scaled64(a, None if keep is None else keep[i * n:(i + 1) * n], case["p"])
        y[i] = out.detach()
        if case["train"]:
            gx, gw, gb = torch.autograd.grad(out, (x, w, b), st["dy"][i].double())
            dx[i] = gx
            dw += gw
            db += gb
    return (y, dx, dw, db) if case["train"] else y
