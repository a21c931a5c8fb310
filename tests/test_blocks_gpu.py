"""The block operators (ldsgnn.ops: keyed_dropout with a residual and in 16-bit
types, group_norm_act, quantize_rows / int8_matmul / int8_linear) against plain
implementations in 64 bits.

Tolerances.  u = 2^-24 is fp32's largest relative rounding error, h(t) that of
the output type (fp32 2^-24, bf16 2^-8, fp16 2^-11; fp16 results below its
smallest normal number are off by up to 2^-25).  They are derived per operator
at its test.
"""
import numpy as np
import pytest
import torch

from oracle import philox

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
KEY = (0x1234567890ABCDEF, (3 << 24) | 5, 77)


@pytest.fixture(scope="module")
def ops():
    from ldsgnn import ops
    return ops


def mask64(key, rows, cols, p):
    """(kept, 1 / (1 - p)) of a rows x cols block; the scale is the fp32 one."""
    keep = np.float32(1.0) - np.float32(p)
    u = philox.uniform(key[0], key[1], key[2], rows, cols)
    scale = float(np.float32(1.0) / keep) if keep > 0 else 0.0
    return torch.from_numpy(u < keep), scale


def dropped64(x, key, p):
    rows, cols = x.numel() // x.shape[-1], x.shape[-1]
    if p == 0.0:
        return x
    kept, scale = mask64(key, rows, cols, p)
    return torch.where(kept.view(x.shape), x * scale, torch.zeros_like(x))


# ---------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------


def plain_dropout(x, key, p, res=None):
    """fp32 as the definition has it: x·scale, + residual, one rounding to the
    type.  Every step is one IEEE operation, so the kernel has the same bits."""
    y = x.float()
    if p > 0.0:
        kept, scale = mask64(key, x.numel() // x.shape[-1], x.shape[-1], p)
        y = torch.where(kept.view(x.shape), y * np.float32(scale), torch.zeros_like(y))
    if res is not None:
        y = y + res.float()
    return y.to(x.dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (1, 1), (3, 5), (4, 8), (37, 50), (2, 3, 33), (5, 1), (1025, 17),
                                   (64, 1433), (2, 2, 3, 16)])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout_add_has_the_definition_bits(device, ops, dtype, shape, residual):
    g = torch.Generator().manual_seed(sum(shape))
    x = torch.randn(shape, generator=g).to(dtype)
    res = torch.randn(shape, generator=g).to(dtype) if residual else None
    for p in (0.0, 0.1, 0.5, 1.0):
        y = ops.keyed_dropout(x.to(device), p, KEY, residual=None if res is None else res.to(device))
        assert y.dtype == dtype and torch.equal(y.cpu(), plain_dropout(x, KEY, p, res)), p


def test_dropout_strides_and_copies(device, ops):
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(6, 40, 70, generator=g).to(torch.bfloat16)
    for cut in (lambda t: t[:, :, 3:36], lambda t: t[:, ::2, :], lambda t: t[1::2, 5:7, 1:2],
                lambda t: t.transpose(1, 2), lambda t: t[:, :, ::3], lambda t: t[0, :1, :1].expand(9, 13),
                lambda t: t[0, 0].expand(5, 70)):
        x, r = cut(wide), cut(wide.neg())
        y = ops.keyed_dropout(cut(wide.to(device)), 0.3, KEY, residual=cut(wide.neg().to(device)))
        assert torch.equal(y.cpu(), plain_dropout(x.contiguous(), KEY, 0.3, r.contiguous()))


def test_dropout_of_nan_and_infinity(device, ops):
    """A dropped element is 0 (plus the residual) whatever x holds there."""
    x = torch.full((8, 33), float("nan"))
    x[::2] = float("inf")
    res = torch.ones(8, 33)
    y = ops.keyed_dropout(x.to(device), 0.5, KEY, residual=res.to(device)).cpu()
    kept, _ = mask64(KEY, 8, 33, 0.5)
    assert torch.equal(y[~kept], torch.ones_like(y[~kept]))
    assert torch.isnan(y[1::2][kept[1::2]]).all() and torch.isinf(y[::2][kept[::2]]).all()


@pytest.mark.parametrize("shape", [(0, 5), (5, 0), (0,), (2, 0, 3)])
def test_dropout_empty(device, ops, shape):
    x = torch.empty(shape, device=device, requires_grad=True)
    y = ops.keyed_dropout(x, 0.5, KEY, residual=torch.empty(shape, device=device))
    y.sum().backward()
    assert y.shape == x.shape == x.grad.shape


@pytest.mark.parametrize("dtype", DTYPES)
def test_dropout_gradients(device, ops, dtype):
    """dx = the same mask on dy (the definition's bits), dres = dy; the second
    order is the mask again; a broadcast residual's gradient is summed by its
    own expansion."""
    g = torch.Generator().manual_seed(9)
    x, dy = (torch.randn(41, 27, generator=g).to(dtype) for _ in range(2))
    r = torch.randn(27, generator=g).to(dtype)
    xd, rd = x.to(device).requires_grad_(), r.to(device).requires_grad_()
    y = ops.keyed_dropout(xd, 0.25, KEY, residual=rd.expand(41, 27))
    gx, gr = torch.autograd.grad(y, (xd, rd), dy.to(device), create_graph=True)
    assert torch.equal(gx.detach().cpu(), plain_dropout(dy, KEY, 0.25))
    assert torch.allclose(gr.detach().cpu().double(), dy.double().sum(0), rtol=41 * HALF[dtype], atol=41 * HALF[dtype])
    w = torch.randn(41, 27, generator=g).to(dtype).to(device).requires_grad_()
    xw = xd.detach().requires_grad_()
    y2 = ops.keyed_dropout(xw, 0.25, KEY)
    (g1,) = torch.autograd.grad(y2, xw, w, create_graph=True)
    (g2,) = torch.autograd.grad(g1, w, dy.to(device))
    assert torch.equal(g2.cpu(), plain_dropout(dy, KEY, 0.25))


def test_dropout_of_operands_that_fill_the_cache(device, ops):
    """Three operands of 96 MB are read past the memory-side cache, two are not:
    in fp32 the residual's sum is one IEEE operation, so both have the same bits."""
    g = torch.Generator(device=device).manual_seed(12)
    x, r = (torch.randn(46003, 521, generator=g, device=device) for _ in range(2))
    both = ops.keyed_dropout(x, 0.3, KEY, residual=r)
    alone = ops.keyed_dropout(x, 0.3, KEY)
    assert torch.equal(both, alone + r)
    assert torch.equal(alone[:64].cpu(), plain_dropout(x[:64].cpu(), KEY, 0.3))
    assert torch.equal(ops.keyed_dropout(x, 0.0, None, residual=r), x + r)


@pytest.mark.parametrize("cols", [1, 3, 4, 5, 7, 8, 257])
def test_dropout_in_place(device, cols):
    """lds_dropout over its own input, and into a block that begins inside it:
    what two threads read of a row's last vector is not what the other wrote."""
    from ldsgnn import _native as nat
    g = torch.Generator().manual_seed(cols)
    x = torch.randn(1031, cols, generator=g)
    want = plain_dropout(x, KEY, 0.5)
    y = x.to(device)
    nat.call("lds_dropout", y.data_ptr(), cols, y.data_ptr(), cols, 1031, cols, 0.5, 2.0, *KEY, nat.stream_of(y.device))
    assert torch.equal(y.cpu(), want)
    wide = torch.full((1031, 2 * cols + 1), 7.0)  # input and result side by side in one block's rows
    wide[:, :cols] = x
    wide = wide.to(device)
    nat.call("lds_dropout", wide.data_ptr(), 2 * cols + 1, wide.data_ptr() + 4 * (cols + 1), 2 * cols + 1, 1031, cols,
             0.5, 2.0, *KEY, nat.stream_of(wide.device))
    assert torch.equal(wide[:, cols + 1:].cpu(), want) and torch.equal(wide[:, :cols].cpu(), x)
    assert (wide[:, cols] == 7.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_dropout_gradients_without_a_mask(device, ops, dtype):
    """p = 0: dx = dres = dy, at both orders, and each leaf's gradient has memory
    of its own (adding to one leaves the other and dy as they were)."""
    g = torch.Generator().manual_seed(10)
    x, r, dy = (torch.randn(13, 9, generator=g).to(dtype).to(device) for _ in range(3))
    x.requires_grad_(), r.requires_grad_()
    y = ops.keyed_dropout(x, 0.0, None, residual=r)
    assert torch.equal(y, (x.float() + r.float()).to(dtype))
    given = dy.clone()
    y.backward(dy)
    assert torch.equal(x.grad, given) and torch.equal(r.grad, given)
    x.grad.add_(1.0)
    assert torch.equal(r.grad, given) and torch.equal(dy, given)
    w = dy.clone().requires_grad_()
    (g1,) = torch.autograd.grad(ops.keyed_dropout(x, 0.0, None), x, w, create_graph=True)
    (g2,) = torch.autograd.grad(g1, w, given)
    assert torch.equal(g1, given) and torch.equal(g2, given)


def test_dropout_entries_at_the_ends(device):
    """lds_dropout and lds_dropout_add take the scale at its word: keep 1 scales
    every element, keep 0 leaves none; lds_dropout takes any keep."""
    from ldsgnn import _native as nat
    x = torch.randn(9, 21, device=device)
    y = torch.empty_like(x)
    st = nat.stream_of(x.device)
    for keep, ref in ((1.0, x * 3), (0.0, x * 0), (1.5, x * 3), (-0.5, x * 0)):
        nat.call("lds_dropout", x.data_ptr(), 21, y.data_ptr(), 21, 9, 21, keep, 3.0, 1, 2, 3, st)
        assert torch.equal(y, ref), keep
        if 0.0 <= keep <= 1.0:
            nat.call("lds_dropout_add", x.data_ptr(), 21, 0, 0, y.data_ptr(), 21, 9, 21, 0, keep, 3.0, 1, 2, 3, st)
            assert torch.equal(y, ref), keep


def test_offsets_past_32_bits(device, ops):
    """More than 2^31 elements: the last rows are the definition's."""
    rows, cols = 70001, 32768
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=device)
    x.copy_(torch.arange(cols, device=device).remainder(251).to(torch.bfloat16)[None, :])
    y = ops.keyed_dropout(x, 0.5, KEY, residual=x)
    tail = 5  # rows 69996 ..: the mask of the last two row quads
    c = np.arange(cols)
    ref = torch.empty(tail, cols)
    for i in range(tail):
        r = rows - tail + i
        w = philox.philox4x32_10(c, r >> 2, KEY[1], KEY[2], KEY[0] & 0xFFFFFFFF, KEY[0] >> 32)[r & 3]
        kept = torch.from_numpy((w >> np.uint64(8)).astype(np.float64) * 2.0 ** -24 < 0.5)
        xr = x[r].cpu().float()
        ref[i] = torch.where(kept, xr * 2, torch.zeros_like(xr)) + xr
    assert torch.equal(y[-tail:].cpu(), ref.to(torch.bfloat16))
    del y
    # group norm: the last group of the last sample; its gradient of ones through a constant is 0
    x3 = x[:70000].view(2, 35000, cols)
    x3[1, :, -64:] = torch.randn(35000, 64, device=device).to(torch.bfloat16)
    z = ops.group_norm_act(x3, cols // 64, act="silu")
    v = x3[1, :, -64:].double()
    zr = (v - v.mean()) / (v.var(unbiased=False) + 1e-5).sqrt()
    ref = zr * torch.sigmoid(zr)
    assert ((z[1, :, -64:].double() - ref).abs() <= HALF[torch.bfloat16] * ref.abs() + 1e-5).all()
    stats = ops._norm_forward(x3, None, None, ops._NormPlan(cols // 64, 2, 1e-5, 1.0, 1.0, None))[1]
    del z
    dy = torch.ones_like(x3)
    dx, _, _ = ops._norm_backward(dy, x3, None, None, stats, ops._NormPlan(cols // 64, 0, 1e-5, 1.0, 1.0, None),
                                  (True, False, False))
    # h = 1: dx = r (1 - 1 - x̂ mean(x̂)), which is 0 to the roundings of the two means
    assert float(dx[1, :, -64:].abs().max()) <= 1e-4
    del dx, dy, x3, x
    a = torch.randint(-127, 128, (rows, 64), dtype=torch.int8, device=device)
    b = torch.randint(-127, 128, (cols, 64), dtype=torch.int8, device=device)
    one = torch.ones(rows, device=device)
    p = ops.int8_matmul(a, one, b, one[:cols], out_dtype=torch.bfloat16)
    ref = a[-300:].double() @ b.double().t()
    assert torch.equal(p[-300:], ref.float().to(torch.bfloat16))


@pytest.mark.parametrize("samples,groups,cg,dtype", [(70_000_001, 1, 8, torch.bfloat16),
                                                     (25_000_003, 3, 2, torch.float16)])
def test_group_norm_of_more_samples_than_a_launch_holds(device, ops, samples, groups, cg, dtype):
    """Single nodes as samples, whose blocks have more than 2^32 threads, with a
    sample's groups in one block and across blocks: y and dx, from the first
    sample to the last, against 64 bits."""
    c = groups * cg
    g = torch.Generator(device=device).manual_seed(5)
    x = torch.randn(samples, 1, c, generator=g, device=device, dtype=dtype)
    dy = torch.randn(samples, 1, c, generator=g, device=device, dtype=dtype)
    pl = ops._NormPlan(groups, ops.ACTIVATIONS["silu"], 1e-5, 1.0, 1.0, None)
    y, stats = ops._norm_forward(x, None, None, pl)
    dx = ops._norm_backward(dy, x, None, None, stats, pl, (True, False, False))[0]
    pick = torch.cat([torch.randint(0, samples, (5000,), generator=g, device=device),
                      torch.arange(samples - 100, samples, device=device), torch.arange(100, device=device)])
    xs, ds = x[pick].cpu(), dy[pick].cpu()
    one, zero = torch.ones(c).double(), torch.zeros(c).double()
    ref, z = norm64(xs.double(), groups, None, None, "silu", 1e-5, KEY, 0.0)
    dz, _, _ = norm_bounds(xs.double(), groups, None, None, 1e-5)
    tol = HALF[dtype] * ref.abs() + TINY[dtype] + 1.1 * dz + 8 * U * z.abs()
    assert ((y[pick].cpu().double() - ref).abs() <= tol).all()
    rx = norm_grads64(xs, groups, one, zero, "silu", 0.0, ds)[0][0]
    tx = grad_bounds(xs, groups, one, zero, "silu", 0.0, ds)[0]
    assert ((dx[pick].cpu().double() - rx).abs() <= HALF[dtype] * rx.abs() + TINY[dtype] + tx).all()


def test_quantize_more_rows_than_a_launch_holds(device, ops):
    """300 million rows of one value: q = 127 times its sign, scale = |x| / 127 (in 64
    bits, then rounded: torch divides an fp32 tensor by a number as a product with
    the number's rounded reciprocal.  A quotient by 127 is 2^-32 or more of itself
    away from the middle of two fp32 values, 64 bits err by 2^-52.)"""
    x = torch.rand(300_000_001, 1, device=device).sub_(0.5)
    q, s = ops.quantize_rows(x)
    for i in range(0, x.size(0), 50_000_000):
        v = x[i:i + 50_000_000, 0]
        assert torch.equal(q[i:i + 50_000_000, 0].float(), v.sign() * 127)
        assert torch.equal(s[i:i + 50_000_000], (v.abs().double() / 127).float())


def test_int8_linear_of_more_columns_than_a_launch_holds(device, ops):
    """One row times 135 million rows of w: the one-launch form would need more
    than 2^32 threads."""
    n, k = 135_000_003, 16
    wq = torch.randint(-127, 128, (n, k), dtype=torch.int8, device=device)
    x = torch.arange(k, device=device).float().sub_(8)[None]
    x[0, 3] = 127
    with torch.no_grad():
        y = ops.int8_linear(x, wq, torch.ones(1, device=device).expand(n))
    for i in range(0, n, 20_000_000):
        assert torch.equal(y[0, i:i + 20_000_000], (wq[i:i + 20_000_000].float() * x).sum(1))


# ---------------------------------------------------------------------------
# group norm + activation
# ---------------------------------------------------------------------------


def norm64(x, groups, w, b, act, eps, key, p):
    c = x.shape[-1]
    v = x.reshape(-1, x.shape[-2], groups, c // groups)
    d = v - v.mean((1, 3), keepdim=True)
    r = 1.0 / (d.square().mean((1, 3), keepdim=True) + eps).sqrt()
    z = (d * r).reshape(x.shape)
    if w is not None:
        z = z * w
    if b is not None:
        z = z + b
    a = torch.relu(z) if act == "relu" else z * torch.sigmoid(z) if act == "silu" else z
    return dropped64(a, key, p), z


def norm_bounds(x64, groups, w, b, eps):
    """Per element, how far the kernel's fp32 z may be from z in 64 bits:
    mean is rounded once and comes from sums good to a few u of the values
    about it, so x - mean is off by u (|mean| + 4 sd + |x - mean|) and x̂ by r
    times that and 6 u |x̂| (rstd's own error and two roundings); the product
    with γ and the sum with β round once more each.  Doubled for the sums."""
    c = x64.shape[-1]
    v = x64.reshape(-1, x64.shape[-2], groups, c // groups)
    mu = v.mean((1, 3), keepdim=True)
    d = v - mu
    var = d.square().mean((1, 3), keepdim=True)
    r = 1.0 / (var + eps).sqrt()
    xe = (r * (mu.abs() + 4 * var.sqrt() + d.abs()) + 6 * (d * r).abs()) * U
    wabs = 1.0 if w is None else w.abs()
    z = (d * r).abs().reshape(x64.shape) * wabs
    babs = 0.0 if b is None else b.abs()
    return 2 * (xe.reshape(x64.shape) * wabs + 2 * U * (z + babs)), r, (d * r).reshape(x64.shape)


NORM_SHAPES = [  # samples, n, groups, channels per group
    (1, 1, 1, 1), (1, 1, 32, 8), (3, 1, 2, 3), (2, 7, 4, 5), (1, 5, 1, 2), (5, 33, 3, 16), (2, 100, 1, 700),
    (1, 9, 2, 4096), (1, 3, 1, 2051), (4, 515, 12, 5), (1, 2708, 4, 4), (2, 600, 32, 8), (17, 2, 300, 2),
    (9, 1501, 3, 7), (1, 9001, 2, 4), (2, 5003, 2, 16), (1, 40, 1, 8200),
    (2, 6001, 3, 7), (1, 7011, 12, 5), (3, 5001, 5, 3), (1, 4502, 4, 12), (1, 18000, 1, 9), (2, 1500, 1, 33),
]


def norm_inputs(s, n, groups, cg, dtype, seed=0, offset=0.3):
    g = torch.Generator().manual_seed(1000 * seed + 7 * n + groups + cg)
    c = groups * cg
    x = (torch.randn(s, n, c, generator=g) * 1.5 + offset).to(dtype)
    w = torch.randn(c, generator=g) * 0.3 + 1.0
    b = torch.randn(c, generator=g) * 0.3
    dy = torch.randn(s, n, c, generator=g).to(dtype)
    return x, w, b, dy


@pytest.mark.parametrize("shape", NORM_SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act,p", [("none", 0.0), ("relu", 0.5), ("silu", 0.0), ("silu", 0.1)])
def test_group_norm_forward(device, ops, shape, dtype, act, p):
    """|y - y64| <= h |y64| + scale (1.1 δz + 8 u |a|): δz the bound of
    norm_bounds, 1.1 the steepest slope of the activations, 8 u for exp, the
    reciprocal and the products of silu."""
    s, n, groups, cg = shape
    x, w, b, _ = norm_inputs(s, n, groups, cg, dtype)
    y = ops.group_norm_act(x.to(device), groups, w.to(device), b.to(device), act=act, p=p, key=KEY).cpu()
    ref, z = norm64(x.double(), groups, w.double(), b.double(), act, 1e-5, KEY, p)
    dz, _, _ = norm_bounds(x.double(), groups, w.double(), b.double(), 1e-5)
    scale = 1.0 if p == 0.0 else 1.0 / (1.0 - p)
    tol = HALF[dtype] * ref.abs() + TINY[dtype] + scale * (1.1 * dz + 8 * U * z.abs())
    assert y.dtype == dtype and y.shape == x.shape
    assert ((y.double() - ref).abs() <= tol).all()


def norm_grads64(x, groups, w, b, act, p, dy):
    leaves = [t.double().requires_grad_() for t in (x, w, b)]
    y, z = norm64(leaves[0], groups, leaves[1], leaves[2], act, 1e-5, KEY, p)
    return torch.autograd.grad(y, leaves, dy.double()), z.detach()


def grad_bounds(x, groups, w, b, act, p, dy):
    """(dx, dγ, dβ) bounds.  h = dy·scale·act'(z): act' is off by δz (its slope is
    at most 1/2 for silu, 0 else) and by 12 u (1 + |z|) of its own roundings,
    so δh <= scale |dy| (δz + 12 u (1 + |z|)) =: e, with |h| <= 1.1 scale |dy|.
    A sum of k terms in any order is within k u of the sum of their
    magnitudes; a thread adds at most n values and a block at most 256 such
    sums in a row, the rest is fp64: with x̂ off by δx̂ (norm_bounds / |γ|),
      δ(Σ h x̂) <= Σ (e |x̂| + |h| δx̂) + (n + 258) u Σ |h x̂|.
    dx = r (γ h - m1 - x̂ m2) adds the elementwise and the two means' errors and
    4 roundings."""
    s, n, c = x.shape
    cg = c // groups
    scale = 1.0 if p == 0.0 else 1.0 / (1.0 - p)
    x64, w64, b64, g = x.double(), w.double(), b.double(), dy.double().abs() * scale
    dz, r, xh = norm_bounds(x64, groups, w64, b64, 1e-5)
    dxh, _, _ = norm_bounds(x64, groups, None, None, 1e-5)
    z = (xh * w64 + b64).abs()
    e = g * (dz + 12 * U * (1 + z)) if act == "silu" else g * 2 * U
    h, xa = 1.1 * g, xh.abs()
    sh = e.sum((0, 1)) + (n + 258) * U * h.sum((0, 1))
    shx = (e * xa + h * dxh).sum((0, 1)) + (n + 258) * U * (h * xa).sum((0, 1))

    def mean(t):
        return t.reshape(s, n, groups, cg).mean((1, 3), keepdim=True).expand(s, n, groups, cg).reshape(s, n, c)

    wa = w64.abs()
    m1, m2 = mean(wa * h), mean(wa * h * xa)
    e1 = mean(wa * e) + (n + 260) * U * m1
    e2 = mean(wa * (e * xa + h * dxh)) + (n + 260) * U * m2
    rr = r.expand(s, n, groups, cg).reshape(s, n, c)
    dx = rr * (wa * e + e1 + xa * e2 + dxh * m2 + 12 * U * (wa * h + m1 + xa * m2))
    return dx, shx + U * 4 * (h * xa).sum((0, 1)), sh + U * 4 * h.sum((0, 1))


@pytest.mark.parametrize("shape", NORM_SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act,p", [("none", 0.1), ("relu", 0.5), ("silu", 0.0), ("silu", 0.1)])
def test_group_norm_backward(device, ops, shape, dtype, act, p):
    s, n, groups, cg = shape
    x, w, b, dy = norm_inputs(s, n, groups, cg, dtype, seed=1)
    if act == "relu":
        # relu's gradient jumps at 0: values nearer to it than z's own error
        # would be decided by a last bit, so those nodes' channels are moved off it
        for _ in range(20):
            _, z = norm64(x.double(), groups, w.double(), b.double(), act, 1e-5, KEY, 0.0)
            near = z.abs() < 1e-5
            if not near.any():
                break
            x[near] = x[near] * 1.125 + 0.25
        assert not near.any() or n * cg == 1
        if n * cg == 1:
            b = torch.where(b.abs() < 1e-3, torch.full_like(b, 0.5), b)
    leaves = [t.to(device).requires_grad_() for t in (x, w, b)]
    y = ops.group_norm_act(leaves[0], groups, leaves[1], leaves[2], act=act, p=p, key=KEY)
    got = torch.autograd.grad(y, leaves, dy.to(device))
    ref, _ = norm_grads64(x, groups, w, b, act, p, dy)
    tol = grad_bounds(x, groups, w, b, act, p, dy)
    for name, a, e, t, dt in zip(("dx", "dweight", "dbias"), got, ref, tol,
                                 (dtype, torch.float32, torch.float32)):
        assert a.dtype == dt, name
        err = (a.cpu().double() - e).abs() - HALF[dt] * e.abs() - TINY[dt] - t
        assert err.max() <= 0, (name, float(err.max()))


# Long rows whose vectors fill more than one block across (two or three chunks of
# whole groups, the last one shorter): 37 groups of 64 in chunks of 19 and 18 (16-bit)
# or 13, 13 and 11 (fp32); 101 of 12 in 51 and 50; 300 of 2 in two of 150.
NORM_CHUNK_SHAPES = [(2, 601, 37, 64), (1, 3001, 101, 12), (4, 1501, 300, 2)]


@pytest.mark.parametrize("shape", NORM_CHUNK_SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act,p", [("silu", 0.1), ("none", 0.5)])
def test_group_norm_in_chunks(device, ops, shape, dtype, act, p):
    from ldsgnn import _native as nat
    s, n, groups, cg = shape
    code = nat.ELEMENT_CODES[dtype]
    assert nat.lib.lds_group_norm_ws_bytes(s, n, groups * cg, groups, code, 0) > 0  # rows cut into parts
    test_group_norm_forward(device, ops, shape, dtype, act, p)
    test_group_norm_backward(device, ops, shape, dtype, act, p)


def mask_columns(key, rows, cols, p):
    """mask64 at some columns."""
    quads = np.arange((rows + 3) // 4)[:, None]
    words = philox.philox4x32_10(np.asarray(cols)[None, :], quads, key[1], key[2], key[0] & 0xFFFFFFFF, key[0] >> 32)
    u = np.stack([(w >> np.uint64(8)).astype(np.float64) * 2.0 ** -24 for w in words], 1)
    keep = np.float32(1.0) - np.float32(p)
    return torch.from_numpy(u.reshape(-1, len(cols))[:rows] < keep), float(np.float32(1.0) / keep)


@pytest.mark.parametrize("dtype,n", [(torch.bfloat16, 14001), (torch.float32, 7001)])
def test_group_norm_results_past_the_caches(device, ops, dtype, n):
    """147 MB results (y and dx are stored past the caches, x and dy read past
    them) of 41 groups of 64 in two (bf16) or three chunks: forward, dx, dγ and dβ
    of the groups at the chunks' borders against 64 bits, under the bounds of
    test_group_norm_forward and _backward."""
    s, groups, cg, p = 2, 41, 64, 0.2
    c = groups * cg
    g = torch.Generator(device=device).manual_seed(n)
    x = torch.randn(s, n, c, generator=g, device=device).mul_(1.5).add_(0.3).to(dtype).requires_grad_()
    dy = torch.randn(s, n, c, generator=g, device=device).to(dtype)
    w = torch.randn(c, generator=g, device=device).mul_(0.3).add_(1.0).requires_grad_()
    b = torch.randn(c, generator=g, device=device).mul_(0.3).requires_grad_()
    assert x.numel() * x.element_size() > 128 << 20
    y = ops.group_norm_act(x, groups, w, b, act="silu", p=p, key=KEY)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    y = y.detach()
    pick = [0, 13, 14, 20, 21, 40]
    cols = torch.cat([torch.arange(k * cg, (k + 1) * cg) for k in pick])
    kept, scale = mask_columns(KEY, s * n, cols.numpy(), p)
    kept = kept.to(device).view(s, n, -1)
    cut = [t.detach()[..., cols.to(device)] for t in (x, w, b, dy)]
    leaves = [t.double().requires_grad_() for t in cut[:3]]
    a, z = norm64(leaves[0], len(pick), leaves[1], leaves[2], "silu", 1e-5, KEY, 0.0)
    ref = torch.where(kept, a * scale, torch.zeros_like(a))
    refs = torch.autograd.grad(ref, leaves, cut[3].double())
    ref, z = ref.detach(), z.detach()
    dz, _, _ = norm_bounds(leaves[0].detach(), len(pick), leaves[1].detach(), leaves[2].detach(), 1e-5)
    tol = HALF[dtype] * ref.abs() + TINY[dtype] + 1.25 * (1.1 * dz + 8 * U * z.abs())
    assert ((y[..., cols.to(device)].double() - ref).abs() <= tol).all()
    tols = grad_bounds(cut[0], len(pick), cut[1], cut[2], "silu", p, cut[3])
    for name, got, e, t, dt in zip(("dx", "dweight", "dbias"), (dx, dw, db), refs, tols,
                                   (dtype, torch.float32, torch.float32)):
        err = (got[..., cols.to(device)].double() - e).abs() - HALF[dt] * e.abs() - TINY[dt] - t
        assert err.max() <= 0, (name, float(err.max()))


def test_group_norm_gradient_by_differences(device, ops):
    """The gradient against central differences of the kernel's own forward
    (fp32): along a random direction d, (L(x + t d) - L(x - t d)) / 2t with t = 2^-6
    differs from <grad, d> by the third derivative (order t² = 2.5e-4 relative)
    and by the forward's rounding, 2 u |L| sqrt(N) / t; 1e-2 of the gradient's
    norm times the direction's covers both."""
    x, w, b, dy = norm_inputs(2, 50, 3, 8, torch.float32, seed=2)
    g = torch.Generator().manual_seed(4)
    leaves = [t.to(device).requires_grad_() for t in (x, w, b)]

    def loss(*a):
        return (ops.group_norm_act(a[0], 3, a[1], a[2], act="silu", p=0.2, key=KEY).double() *
                dy.to(device).double()).sum()

    grads = torch.autograd.grad(loss(*leaves), leaves)
    for i, gr in enumerate(grads):
        d = torch.randn(gr.shape, generator=g).to(device)
        d = d / d.norm()
        t = 2.0 ** -6
        with torch.no_grad():
            args = [[l.detach() + (sg * t * d if j == i else 0) for j, l in enumerate(leaves)] for sg in (1, -1)]
            num = float(loss(*args[0]) - loss(*args[1])) / (2 * t)
        assert abs(num - float((gr * d).sum())) <= 1e-2 * float(gr.norm()), i


def test_group_norm_strides(device, ops):
    """Slices, transposed samples, expanded samples and gradients with other
    strides: the bits of the contiguous call."""
    g = torch.Generator().manual_seed(6)
    wide = torch.randn(4, 30, 52, generator=g).to(device)
    for cut in (lambda t: t[:, :, 4:28], lambda t: t[:, :, 3:27], lambda t: t[:, 1::3, :24], lambda t: t[::2, :, 28:],
                lambda t: t.transpose(0, 1)[:, :, :24], lambda t: t[:, :, ::2][..., :24],
                lambda t: t[:1, :, :24].expand(3, 30, 24), lambda t: t[2, :, 10:34],
                lambda t: t.view(2, 2, 30, 52)[..., :24]):
        x = cut(wide).detach()
        dy = cut(wide.cos())
        out = []
        for src, gy in ((x, dy), (x.contiguous(), dy.contiguous())):
            leaf = src.detach().requires_grad_()
            w = torch.linspace(0.5, 1.5, 24, device=device).requires_grad_()
            y = ops.group_norm_act(leaf, 4, w, None, act="silu", p=0.3, key=KEY)
            out.append((y,) + torch.autograd.grad(y, (leaf, w), gy))
        for a, b in zip(*out):
            assert torch.equal(a, b)


def test_group_norm_samples_stand_alone(device, ops):
    """A NaN or an infinity in one group of one sample reaches no other group;
    a constant group gives act(β)."""
    x, w, b, _ = norm_inputs(3, 40, 4, 8, torch.float32, seed=5)
    x[0, 3, 9] = float("nan")
    x[1, 7, 17] = float("inf")
    x[2, :, 24:] = 2.5
    y = ops.group_norm_act(x.to(device), 4, w.to(device), b.to(device), act="silu").cpu()
    ref, _ = norm64(x.double(), 4, w.double(), b.double(), "silu", 1e-5, KEY, 0.0)
    bad = torch.zeros(3, 40, 32, dtype=torch.bool)
    bad[0, :, 8:16] = True
    bad[1, :, 16:24] = True
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()
    assert torch.allclose(y[~bad].double(), ref[~bad], rtol=1e-5, atol=1e-5)
    assert torch.allclose(y[2, :, 24:], (b * torch.sigmoid(b))[24:].expand(40, 8), rtol=1e-6, atol=1e-7)


@pytest.mark.parametrize("n,cg", [(700, 8), (9000, 8), (9000, 5)])
def test_group_norm_far_from_zero(device, ops, n, cg):
    """Mean 3000 sd, one outlier among the first values: the bound of
    norm_bounds, whose term in |mean| is the mean's own last bit."""
    x, w, b, _ = norm_inputs(2, n, 2, cg, torch.float32, seed=8, offset=0.0)
    x = x / 1.5 + 3000.0
    x[:, 0, 0] = 9000.0
    y = ops.group_norm_act(x.to(device), 2, w.to(device), b.to(device)).cpu()
    ref, _ = norm64(x.double(), 2, w.double(), b.double(), "none", 1e-5, KEY, 0.0)
    dz, _, _ = norm_bounds(x.double(), 2, w.double(), b.double(), 1e-5)
    assert ((y.double() - ref).abs() <= U * ref.abs() + dz).all()


@pytest.mark.parametrize("shape", [(0, 4), (3, 0, 4), (0, 5, 4), (2, 3, 0)])
def test_group_norm_empty(device, ops, shape):
    x = torch.empty(shape, device=device, requires_grad=True)
    w = torch.ones(shape[-1], device=device, requires_grad=True)
    y = ops.group_norm_act(x, 1 if shape[-1] == 0 else 2, w, None, act="relu")
    y.sum().backward()
    assert y.shape == x.shape and x.grad.shape == x.shape and float(w.grad.sum()) == 0.0


@pytest.mark.parametrize("shape,groups", [((0, 3, 4), 2), ((2, 0, 4), 2), ((2, 3, 0), 1), ((0, 4), 4)])
def test_group_norm_second_order_of_an_empty_tensor(device, ops, shape, groups):
    from tests.test_blocks_cpu import check_empty_second_order
    check_empty_second_order(lambda x, w, b: ops.group_norm_act(x, groups, w, b, act="silu", p=0.5, key=KEY), shape,
                             groups, device)


@pytest.mark.parametrize("weight,bias", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("pdtype", DTYPES)
def test_group_norm_parameter_forms(device, ops, weight, bias, pdtype):
    x, w, b, dy = norm_inputs(2, 19, 2, 6, torch.bfloat16, seed=3)
    w, b = (w.to(pdtype) if weight else None), (b.to(pdtype) if bias else None)
    wd = None if w is None else w.to(device).requires_grad_()
    bd = None if b is None else b.to(device).requires_grad_()
    xd = x.to(device).requires_grad_()
    y = ops.group_norm_act(xd, 2, wd, bd, act="silu")
    got = torch.autograd.grad(y, [t for t in (xd, wd, bd) if t is not None], dy.to(device))
    w64 = torch.ones(12).double() if w is None else w.double()
    b64 = torch.zeros(12).double() if b is None else b.double()
    ref, _ = norm_grads64(x, 2, w64, b64, "silu", 0.0, dy)
    tol = grad_bounds(x, 2, w64, b64, "silu", 0.0, dy)
    rows = [0] + ([1] if weight else []) + ([2] if bias else [])
    for a, i in zip(got, rows):
        assert a.dtype == (torch.bfloat16 if i == 0 else pdtype)
        assert ((a.cpu().double() - ref[i]).abs() <= HALF[a.dtype] * (ref[i].abs() + tol[i]) + tol[i] +
                TINY[a.dtype]).all()


@pytest.mark.parametrize("act,p", [("none", 0.0), ("silu", 0.3), ("relu", 0.0)])
def test_group_norm_second_order(device, ops, act, p):
    """create_graph: the gradient's own gradient against 64-bit autograd.  It
    is composed of fp32 operations; 2e-4 of the largest entry covers their
    few hundred roundings (about 300 u) with the amplification of 1/sd."""
    x, w, b, dy = norm_inputs(2, 15, 2, 4, torch.float32, seed=6)
    g = torch.Generator().manual_seed(1)
    cots = [torch.randn(t.shape, generator=g) for t in (x, w, b)]
    out = []
    for dev, dt in ((device, torch.float32), ("cpu", torch.float64)):
        leaves = [t.to(dev, dt).requires_grad_() for t in (dy, x, w, b)]
        if dev == "cpu":
            y, _ = norm64(leaves[1], 2, leaves[2], leaves[3], act, 1e-5, KEY, p)
        else:
            y = ops.group_norm_act(leaves[1], 2, leaves[2], leaves[3], act=act, p=p, key=KEY)
        first = torch.autograd.grad(y, leaves[1:], leaves[0], create_graph=True)
        total = sum((f * c.to(dev, dt)).sum() for f, c in zip(first, cots))
        out.append(torch.autograd.grad(total, leaves, allow_unused=True))
    for a, e in zip(*out):
        if e is None:
            assert a is None or float(a.abs().max()) == 0.0
            continue
        assert (a.cpu().double() - e).abs().max() <= 2e-4 * max(1.0, float(e.abs().max()))


def test_group_norm_equal_calls_equal_bits(device, ops):
    x, w, b, dy = (t.to(device) for t in norm_inputs(3, 4001, 8, 16, torch.bfloat16, seed=4))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    runs = []
    for _ in range(3):
        y = ops.group_norm_act(*leaves[:1], 8, *leaves[1:], act="silu", p=0.2, key=KEY)
        runs.append((y,) + torch.autograd.grad(y, leaves, dy))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


# ---------------------------------------------------------------------------
# 8-bit product
# ---------------------------------------------------------------------------


def quantize64(x):
    """The definition with the exact quotient's rounding decided in 64 bits:
    x and scale are fp32 values, so a quotient that is not exactly a half is at
    least 2^-32 of itself away from it, and 64 bits tell them apart."""
    x = x.double()
    top = x.abs().max(1).values if x.size(1) else torch.zeros(x.size(0), dtype=torch.float64)
    scale = torch.from_numpy(top.numpy().astype(np.float32) / np.float32(127.0))
    bad = ~torch.isfinite(top)
    scale[bad] = float("nan")
    s = scale.double()[:, None]
    zero = bad[:, None] | (s == 0)
    q = torch.where(zero, torch.zeros_like(x), torch.round(x / torch.where(zero, torch.ones_like(s), s)))
    return q.clamp(-127, 127).to(torch.int8), scale


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 7), (5, 16), (2, 17), (64, 100), (33, 1433), (4, 4096), (2, 9001)])
def test_quantize_rows(device, ops, dtype, rows, k):
    g = torch.Generator().manual_seed(rows + k)
    x = torch.randn(rows, k, generator=g).to(dtype)
    q, s = ops.quantize_rows(x.to(device))
    eq, es = quantize64(x)
    assert q.shape == (rows, k) and q.stride(0) % 16 == 0
    assert torch.equal(s.cpu(), es) and torch.equal(q.cpu(), eq)


def test_quantize_rows_borders(device, ops):
    """Ties, quotients one bit from a tie, zero rows, subnormal scales,
    infinities, NaN."""
    k = 300
    x = torch.zeros(12, k)
    x[0] = (torch.arange(k) - 150).float() + 0.5          # scale 1.1772...; general
    x[1, 0] = 127.0                                        # scale 1: exact ties
    x[1, 1:255] = torch.arange(-127, 127).float() + 0.5
    x[2] = x[1]
    x[2, 1:255] = torch.nextafter(x[1, 1:255], torch.full((254,), 1e9))
    x[3] = x[1]
    x[3, 1:255] = torch.nextafter(x[1, 1:255], torch.full((254,), -1e9))
    x[4] = x[1] * 3.3333333                                # scale with many bits, near ties
    x[6, :3] = torch.tensor([1e-45, -1e-45, 1e-44])        # scale underflows to 0
    x[7, :4] = torch.tensor([2.5e-43, -1.3e-43, 1e-44, 0])  # subnormal scale
    x[8, :4] = torch.tensor([3e-38, -1.7e-38, 1e-39, 0])
    x[9, :2] = torch.tensor([3.4e38, -1.0e38])
    x[10, 5] = float("inf")
    x[11, 6] = float("nan")
    q, s = ops.quantize_rows(x.to(device))
    eq, es = quantize64(x)
    assert torch.equal(s.cpu().isnan(), es.isnan()) and torch.equal(s.cpu().nan_to_num(), es.nan_to_num())
    assert torch.equal(q.cpu(), eq)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [0, 1, 3, 5, 7, 9])
@pytest.mark.parametrize("ldq", [16, 4112, 8208, 12304])
def test_quantize_entry_pads_any_row(device, dtype, cols, ldq):
    """Rows shorter than a vector, or empty, in rows of 8 bits of any length:
    the padding is 0 and nothing but the row is read (x is NULL at cols = 0)."""
    from ldsgnn import _native as nat
    g = torch.Generator().manual_seed(cols)
    x = torch.randn(5, cols, generator=g).to(dtype)
    xd = x.to(device)
    q = torch.full((5, ldq), 85, dtype=torch.int8, device=device)
    scale = torch.full((5,), 7.0, device=device)
    nat.call("lds_quantize_rows", xd.data_ptr() if cols else 0, cols, 5, cols, nat.ELEMENT_CODES[dtype], q.data_ptr(),
             ldq, scale.data_ptr(), nat.stream_of(xd.device))
    eq, es = quantize64(x)
    assert torch.equal(scale.cpu(), es) and torch.equal(q[:, :cols].cpu(), eq)
    assert not q[:, cols:].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,ldq", [(5, 3, 8208), (5, 7, 4112), (2, 5, 16368), (3, 9, 12304)])
def test_int8_linear_entry_with_long_rows_in_the_workspace(device, dtype, m, k, ldq):
    from ldsgnn import _native as nat
    g = torch.Generator().manual_seed(m + k)
    x, w = torch.randn(m, k, generator=g).to(dtype), ints(g, 19, k)
    wq = torch.zeros(19, 16, dtype=torch.int8, device=device)
    wq[:, :k] = w.to(device)
    xd, one, y = x.to(device), torch.ones(19, device=device), torch.empty(m, 19, device=device)
    q, xs = torch.empty(m, ldq, dtype=torch.int8, device=device), torch.empty(m, device=device)
    nat.call("lds_int8_linear", xd.data_ptr(), k, nat.ELEMENT_CODES[dtype], q.data_ptr(), ldq, xs.data_ptr(),
             wq.data_ptr(), 16, one.data_ptr(), 0, 0, m, 19, k, y.data_ptr(), 19, 0, nat.stream_of(xd.device))
    eq, es = quantize64(x)
    assert torch.equal(y.cpu(), (eq.double() @ w.double().t()).float() * es[:, None])


def test_quantize_entry_pads_past_an_int_of_bits(device):
    """Padding that begins 2^26 and more values behind the row: still 0."""
    from ldsgnn import _native as nat
    cols, ldq = 9, (1 << 26) + 4096
    x = torch.arange(1.0, cols + 1.0, device=device)
    q = torch.full((ldq,), 85, dtype=torch.int8, device=device)
    scale = torch.empty(1, device=device)
    nat.call("lds_quantize_rows", x.data_ptr(), cols, 1, cols, 0, q.data_ptr(), ldq, scale.data_ptr(),
             nat.stream_of(x.device))
    assert torch.equal(q[:cols].cpu(), quantize64(x.cpu()[None])[0][0]) and not q[cols:].any()


def ints(g, *shape):
    return torch.randint(-127, 128, shape, generator=g, dtype=torch.int8)


INT8_SHAPES = [  # m, n, k
    (1, 1, 1), (1, 7, 16), (2, 3, 15), (5, 16, 17), (16, 16, 64), (17, 33, 65), (1, 1000, 4096), (3, 257, 1000),
    (33, 31, 129), (64, 64, 256), (100, 7, 1433), (130, 300, 511), (257, 129, 128), (300, 520, 640), (513, 1030, 200),
    (3600, 3590, 200), (3585, 3600, 64), (1100, 1025, 333), (2500, 2300, 65), (1600, 2000, 129), (900, 1700, 700),
    (777, 900, 1000), (2708, 16, 1433), (500, 120, 2049),
]


@pytest.mark.parametrize("m,n,k", INT8_SHAPES)
def test_int8_matmul_whole_numbers(device, ops, m, n, k):
    """Scales 1, no bias: y is the integer sum, rounded to fp32 once."""
    g = torch.Generator().manual_seed(m + n + k)
    a, b = ints(g, m, k), ints(g, n, k)
    one = torch.ones(max(m, n), device=device)
    y = ops.int8_matmul(a.to(device), one[:m], b.to(device), one[:n])
    a127 = a.clone()
    a127[:, 0] = 127  # the scale of the same numbers as fp32 rows is 1: the joint call gives the same
    with torch.no_grad():
        y127 = ops.int8_linear(a127.float().to(device), b.to(device), one[:n])
    assert torch.equal(y127.cpu(), (a127.double() @ b.double().t()).float())
    assert torch.equal(y.cpu(), (a.double() @ b.double().t()).float())


def int8_tile(m, n):
    """The largest tile that gives 192 blocks (lds_int8_matmul's rule), 0: split."""
    for bm, bn in ((256, 256), (256, 128), (128, 128), (128, 64), (64, 64)):
        if -(-m // bm) * -(-n // bn) >= 192:
            return bm, bn
    return 0


@pytest.mark.parametrize("m,n,k,tile", [
    (3590, 3587, 1031, (256, 256)), (3585, 3841, 448, (256, 256)), (2500, 3300, 777, (256, 128)),
    (2561, 3205, 1024, (256, 128)), (1600, 2000, 1000, (128, 128)), (1665, 1793, 833, (128, 128)),
    (1500, 1090, 1033, (128, 64)), (1030, 810, 1409, (64, 64))])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_int8_tiles_in_their_steady_loop(device, ops, m, n, k, tile, dtype):
    """Every tile instance over seven and more steps of 64 bytes, so that its ring
    is refilled in the loop (from six steps on; eight with the longer ring), with
    ends of m, n and k inside a tile, a step and a 16-byte chunk: whole numbers,
    exact."""
    assert int8_tile(m, n) == tile and (k + 63) // 64 >= 7
    g = torch.Generator().manual_seed(m + n + k)
    a, b = (ints(g, r, k).to(device) for r in (m, n))
    one = torch.ones(max(m, n), device=device)
    y = ops.int8_matmul(a, one[:m], b, one[:n], out_dtype=dtype)
    assert torch.equal(y, (a.double() @ b.double().t()).float().to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 33, 70), (40, 50, 600), (129, 258, 300)])
def test_int8_matmul_scales(device, ops, dtype, m, n, k):
    """acc·xs·ws + b: four roundings (of acc to fp32, two products, the sum) and
    the one to the type."""
    g = torch.Generator().manual_seed(1)
    a, b = ints(g, m, k), ints(g, n, k)
    xs, ws, bias = torch.rand(m, generator=g) * 0.1, torch.rand(n, generator=g) * 0.1, torch.randn(n, generator=g)
    for bd in (None, bias, bias.to(torch.bfloat16)):
        y = ops.int8_matmul(a.to(device), xs.to(device), b.to(device), ws.to(device),
                            None if bd is None else bd.to(device), out_dtype=dtype).cpu()
        prod = (a.double() @ b.double().t()) * xs.double()[:, None] * ws.double()
        ref = prod if bd is None else prod + bd.double()
        tol = HALF[dtype] * ref.abs() + 2 * (3 * U * prod.abs() + U * ref.abs()) + TINY[dtype]
        assert y.dtype == dtype and ((y.double() - ref).abs() <= tol).all()


def test_int8_matmul_largest_sum(device, ops):
    k = ops.INT8_MAX_K
    a = torch.full((2, k), -128, dtype=torch.int8, device=device)
    a[1] = 127
    y = ops.int8_matmul(a, torch.ones(2, device=device), a, torch.ones(2, device=device))
    ref = torch.tensor([[k * 16384.0, -k * 16256.0], [-k * 16256.0, k * 16129.0]], dtype=torch.float64)
    assert torch.equal(y.cpu(), ref.float())


def test_int8_matmul_layouts(device, ops):
    """Rows with other bytes behind them, at odd addresses, transposed: what
    lies past k is never used."""
    g = torch.Generator().manual_seed(2)
    m, n, k = 45, 70, 150
    a, b = ints(g, m, k), ints(g, n, k)
    ref = (a.double() @ b.double().t()).float()
    one = torch.ones(100, device=device)

    def wide(t, ld, at):
        buf = torch.full((t.size(0) * ld + at + 64,), 85, dtype=torch.int8, device=device)
        v = buf[at:at + t.size(0) * ld].view(t.size(0), ld)[:, :t.size(1)]
        v.copy_(t.to(device))
        return v

    for va, vb in ((wide(a, 160, 0), wide(b, 176, 16)), (wide(a, 150, 0), wide(b, 160, 3)),
                   (a.t().contiguous().to(device).t(), wide(b, 151, 1)), (wide(a, 192, 32), b.to(device))):
        assert torch.equal(ops.int8_matmul(va, one[:m], vb, one[:n]).cpu(), ref)
    # a row stride of a multiple of 16 whose last row ends with the storage
    tight = torch.empty((m - 1) * 160 + k, dtype=torch.int8, device=device).as_strided((m, k), (160, 1))
    tight.copy_(a)
    assert ops.int8_rows(tight) is not tight
    assert torch.equal(ops.int8_matmul(tight, one[:m], b.to(device), one[:n]).cpu(), ref)


@pytest.mark.parametrize("m,n,k", [(0, 4, 8), (4, 0, 8), (3, 5, 0)])
def test_int8_matmul_empty(device, ops, m, n, k):
    q = torch.zeros((m, k), dtype=torch.int8, device=device)
    w = torch.zeros((n, k), dtype=torch.int8, device=device)
    bias = torch.arange(n, device=device).float()
    y = ops.int8_matmul(q, torch.ones(m, device=device), w, torch.ones(n, device=device), bias)
    assert y.shape == (m, n) and torch.equal(y, bias.expand(m, n))
    with torch.no_grad():
        z = ops.int8_linear(torch.zeros(m, k, device=device), w, torch.ones(n, device=device), bias)
    assert z.shape == (m, n) and torch.equal(z, bias.expand(m, n))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,n", [((1, 64), 16), ((37,), 5), ((1, 1), 1), ((3, 17), 40), ((4, 8200), 33),
                                     ((2, 20000), 7), ((4, 5000), 100), ((1, 40000), 19), ((5, 130), 18), ((2, 9, 100), 33), ((300, 1433), 16), ((1, 4096), 260)])
def test_int8_linear(device, ops, dtype, shape, n):
    """The quantised operands are those of quantize64 exactly; the rest as in
    test_int8_matmul_scales.  Rows of zeros give the bias, rows with a NaN give
    NaN."""
    g = torch.Generator().manual_seed(8)
    k = shape[-1]
    x = torch.randn(shape, generator=g).to(dtype)
    w = torch.randn(n, k, generator=g) / k ** 0.5
    bias = torch.randn(n, generator=g)
    if x.dim() > 1 and x[..., 0].numel() > 2:
        x.view(-1, k)[1] = 0
        x.view(-1, k)[2, k // 2] = float("nan")
    wq, ws = ops.quantize_rows(w.to(device))
    with torch.no_grad():
        y = ops.int8_linear(x.to(device), wq, ws, bias.to(device)).cpu()
    q, s = quantize64(x.reshape(-1, k))
    qw, sw = quantize64(w)
    prod = (q.double() @ qw.double().t()) * s.double()[:, None] * sw.double()
    ref = prod + bias.double()
    y2 = y.view(-1, n).double()
    assert y.shape == shape[:-1] + (n,) and y.dtype == dtype
    assert torch.equal(torch.isnan(y2), torch.isnan(ref))
    tol = HALF[dtype] * ref.abs() + 2 * (3 * U * prod.abs() + U * ref.abs()) + TINY[dtype]
    assert ((y2 - ref).abs() <= tol)[~torch.isnan(ref)].all()


# ---------------------------------------------------------------------------
# streams, graphs
# ---------------------------------------------------------------------------


def _all_ops(ops, x, w, b, dy, wq, ws):
    leaf = x.detach().requires_grad_()
    wl, bl = w.detach().requires_grad_(), b.detach().requires_grad_()
    y = ops.group_norm_act(leaf, 4, wl, bl, act="silu", p=0.25, key=KEY)
    z = ops.keyed_dropout(y, 0.5, KEY, residual=leaf)
    grads = torch.autograd.grad(z, (leaf, wl, bl), dy)
    with torch.no_grad():
        out = ops.int8_linear(z, wq, ws, b[:wq.size(0)])
    return (z.detach(), out) + grads


def _block_inputs(ops, device):
    x, w, b, dy = (t.to(device) for t in norm_inputs(2, 333, 4, 16, torch.bfloat16, seed=12))
    g = torch.Generator().manual_seed(3)
    wq, ws = ops.quantize_rows(torch.randn(48, 64, generator=g).to(device))
    return x, w, b, dy, wq, ws


def test_stream_of_takes_what_names_a_device(device):
    from ldsgnn import _native as nat
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for name in (device, 0, "cuda", "cuda:0", None, torch.device("cuda")):
            assert nat.stream_of(name) == side.cuda_stream, name


def test_side_stream_runs_the_same_bits(device, ops):
    args = _block_inputs(ops, device)
    ref = _all_ops(ops, *args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _all_ops(ops, *args)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(ref, got))


@pytest.mark.parametrize("n,groups,cg", [(5000, 12, 5), (5000, 7, 5), (5000, 4, 8), (60, 7, 5)])
def test_group_norm_entries_in_place(device, n, groups, cg):
    """y over x and dx over dy: the bits of separate results, also where a row's
    last vector shares elements with the one before it."""
    from ldsgnn import _native as nat
    c, half = groups * cg, nat.ELEMENT_CODES[torch.float16]
    g = torch.Generator().manual_seed(n + c)
    x, dy = (torch.randn(3, n, c, generator=g).half().to(device) for _ in range(2))
    stats = torch.empty(2, 3, groups, device=device)
    at, to = stats.data_ptr(), stats.data_ptr() + 4 * 3 * groups
    ws = torch.empty(max(nat.lib.lds_group_norm_ws_bytes(3, n, c, groups, half, k) for k in (0, 1)) + 16,
                     dtype=torch.uint8, device=device)

    def forward(a, y):
        nat.call("lds_group_norm_forward", a.data_ptr(), n * c, c, 3, n, c, groups, half, 0, 0, 0, 1e-5, 2, 0.75,
                 4.0 / 3.0, *KEY, y.data_ptr(), at, to, ws.data_ptr(), nat.stream_of(a.device))
        return y

    def backward(d, dx):
        nat.call("lds_group_norm_backward", d.data_ptr(), n * c, c, x.data_ptr(), n * c, c, 3, n, c, groups, half, 0, 0,
                 0, 2, 0.75, 4.0 / 3.0, *KEY, at, to, dx.data_ptr(), 0, 0, ws.data_ptr(), nat.stream_of(x.device))
        return dx

    y, dx = forward(x, torch.empty_like(x)), backward(dy, torch.empty_like(x))
    here = dy.clone()
    assert torch.equal(backward(here, here), dx)
    here = x.clone()
    assert torch.equal(forward(here, here), y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (7, 3), (1031, 33), (520, 8), (301, 257)])
def test_dropout_add_in_place(device, dtype, rows, cols):
    """y over x, y over the residual, and all three the same: the bits of separate
    tensors."""
    from ldsgnn import _native as nat
    g = torch.Generator().manual_seed(rows + cols)
    x, r = (torch.randn(rows, cols, generator=g).to(dtype) for _ in range(2))
    code = nat.ELEMENT_CODES[dtype]

    def call(a, b, y):
        nat.call("lds_dropout_add", a.data_ptr(), cols, 0 if b is None else b.data_ptr(), cols, y.data_ptr(), cols, rows,
                 cols, code, 0.75, float(np.float32(1.0) / np.float32(0.75)), *KEY, nat.stream_of(y.device))
        return y.cpu()

    a, b = x.to(device), r.to(device)
    want = plain_dropout(x, KEY, 0.25, r)
    assert torch.equal(call(a, b, a), want)
    a = x.to(device)
    assert torch.equal(call(a, b, b), want) and torch.equal(a.cpu(), x)
    a = x.to(device)
    assert torch.equal(call(a, a, a), plain_dropout(x, KEY, 0.25, x))
    a = x.to(device)
    assert torch.equal(call(a, None, a), plain_dropout(x, KEY, 0.25))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("s,n,groups,cg", [(3, 2, 2, 8), (9, 60, 5, 3), (2, 601, 37, 64), (3, 5001, 5, 3), (1, 40, 1, 8200),
                                           (1, 9001, 2, 4)])
def test_group_norm_in_place_in_every_form(device, ops, dtype, s, n, groups, cg):
    """y over x, dx over dy and dx over x, in one launch and in parts, a group per
    vector, vectors across groups and groups across blocks."""
    from ldsgnn import _native as nat
    c, code = groups * cg, nat.ELEMENT_CODES[dtype]
    x, w, b, dy = (t.to(device) for t in norm_inputs(s, n, groups, cg, dtype, seed=21))
    pl = ops._NormPlan(groups, ops.ACTIVATIONS["silu"], 1e-5, 0.75, 4.0 / 3.0, KEY)
    y, stats = ops._norm_forward(x, w, b, pl)
    dx, dw, db = ops._norm_backward(dy, x, w, b, stats, pl, (True, True, True))
    ws = torch.empty(max(nat.lib.lds_group_norm_ws_bytes(s, n, c, groups, code, k) for k in (0, 1)) + 16,
                     dtype=torch.uint8, device=device)
    st, at, to = nat.stream_of(x.device), stats.data_ptr(), stats.data_ptr() + 4 * s * groups
    for over in ("dy", "x"):
        a, d = x.clone(), dy.clone()
        out = d if over == "dy" else a
        ew, eb = torch.empty(c, device=device), torch.empty(c, device=device)
        nat.call("lds_group_norm_backward", d.data_ptr(), n * c, c, a.data_ptr(), n * c, c, s, n, c, groups, code,
                 w.data_ptr(), b.data_ptr(), 0, pl.act, *pl.mask, at, to, out.data_ptr(), ew.data_ptr(), eb.data_ptr(),
                 ws.data_ptr(), st)
        assert torch.equal(out, dx) and torch.equal(ew, dw) and torch.equal(eb, db), over
    nat.call("lds_group_norm_forward", x.data_ptr(), n * c, c, s, n, c, groups, code, w.data_ptr(), b.data_ptr(), 0, 1e-5,
             pl.act, *pl.mask, x.data_ptr(), at, to, ws.data_ptr(), st)
    assert torch.equal(x, y)


@pytest.mark.parametrize("dtype,n", [(torch.bfloat16, 14001), (torch.float32, 7001)])
def test_group_norm_in_place_past_the_caches(device, ops, dtype, n):
    """147 MB over itself: the bits of a result of its own, which is stored past
    the caches."""
    from ldsgnn import _native as nat
    s, groups, c = 2, 41, 41 * 64
    code = nat.ELEMENT_CODES[dtype]
    x, dy = (torch.randn(s, n, c, device=device, dtype=dtype) for _ in range(2))
    pl = ops._NormPlan(groups, ops.ACTIVATIONS["silu"], 1e-5, 0.75, 4.0 / 3.0, KEY)
    y, stats = ops._norm_forward(x, None, None, pl)
    dx = ops._norm_backward(dy, x, None, None, stats, pl, (True, False, False))[0]
    ws = torch.empty(max(nat.lib.lds_group_norm_ws_bytes(s, n, c, groups, code, k) for k in (0, 1)), dtype=torch.uint8,
                     device=device)
    st, at, to = nat.stream_of(x.device), stats.data_ptr(), stats.data_ptr() + 4 * s * groups
    nat.call("lds_group_norm_backward", dy.data_ptr(), n * c, c, x.data_ptr(), n * c, c, s, n, c, groups, code, 0, 0, 0,
             pl.act, *pl.mask, at, to, dy.data_ptr(), 0, 0, ws.data_ptr(), st)
    assert torch.equal(dy, dx)
    nat.call("lds_group_norm_forward", x.data_ptr(), n * c, c, s, n, c, groups, code, 0, 0, 0, 1e-5, pl.act, *pl.mask,
             x.data_ptr(), at, to, ws.data_ptr(), st)
    assert torch.equal(x, y)


def test_captured_run_replays_the_eager_bits(device, ops):
    """Forward, backward and the 8-bit product in one captured graph, replayed
    with new inputs and eager work in between; kernel nodes only."""
    import ldsgnn._native as nat
    static = [t.clone() for t in _block_inputs(ops, device)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _all_ops(ops, *static)
    torch.cuda.current_stream().wait_stream(side)
    graph = nat.new_graph()
    with torch.cuda.graph(graph):
        out = _all_ops(ops, *static)
    nat.seal_graph(graph, "block operators")
    for i in range(4):
        static[0].copy_(torch.randn_like(static[0].float()).mul_(1.0 + i))
        static[3].copy_(torch.randn_like(static[3].float()))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        ref = _all_ops(ops, *static)
        assert all(torch.equal(a, b) for a, b in zip(ref, got)), i
