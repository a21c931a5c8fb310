"""The block operators' refusals: raised on the host, before any launch."""
import pytest
import torch

from ldsgnn import _native as nat
from ldsgnn import ops

FAKE = 1 << 20  # never dereferenced: the argument checks run first
KEY = (1, 2, 3)


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 8)
    q = torch.zeros(4, 16, dtype=torch.int8)
    one = torch.ones(4)
    for call in (lambda: ops.keyed_dropout(x, 0.5, KEY), lambda: ops.group_norm_act(x, 2),
                 lambda: ops.quantize_rows(x), lambda: ops.int8_matmul(q, one, q, one),
                 lambda: ops.int8_linear(x, q, one), lambda: ops.int8_rows(q)):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()


def test_dropout_arguments():
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError, match="p must lie"):
            ops.keyed_dropout(torch.randn(4, 8), p, KEY)
    with pytest.raises(ValueError, match="key"):
        ops.keyed_dropout(torch.randn(4, 8), 0.5, None)


def test_group_norm_arguments():
    with pytest.raises(ValueError, match="activation"):
        ops.group_norm_act(torch.randn(4, 8), 2, act="tanh")


def test_no_gradient_through_the_8_bit_product():
    x = torch.randn(4, 16, requires_grad=True)
    q = torch.zeros(4, 16, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.int8_linear(x, q, torch.ones(4))
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.int8_matmul(q, torch.ones(4), q, torch.ones(4), bias=torch.zeros(4, requires_grad=True))


def check_empty_second_order(norm, shape, groups, device):
    """The second derivative of an empty tensor: zeros, as the first order gives."""
    leaves = [torch.randn(s, device=device, requires_grad=True) for s in (shape, shape[-1:], shape[-1:])]
    dy = torch.randn(shape, device=device, requires_grad=True)
    y = norm(*leaves)
    first = torch.autograd.grad(y, leaves, dy, create_graph=True)
    total = sum((f * torch.ones_like(f)).sum() for f in first)
    for t, g in zip([dy] + leaves, torch.autograd.grad(total, [dy] + leaves)):
        assert g.shape == t.shape and not g.any()


@pytest.mark.parametrize("shape,groups", [((0, 3, 4), 2), ((2, 0, 4), 2), ((2, 3, 0), 1), ((0, 4), 4), ((0, 0, 0), 3)])
@pytest.mark.parametrize("act,p", [("none", 0.0), ("silu", 0.5), ("relu", 1.0)])
def test_second_order_of_an_empty_norm(shape, groups, act, p):
    keep = 1.0 - p
    pl = ops._NormPlan(groups, ops.ACTIVATIONS[act], 1e-5, keep, 1.0 / keep if keep else 0.0, KEY)
    check_empty_second_order(lambda x, w, b: ops._GroupNormAct.apply(x, w, b, pl), shape, groups, "cpu")


@pytest.mark.parametrize("which", ["x", "residual", "norm x", "weight", "bias", "quantize", "matmul scale", "linear x",
                                   "linear bias", "aggregate"])
def test_tangents_are_refused(which):
    """A forward-mode derivative is not computed, so it is not dropped in silence
    either: the refusal comes before any other check."""
    from torch.autograd import forward_ad
    x, c = torch.randn(4, 8), torch.ones(8)
    q, one = torch.zeros(4, 16, dtype=torch.int8), torch.ones(4)
    calls = {"x": lambda d: ops.keyed_dropout(d(x), 0.5, KEY), "residual": lambda d: ops.keyed_dropout(x, 0.5, KEY, d(x)),
             "norm x": lambda d: ops.group_norm_act(d(x), 2), "weight": lambda d: ops.group_norm_act(x, 2, d(c)),
             "bias": lambda d: ops.group_norm_act(x, 2, c, d(c)), "quantize": lambda d: ops.quantize_rows(d(x)),
             "matmul scale": lambda d: ops.int8_matmul(q, d(one), q, one), "linear x": lambda d: ops.int8_linear(d(x), q, one),
             "linear bias": lambda d: ops.int8_linear(x, q, one, d(one)), "aggregate": lambda d: ops.aggregate(d(x), None)}
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            calls[which](lambda t: forward_ad.make_dual(t, torch.ones_like(t)))
        with pytest.raises((RuntimeError, AttributeError)) as other:  # no tangent: the next check (no device here)
            calls[which](lambda t: t)
        assert not isinstance(other.value, NotImplementedError)


def test_8_bit_evaluation_does_not_ignore_weights():
    """empirical_mean_loss with weights for a model that already holds its own."""
    from collections import OrderedDict

    from ldsgnn.models.gcn import Int8DenseGCN
    from ldsgnn.utils.evaluation import empirical_mean_loss
    model = Int8DenseGCN.__new__(Int8DenseGCN)
    torch.nn.Module.__init__(model)
    with pytest.raises(ValueError, match="own weights"):
        empirical_mean_loss(model, torch.nn.Module(), 0, None, model_parameters=OrderedDict(), int8=True)


def _drop(**kw):
    a = dict(x=FAKE, ldx=8, res=0, ldr=0, y=FAKE, ldy=8, rows=4, cols=8, dtype=0, keep=0.5, scale=2.0)
    a.update(kw)
    return nat.lib.lds_dropout_add(*a.values(), 1, 2, 3, None)


@pytest.mark.parametrize("kw", [dict(x=0), dict(y=0), dict(ldx=7), dict(ldy=7), dict(rows=-1), dict(cols=-1),
                                dict(dtype=3), dict(dtype=-1), dict(keep=1.5), dict(keep=-0.5), dict(res=FAKE, ldr=7),
                                dict(rows=1 << 31)])
def test_dropout_entry_refuses(kw):
    assert _drop(**kw) == 1


def test_empty_calls_launch_nothing():
    assert _drop(rows=0) == 0 and _drop(cols=0, ldx=0, ldy=0) == 0
    assert _norm(n=0) == 0 and _norm(samples=0) == 0
    assert _quant(rows=0) == 0
    assert _mul(m=0) == 0 and _mul(n=0) == 0


def _norm(back=False, **kw):
    a = dict(x=FAKE, sx=64, ldx=8, samples=2, n=8, c=8, groups=2, dtype=0, w=0, b=0, pt=0, eps=1e-5, act=0, keep=1.0,
             scale=1.0, seed=1, tag=2, counter=3, y=FAKE, mean=FAKE, rstd=FAKE, ws=FAKE)
    a.update(kw)
    if not back:
        return nat.lib.lds_group_norm_forward(*a.values(), None)
    return nat.lib.lds_group_norm_backward(
        a["y"], 64, 8, a["x"], a["sx"], a["ldx"], a["samples"], a["n"], a["c"], a["groups"], a["dtype"], a["w"],
        a["b"], a["pt"], a["act"], a["keep"], a["scale"], 1, 2, 3, a["mean"], a["rstd"], FAKE, 0, 0, a["ws"], None)


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("kw", [dict(x=0), dict(y=0), dict(mean=0), dict(rstd=0), dict(ws=0, n=200000), dict(ldx=7),
                                dict(groups=3), dict(groups=0), dict(groups=-2), dict(dtype=3), dict(act=3),
                                dict(act=-1), dict(pt=5), dict(keep=-1.0), dict(keep=float("nan")), dict(n=-1),
                                dict(samples=-1), dict(c=-8), dict(samples=1 << 16, n=1 << 16), dict(sx=-1)])
def test_group_norm_entries_refuse(back, kw):
    assert _norm(back, **kw) == 1


def test_group_norm_forward_refuses_eps():
    assert _norm(eps=-1.0) == 1 and _norm(eps=float("nan")) == 1


def test_group_norm_workspace_sizes():
    size = nat.lib.lds_group_norm_ws_bytes
    assert size(1, 0, 8, 2, 0, 0) == 0 and size(0, 8, 8, 2, 0, 1) == 0
    assert size(1, 8, 8, 3, 0, 0) == -1 and size(1, 8, 8, 2, 7, 0) == -1 and size(-1, 8, 8, 2, 0, 0) == -1
    for dt in (0, 1, 2):
        # rows that a block holds need no workspace; longer ones do
        assert size(1, 1, 8, 2, dt, 0) == 0 and size(1, 1, 8, 2, dt, 1) == 0
        assert size(2, 1, 8, 2, dt, 1) == 2 * 8 * 8
        assert size(8, 20000, 256, 32, dt, 0) > 0 and size(8, 20000, 256, 32, dt, 1) > 0


def _quant(**kw):
    a = dict(x=FAKE, ldx=20, rows=3, cols=20, dtype=0, q=FAKE, ldq=32, scale=FAKE)
    a.update(kw)
    return nat.lib.lds_quantize_rows(*a.values(), None)


@pytest.mark.parametrize("kw", [dict(x=0), dict(q=0), dict(q=FAKE + 8), dict(scale=0), dict(ldq=20), dict(ldq=16),
                                dict(ldx=19), dict(rows=-1), dict(cols=-1), dict(dtype=4)])
def test_quantize_entry_refuses(kw):
    assert _quant(**kw) == 1


def _mul(**kw):
    a = dict(xq=FAKE, ldx=32, xs=FAKE, wq=FAKE, ldw=32, ws=FAKE, bias=0, pt=0, m=3, n=5, k=20, y=FAKE, ldy=5, dtype=0)
    a.update(kw)
    return nat.lib.lds_int8_matmul(*a.values(), None)


@pytest.mark.parametrize("kw", [dict(xq=0), dict(wq=0), dict(xs=0), dict(ws=0), dict(y=0), dict(ldx=20), dict(ldw=24),
                                dict(ldx=16), dict(ldy=4), dict(xq=FAKE + 4), dict(wq=FAKE + 8), dict(k=131072),
                                dict(k=-1), dict(m=-1), dict(n=-1), dict(dtype=3), dict(pt=9)])
def test_int8_matmul_entry_refuses(kw):
    assert _mul(**kw) == 1


@pytest.mark.parametrize("kw", [dict(x=0), dict(xq=0), dict(wq=0), dict(xs=0), dict(ws=0), dict(y=0), dict(ldq=20),
                                dict(ldw=24), dict(ldx=16), dict(ldy=4), dict(xq=FAKE + 4), dict(k=131072),
                                dict(m=-1), dict(xdt=3), dict(dtype=3), dict(pt=-1)])
def test_int8_linear_entry_refuses(kw):
    a = dict(x=FAKE, ldx=20, xdt=0, xq=FAKE, ldq=32, xs=FAKE, wq=FAKE, ldw=32, ws=FAKE, bias=0, pt=0, m=3, n=5, k=20,
             y=FAKE, ldy=5, dtype=0)
    a.update(kw)
    assert nat.lib.lds_int8_linear(*a.values(), None) == 1
