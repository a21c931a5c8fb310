"""The models and paths that run the block operators: the GCN with a normalised
hidden layer (forward, gradients, the differentiable inner step, the fused
engine's refusal) and the GCN evaluated with 8-bit products."""
from collections import OrderedDict

import pytest
import torch

from oracle import philox

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def small_graph(n=60, seed=0, p=0.15):
    g = torch.Generator().manual_seed(seed)
    a = (torch.rand(n, n, generator=g) < p).float().triu(1)
    return a + a.t()


def tiny_data(device, n=96, f_in=24, classes=4, seed=1):
    from ldsgnn.utils.graph import DenseData
    g = torch.Generator().manual_seed(seed)
    x = torch.rand(n, f_in, generator=g)
    masks = [torch.zeros(n, dtype=torch.bool) for _ in range(3)]
    perm = torch.randperm(n, generator=g)
    for m, rows in zip(masks, (perm[:30], perm[30:60], perm[60:])):
        m[rows] = True
    return DenseData(x=x, y=torch.randint(0, classes, (n,), generator=g), dense_adj=small_graph(n, seed),
                     train_mask=masks[0], val_mask=masks[1], test_mask=masks[2], num_classes=classes).to(device)


def a_hat64(adj):
    a = adj.double().clone()
    a.fill_diagonal_(1.0)
    s = a.sum(1).rsqrt()
    return s[:, None] * a * s[None, :]


def keep64(seed, kind, counter, rows, cols, p):
    u = torch.from_numpy(philox.uniform(seed, kind, counter, rows, cols).astype("float64"))
    return (u < 1.0 - p).double() / (1.0 - p)


def gcn64(x, a, w, groups, act, masks):
    """log_softmax(Â (m act(norm(Â (m x W0ᵀ + b0))) W1ᵀ + b1)) in 64 bits."""
    mx, mh = masks if masks is not None else (1.0, 1.0)
    h = a @ ((x * mx) @ w["layer_in.fc.weight"].t() + w["layer_in.fc.bias"])
    n, c = h.shape
    v = h.reshape(n, groups, c // groups)
    d = v - v.mean((0, 2), keepdim=True)
    h = (d / (d.square().mean((0, 2), keepdim=True) + 1e-5).sqrt()).reshape(n, c)
    h = h * w["layer_in.norm.weight"] + w["layer_in.norm.bias"]
    h = torch.relu(h) if act == "relu" else h * torch.sigmoid(h)
    o = a @ ((h * mh) @ w["layer_out.fc.weight"].t() + w["layer_out.fc.bias"])
    return torch.log_softmax(o, 1)


def build(device, act, dropout, f_in=24, hidden=16, classes=4, seed=3):
    from ldsgnn.models.gcn import MetaDenseGCN
    from ldsgnn.rng import Generator
    torch.manual_seed(seed)
    gen = Generator(11, 2)
    gcn = MetaDenseGCN(f_in, hidden, classes, dropout=dropout, generator=gen, norm_groups=4, norm_act=act).to(device)
    with torch.no_grad():
        gcn.layer_in.norm.weight.add_(torch.randn(hidden).to(device) * 0.2)
        gcn.layer_in.norm.bias.add_(torch.randn(hidden).to(device) * 0.2)
    return gcn, gen


@pytest.mark.parametrize("act,dropout", [("silu", 0.0), ("silu", 0.5), ("relu", 0.0)])
def test_normalised_gcn_and_its_inner_step(device, act, dropout):
    """Forward, then one SGD step of the parameters with create_graph and the
    gradient of the loss after it with respect to x and the first parameters
    (the double backward that the hyper step takes), against 64-bit autograd.
    fp32 through two aggregations and products of width <= 60 and three
    passes: some thousand roundings of 6e-8 in all, 5e-4 of the largest entry."""
    from ldsgnn.ops import csr_graph_from_dense
    from ldsgnn.rng import TAG_DROP_H, TAG_DROP_X
    n, f_in, hidden = 60, 24, 16
    adj = small_graph(n)
    gcn, gen = build(device, act, dropout)
    g = torch.Generator().manual_seed(5)
    x, y = torch.randn(n, f_in, generator=g), torch.randint(0, 4, (n,), generator=g)
    graph = csr_graph_from_dense(adj.to(device))
    gcn.train()
    results = []
    for dev, dt in ((device, torch.float32), ("cpu", torch.float64)):
        xd = x.to(dev, dt).requires_grad_()
        w0 = OrderedDict((k, v.detach().to(dev, dt).requires_grad_()) for k, v in gcn.named_parameters())
        gen.manual_seed(11, 2)
        a64 = a_hat64(adj)
        counter = 0

        def forward(w):
            nonlocal counter
            if dev != "cpu":
                return gcn(xd, graph, params=w)
            masks = None
            if dropout > 0:
                masks = (keep64(11, TAG_DROP_X | 2, counter, n, f_in, dropout),
                         keep64(11, TAG_DROP_H | 2, counter, n, hidden, dropout))
            counter += 1
            return gcn64(xd, a64, w, 4, act, masks)

        out = forward(w0)
        yd = y.to(dev)
        loss = torch.nn.functional.nll_loss(out, yd)
        grads = torch.autograd.grad(loss, list(w0.values()), create_graph=True)
        w1 = OrderedDict((k, v - 0.5 * gr) for (k, v), gr in zip(w0.items(), grads))
        loss2 = torch.nn.functional.nll_loss(forward(w1), yd)
        second = torch.autograd.grad(loss2, [xd] + list(w0.values()))
        results.append([out] + list(grads) + [loss2] + list(second))
    for i, (a, e) in enumerate(zip(*results)):
        e = e.detach()
        assert (a.detach().cpu().double() - e).abs().max() <= 5e-4 * max(float(e.abs().max()), 1e-3), i


def test_normalised_gcn_trains_in_the_bilevel_trainers(device):
    """The norm's parameters are among the inner optimizer's (with layer_in's)
    and move; a hyper step reaches theta through them; the fused engine refuses
    the model."""
    from ldsgnn.fused import engine_from_trainers
    from ldsgnn.models.gcn import MetaDenseGCN
    from ldsgnn.models.graph import BernoulliGraphModel
    from ldsgnn.trainers.inner import InnerProblemTrainer
    from ldsgnn.trainers.outer import OuterProblemTrainer
    torch.manual_seed(0)
    data = tiny_data(device)
    gcn = MetaDenseGCN(data.num_features, 16, data.num_classes, dropout=0.3, norm_groups=2, norm_act="silu").to(device)
    gm = BernoulliGraphModel(data.dense_adj * 0.6 + 0.02)
    inner = InnerProblemTrainer(gcn, data, lr=0.01, weight_decay=5e-4)
    outer = OuterProblemTrainer(torch.optim.SGD(gm.parameters(), lr=0.1), data, data.val_mask, gm)
    before = {k: v.detach().clone() for k, v in inner.model_params.items()}
    theta = gm.probs.detach().clone()
    assert "layer_in.norm.weight" in before
    for _ in range(2):
        inner.train_step(outer.sample())
    outer.train_step(inner.model_forward)
    assert all(not torch.equal(before[k], v.detach()) for k, v in inner.model_params.items())
    assert torch.isfinite(gm.probs.grad).all() and not torch.equal(theta, gm.probs.detach())
    inner.detach()
    with pytest.raises(NotImplementedError, match="norm layer"):
        engine_from_trainers(inner, outer, tau=2)


def quant_error(x, w):
    """Bound of |x wᵀ - (its 8-bit form)|: x = s q + e with |e| <= s / 2 (s a row's
    largest value / 127), and likewise w."""
    sx = x.abs().max(1).values[:, None] / 127 * 0.5 * (1 + 2 ** -10)
    sw = w.abs().max(1).values[None, :] / 127 * 0.5 * (1 + 2 ** -10)
    return x.abs().sum(1)[:, None] * sw + sx * w.abs().sum(1)[None, :] + x.size(1) * sx * sw


@pytest.mark.parametrize("norm", [0, 4])
def test_int8_gcn(device, norm):
    """The 8-bit form against the same model in 64 bits.  Without a norm the
    bound follows from quant_error through the two layers: relu and Â (whose
    entries are not negative) carry a bound B of |h - h'| to Â B, the hidden
    rows' own quantisation adds quant_error at |h| + B, and log_softmax moves by at
    most twice the largest change of its inputs; 1e-5 covers fp32.  With a norm
    the first layer's bound is multiplied by the norm's slope, bounded by
    |weight| / sd times 1 + 1 + |x̂|max² / 1 (the change of mean and sd)."""
    from ldsgnn.models.gcn import Int8DenseGCN, MetaDenseGCN
    from ldsgnn.ops import csr_graph_from_dense
    torch.manual_seed(4)
    n, f_in = 60, 33
    adj = small_graph(n, seed=2)
    gcn = MetaDenseGCN(f_in, 16, 5, dropout=0.5, norm_groups=norm).to(device).eval()
    x = torch.rand(n, f_in)
    x[7] = 0.0
    w = {k: v.detach().cpu().double() for k, v in gcn.named_parameters()}
    model8 = Int8DenseGCN(gcn)
    graph = csr_graph_from_dense(adj.to(device))
    out = model8(x.to(device), graph).cpu().double()
    assert torch.equal(model8(x.to(device), adj.to(device)).cpu().double(), out)  # a dense 0/1 graph: the same form
    a, xd = a_hat64(adj), x.double()
    w0, b0, w1, b1 = (w[k] for k in ("layer_in.fc.weight", "layer_in.fc.bias", "layer_out.fc.weight",
                                     "layer_out.fc.bias"))
    z = a @ (xd @ w0.t() + b0)
    bound = a @ quant_error(xd, w0)
    if norm:
        v = z.reshape(n, norm, -1)
        d = v - v.mean((0, 2), keepdim=True)
        sd = (d.square().mean((0, 2), keepdim=True) + 1e-5).sqrt()
        xh = d / sd
        group = bound.reshape(n, norm, -1).amax((0, 2), keepdim=True)
        assert (sd > 2 * group).all()
        slope = 2 * (1 + xh.abs().amax((0, 2), keepdim=True)) / (sd - 2 * group)
        bound = (group * slope).expand_as(v).reshape(n, -1)
        z = xh.reshape(n, -1)
    h = torch.relu(z)
    top = h.abs() + bound
    err = a @ (quant_error(top, w1) + bound @ w1.abs().t())
    ref = torch.log_softmax(a @ (h @ w1.t() + b1), 1)
    assert ((out - ref).abs() <= 2 * err.amax(1, keepdim=True) + 1e-5).all()
    with pytest.raises(ValueError, match="own weights"):
        model8(x.to(device), graph, params={})


def test_int8_evaluation_paths(device):
    """evaluate() and empirical_mean_loss() with int8=True run the 8-bit form:
    the metrics of the model built by hand, with the trainer's weights."""
    from ldsgnn.models.gcn import Int8DenseGCN, MetaDenseGCN
    from ldsgnn.models.graph import BernoulliGraphModel
    from ldsgnn.rng import manual_seed
    from ldsgnn.utils.evaluation import empirical_mean_loss, evaluate
    torch.manual_seed(1)
    data = tiny_data(device, seed=2)
    gcn = MetaDenseGCN(data.num_features, 16, data.num_classes, dropout=0.5).to(device)
    params = OrderedDict((k, v.detach() * 1.1) for k, v in gcn.named_parameters())
    by_hand = Int8DenseGCN(gcn)
    assert evaluate(gcn, data, int8=True) == evaluate(by_hand, data)
    gm = BernoulliGraphModel(data.dense_adj * 0.6 + 0.02)
    manual_seed(3)
    a = empirical_mean_loss(gcn, gm, 3, data, model_parameters=params, int8=True)
    manual_seed(3)
    b = empirical_mean_loss(Int8DenseGCN(gcn, params), gm, 3, data)
    manual_seed(3)
    c = empirical_mean_loss(gcn, gm, 3, data, model_parameters=params)
    assert [m.loss for m in a] == [m.loss for m in b]
    assert all(abs(p.loss - q.loss) < 0.05 for p, q in zip(a, c))
