"""Balance loss of a router, its counts, mean probabilities and gradient, against the definition in 64 bits.

Tolerances.  A probability is an exponential (2 steps, of a difference rounded once: at most 2^-24 |x|) over a sum of E of them: 2^-22 (4 + |x|
largest) of its size, with sums over a lane's rows in fp32 2^-24 of them each.  A gradient p (c - p.c) is that of p times two
sizes, and half a step of the logits' type."""
import pytest
import torch

from piper_b200 import ops
from piper_b200.ops import moe, native

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
INF = float("inf")


def _inputs(T, E, k, dtype, device, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, E, generator=g) * 2 + torch.randn(E, generator=g)).to(dtype)
    idx = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :k].to(torch.int32).contiguous()
    mask = torch.rand(T, generator=g) < 0.8
    return x.to(device), idx.to(device), mask.to(device)


def _check(x, idx, mask, r, d, up):
    T, E = x.shape
    k = idx.shape[1]
    x64 = x.detach().double().cpu()
    on = torch.ones(T, dtype=torch.bool) if mask is None else mask.cpu()
    n = max(1, int(on.sum()))
    nothing = torch.isneginf(x64).all(1, keepdim=True)
    p = torch.softmax(torch.where(nothing, 0.0, x64), 1) * ~nothing
    counts = torch.bincount(idx.cpu()[on].reshape(-1).long(), minlength=E)
    P, f = p[on].sum(0) / n, counts.double() / (n * k)
    rel = 2.0 ** -22 * (4 + float(x64[torch.isfinite(x64)].abs().max() if x64.numel() else 0)) + T * 2.0 ** -24 / (1 if T < 4096 else 8)
    assert torch.equal(r.counts.cpu().long(), counts) and r.counts.dtype == torch.int32
    assert bool(((r.prob.double().cpu() - P).abs() <= rel * P + 1e-30).all())
    loss = float(E * (f * P).sum())
    assert abs(float(r.loss) - loss) <= rel * loss
    c = E / n * f * up
    want = p * (c - (p * c).sum(1, keepdim=True)) * on.unsqueeze(1)
    size = p * (c.abs() + (p * c.abs()).sum(1, keepdim=True))
    off = (d.double().cpu() - want).abs()
    bound = torch.finfo(x.dtype).eps / 2 * want.abs() + 2.0 ** -21 * (6 + float(x64[torch.isfinite(x64)].abs().max() if x64.numel() else 0)) * size
    assert bool((off <= bound * 1.01 + 1e-37).all()), float((off - bound).max())
    assert not bool(d[~on.to(d.device)].any())


def _pass(x, idx, mask, up=0.7):
    leaf = x.detach().requires_grad_(True)
    r = moe.moe_balance_loss(leaf, idx, mask=mask)
    (d,) = torch.autograd.grad(r.loss, leaf, torch.tensor(up, device=x.device))
    return r, d


SHAPES = [(1, 1, 1), (1, 8, 2), (3, 7, 7), (31, 9, 2), (64, 16, 4), (65, 64, 8), (130, 60, 3), (257, 128, 8), (40, 255, 5), (33, 256, 8),
          (2000, 128, 2), (1500, 33, 4)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,E,k", SHAPES)
def test_loss_counts_and_gradient(T, E, k, dtype, device):
    x, idx, mask = _inputs(T, E, k, dtype, device, T + E)
    for m in (None, mask):
        r, d = _pass(x, idx, m)
        _check(x, idx, m, r, d, 0.7)
    if device == "cuda":
        native.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("T,E", [(512, 128), (513, 128), (1025, 128), (8192, 8), (8200, 8), (30000, 60), (70000, 256)])
def test_both_sides_of_the_cluster_limit(T, E):
    x, idx, mask = _inputs(T, E, 4, torch.bfloat16, "cuda", 1)
    for m in (None, mask):
        r, d = _pass(x, idx, m, -3.0)
        _check(x, idx, m, r, d, -3.0)
        again, d2 = _pass(x, idx, m, -3.0)
        assert torch.equal(r.loss, again.loss) and torch.equal(r.prob, again.prob) and torch.equal(d, d2)
    native.check_status()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_experts_and_masked_tokens(dtype, device):
    """Experts masked by -inf or by the type's lowest value, rows that have none left, anything at tokens that do not count."""
    x, idx, mask = _inputs(100, 24, 3, dtype, device, 2)
    x[:, 5] = -INF
    x[:, 7] = torch.finfo(dtype).min
    x[3], mask[3] = -INF, True
    mask[10:20] = False
    r, d = _pass(x, idx, mask)
    _check(torch.where(torch.isneginf(x) | (x > -1e30), x, torch.full_like(x, -INF)), idx, mask, r, d, 0.7)
    assert not bool(d[3].any()) and not bool(d[:, 5].any()) and not bool(d[:, 7].any())
    for value in (float("nan"), INF, -INF):
        y, other = x.clone(), idx.clone()
        y[~mask] = value
        other[~mask] = 1 << 20
        r2, d2 = _pass(y, other, mask)
        assert all(torch.equal(a, b) for a, b in zip((*r, d), (*r2, d2)))
    r, d = _pass(x, idx, torch.zeros_like(mask))
    assert float(r.loss) == 0 and not bool(r.counts.any()) and not bool(r.prob.any()) and not bool(d.any())
    r, d = _pass(x[:0], idx[:0], None)
    assert float(r.loss) == 0 and not bool(r.counts.any()) and d.shape == (0, 24)
    if device == "cuda":
        native.check_status()


@pytest.mark.parametrize("device", DEVICES)
def test_even_routing_has_loss_one(device):
    E, k = 16, 2
    x = torch.zeros(8, E, device=device)
    idx = torch.arange(E, device=device, dtype=torch.int32).view(8, k)
    r, d = _pass(x, idx, None)
    assert float(r.loss) == 1.0 and float(d.abs().max()) <= 2.0 ** -23 / 8


@pytest.mark.parametrize("device", DEVICES)
def test_what_is_refused(device):
    x, idx, mask = _inputs(10, 8, 2, torch.float32, device, 3)
    wide = torch.zeros(2, 257, device=device)
    bad = [(x, idx.long(), None), (x, idx[:9], None), (x, idx[:, :0], None), (x[0], idx, None), (wide, idx[:2], None),
           (x[:, :1], idx, None), (x, idx, mask[:9]), (x, idx, mask.int()), (x.long(), idx, None), (x, idx[0], None)]
    if device == "cuda":
        bad += [(x, idx.cpu(), None), (x, idx, mask.cpu()), (x.half(), idx, None)]
    for args in bad:
        with pytest.raises((ValueError, TypeError)):
            moe.moe_balance_loss(args[0], args[1], mask=args[2])


def test_choices_that_are_no_experts_are_refused_on_the_cpu():
    x, idx, _ = _inputs(10, 8, 2, torch.float32, "cpu", 4)
    for value in (-1, 8):
        idx[4, 1] = value
        with pytest.raises(ValueError):
            moe.moe_balance_loss(x, idx)


@pytest.mark.gpu
def test_choices_that_are_no_experts_are_reported_on_the_gpu():
    x, idx, _ = _inputs(10, 8, 2, torch.float32, "cuda", 4)
    for value in (-1, 8, 1 << 30):
        idx[4, 1] = value
        r = moe.moe_balance_loss(x, idx)
        assert int(r.counts.sum()) == 19
        with pytest.raises(native.PiperKernelError):
            native.check_status()
    native.check_status()


@pytest.mark.parametrize("device", DEVICES)
def test_gradient_against_differences_and_no_second_one(device):
    g = torch.Generator().manual_seed(5)
    x, idx, mask = _inputs(6, 5, 2, torch.float32, device, 5)
    leaf = x.clone().requires_grad_(True)
    r = moe.moe_balance_loss(leaf, idx, mask=mask)
    (d,) = torch.autograd.grad(r.loss, leaf, create_graph=True)
    h = 2.0 ** -6
    for _ in range(4):
        v = torch.randn(x.shape, generator=g).to(device)
        up, down = (moe.moe_balance_loss(x + s * h * v, idx, mask=mask).loss for s in (1, -1))
        # losses below 5 rounded, over 2h; h^2 / 6 of a third derivative below 30 x 5
        assert abs(float(up - down) / (2 * h) - float((d * v).sum())) < 5 * 2.0 ** -22 / (2 * h) * 4 + h * h * 25
    with pytest.raises(RuntimeError):
        d.sum().backward()


@pytest.mark.gpu
def test_native_formulas_do_what_the_python_ones_do():
    lib = native.lib()
    for T, E in ((50, 24), (3000, 128)):
        x, idx, mask = _inputs(T, E, 2, torch.bfloat16, "cuda", 6)
        odd = torch.zeros(T * E + 1, device="cuda", dtype=torch.bfloat16)
        odd[1:] = x.reshape(-1)
        r, d = _pass(x, idx, mask)
        for y in (x, odd[1:].view(T, E), x.t().contiguous().t()):          # unaligned, strided
            r3, d3 = _pass(y, idx, mask)
            assert all(torch.equal(a, b) for a, b in zip((*r, d), (*r3, d3)))
        lib.native_op_remove("moe_balance_fwd")
        try:
            r2, d2 = _pass(x, idx, mask)
        finally:
            lib.native_op_install("moe_balance_fwd")
        assert all(torch.equal(a, b) for a, b in zip((*r, d), (*r2, d2)))


@pytest.mark.gpu
def test_streams_and_graphs():
    sets = [_inputs(700, 32, 4, torch.bfloat16, "cuda", 7), _inputs(9000, 128, 8, torch.float32, "cuda", 8)]
    want = [_pass(*s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(4):
        for stream, s in zip(streams, sets):
            with torch.cuda.stream(stream):
                got.append(_pass(*s))
    torch.cuda.synchronize()
    up = torch.tensor(0.7, device="cuda")
    graphs = []
    for x, idx, mask in sets:
        leaf = x.detach().requires_grad_(True)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = moe.moe_balance_loss(leaf, idx, mask=mask)
            (d,) = torch.autograd.grad(r.loss, leaf, up)
        graphs.append((graph, r, d))
    for stream, (graph, _r, _d) in zip(streams, graphs):
        with torch.cuda.stream(stream):
            graph.replay()
    torch.cuda.synchronize()
    for i, (r, d) in enumerate(got + [(r, d) for _g, r, d in graphs]):
        w = want[i % 2]
        assert all(torch.equal(a, b) for a, b in zip((*r, d), (*w[0], w[1])))
    native.check_status()


@pytest.mark.parametrize("device", DEVICES)
def test_a_model_with_a_balance_loss(device):
    """Qwen3Config.balance_coef: the model's loss stays, the gates' gradients are those of the loss and coef x the balance losses."""
    from piper_b200.models.qwen3 import MoE, Qwen3Config

    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    torch.manual_seed(0)
    layers = [MoE(Qwen3Config(dim=64, num_experts=8, top_k=2, moe_hidden=64, balance_coef=c)).to(device).to(dtype) for c in (0.0, 2.0)]
    with torch.no_grad():
        for p in layers[0].parameters():
            p.copy_(torch.randn(p.shape) * 0.2)
    layers[1].load_state_dict(layers[0].state_dict())
    x, dy = (torch.randn(50, 64).to(device).to(dtype) for _ in range(2))
    outs, grads = [], []
    for layer in layers:
        out = layer(x)
        outs.append(out.detach())
        (out * dy).sum().backward()
        grads.append(layer.gate.weight.grad.double().cpu())
    assert torch.equal(*outs)
    logits = layers[0].gate(x).detach().requires_grad_(True)
    _w, idx, _c = moe.moe_route(logits, 2, True)
    (d,) = torch.autograd.grad(moe.moe_balance_loss(logits, idx).loss, logits)
    want = 2.0 * (d.double().t() @ x.double()).cpu()
    half = torch.finfo(dtype).eps / 2
    # logits' gradients of both terms are rounded and added once more, weights' gradients rounded on both sides
    size = (d.double().abs() * 2).t() @ x.double().abs()
    route = torch.autograd.grad((layers[0](x) * dy).sum(), layers[0].gate.weight)[0].double().abs()
    tol = half * 4 * (size.cpu() + grads[0].abs() + grads[1].abs() + route.cpu()) + half * 4 * _route_size(layers[0], x, dy)
    assert bool(((grads[1] - grads[0] - want).abs() <= tol).all())
    if device == "cpu":                          # in bf16 the roundings of the model's own gradient are larger than what is added to it
        assert float(want.abs().max()) > 10 * float(tol.min())
    # nothing of the model's own: the gradient of the balance loss alone
    layers[1].zero_grad()
    (layers[1](x) * torch.zeros_like(dy)).sum().backward()
    got = layers[1].gate.weight.grad.double().cpu()
    assert bool(((got - want).abs() <= half * 4 * size.cpu() + half * want.abs()).all())
    worst, least = float((half * 4 * size.cpu() + half * want.abs()).max()), float(want.abs().max())
    assert least > 4 * worst


def _route_size(layer, x, dy):
    """Magnitudes that the gate's gradient of the model's own loss is summed from."""
    logits = layer.gate(x).detach().requires_grad_(True)
    w, idx, counts = moe.moe_route(logits, layer.top_k, layer.renorm)
    rows, pos, g_start, g_len, c = moe.moe_dispatch(x, idx, counts)
    out = moe.moe_combine(layer.experts(rows, c), pos, w, g_start, g_len, counts)
    (d,) = torch.autograd.grad((out * dy).sum(), logits)
    return (d.double().abs().t() @ x.double().abs()).cpu()
