"""Clipped policy loss with a KL term against its definition in 64 bits.

Tolerances.  A ratio is the exponential (2 steps) of a difference rounded once, its gradient two products more: 2^-23 (8 + |d|) of its size,
and the same of the KL term's; their sum is bounded by the sum of both sizes.  Sums are in 64 bits, results rounded once: a mean
is off by its terms' errors and 2^-24 of itself."""
import math

import pytest
import torch

from piper_b200 import nn, ops
from piper_b200.ops import native

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
INF, NAN = float("inf"), float("nan")


def _offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return torch.tensor(out)


def _inputs(T, device, seed, far=0.05):
    g = torch.Generator().manual_seed(seed)
    old = -torch.rand(T, generator=g) * 6 - 0.01
    new = old + torch.randn(T, generator=g) * 0.2
    new = torch.where(torch.rand(T, generator=g) < far, new + torch.randn(T, generator=g) * 4, new)
    ref = old + torch.randn(T, generator=g) * 0.3
    adv = torch.randn(T, generator=g)
    adv[torch.rand(T, generator=g) < 0.05] = 0.0
    mask = torch.rand(T, generator=g) < 0.7
    return [t.to(device) for t in (new, old, adv, ref, mask)]


def _definition(new, old, adv, ref, mask, lens, clip, kl_coef):
    """(loss, kl, clipped, gradient), then the bounds of loss, kl and gradient."""
    new, old, adv = (t.detach().double().cpu() for t in (new, old, adv))
    T = new.numel()
    on = torch.ones(T, dtype=torch.bool) if mask is None else mask.cpu()
    w = torch.zeros(T, dtype=torch.float64)
    if lens is None:
        groups = [(0, T)]
    else:
        at = _offsets(lens).tolist()
        groups = list(zip(at, at[1:]))
    live = [(a, b) for a, b in groups if bool(on[a:b].any())]
    for a, b in live:
        w[a:b] = 1.0 / int(on[a:b].sum()) / len(live)
    on = on & (w > 0)
    res = [0.0, 0.0, 0, torch.zeros(T, dtype=torch.float64), 0.0, 0.0, torch.zeros(T, dtype=torch.float64)]
    for t in on.nonzero().squeeze(1).tolist():
        A, d = float(adv[t]), float(new[t]) - float(old[t])
        r = math.exp(min(d, 700))
        clipped = (A > 0 and r > 1 + clip[1]) or (A < 0 and r < 1 - clip[0])
        each = -A * min(max(r, 1 - clip[0]), 1 + clip[1]) if clipped else (-A * r if A else 0.0)
        grad = 0.0 if clipped or not A else -A * r
        size = (abs(each) + abs(grad)) * (8 + abs(d))
        res[2] += clipped
        if ref is not None:
            u = float(ref[t]) - float(new[t])
            kl = math.expm1(u) - u if abs(u) > 1e-2 else sum(u ** i / math.factorial(i) for i in range(2, 9))
            each, grad = each + kl_coef * kl, grad - kl_coef * math.expm1(u)
            res[1] += float(w[t]) * kl
            res[5] += float(w[t]) * kl * (8 + abs(u))
            size += abs(kl_coef) * (abs(math.expm1(u)) + kl) * (8 + abs(u))
        res[0] += float(w[t]) * each
        res[4] += float(w[t]) * size
        res[3][t], res[6][t] = grad * float(w[t]), size * float(w[t])
    res[2] /= max(1, int(on.sum()))
    return res


def _check(r, d, want, up=1.0):
    loss, kl, clipped, grad, e_loss, e_kl, e_grad = want
    step = 2.0 ** -23
    assert abs(float(r.loss) - loss) <= step * (e_loss + abs(loss)), (float(r.loss), loss)
    assert abs(float(r.kl) - kl) <= step * (e_kl + abs(kl)), (float(r.kl), kl)
    assert abs(float(r.clipped) - clipped) <= step * clipped
    off = (d.double().cpu().reshape(-1) - up * grad).abs()
    assert bool((off <= abs(up) * step * (e_grad + 4 * grad.abs()) + 2.0 ** -140).all()), float(off.max())


SHAPES = [(1, None), (7, None), (127, None), (128, None), (129, [129]), (300, [0, 100, 0, 1, 140]), (5000, None), (5000, [4000, 3, 900]),
          (4100, [7] * 500), (700, [300, 400])]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kl_coef", [0.0, 0.05])
@pytest.mark.parametrize("T,lens", SHAPES, ids=lambda v: str(v) if isinstance(v, int) or v is None else f"{len(v)}x{max(v)}")
def test_loss_and_gradient(T, lens, kl_coef, device):
    new, old, adv, ref, mask = _inputs(T, device, T)
    s = None if lens is None else ops.pack_sequences(_offsets(lens), T, device=device)
    for m in (mask, None):
        for use_ref in (True, False):
            if kl_coef and not use_ref:
                continue
            x = new.clone().requires_grad_(True)
            r = ops.clipped_policy_loss(x, old, adv, ref_logprob=ref if use_ref else None, mask=m, sequences=s, clip=(0.2, 0.3),
                                        kl_coef=kl_coef)
            (d,) = torch.autograd.grad(r.loss, x, torch.tensor(-0.5, device=device))
            _check(r, d, _definition(new, old, adv, ref if use_ref else None, m, lens, (0.2, 0.3), kl_coef), -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("T,lens", [(4096, None), (4097, None), (4000, [2000, 1, 1999]), (4096, [7] * 500), (65536, None), (70000, [30000, 1, 39000]), (66000, [100] * 650), (300000, None)])
def test_both_sides_of_the_limit_of_one_launch(T, lens):
    new, old, adv, ref, mask = _inputs(T, "cuda", 1)
    s = None if lens is None else ops.pack_sequences(_offsets(lens), T, device="cuda")
    x = new.clone().requires_grad_(True)
    r = ops.clipped_policy_loss(x, old, adv, ref_logprob=ref, mask=mask, sequences=s, kl_coef=0.1)
    (d,) = torch.autograd.grad(r.loss, x)
    _check(r, d, _definition(new, old, adv, ref, mask, lens, (0.2, 0.2), 0.1))
    if lens is not None:                          # offsets that only the GPU knows: more blocks in the table's memory than in use
        s = ops.pack_sequences(_offsets(lens).cuda(), T)
        again = ops.clipped_policy_loss(x, old, adv, ref_logprob=ref, mask=mask, sequences=s, kl_coef=0.1)
        (d2,) = torch.autograd.grad(again.loss, x)
        assert torch.equal(d2, d) and abs(float(again.loss - r.loss)) <= 2.0 ** -23 * abs(float(r.loss))
    native.check_status()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lens", [None, [100, 50, 50]])
def test_what_does_not_count_reaches_nothing(lens, device):
    T = 230
    new, old, adv, ref, mask = _inputs(T, device, 3)
    mask[100:150] = False
    s = None if lens is None else ops.pack_sequences(_offsets(lens), T, device=device)
    left_out = ~mask
    if lens is not None:
        left_out[200:] = True
    results = []
    for value in (0.0, NAN, INF, -INF):
        args = [torch.where(left_out, value, t) for t in (new, old, adv, ref)]
        x = args[0].requires_grad_(True)
        r = ops.clipped_policy_loss(x, args[1], args[2], ref_logprob=args[3], mask=mask, sequences=s, kl_coef=0.1)
        (d,) = torch.autograd.grad(r.loss, x)
        assert not bool(d[left_out].any())
        results.append((r.loss.detach(), r.kl, r.clipped, d))
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))
    _check(ops.PolicyLoss(*results[0][:3]), results[0][3], _definition(new, old, adv, ref, mask, lens, (0.2, 0.2), 0.1))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T", [0, 1, 200])
def test_nothing_counts(T, device):
    new, old, adv, ref, mask = _inputs(T, device, 4)
    mask[:] = False
    for s in (None, ops.pack_sequences(torch.tensor([0]), T, device=device), ops.pack_sequences(torch.tensor([0, 0, T]), T, device=device)):
        x = new.clone().requires_grad_(True)
        r = ops.clipped_policy_loss(x, old, adv, ref_logprob=ref, mask=mask, sequences=s, kl_coef=0.1)
        (d,) = torch.autograd.grad(r.loss, x)
        assert [float(v) for v in r] == [0.0, 0.0, 0.0] and d.shape == x.shape and not bool(d.any())


@pytest.mark.parametrize("device", DEVICES)
def test_borders_and_extremes(device):
    """A ratio at a border by fp32 rounding goes by its exact difference; ratios that overflow are clipped or infinite."""
    high, low = math.log(1.2), math.log(0.8)
    old = torch.tensor([-2.0, -2.0, -2.0, -2.0, -300.0, -300.0, -1.0, -1.0, -100.0])
    new = torch.tensor([0.0] * 9)
    new[0] = torch.nextafter(torch.tensor(-2.0 + high), torch.tensor(1.0))
    new[1] = torch.nextafter(torch.tensor(-2.0 + high), torch.tensor(-9.0))
    new[2] = torch.nextafter(torch.tensor(-2.0 + low), torch.tensor(1.0))
    new[3] = torch.nextafter(torch.tensor(-2.0 + low), torch.tensor(-9.0))
    new[6], new[7] = -INF, -INF
    adv = torch.tensor([1.0, 1.0, -1.0, -1.0, 1.0, -1.0, 1.0, -1.0, 0.0])
    new, old, adv = (t.to(device) for t in (new, old, adv))
    x = new.clone().requires_grad_(True)
    for i in range(9):
        mask = torch.zeros(9, dtype=torch.bool, device=device)
        mask[i] = True
        r = ops.clipped_policy_loss(x, old, adv, mask=mask)
        (d,) = torch.autograd.grad(r.loss, x)
        diff = float(new[i].double() - old[i].double())
        if i == 5:                                # r = inf, not clipped: -A r
            assert float(r.loss) == INF and float(r.clipped) == 0
            continue
        clipped = diff > high if float(adv[i]) > 0 else diff < low if float(adv[i]) < 0 else False
        assert bool(r.clipped) == clipped, i
        want = -float(adv[i]) * ((1.2 if float(adv[i]) > 0 else 0.8) if clipped else math.exp(min(diff, 600)))
        assert float(r.loss) == pytest.approx(want if float(adv[i]) else 0.0, rel=2.0 ** -20)
        assert float(d[i]) == pytest.approx(0.0 if clipped or not float(adv[i]) else want, rel=2.0 ** -20)


@pytest.mark.parametrize("device", DEVICES)
def test_small_and_large_divergences(device):
    """e^u - 1 - u keeps its digits on both sides of where the series ends."""
    u = torch.tensor([0.0, 1e-30, 1e-6, -1e-3, 0.1, -0.49999, 0.49999, 0.50001, -0.50001, 3.0, -20.0, 60.0], device=device)
    zero = torch.zeros_like(u)
    for i in range(len(u)):
        mask = torch.zeros(len(u), dtype=torch.bool, device=device)
        mask[i] = True
        v = float(u[i])
        want = sum(v ** k / math.factorial(k) for k in range(2, 18)) if abs(v) < 1 else math.expm1(v) - v
        x = zero.clone().requires_grad_(True)
        r = ops.clipped_policy_loss(x, zero, zero, ref_logprob=u, mask=mask, kl_coef=1.0)
        (d,) = torch.autograd.grad(r.loss, x)
        # six roundings of the series, or 2 steps of expm1 and one of the difference, below 4 times the result above 0.5; results are
        # fp32 numbers, whose smallest step is 2^-149 (u = 1e-30: 5e-61 is none but 0)
        assert abs(float(r.kl) - want) <= 2.0 ** -21 * want + 2.0 ** -149 and float(r.loss) == float(r.kl)
        assert abs(float(d[i]) + math.expm1(v)) <= 2.0 ** -22 * abs(math.expm1(v))


@pytest.mark.parametrize("device", DEVICES)
def test_shapes_and_what_is_refused(device):
    new, old, adv, ref, mask = _inputs(60, device, 5)
    flat = ops.clipped_policy_loss(new, old, adv, ref_logprob=ref, mask=mask, kl_coef=0.1)
    x = new.view(4, 15).t().contiguous().t().requires_grad_(True)                   # strided
    r = ops.clipped_policy_loss(x, old.view(4, 15), adv.view(4, 15), ref_logprob=ref.view(4, 15), mask=mask.view(4, 15), kl_coef=0.1)
    (d,) = torch.autograd.grad(r.loss, x)
    assert torch.equal(flat.loss, r.loss) and d.shape == x.shape
    s = ops.pack_sequences(torch.tensor([0, 59]), 59, device=device)
    bad = [dict(old_logprob=old[:59]), dict(advantages=adv.double()), dict(mask=mask.int()), dict(logprob=new.to(torch.bfloat16)),
           dict(clip=(-0.1, 0.2)), dict(clip=(1.1, 0.2)), dict(clip=(0.2, -0.1)), dict(clip=(0.2, INF)), dict(clip=(NAN, 0.2)),
           dict(kl_coef=0.1, ref_logprob=None), dict(kl_coef=NAN), dict(sequences=s), dict(ref_logprob=ref.view(4, 15))]
    if device == "cuda":
        bad += [dict(mask=mask.cpu()), dict(old_logprob=old.cpu()), dict(sequences=ops.pack_sequences(torch.tensor([0, 60]), 60))]
    for change in bad:
        args = {**dict(logprob=new, old_logprob=old, advantages=adv, ref_logprob=ref, mask=mask), **change}
        with pytest.raises((ValueError, TypeError)):
            ops.clipped_policy_loss(**args)


@pytest.mark.parametrize("device", DEVICES)
def test_gradient_against_differences_and_no_second_one(device):
    """Central differences of the fp32 loss of a few tokens, none within 0.01 of a border."""
    old = torch.tensor([-1.0, -2.0, -0.5, -3.0], device=device)
    new = old + torch.tensor([0.05, 0.5, -0.6, 0.1], device=device)
    adv, ref = torch.tensor([1.0, 1.0, -1.0, -2.0], device=device), old + 0.2
    x = new.clone().requires_grad_(True)
    r = ops.clipped_policy_loss(x, old, adv, ref_logprob=ref, kl_coef=0.5)
    (d,) = torch.autograd.grad(r.loss, x, create_graph=True)
    h = 2.0 ** -8
    for i in range(4):
        e = torch.zeros_like(new)
        e[i] = h
        up, down = (ops.clipped_policy_loss(v, old, adv, ref_logprob=ref, kl_coef=0.5).loss for v in (new + e, new - e))
        # a loss below 2 rounded to 2^-24 of it twice, over 2h; h^2 / 6 of a third derivative below 4
        assert abs(float(up - down) / (2 * h) - float(d[i])) < 4 * 2.0 ** -24 / (2 * h) * 4 + h * h
    with pytest.raises(RuntimeError):
        d.sum().backward()


@pytest.mark.gpu
def test_native_formulas_do_what_the_python_ones_do():
    new, old, adv, ref, mask = _inputs(400, "cuda", 6)
    s = ops.pack_sequences(torch.tensor([0, 150, 390]), 400, device="cuda")
    lib = native.lib()

    def results():
        x = new.clone().requires_grad_(True)
        r = ops.clipped_policy_loss(x, old, adv, ref_logprob=ref, mask=mask, sequences=s, kl_coef=0.1)
        return [v.detach() for v in r] + list(torch.autograd.grad(r.loss, x))

    want = results()
    lib.native_op_remove("clipped_policy_fwd")
    try:
        got = results()
    finally:
        lib.native_op_install("clipped_policy_fwd")
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_streams_and_graphs():
    new, old, adv, ref, mask = _inputs(3000, "cuda", 7)
    x = new.clone().requires_grad_(True)

    def step(s):
        r = ops.clipped_policy_loss(x, old, adv, ref_logprob=ref, mask=mask, sequences=s, kl_coef=0.1)
        return r.loss.detach(), r.kl, r.clipped, torch.autograd.grad(r.loss, x)[0]

    both = [None, ops.pack_sequences(torch.tensor([0, 1000, 2500]), 3000, device="cuda")]
    want = [step(s) for s in both]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(4):
        for stream, s in zip(streams, both):
            with torch.cuda.stream(stream):
                got.append(step(s))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))
    graphs = []
    for s in both:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(s)
        graphs.append((graph, out))
    for stream, (graph, _out) in zip(streams, graphs):
        with torch.cuda.stream(stream):
            graph.replay()
    torch.cuda.synchronize()
    for (_graph, out), w in zip(graphs, want):
        assert all(torch.equal(a, b) for a, b in zip(out, w))


@pytest.mark.parametrize("device", DEVICES)
def test_from_logits(device):
    """nn.clipped_policy_loss: log probabilities of the tokens, then the loss; ids that do not count are left out."""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    g = torch.Generator().manual_seed(8)
    logits = torch.randn(2, 40, 97, generator=g).to(dtype).to(device).requires_grad_(True)
    tokens = torch.randint(0, 97, (2, 40), generator=g).to(device)
    tokens[:, :7] = -100
    tokens[1, 30] = 97
    new, old, adv, ref, mask = _inputs(80, device, 9)
    s = ops.pack_sequences(torch.tensor([0, 33, 70]), 80, device=device)
    loss = nn.clipped_policy_loss(logits, tokens, adv.view(2, 40), old.view(2, 40), ref_logprob=ref.view(2, 40), mask=mask.view(2, 40),
                                  sequences=s, clip=(0.2, 0.3), kl_coef=0.1, temperature=0.8)
    (d,) = torch.autograd.grad(loss, logits)
    lp = ops.token_logprobs(logits, tokens, temperature=0.8).logprob.detach().reshape(-1)
    counted = mask & (tokens.reshape(-1) >= 0) & (tokens.reshape(-1) < 97)
    want = _definition(lp, old, adv, ref, counted, [33, 37], (0.2, 0.3), 0.1)
    assert abs(float(loss) - want[0]) <= 2.0 ** -23 * (want[4] + abs(want[0]))
    assert bool((d.view(80, 97)[~counted] == 0).all()) and bool((d.view(80, 97)[70:] == 0).all())
    z = torch.log_softmax(logits.detach().double().cpu().view(80, 97) / 0.8, 1)
    onehot = torch.nn.functional.one_hot(tokens.cpu().reshape(-1).clamp(0, 96), 97)
    grad = want[3].unsqueeze(1) * (onehot - z.exp()) / 0.8
    half = torch.finfo(dtype).eps / 2
    size = (want[3].abs() + 2.0 ** -23 * want[6]).unsqueeze(1) * (onehot + z.exp()) / 0.8
    off = (d.double().cpu().view(80, 97) - grad).abs()
    assert bool((off <= half * grad.abs() + 2.0 ** -18 * size + 1e-30).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lens", [None, [2, 1]])
def test_divergences_without_bound(lens, device):
    """A token that counts and whose log probability is -inf, as a masked id's, is infinitely far from a reference that gives it one, not NaN."""
    old, ref = torch.tensor([-1.0, -2.0, -3.0], device=device), torch.tensor([-1.5, -2.0, -2.5], device=device)
    adv = torch.tensor([1.0, 0.0, -1.0], device=device)
    s = None if lens is None else ops.pack_sequences(_offsets(lens), 3, device=device)
    for at, value, grad in ((0, -INF, -INF), (1, -INF, -INF), (2, -INF, -INF), (0, INF, None), (1, INF, None)):
        x, y = old.clone(), ref.clone()
        if grad is None:                          # a reference of -inf: u = -inf, whose gradient is that of -u
            y[at] = -INF
        else:
            x[at] = value
        x.requires_grad_(True)
        for kl_coef in (0.5, 0.0):
            r = ops.clipped_policy_loss(x, old, adv, ref_logprob=y, sequences=s, kl_coef=kl_coef)
            (d,) = torch.autograd.grad(r.loss, x)
            assert float(r.kl) == INF
            assert float(r.loss) == INF if kl_coef else math.isfinite(float(r.loss))
            assert bool(torch.isfinite(d[torch.arange(3, device=device) != at]).all())
            if kl_coef and grad is not None:
                assert float(d[at]) == grad
            else:
                assert math.isfinite(float(d[at]))
    if device == "cuda":
        native.check_status()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("diff", [-1.0, 0.0, 1.0])
def test_advantages_that_are_nan_leave_a_trace(diff, device):
    """Below, between and above the borders: the loss and the token's gradient are NaN, and no border is its."""
    old = torch.tensor([-2.0, -2.0, -2.0], device=device)
    new = old + torch.tensor([0.1, diff, 0.1], device=device)
    adv = torch.tensor([1.0, NAN, -1.0], device=device)
    x = new.requires_grad_(True)
    r = ops.clipped_policy_loss(x, old, adv)
    (d,) = torch.autograd.grad(r.loss, x)
    assert torch.isnan(r.loss) and torch.isnan(d).tolist() == [False, True, False] and float(r.clipped) == 0
    on = torch.tensor([True, False, True], device=device)
    r = ops.clipped_policy_loss(x, old, adv, mask=on)         # nor where the token does not count
    (d,) = torch.autograd.grad(r.loss, x)
    assert torch.isfinite(r.loss) and float(d[1]) == 0 and bool(torch.isfinite(d).all())


@pytest.mark.gpu
@pytest.mark.parametrize("T,lens", [(600, [1, 2, 0, 1] * 125), (700, [3] * 40 + [580]), (9000, None)])
def test_the_gradient_has_a_warp_for_every_block(T, lens, tmp_path):
    """Blocks are of 128 tokens or, in a packed batch, of a sequence: many short ones are more than their tokens would say."""
    import json
    new, old, adv, ref, mask = _inputs(T, "cuda", 10)
    s = None if lens is None else ops.pack_sequences(_offsets(lens), T, device="cuda")
    blocks = (T + 127) // 128 if lens is None else sum((n + 127) // 128 for n in lens)
    x = new.requires_grad_(True)

    def step():
        r = ops.clipped_policy_loss(x, old, adv, ref_logprob=ref, mask=mask, sequences=s, kl_coef=0.05)
        return r, torch.autograd.grad(r.loss, x)[0]

    _check(*step(), _definition(new, old, adv, ref, mask, lens, (0.2, 0.2), 0.05))
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        step()
        torch.cuda.synchronize()
    prof.export_chrome_trace(str(tmp_path / "trace.json"))
    grids = [e["args"]["grid"][0] for e in json.loads((tmp_path / "trace.json").read_text())["traceEvents"]
             if e.get("cat") == "kernel" and "policy_bwd" in e["name"]]
    assert grids and all(8 * g >= blocks for g in grids)
