"""Log probabilities of tokens, entropy and alternatives against their definition in 64 bits.

Tolerances.  Sums run over a thread's V / 512 elements (all V in a plain sum on the CPU) and about twenty merges; a term's
relative error is a few 2^-23 and that of its exponent.  So log S is off by less than 2^-24 (depth + 40), a log probability by
that and three roundings of its own size, the entropy by the same relative to its largest term.  A gradient is
-p (a + b log p), whose two addends may cancel: its error is 2^-20 of their absolute sum, and half a step of its type."""
import math

import pytest
import torch

from piper_b200 import ops

INF = float("inf")
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _definition(x, tokens, top, temperature, ignore_index=-100):
    """In 64 bits, row by row of the formulas; ids by sorting (value falling, id rising)."""
    x = x.detach().double().cpu()
    tokens = tokens.cpu()
    V = x.shape[-1]
    left = torch.isfinite(x).any(-1, keepdim=True)
    z = torch.where(left, x - x.amax(-1, keepdim=True), x) / temperature
    logp = torch.where(left, z - torch.logsumexp(z, -1, keepdim=True), torch.full_like(z, -INF))
    p = logp.exp()
    H = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
    on = (tokens != ignore_index) & (tokens >= 0) & (tokens < V)
    lp = torch.where(on, logp.gather(-1, tokens.clamp(0, V - 1).unsqueeze(-1)).squeeze(-1), 0.0)
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :top]
    return logp, p, H, on, lp, ids, left


def _gradient(x, tokens, top, temperature, dlp, dH, dtop):
    logp, p, H, on, _lp, ids, left = _definition(x, tokens, top, temperature)
    up = torch.zeros_like(p)
    V = p.shape[-1]
    up.scatter_add_(-1, tokens.cpu().clamp(0, V - 1).unsqueeze(-1), (dlp.double().cpu() * on).unsqueeze(-1))
    if top:
        up.scatter_add_(-1, ids, dtop.double().cpu())
    u = torch.where(p > 0, logp, torch.zeros_like(p))
    dh = dH.double().cpu().unsqueeze(-1)
    g = up.sum(-1, keepdim=True)
    d = (up - p * g - dh * p * (u + H.unsqueeze(-1))) / temperature
    size = (up.abs() + p * (up.abs().sum(-1, keepdim=True) + dh.abs() * (u.abs() + H.unsqueeze(-1)))) / temperature
    return torch.where(left, d, torch.zeros_like(d)), size


def _check(x, tokens, top, temperature, out, d=None, gradients=None):
    V = x.shape[-1]
    eps = 2.0 ** -24
    depth = (V if not x.is_cuda else V / 512 + 20) + 40
    logp, p, H, on, lp, ids, left = _definition(x, tokens, top, temperature)
    row = eps * depth

    def close(got, want, tol):
        got = got.double().cpu()
        same = (got == want) | ((got - want).abs() <= tol)
        assert bool(same.all()), (got[~same][:5], want[~same][:5])

    close(out.logprob, lp, row + 6 * eps * lp.abs().nan_to_num(posinf=0))
    close(out.entropy, H, row * (1 + H) + 8 * eps * math.log(V + 1))
    assert torch.equal(out.top_id.cpu(), ids)
    want = logp.gather(-1, ids)
    close(out.top_logprob, want, row + 6 * eps * want.abs().nan_to_num(posinf=0))
    if d is not None:
        want, size = _gradient(x, tokens, top, temperature, *gradients)
        half = torch.finfo(x.dtype).eps / 2
        tiny = torch.finfo(x.dtype).tiny
        close(d, want, half * want.abs() + (2.0 ** -20 + 2 * row) * size + tiny)


def _logits(T, V, dtype, device, seed, std=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, V, generator=g) * std).to(dtype)
    tokens = torch.randint(0, V, (T,), generator=g)
    return x.to(device), tokens.to(device)


SHAPES = [(1, 1, 0), (1, 1, 1), (3, 7, 7), (2, 31, 20), (5, 33, 32), (4, 257, 5), (2, 4099, 32), (3, 8191, 3), (1, 128256, 20),
          (2, 40000, 32), (300, 2048, 4), (40, 32003, 6), (0, 50, 3)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V,top", SHAPES)
def test_values_and_gradients(T, V, top, dtype, device):
    for temperature in (1.0, 0.7):
        x, tokens = _logits(T, V, dtype, device, 3 * T + V)
        if T > 2:
            tokens[1], tokens[2] = -100, V
        x.requires_grad_(True)
        out = ops.token_logprobs(x, tokens, top=top, temperature=temperature)
        g = torch.Generator().manual_seed(5)
        gradients = [torch.randn(s, generator=g).to(device) for s in ((T,), (T,), (T, top))]
        (d,) = torch.autograd.grad([out.logprob, out.entropy, out.top_logprob], x, gradients)
        assert d.dtype == dtype and d.shape == x.shape
        _check(x, tokens, top, temperature, out, d, gradients)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [9, 600, 10007])
def test_rows_that_are_special(V, dtype, device):
    low = torch.finfo(dtype).min
    x, tokens = _logits(8, V, dtype, device, V)
    x[0] = -INF                                   # nothing left
    x[1] = low                                    # all equal, at the type's lowest value
    x[2] = low
    x[2, V - 1] = 2.0                             # one token has all
    x[3, ::2] = -INF
    x[4] = -INF
    x[4, V // 2] = -7.0                           # a single one left
    x[5] = 0.0
    x[5, 1::2] = -0.0                             # equal numbers of two signs
    x[6] = x[6].round()                           # many ties
    x[7, 0] = low
    tokens[2], tokens[3], tokens[4] = 0, 0, V // 2
    x.requires_grad_(True)
    top = min(V, 8)
    out = ops.token_logprobs(x, tokens, top=top)
    gradients = [torch.ones(8, device=device), torch.full((8,), 0.5, device=device), torch.full((8, top), 0.1, device=device)]
    (d,) = torch.autograd.grad([out.logprob, out.entropy, out.top_logprob], x, gradients)
    assert bool(torch.isfinite(d).all())
    _check(x, tokens, top, 1.0, out, d, gradients)
    assert out.entropy[0] == 0 and out.logprob[0] == -INF and not d[0].any()
    assert out.top_id[0].tolist() == list(range(top))


MASKS = [-1e4, -7e8, -1e9, -1e10, -1e20, -7e29, -3e38]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V,offset", [(1, 9, 0), (1, 32003, 1), (6, 4099, 0), (6, 17003, 0), (600, 515, 3)])
def test_rows_that_are_masked_by_large_numbers(T, V, offset, dtype, device):
    """Masks that are finite, over most of a row, all of it, its first half and around single ids: a masked id has probability 0 beside
    one that is not, and a row of nothing else is uniform.  Log probabilities below the smallest fp32 number are -inf."""
    few = 4
    for mask in MASKS:
        for temperature in (0.1, 0.3, 0.6, 0.8, 1.0) if T * V < 50000 else (0.3, 0.6, 1.0):
            x, tokens = _logits(T, V, dtype, "cpu", V)
            real = x.clone()
            for r in range(T):
                if r % 6 == 0:
                    x[r, :V - few - 1] = mask                 # all but a few at the end, one more behind them
                    x[r, V - 1] = mask
                    tokens[r] = V - 2
                elif r % 6 == 1:
                    x[r] = mask
                elif r % 6 == 2:
                    x[r, :V // 2] = mask
                elif r % 6 == 3:
                    x[r, few:] = mask                         # all but a few in front
                elif r % 6 == 4:
                    x[r] = mask
                    x[r, V // 3] = real[r, V // 3]            # a single one left
                else:
                    x[r, :V // 2] = mask
                    x[r, V // 2:V // 2 + few] = 2 * mask if mask > -1e38 else -INF
            store = torch.zeros(T * V + 8, dtype=dtype, device=device)
            x = store[offset:offset + T * V].copy_(x.reshape(-1)).view(T, V).requires_grad_(True)
            tokens = tokens.to(device)
            out = ops.token_logprobs(x, tokens, top=few, temperature=temperature)
            g = torch.Generator().manual_seed(6)
            gradients = [torch.randn(s, generator=g).to(device) for s in ((T,), (T,), (T, few))]
            (d,) = torch.autograd.grad([out.logprob, out.entropy, out.top_logprob], x, gradients)
            logp, _p, H, _on, lp, ids, _left = _definition(x, tokens, few, temperature)
            assert torch.equal(out.top_id.cpu(), ids)
            eps, row = 2.0 ** -24, 2.0 ** -24 * ((V if device == "cpu" else V / 512 + 20) + 40)
            for got, want, extra in ((out.logprob, lp, 0), (out.top_logprob, logp.gather(-1, ids), 0), (out.entropy, H, row * H + 8 * eps * math.log(V + 1))):
                got, want = got.double().cpu(), want.float().double()
                assert bool(((got == want) | ((got - want).abs() <= row + extra + 6 * eps * want.abs().nan_to_num(posinf=0))).all()), \
                    (mask, temperature, got[got != want][:4], want[got != want][:4])
            want, size = _gradient(x, tokens, few, temperature, *gradients)
            # p = 2^u with u = (x - M) c2 - log S: four roundings (the difference, 1 / temperature, c2, the sum) and log2(e)'s own of
            # numbers up to |u| are 5 2^-24 |log p| of p.  A p below the normal numbers is 0, which loses less than the
            # smallest of them times what p is multiplied by.
            u = torch.where(logp.isfinite(), logp, 0.0).abs()
            d_logprob, d_entropy, d_top = (t.double().cpu().abs().view(T, -1) for t in gradients)
            times = (d_logprob + d_top.sum(1, keepdim=True) + d_entropy * (u + H.unsqueeze(1))) / temperature
            bound = (torch.finfo(dtype).eps / 2 * want.abs() + (2.0 ** -20 + 2 * row + 5 * eps * u) * size
                     + torch.finfo(dtype).tiny * (1 + times))
            far = (d.double().cpu() - want).abs() > bound
            assert not bool(far.any()), (mask, temperature, d.cpu()[far][:4], want[far][:4])


@pytest.mark.parametrize("device", DEVICES)
def test_rows_without_numbers_are_nan(device):
    for bad in (float("nan"), INF):
        x, tokens = _logits(3, 700, torch.float32, device, 1)
        x[1, 300] = bad
        out = ops.token_logprobs(x, tokens, top=3)
        for t in (out.logprob, out.entropy, out.top_logprob):
            assert bool(torch.isnan(t[1]).all()) and not bool(torch.isnan(t[0]).any()) and not bool(torch.isnan(t[2]).any())
        assert bool((out.top_id >= 0).all()) and bool((out.top_id < 700).all())
        assert len(set(out.top_id[1].tolist())) == 3


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V,masked,where", [(3, 7, None, [3]), (3, 7, None, [0]), (3, 7, 1, [6]), (2, 1000, 256, [300]), (3, 1000, None, range(16, 24)),
                                              (3, 1000, 0, range(1000)), (2, 4000, 100, [3999]), (600, 4000, 256, [1300]),
                                              (1, 128256, None, range(64, 72)), (1, 128256, 4096, [100000])])
def test_a_nan_wherever_it_is(T, V, masked, where, dtype, device):
    """Alone in a thread's elements, among masked ids, a whole vector of them, in a piece of a row that is cut: the row is NaN."""
    for mask in (-INF, -1e9):
        x, tokens = _logits(T, V, dtype, "cpu", 2)
        if masked is not None:
            x[0, masked:] = mask
        x[0, list(where)] = float("nan")
        for top in (0, 3):
            out = ops.token_logprobs(x.to(device), tokens.to(device), top=top)
            for t in (out.logprob, out.entropy, out.top_logprob):
                assert bool(torch.isnan(t[0]).all()) and not bool(torch.isnan(t[1:]).any())
            assert bool((out.top_id >= 0).all()) and bool((out.top_id < V).all())
            assert len(set(out.top_id[0].tolist())) == top


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V,offset", [(6, 9, 0), (6, 10007, 1), (600, 1031, 3)])
def test_rows_that_nothing_asks_for_have_no_gradient(T, V, offset, dtype, device):
    """Padding, whatever its logits are (0 x NaN is NaN in the formula): by an ignored token, by gradients of zero; and what the
    gradient's memory held shows nowhere, other rows are as without padding."""
    g = torch.Generator().manual_seed(5)
    x = (torch.randn(T, V, generator=g) * 3).to(dtype)
    tokens = torch.randint(0, V, (T,), generator=g)
    tokens[1::3] = -100
    tokens[2::3] = V + 7
    dlp, dH, dtop = torch.randn(T, generator=g), torch.randn(T, generator=g), torch.randn(T, 3, generator=g)
    padded = torch.arange(T) % 3 != 0
    dlp[padded] = float("nan")             # behind a token that does not count
    dH[padded] = 0
    dtop[padded] = 0
    bad = x.clone()
    bad[1::3, V // 2] = float("nan")
    bad[2::3, :] = INF
    grads = []
    for values in (x, bad):
        room = torch.zeros(T, V + 8, dtype=dtype, device=device)
        leaf = room[:, offset:offset + V]
        leaf.copy_(values)
        leaf.requires_grad_(True)
        r = ops.token_logprobs(leaf, tokens.to(device), top=3)
        dirty = torch.full((T, V), float("nan"), dtype=dtype, device=device)
        del dirty
        (d,) = torch.autograd.grad((r.logprob, r.entropy, r.top_logprob), leaf, (dlp.to(device), dH.to(device), dtop.to(device)))
        grads.append(d.cpu())
    assert all(bool((d[padded] == 0).all()) for d in grads)
    assert bool((grads[0][~padded] == grads[1][~padded]).all()) and bool((grads[0][~padded] != 0).any())


@pytest.mark.parametrize("device", DEVICES)
def test_largest_values_in_one_threads_elements(device):
    """The alternatives all at one place of the pattern in which threads take vectors, and in an order that keeps replacing them."""
    V = 65536
    for dtype, vec in ((torch.bfloat16, 8), (torch.float32, 4)):
        x = torch.zeros(1, V, dtype=dtype, device=device)
        at = torch.arange(0, V, 512 * vec, device=device)
        x[0, at] = torch.arange(1, len(at) + 1, device=device).to(dtype)
        x[0, at + 1] = torch.arange(1, len(at) + 1, device=device).to(dtype)
        tokens = torch.zeros(1, dtype=torch.int64, device=device)
        _check(x, tokens, 20, 1.0, ops.token_logprobs(x, tokens, top=20))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,offset", [(32003, 0), (32003, 1), (5003, 3), (70001, 7)])
def test_where_the_largest_values_are(V, offset, dtype, device):
    """The alternatives, one after the other: in one vector; in one thread's vectors near each other, and far apart; in front of the first
    whole vector and behind the last; the largest alone in its thread and the next ones together in another."""
    vec = 128 // torch.finfo(dtype).bits
    step = 512 * vec
    head = (-offset) % vec
    starts = [[head + 5 * vec + q for q in range(vec)], [head + 9 * vec + j * step for j in range(4)],
              [head + 9 * vec + j * step + j % vec for j in range(0, (V - 100) // step, 3)], [0, 1, V - 1, V - 2, V - 3],
              [head + 40 * vec, head + 77 * vec, head + 77 * vec + step, head + 77 * vec + 1],
              [head, V // 2, V - 1] + [head + 200 * vec + j * step for j in range(2, 14, 4)]]
    g = torch.Generator().manual_seed(11)
    room = torch.zeros(2 * len(starts), V + 8, dtype=dtype)
    x = room[:, offset:offset + V]
    x.copy_(torch.rand(2 * len(starts), V, generator=g))
    for r, places in enumerate(starts):
        at = torch.tensor([p for p in places if p < V])
        x[2 * r, at] = torch.arange(2, 2 + len(at)).to(dtype)                # rising, and equal
        x[2 * r + 1, at] = torch.full((len(at),), 3.0, dtype=dtype)
    room = room.to(device)
    x = room[:, offset:offset + V]
    tokens = torch.zeros(len(x), dtype=torch.int64, device=device)
    for top in (1, 5, 20, 32):
        _check(x, tokens, top, 1.0, ops.token_logprobs(x, tokens, top=top))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V,top", [(1000, 4099, 0), (1000, 4099, 20), (700, 7, 0), (900, 1, 0), (460, 33000, 0)])
def test_more_rows_than_are_read_at_a_time(T, V, top, dtype):
    room = torch.randn(T, V + 5, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    x = room[:, 3:3 + V]
    tokens = torch.randint(0, V, (T,), generator=torch.Generator().manual_seed(4)).cuda()
    _check(x, tokens, top, 0.7, ops.token_logprobs(x, tokens, top=top, temperature=0.7))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_peaked_rows_keep_their_last_digits(dtype, device):
    """Nearly all of the probability in one token, far above what a thread has seen before it: log S is close to 0, so an absolute
    error of a few steps of 1 is what S itself has, and every other term keeps its own relative one."""
    V = 32003
    x, tokens = _logits(6, V, dtype, device, 12, std=1.0)
    for i, (at, height) in enumerate([(0, 12.0), (V - 1, 15.0), (20000, 18.0), (4097, 24.0), (31000, 30.0), (9, 60.0)]):
        x[i, at] = height
        tokens[i] = at
    for temperature in (0.7, 1.0):
        out = ops.token_logprobs(x, tokens, top=2, temperature=temperature)
        _logp, _p, H, _on, lp, _ids, _left = _definition(x, tokens, 2, temperature)
        depth = (V if device == "cpu" else V / 512 + 20) + 40
        for got, want in ((out.entropy, H), (out.logprob, lp)):
            err = (got.double().cpu() - want).abs()
            assert bool((err <= 2.0 ** -24 * (8 + depth * want.abs())).all()), (err, want)


@pytest.mark.parametrize("device", DEVICES)
def test_extreme_temperatures(device):
    x, tokens = _logits(5, 3000, torch.float32, device, 3)
    x[2, 100:] = -INF
    x.requires_grad_(True)
    for temperature in (1e-6, 1e-3, 1e3, 1e6):
        out = ops.token_logprobs(x, tokens, top=3, temperature=temperature)
        gradients = [torch.ones(5), torch.ones(5), torch.ones(5, 3)]
        (d,) = torch.autograd.grad([out.logprob, out.entropy, out.top_logprob], x, [g.to(device) for g in gradients])
        logp, _p, H, on, lp, ids, _left = _definition(x, tokens, 3, temperature)
        # the temperature's inverse and log2(e) are rounded: a log probability is off by so many steps of itself
        err = (out.logprob.double().cpu() - lp).abs()
        assert bool(((err <= 2.0 ** -24 * (3100 + 8 * lp.abs())) | (out.logprob.double().cpu() == lp)).all())
        assert torch.equal(out.top_id.cpu(), ids) and bool(torch.isfinite(d).all())


@pytest.mark.parametrize("device", DEVICES)
def test_strides_offsets_and_shapes(device):
    base = torch.randn(6, 1003, generator=torch.Generator().manual_seed(2)).to(device)
    for dtype in (torch.bfloat16, torch.float32):
        wide = base.to(dtype)
        tokens = torch.tensor([0, 5, 900, -100, 1, 2], device=device)
        for x in (wide[:, 1:], wide[:, 3:904], wide[:, :1000], wide.t().contiguous().t(), wide[:, 17:18].expand(6, 40)):
            leaf = x.detach().requires_grad_(True)
            out = ops.token_logprobs(leaf, tokens, top=4)
            _check(x, tokens, 4, 1.0, out)
            (d,) = torch.autograd.grad(out.logprob.sum(), leaf)
            want, size = _gradient(x, tokens, 0, 1.0, torch.ones(6), torch.zeros(6), torch.zeros(6, 0))
            assert bool(((d.double().cpu() - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + 2 ** -18 * size).all())
    x = base.view(2, 3, 1003)
    out = ops.token_logprobs(x, tokens.view(2, 3), top=2)
    assert out.logprob.shape == (2, 3) and out.top_id.shape == (2, 3, 2)
    one = ops.token_logprobs(base[0], tokens[0], top=2)
    assert one.logprob.shape == () and torch.equal(one.top_id, out.top_id[0, 0])
    assert torch.equal(one.logprob, out.logprob[0, 0])


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_that_do_not_arrive(device):
    x, tokens = _logits(4, 500, torch.float32, device, 9)
    x.requires_grad_(True)
    zero = [torch.zeros(4), torch.zeros(4), torch.zeros(4, 3)]
    for which in range(3):
        out = ops.token_logprobs(x, tokens, top=3)
        picked = [out.logprob, out.entropy, out.top_logprob][which]
        (d,) = torch.autograd.grad(picked.sum(), x)
        gradients = list(zero)
        gradients[which] = torch.ones_like(gradients[which])
        _check(x, tokens, 3, 1.0, out, d, gradients)
    with torch.no_grad():
        assert not ops.token_logprobs(x, tokens).logprob.requires_grad


def test_gradient_against_differences():
    x, tokens = _logits(3, 11, torch.float32, "cpu", 4, std=1.0)
    x = x.double().requires_grad_(True)
    weights = torch.linspace(0.5, 1.5, 3)

    def loss(v):
        out = ops.token_logprobs(v, tokens, top=2, temperature=0.8)
        return (weights * (out.logprob + 0.3 * out.entropy + out.top_logprob.sum(-1))).sum().double()

    (d,) = torch.autograd.grad(loss(x), x)
    h = 2.0 ** -9                                # error h^2 of the difference, 2^-22 / h of the loss in fp32
    for i in range(3):
        for j in range(11):
            e = torch.zeros_like(x)
            e[i, j] = h
            with torch.no_grad():
                slope = (loss(x + e) - loss(x - e)) / (2 * h)
            assert abs(float(slope) - float(d[i, j])) < 20 * (h * h + 2.0 ** -22 / h)


def test_agrees_with_cross_entropy():
    x, tokens = _logits(6, 300, torch.float32, "cpu", 8)
    tokens[2] = -100
    lp = ops.token_logprobs(x, tokens).logprob
    loss = ops.cross_entropy(x, tokens, reduction="none")
    assert bool(((lp + loss).abs() <= 2.0 ** -20 * (1 + loss.abs())).all())


def test_refusals():
    x, tokens = _logits(4, 50, torch.float32, "cpu", 1)
    for bad in (dict(top=-1), dict(top=33), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")),
                dict(temperature=INF), dict(temperature=1e-7), dict(temperature=1e7)):
        with pytest.raises(ValueError):
            ops.token_logprobs(x, tokens, **bad)
    with pytest.raises(ValueError):
        ops.token_logprobs(x[:, :5], tokens, top=6)
    with pytest.raises(ValueError):
        ops.token_logprobs(x, tokens[:3])
    with pytest.raises(ValueError):
        ops.token_logprobs(x, tokens.int())
    with pytest.raises(ValueError):
        ops.token_logprobs(x[:, :0], tokens)
    with pytest.raises(TypeError):
        ops.token_logprobs(x.long(), tokens)


def test_a_vocabulary_that_is_too_large_is_refused():
    x = torch.zeros(1, 1, dtype=torch.bfloat16).expand(2, (1 << 30) + 1)        # no memory behind it
    with pytest.raises(ValueError):
        ops.token_logprobs(x, torch.zeros(2, dtype=torch.int64))


@pytest.mark.gpu
def test_refusals_on_the_device():
    x, tokens = _logits(4, 50, torch.float32, "cuda", 1)
    with pytest.raises(TypeError):
        ops.token_logprobs(x.half(), tokens)
    with pytest.raises(TypeError):
        ops.token_logprobs(x.double(), tokens)
    with pytest.raises(ValueError):
        ops.token_logprobs(x, tokens.cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("lead", [(4,), (2, 2)])
def test_the_same_refusals_by_the_library(lead):
    x, tokens = _logits(4, 50, torch.float32, "cuda", 1)
    x, tokens = x.detach().view(*lead, 50), tokens.view(lead)
    for bad in (dict(top=-1), dict(top=33), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")),
                dict(temperature=INF), dict(temperature=1e-7), dict(temperature=1e7)):
        with pytest.raises(ValueError):
            ops.token_logprobs(x, tokens, **bad)
    for a, b, top in ((x[..., :5], tokens, 6), (x, tokens[:1], 0), (x, tokens.int(), 0), (x, tokens.unsqueeze(0), 0), (x[..., :0], tokens, 0),
                      (x, tokens.cpu(), 0), (x[:1, ..., :1].expand(*lead, (1 << 30) + 1), tokens, 0)):
        with pytest.raises(ValueError):
            ops.token_logprobs(a, b, top=top)
    for a in (x.long(), x.half(), x.double()):
        with pytest.raises(TypeError):
            ops.token_logprobs(a, tokens)
    assert ops.token_logprobs(x, tokens, temperature=1).logprob.shape == lead


@pytest.mark.gpu
def test_same_bits_on_streams_and_in_a_captured_graph():
    for T, V in ((1, 128256), (70, 32003)):
        x, tokens = _logits(T, V, torch.bfloat16, "cuda", 6)
        x.requires_grad_(True)

        def step():
            out = ops.token_logprobs(x, tokens, top=5)
            (d,) = torch.autograd.grad(out.logprob.sum() + out.entropy.sum(), x)
            return [t.detach() for t in out] + [d]

        want = step()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = []
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(step())
        torch.cuda.synchronize()
        for r in got:
            assert all(torch.equal(a, b) for a, b in zip(want, r))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = step()
        other, _ = _logits(T, V, torch.bfloat16, "cuda", 7)
        with torch.no_grad():
            x.copy_(other)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in kept]
        assert all(torch.equal(a, b) for a, b in zip(replayed, step()))


def test_traced_programs_record_one_op():
    x, tokens = _logits(4, 60, torch.float32, "cpu", 2)
    x.requires_grad_(True)

    def f(v):
        r = ops.token_logprobs(v, tokens, top=2)
        return (r.logprob + 0.1 * r.entropy).sum() + r.top_logprob.sum()

    (want,) = torch.autograd.grad(f(x), x)
    for backend in ("eager", "aot_eager"):
        compiled = torch.compile(f, backend=backend, fullgraph=True)
        (d,) = torch.autograd.grad(compiled(x), x)
        assert torch.allclose(d, want)
    torch.library.opcheck(torch.ops.piper.token_logprobs_fwd.default, (x, tokens, 2, 1.0, -100))


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_of_the_gradient(device):
    """On the CPU those of the plain formula; kernels' gradients have none, and say so in place of being left out."""
    x, tokens = _logits(5, 40, torch.float32, device, 9, std=1.0)
    x.requires_grad_(True)
    g = torch.Generator().manual_seed(2)
    up, v = torch.randn(5, generator=g).to(device), torch.randn(5, 40, generator=g).to(device)

    def first(create):
        out = ops.token_logprobs(x, tokens, top=3, temperature=0.7)
        loss = (out.logprob * up).sum() + out.entropy.square().sum() + 0.3 * out.top_logprob.sum()
        return torch.autograd.grad(loss, x, create_graph=create)[0]

    d = first(True)
    assert torch.equal(d.detach(), first(False)) and not first(False).requires_grad
    if device == "cuda":
        with pytest.raises(RuntimeError, match="no derivative"):
            torch.autograd.grad((d * v).sum() + x.sum(), x)
        return
    (got,) = torch.autograd.grad((d * v).sum(), x)
    y = x.detach().double().requires_grad_(True)
    logp = torch.log_softmax(y / 0.7, -1)
    entropy = -(logp.exp() * logp).sum(-1)
    ids = torch.sort(x.detach(), dim=-1, descending=True, stable=True).indices[:, :3]
    loss = (logp.gather(1, tokens.unsqueeze(1)).squeeze(1) * up).sum() + entropy.square().sum() + 0.3 * logp.gather(1, ids).sum()
    (d,) = torch.autograd.grad(loss, y, create_graph=True)
    (want,) = torch.autograd.grad((d * v.double()).sum(), y)
    # some 40 operations on numbers of at most 100 times the result's size
    assert float((got - want).abs().max()) <= 4000 * 2.0 ** -24 * float(want.abs().max())
