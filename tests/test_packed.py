"""Packed batches: their table, and attention within every sequence against its definition in 64 bits.

Tolerances.  Inputs are bf16, their products in fp32 exact, sums of them 2^-22 of the magnitudes.  A probability is off by that of
its exponent (z: the largest score) and rounded to bf16 (2^-8) as an operand, an output is rounded once more; on the CPU all but the last
is in fp32.  With D = dO . O, of the rounded output, a score gradient P (dP - D) has the errors of P, dP and D and is rounded to bf16.
Bounds are sums of magnitudes with these factors, element by element."""
import random

import pytest
import torch

from piper_b200 import ops
from piper_b200.ops import native, packed
from piper_b200.ops.packed import _table_ref

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
HALF = 2.0 ** -8


def _offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return torch.tensor(out)


def _definition(qkv, dout, lens, Hq, Hkv, hd, scale):
    """Output and gradient in fp64 and their bounds."""
    T = qkv.shape[0]
    x, d = qkv.detach().double().cpu().view(T, Hq + 2 * Hkv, hd), dout.detach().double().cpu().view(T, Hq, hd)
    out, dx = torch.zeros(T, Hq, hd, dtype=torch.float64), torch.zeros_like(x)
    eo, ex = torch.zeros_like(out), torch.zeros_like(x)
    a = 0
    for n in lens:
        r = slice(a, a + n)
        a += n
        if n == 0:
            continue
        for h in range(Hq):
            kv = Hq + h // (Hq // Hkv)
            q, k, v, g = x[r, h], x[r, kv], x[r, kv + Hkv], d[r, h]
            s = (q @ k.t()) * scale
            s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -float("inf"))
            p = torch.softmax(s, -1)
            o = p @ v
            z = 1 + s.abs().masked_fill(s.isinf(), 0).amax(1, keepdim=True) + (q.abs() @ k.abs().t()).amax(1, keepdim=True) * scale
            tiny = 2.0 ** -21 * z                                # of a probability, by its exponent
            so = (p * (HALF + tiny)) @ v.abs() + 2.0 ** -22 * (p @ v.abs())
            out[r, h], eo[r, h] = o, so + HALF * (o.abs() + so)
            dp, D = g @ v.t(), (g * o).sum(1, keepdim=True)
            eD = (g.abs() * eo[r, h]).sum(1, keepdim=True) + 2.0 ** -21 * (g * o).abs().sum(1, keepdim=True)
            ds = p * (dp - D)
            es = ds.abs() * (HALF + tiny) + p * (1 + HALF) * (eD + 2.0 ** -21 * (g.abs() @ v.abs().t()))
            dx[r, h] = ds @ k * scale
            ex[r, h] += (es + 2.0 ** -22 * ds.abs()) @ k.abs() * scale
            dx[r, kv] += ds.t() @ q * scale
            ex[r, kv] += (es + 2.0 ** -22 * ds.abs()).t() @ q.abs() * scale
            dx[r, kv + Hkv] += p.t() @ g
            ex[r, kv + Hkv] += (p * (HALF + tiny + 2.0 ** -22)).t() @ g.abs()
    ex = ex * (1 + HALF) + HALF * dx.abs()
    return out.view(T, -1), eo.view(T, -1), dx.view(T, -1), ex.view(T, -1)


def _inputs(T, Hq, Hkv, hd, device, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(T, (Hq + 2 * Hkv) * hd, generator=g) * std).to(torch.bfloat16)
    dout = torch.randn(T, Hq * hd, generator=g).to(torch.bfloat16)
    return qkv.to(device), dout.to(device)


def _pass(qkv, dout, seqs, Hq, Hkv, hd, scale=None):
    x = qkv.detach().requires_grad_(True)
    out = ops.packed_attention(x, seqs, Hq, Hkv, hd, hd ** -0.5 if scale is None else scale)
    (d,) = torch.autograd.grad(out, x, dout)
    if qkv.is_cuda:
        native.check_status()
    return out.detach(), d


def _close(got, want, bound):
    off = (got.double().cpu() - want).abs()
    bad = ~(off <= bound + 1e-30)
    assert not bool(bad.any()), (int(bad.sum()), off[bad][:4], bound[bad][:4], bad.nonzero()[:4])


# ------------------------------------------------------------------ table
TABLES = [[], [0], [1], [128], [129], [0, 0, 5, 0], [300, 1, 128, 129, 0, 300, 300, 257], [1] * 2100, [2000] + [3] * 40]


@pytest.mark.parametrize("lens", TABLES, ids=lambda v: f"{len(v)}-{sum(v)}")
@pytest.mark.parametrize("behind", [0, 130])
def test_table_on_the_cpu(lens, behind):
    T = sum(lens) + behind
    s = ops.pack_sequences(_offsets(lens), T)
    rows = s.table.tolist()
    assert rows[0] == [sum((n + 127) // 128 for n in lens), sum(lens), T, sum(n > 0 for n in lens)] and len(rows) == rows[0][0] + 1
    blocks, at = {}, 0
    for a, n in zip(_offsets(lens).tolist(), lens):
        for i in range((n + 127) // 128):
            blocks[(a, n, i, at * 128)] = i
        at += (n + 127) // 128
    assert {tuple(r) for r in rows[1:]} == set(blocks)
    assert [r[2] for r in rows[1:]] == sorted(blocks.values(), reverse=True)
    assert s.longest == max([(n + 127) // 128 for n in lens], default=0)
    want = [i for n in lens for i in range(n)] + [0] * behind
    assert s.positions().tolist() == want


@pytest.mark.gpu
@pytest.mark.parametrize("lens", TABLES + [[random.Random(i).randrange(0, 700) for i in range(1500)], [1 << 17, 5, 1 << 16]],
                         ids=lambda v: f"{len(v)}-{sum(v)}")
@pytest.mark.parametrize("behind", [0, 130])
def test_table_on_the_gpu(lens, behind):
    T = sum(lens) + behind
    want = ops.pack_sequences(_offsets(lens), T)
    here = ops.pack_sequences(_offsets(lens), T, device="cuda")                  # offsets from the host
    there = ops.pack_sequences(_offsets(lens).cuda(), T)                          # offsets that are on the GPU
    native.check_status()
    assert torch.equal(here.table.cpu(), want.table) and here[4:] == want[4:] and (here.own is None) == (want.own is None)
    used = want.table.shape[0]
    assert there.table.shape[0] >= used and torch.equal(there.table[:used].cpu(), want.table)
    if want.own is not None:                     # rows of blocks that are no groups are not written
        used = want.tiles.shape[0]
        for s in (here, there) if there.own is not None else (here,):
            assert s.own.shape[0] == 128 * (s.tiles.shape[0] - 1) and torch.equal(s.tiles[:used].cpu(), want.tiles)
            for _a, n, _i, at in want.tiles[1:].tolist():
                if at % 2:
                    assert torch.equal(s.own[at - 1:at - 1 + n].cpu(), want.own[at - 1:at - 1 + n])
    assert torch.equal(there.positions().cpu(), want.positions())


@pytest.mark.parametrize("lens", TABLES + [[40, 50, 1, 30, 100, 28, 0, 300, 10, 0, 20], [64] * 200, [1, 127, 128, 0, 2, 126, 1]],
                         ids=lambda v: f"{len(v)}-{sum(v)}")
def test_short_neighbours_share_blocks(lens):
    """Every row of a sequence is in one block, in one piece; a block has a sequence or a group of whole ones; no two neighbouring
    groups of one part of the sequences would fit one block."""
    at = _offsets(lens).tolist()
    from piper_b200.ops.packed import _groups, _groups_ref, _sequences
    tiles, own = _groups_ref(at, sum(lens), len(lens) + sum(lens) // 128)
    assert sorted((a, n) for a, n, _ in _sequences(tiles, own)) == [(a, n) for a, n in zip(at, lens) if n]
    places = sorted((p, p + n) for _a, n, p in _sequences(tiles, own))
    assert all(b <= c for (_, b), (c, _) in zip(places, places[1:]))
    groups = _groups(at)
    assert [i for g in groups for i in g] == [i for i, n in enumerate(lens) if n]
    s = ops.pack_sequences(_offsets(lens), sum(lens))                        # of these, none is near the border
    assert (s.own is not None) == (s.tiles is not None) == (len(groups) * 10 < 7 * sum(n > 0 for n in lens))
    chunk = max(64, -(-len(lens) // 32))
    for g, h in zip(groups, groups[1:]):
        assert len(g) == 1 or at[g[-1] + 1] - at[g[0]] <= 128
        assert g[0] // chunk != h[0] // chunk or at[h[0] + 1] - at[g[0]] > 128


@pytest.mark.parametrize("offsets,tokens", [([1, 2], 5), ([0, 3, 2], 5), ([0, 6], 5), ([0, -1], 5), ([-1, 3], 5)])
def test_offsets_that_do_not_rise_are_refused(offsets, tokens):
    with pytest.raises(ValueError):
        ops.pack_sequences(torch.tensor(offsets), tokens)


def test_what_is_no_batch_is_refused():
    for bad in (lambda: ops.pack_sequences(torch.tensor([0.0, 1.0]), 5), lambda: ops.pack_sequences(torch.zeros(2, 2).long(), 5),
                lambda: ops.pack_sequences(torch.zeros(0).long(), 5), lambda: ops.pack_sequences(torch.tensor([0]), -1),
                lambda: ops.pack_sequences(torch.tensor([0]), (1 << 21) + 1)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("device", DEVICES)
def test_attention_refuses_what_does_not_fit(device):
    s = ops.pack_sequences(_offsets([3, 4]), 7, device=device)
    x = torch.zeros(7, 256, dtype=torch.bfloat16, device=device)
    calls = [lambda: ops.packed_attention(x[:6], s, 2, 1, 64, 1.0), lambda: ops.packed_attention(x, s, 3, 2, 64, 1.0),
             lambda: ops.packed_attention(x, s, 2, 0, 64, 1.0), lambda: ops.packed_attention(x.view(7, 4, 64), s, 2, 1, 64, 1.0),
             lambda: ops.packed_attention(x, s, 2, 2, 64, 1.0), lambda: ops.packed_attention(x, s, 2, 1, 64, 0.0),
             lambda: ops.packed_attention(x, s, 2, 1, 64, -1.0), lambda: ops.packed_attention(x, s, 2, 1, 64, float("nan"))]
    if device == "cuda":
        calls += [lambda: ops.packed_attention(x, s, 14, 1, 16, 1.0), lambda: ops.packed_attention(x.float(), s, 2, 1, 64, 1.0),
                  lambda: ops.packed_attention(x, ops.pack_sequences(_offsets([3, 4]), 7), 2, 1, 64, 1.0)]
    for call in calls:
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("offsets", [[0, 300, 200], [5, 300], [0, 301], [0, -5, 3]])
def test_bad_offsets_on_the_gpu_give_an_empty_batch_and_an_error(offsets):
    s = ops.pack_sequences(torch.tensor(offsets, device="cuda"), 300)
    qkv, dout = _inputs(300, 4, 2, 64, "cuda", 0)
    x = qkv.requires_grad_(True)
    out = ops.packed_attention(x, s, 4, 2, 64, 0.125)
    (d,) = torch.autograd.grad(out, x, dout)
    assert not bool(out.any()) and not bool(d.any())
    with pytest.raises(native.PiperKernelError):
        native.check_status()
    native.check_status()


# ------------------------------------------------------------------ attention
CASES = [
    ([1], 4, 4, 64), ([1, 1, 1], 4, 2, 128), ([2, 0, 127, 1], 8, 1, 64), ([128], 4, 2, 128), ([129, 63, 64, 65], 4, 4, 64),
    ([0, 5, 0, 300, 1, 0], 6, 2, 128), ([200, 333, 17, 400], 4, 2, 64), ([16, 15, 17, 112, 113, 111], 2, 1, 128),
    ([512], 32, 4, 128), ([700, 3], 16, 1, 64), ([193, 257, 320], 3, 1, 128), ([1300, 40, 700], 8, 2, 128), ([1025, 900], 12, 4, 64), ([30, 31, 33, 34, 64, 64, 1, 127], 4, 2, 128), ([5] * 70 + [129], 8, 2, 64),
    ([40, 50, 1, 30, 100, 28, 0, 300, 10, 0, 20], 12, 2, 128), ([64, 65, 63, 1, 128, 3], 6, 2, 64), ([60] * 31, 32, 4, 128),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lens,Hq,Hkv,hd", CASES, ids=lambda v: str(v).replace(" ", ""))
def test_attention(lens, Hq, Hkv, hd, device, monkeypatch):
    if device == "cpu" and (sum(lens) * Hq > 2000 or len(lens) > 12):
        pytest.skip("long on the CPU")
    T = sum(lens) + 3
    qkv, dout = _inputs(T, Hq, Hkv, hd, device, len(lens) + hd)
    want = _definition(qkv, dout, lens, Hq, Hkv, hd, hd ** -0.5)
    out, d = _pass(qkv, dout, ops.pack_sequences(_offsets(lens), T, device=device), Hq, Hkv, hd)
    _close(out, *want[:2])
    _close(d, *want[2:])
    monkeypatch.setattr(packed, "GROUP_GAIN", 0.0)         # groups wherever there are any
    monkeypatch.setattr(packed, "GROUP_BLOCKS", 0)
    s = ops.pack_sequences(_offsets(lens), T, device=device)
    assert s.own is not None
    out, d = _pass(qkv, dout, s, Hq, Hkv, hd)
    _close(out, *want[:2])
    _close(d, *want[2:])
    if device == "cuda":                                   # launch shapes of a batch that the host does not know
        out, d = _pass(qkv, dout, ops.pack_sequences(_offsets(lens).cuda(), T), Hq, Hkv, hd)
        _close(out, *want[:2])
        _close(d, *want[2:])


@pytest.mark.gpu
@pytest.mark.parametrize("n,Hq,Hkv,hd", [(40, 32, 8, 128), (40, 32, 8, 64), (60, 24, 8, 128), (25, 16, 2, 64)])
def test_attention_over_many_sequences(n, Hq, Hkv, hd):
    """More tiles than SMs: two heads to a CTA, where groups are even."""
    rng = random.Random(n + hd)
    lens = [rng.choice([1, 30, 128, 129, 200, 384, 500]) for _ in range(n)]
    T = sum(lens) + 9
    qkv, dout = _inputs(T, Hq, Hkv, hd, "cuda", n)
    want = _definition(qkv, dout, lens, Hq, Hkv, hd, 0.07)
    out, d = _pass(qkv, dout, ops.pack_sequences(_offsets(lens), T, device="cuda"), Hq, Hkv, hd, 0.07)
    _close(out, *want[:2])
    _close(d, *want[2:])


@pytest.mark.gpu
def test_large_scores_and_launch_shapes_of_skewed_batches():
    lens = [900] + [7] * 60
    T = sum(lens)
    qkv, dout = _inputs(T, 8, 2, 128, "cuda", 3, std=3.0)
    want = _definition(qkv, dout, lens, 8, 2, 128, 128 ** -0.5)
    for s in (ops.pack_sequences(_offsets(lens), T, device="cuda"), ops.pack_sequences(_offsets(lens).int().cuda(), T)):
        out, d = _pass(qkv, dout, s, 8, 2, 128)
        _close(out, *want[:2])
        _close(d, *want[2:])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_nothing_of_a_sequence_reaches_another(device, hd, value):
    """Infinities and NaN in one sequence, behind the last one and in their gradients: the other sequences keep their bits."""
    if device == "cpu" and (hd != 64 or value == value):
        pytest.skip("one of them on the CPU")
    lens = [70, 130, 1, 129, 60]
    T, Hq, Hkv = sum(lens) + 40, 4, 2
    qkv, dout = _inputs(T, Hq, Hkv, hd, device, 5)
    s = ops.pack_sequences(_offsets(lens), T, device=device)
    want = _pass(qkv, dout, s, Hq, Hkv, hd)
    at = _offsets(lens).tolist()
    for bad in (1, 2, 4):
        q2, d2 = qkv.clone(), dout.clone()
        for x in (q2, d2):
            x[at[bad]:at[bad + 1]] = value
            x[at[-1]:] = value
        got = _pass(q2, d2, s, Hq, Hkv, hd)
        for g, w in zip(got, want):
            for i in range(len(lens)):
                if i != bad:
                    assert torch.equal(g[at[i]:at[i + 1]], w[at[i]:at[i + 1]]), (bad, i)
            assert not bool(g[at[-1]:].any())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_nothing_of_a_sequence_reaches_others_of_its_block(device, hd, value, monkeypatch):
    """Sequences that share a block: what is not finite in one of them, in all of its row or in queries, keys, values or output gradients
    alone, leaves the others as exact as they were, and does what it does to its own."""
    if device == "cpu" and (hd != 64 or value == value):
        pytest.skip("one of them on the CPU")
    lens = [40, 50, 1, 37, 100, 28, 130, 10, 20, 64]
    T, Hq, Hkv = sum(lens) + 2, 4, 2
    monkeypatch.setattr(packed, "GROUP_BLOCKS", 0)
    qkv, dout = _inputs(T, Hq, Hkv, hd, device, 6)
    s = ops.pack_sequences(_offsets(lens), T, device=device)
    assert s.own is not None
    want = _definition(qkv, dout, lens, Hq, Hkv, hd, hd ** -0.5)
    at = _offsets(lens).tolist()
    for bad in (1, 2, 4, 8):
        for part in ("all", "q", "k", "v", "dout"):
            q2, d2 = qkv.clone(), dout.clone()
            x = q2.view(T, Hq + 2 * Hkv, hd)
            row = at[bad] + lens[bad] // 2
            if part == "all":
                q2[at[bad]:at[bad + 1]], d2[at[bad]:at[bad + 1]] = value, value
            elif part == "dout":
                d2[row, 3] = value
            else:
                x[row, {"q": 1, "k": Hq, "v": Hq + Hkv}[part], 5] = value
            out, d = _pass(q2, d2, s, Hq, Hkv, hd)
            for i in range(len(lens)):
                r = slice(at[i], at[i + 1])
                if i != bad:
                    _close(out[r], want[0][r], want[1][r])
                    _close(d[r], want[2][r], want[3][r])
            own = slice(row, at[bad + 1])
            broken = {"all": out[own], "v": out[own], "q": out[row], "k": d[own], "dout": d[own]}[part]
            assert not bool(torch.isfinite(broken.float()).all()), (bad, part)
    assert bool(torch.isfinite(_pass(qkv, dout, s, Hq, Hkv, hd)[1].float()).all())


@pytest.mark.gpu
def test_attention_is_reproducible_and_takes_strided_and_unaligned_inputs():
    lens = [400, 129, 333]
    T, Hq, Hkv, hd = sum(lens), 8, 2, 64
    qkv, dout = _inputs(T, Hq, Hkv, hd, "cuda", 8)
    s = ops.pack_sequences(_offsets(lens), T, device="cuda")
    want = _pass(qkv, dout, s, Hq, Hkv, hd)
    wide = torch.zeros(T, qkv.shape[1] + 8, device="cuda", dtype=torch.bfloat16)
    wide[:, 3:3 + qkv.shape[1]] = qkv
    flat = torch.zeros(qkv.numel() + 1, device="cuda", dtype=torch.bfloat16)
    flat[1:] = qkv.reshape(-1)
    flat_d = torch.zeros(dout.numel() + 1, device="cuda", dtype=torch.bfloat16)
    flat_d[1:] = dout.reshape(-1)
    for x, d in ((qkv, dout), (wide[:, 3:3 + qkv.shape[1]], dout.t().contiguous().t()),
                 (flat[1:].view(qkv.shape), flat_d[1:].view(dout.shape))):
        got = _pass(x, d, s, Hq, Hkv, hd)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    none = torch.zeros(0, qkv.shape[1], device="cuda", dtype=torch.bfloat16)
    out, d = _pass(none, none[:, :Hq * hd], ops.pack_sequences(torch.tensor([0, 0]), 0, device="cuda"), Hq, Hkv, hd)
    assert out.shape == (0, Hq * hd) and d.shape == none.shape


@pytest.mark.gpu
def test_attention_on_other_streams_and_in_a_graph():
    """Two batches at once on two streams; one captured with its layout, whose offsets change between replays."""
    Hq, Hkv, hd, T = 8, 2, 128, 700
    batches = [[300, 400], [699, 1]]
    qkv, dout = _inputs(T, Hq, Hkv, hd, "cuda", 9)
    want = [_pass(qkv, dout, ops.pack_sequences(_offsets(b).cuda(), T), Hq, Hkv, hd) for b in batches]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in batches], []
    for _ in range(3):
        for stream, b in zip(streams, batches):
            with torch.cuda.stream(stream):
                x = qkv.detach().requires_grad_(True)
                out = ops.packed_attention(x, ops.pack_sequences(_offsets(b).cuda(), T), Hq, Hkv, hd, hd ** -0.5)
                got.append((out.detach(), torch.autograd.grad(out, x, dout)[0]))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))
    offsets = _offsets(batches[0]).int().cuda()
    x = qkv.detach().clone().requires_grad_(True)

    def step():
        out = ops.packed_attention(x, ops.pack_sequences(offsets, T), Hq, Hkv, hd, hd ** -0.5)
        return out.detach(), torch.autograd.grad(out, x, dout)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for b, w in list(zip(batches, want)) * 2:
        offsets.copy_(_offsets(b))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], w[0]) and torch.equal(out[1], w[1])
    native.check_status()


@pytest.mark.gpu
def test_groups_in_a_graph_whose_offsets_change():
    """Short sequences with offsets on the GPU, in groups: captured with their layout, replayed with other offsets, on two streams at once."""
    Hq, Hkv, hd, T, n = 32, 8, 64, 700, 40
    rng = random.Random(2)
    batches = []
    for _ in range(3):
        cuts = sorted(rng.randrange(0, T + 1) for _ in range(n - 1))
        batches.append([b - a for a, b in zip([0, *cuts], [*cuts, T])])
    qkv, dout = _inputs(T, Hq, Hkv, hd, "cuda", 9)
    assert ops.pack_sequences(_offsets(batches[0]).cuda(), T).own is not None
    want = [_definition(qkv, dout, b, Hq, Hkv, hd, hd ** -0.5) for b in batches]
    offsets = [_offsets(batches[0]).int().cuda() for _ in range(2)]
    x = qkv.detach().clone().requires_grad_(True)
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for o in offsets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.packed_attention(x, ops.pack_sequences(o, T), Hq, Hkv, hd, hd ** -0.5)
            outs.append((out, *torch.autograd.grad(out, x, dout)))
        graphs.append(graph)
    for i in range(3):
        for j in range(2):
            offsets[j].copy_(_offsets(batches[(i + j) % 3]))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for j in range(2):
            w = want[(i + j) % 3]
            _close(outs[j][0].detach(), *w[:2])
            _close(outs[j][1], *w[2:])
    native.check_status()


@pytest.mark.gpu
def test_batches_of_more_than_2_to_the_31_elements():
    """The last sequences of a batch whose rows lie beyond 2^31 elements, and the rows behind them."""
    Hq, Hkv, hd, tail = 64, 8, 128, [300, 40, 50, 513]
    lens = [777] * 360 + tail
    T = sum(lens) + 100
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * hd, generator=g, device="cuda", dtype=torch.bfloat16)
    dout = torch.randn(T, Hq * hd, generator=g, device="cuda", dtype=torch.bfloat16)
    first = sum(lens) - sum(tail)
    assert first * qkv.shape[1] > 2 ** 31
    out, d = _pass(qkv, dout, ops.pack_sequences(_offsets(lens), T, device="cuda"), Hq, Hkv, hd)
    want = _definition(qkv[first:first + sum(tail)], dout[first:first + sum(tail)], tail, Hq, Hkv, hd, hd ** -0.5)
    _close(out[first:first + sum(tail)], *want[:2])
    _close(d[first:first + sum(tail)], *want[2:])
    assert not bool(out[sum(lens):].any()) and not bool(d[sum(lens):].any())


@pytest.mark.gpu
def test_a_table_of_another_batch_gives_zeros_and_an_error():
    a, b = ops.pack_sequences(_offsets([100, 60]), 200, device="cuda"), ops.pack_sequences(_offsets([130, 5]), 190, device="cuda")
    qkv, dout = _inputs(200, 4, 2, 64, "cuda", 0)
    x = qkv.requires_grad_(True)
    out = ops.packed_attention(x, a._replace(table=b.table), 4, 2, 64, 0.125)
    (d,) = torch.autograd.grad(out, x, dout)
    assert not bool(out.any()) and not bool(d.any())
    with pytest.raises(native.PiperKernelError):
        native.check_status()


@pytest.mark.gpu
def test_native_formulas_do_what_the_python_ones_do():
    lens = [200, 77]
    T = sum(lens) + 5
    qkv, dout = _inputs(T, 4, 2, 64, "cuda", 4)
    s = ops.pack_sequences(_offsets(lens), T, device="cuda")
    want = _pass(qkv, dout, s, 4, 2, 64)
    lib = native.lib()
    lib.native_op_remove("packed_attention_fwd")
    try:
        got = _pass(qkv, dout, s, 4, 2, 64)
    finally:
        lib.native_op_install("packed_attention_fwd")
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("device", DEVICES)
def test_the_gradient_has_no_derivative(device):
    qkv, dout = _inputs(9, 2, 1, 64, device, 2)
    x = qkv.requires_grad_(True)
    out = ops.packed_attention(x, ops.pack_sequences(_offsets([4, 5]), 9, device=device), 2, 1, 64, 0.1)
    (d,) = torch.autograd.grad(out, x, dout, create_graph=True)
    with pytest.raises(RuntimeError):
        d.float().square().sum().backward()


def test_attention_gradient_against_differences():
    """On the CPU, fp32 throughout: central differences along random directions."""
    lens, Hq, Hkv, hd = [5, 1, 7], 2, 1, 8
    T = sum(lens)
    g = torch.Generator().manual_seed(1)
    x, dout = torch.randn(T, 4 * hd, generator=g), torch.randn(T, Hq * hd, generator=g)
    s = ops.pack_sequences(_offsets(lens), T)
    leaf = x.clone().requires_grad_(True)
    (d,) = torch.autograd.grad(ops.packed_attention(leaf, s, Hq, Hkv, hd, 0.4), leaf, dout)
    for i in range(4):
        v = torch.randn(x.shape, generator=g)
        h = 2.0 ** -6
        up, down = (ops.packed_attention(x + sign * h * v, s, Hq, Hkv, hd, 0.4) for sign in (1, -1))
        change = float(((up - down).double() * dout).sum()) / (2 * h)
        # fp32 rounding of some 100 terms of size 1 over 2h, and h^2 / 6 of a third derivative below 64 x 100
        assert abs(change - float((d * v).sum())) < 100 * 2.0 ** -22 / (2 * h) * 8 + h * h / 6 * 6400


def test_reference_table_is_the_ops():
    assert torch.equal(_table_ref([0, 130, 135], 140, 4)[:4], ops.pack_sequences(torch.tensor([0, 130, 135]), 140).table)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_a_layout_keeps_the_offsets_that_it_was_made_of(dtype, device):
    """A program that fills the same buffer for its next batch changes nothing of this one."""
    offsets = torch.tensor([0, 3, 10], dtype=dtype, device=device)
    s = ops.pack_sequences(offsets, 12)
    positions, inside = s.positions(), s.inside()
    offsets.copy_(torch.tensor([0, 7, 12]))
    assert torch.equal(s.positions(), positions) and torch.equal(s.inside(), inside)
    assert s.positions().tolist() == [0, 1, 2, 0, 1, 2, 3, 4, 5, 6, 0, 0]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("lens", [[64], [70], [128, 3], [333, 20, 30], [1, 200, 5]], ids=str)
def test_keys_that_no_query_sees_by_their_scores(lens, grouped, hd, device, monkeypatch):
    """A key of -inf where all queries are positive has probabilities of 0: outputs and the gradients of keys and values are those
    beside a key whose scores are so far down that its probabilities are 0 too, whatever the sequence's length."""
    if device == "cpu" and hd != 64:
        pytest.skip("one of them on the CPU")
    Hq, Hkv, T = 4, 2, sum(lens)
    if grouped:
        monkeypatch.setattr(packed, "GROUP_GAIN", 0.0)
        monkeypatch.setattr(packed, "GROUP_BLOCKS", 0)
    s = ops.pack_sequences(_offsets(lens), T, device=device)
    qkv, dout = _inputs(T, Hq, Hkv, hd, device, 11)
    x = qkv.view(T, Hq + 2 * Hkv, hd)
    x[:, :Hq, 0] = x[:, :Hq, 0].abs() + 1
    at = _offsets(lens).tolist()
    results = []
    for value in (-float("inf"), -2.0 ** 16):                # at most -2^16 / 2^4 beside scores below 2^7
        for a, b in zip(at, at[1:]):
            if b - a > 5:                                    # not the first key, which is all that the first query has
                x[a + 5, Hq:Hq + Hkv, 0] = value
        out, d = _pass(qkv, dout, s, Hq, Hkv, hd)
        results.append((out, d.view(T, Hq + 2 * Hkv, hd)[:, Hq:]))
    (out, d), (want, dwant) = results
    assert bool(torch.isfinite(out.float()).all()) and bool(torch.isfinite(d.float()).all())
    assert torch.equal(out, want) and torch.equal(d, dwant)
