"""Products in e4m3 with power-of-two scales against their definition in 64 bits.

Codes are exact: scaling by a power of two is, and an element is then rounded once, ties to even.  A product's sum is kept in
fp32: the tensor core adds 32 products at a time, and each of the K / 32 additions (and the alignment of the products within one)
is off by at most 2^-22 of the sum of the products' magnitudes; the result is rounded to bf16 once, 2^-8 of itself (the CPU's
plain form stays in fp32, and is cast to the type of x)."""
import pytest
import torch

from piper_b200 import ops
from piper_b200.ops import fp8 as fp8_ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _pow2(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _rounded(x, square=False):
    """x on its e4m3 grid, in 64 bits: four significant bits, none below 2^-9 of the scale, ties to even."""
    x = x.detach().double().cpu()
    rows, cols = x.shape
    h = 128 if square else 1
    out = torch.empty_like(x)
    for i in range(0, rows, h):
        for j in range(0, cols, 128):
            part = x[i:i + h, j:j + 128]
            m, e = torch.frexp(part.abs().max() / 448)
            e = max(int(e) - (float(m) == 0.5), -127)
            y = part / _pow2(torch.tensor(e))
            ulp = _pow2((torch.frexp(y).exponent - 1).clamp(min=-6) - 3)
            out[i:i + h, j:j + 128] = torch.round(y / ulp) * ulp * _pow2(torch.tensor(e))
    return out


def _matrix(rows, cols, device, seed, std=1.0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * std
    x *= 2.0 ** torch.randint(-6, 7, (rows, 1), generator=g)
    return x.to(dtype).to(device)


def _close(got, a, b, dtype=torch.bfloat16, scale=1.0):
    """got against a [M, K] b [N, K]^T of rounded operands in 64 bits."""
    want, size = scale * (a @ b.t()), a.abs() @ b.abs().t()
    K = a.shape[1]
    tol = torch.finfo(dtype).eps / 2 * want.abs() + scale * (K / 32 + 4) * 2.0 ** -22 * size
    got = got.detach().double().cpu()
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol.clamp(min=1e-300)).max())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,cols", [(1, 16), (3, 128), (128, 128), (129, 144), (200, 640), (16, 2064), (300, 48)])
def test_codes(rows, cols, device):
    x = _matrix(rows, cols, device, rows + cols)
    x[0, 0] = 3e38                                # the largest magnitudes, and the smallest
    if rows > 2:
        x[1] = x[1] * 1e-38
        x[2] = 0
    for square in (False, True):
        q = ops.fp8_quantize(x, square=square)
        assert q.shape == (rows, cols) and torch.equal(q.dequantize().double().cpu(), _rounded(x, square))
        t = ops.fp8_quantize(x, square=square, transpose=True)
        assert t.shape == (cols, rows) and torch.equal(t.dequantize().double().cpu(), _rounded(x.t(), square))
        if square:
            assert torch.equal(t.dequantize().t(), q.dequantize())
    if device == "cuda":                          # words of scales and unused bytes too
        for square in (False, True):
            for transpose in (False, True):
                a, b = (ops.fp8_quantize(y, square=square, transpose=transpose) for y in (x, x.cpu()))
                assert torch.equal(a.codes.cpu(), b.codes) and torch.equal(a.scales.cpu(), b.scales)


@pytest.mark.parametrize("device", DEVICES)
def test_largest_magnitudes_at_the_borders(device):
    """448 times a power of two is the last number of its scale; every bf16 number of two binades as the largest one."""
    bits = torch.arange(0x4380, 0x4480, dtype=torch.int32).to(torch.int16)       # 256.0 to 1016
    x = torch.zeros(256, 128)
    x[:, 5] = bits.view(torch.bfloat16).float()
    x[:, 6] = x[:, 5] / 3
    x = x.to(torch.bfloat16).to(device)
    q = ops.fp8_quantize(x)
    assert torch.equal(q.dequantize().double().cpu(), _rounded(x))
    biased = q.scales[0, :256].cpu() & 255
    largest = x[:, 5].float().cpu()
    assert torch.equal(biased, 127 + (largest > 448).int() + (largest > 896).int())


@pytest.mark.parametrize("device", DEVICES)
def test_groups_without_numbers(device):
    x = _matrix(4, 256, device, 3)
    x[1, 7], x[2, 200] = float("nan"), float("-inf")
    v = ops.fp8_quantize(x).dequantize().cpu()
    bad = torch.zeros(4, 256, dtype=torch.bool)
    bad[1, :128] = bad[2, 128:] = True
    assert torch.equal(torch.isnan(v), bad)
    w = _matrix(32, 256, device, 4)
    y = ops.fp8_linear(x, w)
    assert bool(torch.isnan(y[1:3]).all()) and bool(torch.isfinite(y[[0, 3]]).all())


PRODUCTS = [(1, 16, 16), (5, 48, 32), (128, 32, 128), (24, 512, 512), (130, 80, 528), (257, 224, 1040), (256, 448, 384),
            (1000, 336, 272), (64, 2064, 640), (700, 3008, 144), (2048, 2048, 256)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_products(M, N, K, device):
    if device == "cpu" and M * N * K > 1 << 27:
        pytest.skip("the plain form at sizes of the kernel's tiles")
    a, b = _matrix(M, K, device, M + N), _matrix(N, K, device, K, std=0.1)
    dtype = torch.bfloat16 if device == "cuda" else torch.float32
    for square in (False, True):
        y = ops.fp8_matmul(ops.fp8_quantize(a), ops.fp8_quantize(b, square=square))
        assert y.dtype == dtype and y.shape == (M, N)
        _close(y, _rounded(a), _rounded(b, square), dtype)


@pytest.mark.gpu
def test_scales_reach_every_row_and_block():
    """Operands of ones, a scale of its own for every row and block: a sum over blocks of powers of two is exact."""
    M, N, K = 300, 272, 1536
    a, b = torch.ones(M, K), torch.ones(N, K)
    ea = (torch.arange(M)[:, None] * 7 + torch.arange(12)[None, :] * 3) % 9 - 4
    eb = (torch.arange(N)[:, None] * 5 + torch.arange(12)[None, :] * 2) % 7 - 3
    a, b = (t * (2.0 ** e).repeat_interleave(128, 1) for t, e in ((a, ea), (b, eb)))
    a, b = a.bfloat16().cuda(), b.bfloat16().cuda()
    y = ops.fp8_matmul(ops.fp8_quantize(a), ops.fp8_quantize(b))
    want = (a.double() @ b.double().t()).to(torch.bfloat16)
    assert torch.equal(y, want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T,K,N", [(1, 16, 16), (7, 256, 96), (129, 144, 272), (300, 688, 256), (0, 64, 32), (513, 64, 1376)])
def test_linear_and_its_gradients(T, K, N, device):
    x = _matrix(T, K, device, 1).requires_grad_(True)
    w = _matrix(N, K, device, 2, std=K ** -0.5).requires_grad_(True)
    dy = _matrix(T, N, device, 3, std=1e-4)
    y = ops.fp8_linear(x, w)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    assert y.dtype == x.dtype and dx.shape == x.shape and dw.shape == w.shape
    if T == 0:
        assert not dw.any()
        return
    _close(y, _rounded(x), _rounded(w, True))
    _close(dx, _rounded(dy), _rounded(w, True).t())
    _close(dw, _rounded(dy.t()), _rounded(x.t()))
    with torch.no_grad():
        kept = ops.fp8_quantize(w, square=True)
        assert torch.equal(ops.fp8_linear(x, kept), y)
        assert torch.equal(ops.fp8_linear(x, w), y)
    only_x = torch.autograd.grad(ops.fp8_linear(x, w.detach()), x, dy)[0]
    only_w = torch.autograd.grad(ops.fp8_linear(x.detach(), w), w, dy)[0]
    assert torch.equal(only_x, dx) and torch.equal(only_w, dw)


def test_gradient_is_that_of_the_rounded_product():
    """In fp32 on the CPU, where operands that are on their grids already make the layer exactly linear: differences of the
    output along a direction are the gradient's product with it."""
    g = torch.Generator().manual_seed(0)
    x = torch.randint(-8, 9, (6, 32), generator=g).float().requires_grad_(True)
    w = torch.randint(-4, 5, (16, 32), generator=g).float().requires_grad_(True)
    dy = torch.randint(-3, 4, (6, 16), generator=g).float()
    dx, dw = torch.autograd.grad(ops.fp8_linear(x, w), [x, w], dy)
    for leaf, grad in ((x, dx), (w, dw)):
        for i, j in ((0, 0), (3, 17), (5, 31)):
            e = torch.zeros_like(leaf)
            e[i, j] = 1.0
            with torch.no_grad():
                plus, minus = (ops.fp8_linear(*((x + s * e, w) if leaf is x else (x, w + s * e))) for s in (1, -1))
                assert float((dy * (plus - minus)).sum() / 2) == float(grad[i, j])


@pytest.mark.parametrize("device", DEVICES)
def test_strides_offsets_and_shapes(device):
    base = _matrix(40, 1056, device, 5)
    w = _matrix(64, 256, device, 6, std=0.1)
    for x in (base[:, :256], base[:, 16:272], base[:, 3:259], base[::2, :256], base[:32, :256].reshape(2, 16, 256),
              base[:256 // 8, :40].t().contiguous().t()[:, :32]):
        weight = w if x.shape[-1] == 256 else w[:, :32].contiguous()
        want = ops.fp8_linear(x.reshape(-1, x.shape[-1]).contiguous(), weight)
        got = ops.fp8_linear(x, weight)
        assert got.shape == (*x.shape[:-1], 64) and torch.equal(got.reshape(-1, 64), want)
    leaf = base[0, :256].clone().requires_grad_(True)
    y = ops.fp8_linear(leaf, w)
    assert y.shape == (64,)
    (d,) = torch.autograd.grad(y, leaf, torch.ones(64, dtype=y.dtype, device=device).expand(64))
    assert d.shape == (256,)
    (d2,) = torch.autograd.grad(ops.fp8_linear(leaf.view(1, 256), w), leaf, torch.ones(1, 1, dtype=y.dtype, device=device).expand(1, 64))
    assert torch.equal(d, d2)


@pytest.mark.parametrize("device", DEVICES)
def test_weight_gradients_go_into_buckets(device):
    x, w = _matrix(200, 256, device, 1), _matrix(96, 256, device, 2, std=0.1).requires_grad_(True)
    dy = _matrix(200, 96, device, 3)
    (plain,) = torch.autograd.grad(ops.fp8_linear(x, w), w, dy)
    sink = torch.full((96, 256), 3.0, device=device)
    ops.grad_sinks.register(w, sink)
    try:
        assert torch.autograd.grad(ops.fp8_linear(x, w), w, dy, allow_unused=True)[0] is None
        once = sink - 3.0
        queue = ops.wgrad_store.begin()
        try:
            torch.autograd.grad(ops.fp8_linear(x, w), w, dy, allow_unused=True)
            assert torch.equal(sink - 3.0, once) and len(queue) == 1
        finally:
            ops.wgrad_store.end()
        assert ops.wgrad_store.drain(queue) == []
    finally:
        ops.grad_sinks.unregister(w)
    _close(once, _rounded(dy.t()), _rounded(x.t()), torch.bfloat16)
    assert bool(((sink - 3.0 - 2 * once).abs() <= 2.0 ** -21 * (sink.abs() + 3)).all())
    assert bool(((once - plain.float()).abs() <= 2.0 ** -8 * once.abs() + 2.0 ** -20 * 3).all())


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x, w = _matrix(4, 64, device, 1), _matrix(32, 64, device, 2)
    for a, b in ((x[:, :32], w), (x[:, :24], w[:, :24]), (x, w[:24]), (x, w[:0]), (x[:, :0], w[:, :0])):
        with pytest.raises(ValueError):
            ops.fp8_linear(a, b)
    with pytest.raises(TypeError):
        ops.fp8_linear(x, w.float())
    with pytest.raises(TypeError):
        ops.fp8_linear(x.half(), w.half())
    for bad in (x[0], x[:, :24], x[:0]):
        with pytest.raises(ValueError):
            ops.fp8_quantize(bad)
    qx, qw = ops.fp8_quantize(x), ops.fp8_quantize(w, square=True)
    with pytest.raises(ValueError):
        ops.fp8_matmul(qx, ops.fp8_quantize(w[:, :32].contiguous()))
    with pytest.raises(ValueError):
        ops.fp8_matmul(qx, ops.fp8_quantize(w[:3]))
    with pytest.raises(ValueError):
        ops.fp8_linear(x.clone().requires_grad_(True), qw)
    if device == "cuda":
        with pytest.raises(ValueError):
            ops.fp8_linear(x.cpu(), w)
        with pytest.raises(TypeError):
            ops.fp8_linear(x.float(), w.float())


@pytest.mark.gpu
@pytest.mark.parametrize("N,K", [(1376, 256), (4096, 1024), (6144, 4096)])
def test_a_row_has_the_same_bits_in_a_batch_of_any_size(N, K):
    """Tiles of every width and height add along the contraction in one order."""
    x, w = _matrix(4096, K, "cuda", 1), _matrix(N, K, "cuda", 2, std=0.05)
    kept = ops.fp8_quantize(w, square=True)
    whole = ops.fp8_linear(x, w)
    for T in (1, 3, 24, 64, 100, 129, 300, 700, 1000, 2048):
        assert torch.equal(ops.fp8_linear(x[:T], w), whole[:T]), T
        assert torch.equal(ops.fp8_linear(x[4096 - T:], kept), whole[4096 - T:]), T


@pytest.mark.gpu
@pytest.mark.parametrize("lead", [(6,), (2, 3)])
def test_the_same_refusals_by_the_library(lead):
    x, w = (torch.ones(*n, dtype=torch.bfloat16, device="cuda") for n in ((*lead, 64), (32, 64)))
    for a, b in ((x[..., :48], w), (x[..., :40], w[:, :40]), (x, w[:24]), (x, w[:0]), (x[..., :0], w[:, :0]), (x, w.cpu()), (x.cpu(), w)):
        with pytest.raises(ValueError):
            ops.fp8_linear(a, b)
        with pytest.raises(ValueError):
            ops.fp8_linear(a, b.clone().requires_grad_(True))
    for a, b in ((x.float(), w), (x, w.float()), (x.half(), w.half()), (x, w.half())):
        with pytest.raises(TypeError):
            ops.fp8_linear(a, b)
    kept = ops.fp8_quantize(w, square=True)
    for a in (x[..., :48], x.cpu(), x.clone().requires_grad_(True)):
        with pytest.raises(ValueError):
            ops.fp8_linear(a, kept)
    assert ops.fp8_linear(x, kept).shape == (*lead, 32) and ops.fp8_linear(x[:0], w).shape == (0, *lead[1:], 32)


@pytest.mark.gpu
def test_captured_products_share_no_counters():
    """Graphs captured 4,096 launches apart, the number of places in which launches count their tiles, and an eager launch on a third
    stream, all in flight at once: several rounds of tiles each, every one of them written."""
    g = torch.Generator().manual_seed(7)
    a, b = (ops.fp8_quantize(torch.randn(n, 128, generator=g).bfloat16().cuda()) for n in (4096, 4096))
    want = ops.fp8_matmul(a, b)
    lib, status = ops.native.lib(), ops.native.status_tensor(want.device)
    streams = [torch.cuda.Stream() for _ in range(3)]
    graphs, outs = [], [torch.empty_like(want) for _ in range(3)]
    small = ops.fp8_quantize(torch.ones(16, 16, dtype=torch.bfloat16, device="cuda"))
    few = torch.empty(16, 16, dtype=torch.bfloat16, device="cuda")
    for out in outs[:2]:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            for _ in range(3):
                lib.fp8_gemm(a.data, b.data, out, 128, status)
        graphs.append(graph)
        for _ in range(4093):
            lib.fp8_gemm(small.data, small.data, few, 16, status)
    torch.cuda.synchronize()
    for _ in range(20):
        for out in outs:
            out.fill_(float("nan"))
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            for _ in range(3):
                lib.fp8_gemm(a.data, b.data, outs[2], 128, status)
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for out in outs)
    ops.native.check_status()


@pytest.mark.gpu
def test_a_product_that_waited_while_thousands_ran_on_another_stream():
    """Streams count their tiles by themselves: a product that was launched long before the others and runs beside them has all its tiles,
    and so have those on the default stream and on more streams than one."""
    a, b = (ops.fp8_quantize(_matrix(r, 128, "cuda", r)) for r in (4096, 2048))
    want = ops.fp8_matmul(a, b)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    held = torch.cuda.Event()
    with torch.cuda.stream(streams[0]):
        torch.cuda._sleep(100_000_000)                     # some 50 ms
        held.record()
    waiting = []
    for s in streams[:2]:
        with torch.cuda.stream(s):
            s.wait_event(held)
            waiting.append(ops.fp8_matmul(a, b))
    with torch.cuda.stream(streams[2]):
        last = [ops.fp8_matmul(a, b) for _ in range(4200)][-50:]
    last += [ops.fp8_matmul(a, b) for _ in range(10)]
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in waiting + last)
    ops.native.check_status()


@pytest.mark.gpu
def test_same_bits_on_streams_and_in_a_captured_graph():
    x = _matrix(700, 1024, "cuda", 1).requires_grad_(True)
    w = _matrix(1376, 1024, "cuda", 2, std=0.03).requires_grad_(True)
    dy = _matrix(700, 1376, "cuda", 3)

    def step():
        y = ops.fp8_linear(x, w)
        return [y.detach(), *torch.autograd.grad(y, [x, w], dy)]

    want = step()
    torch.cuda.synchronize()
    results = []
    for s in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(s):
            results.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in results for a, b in zip(want, r))
    graphs, kept = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept.append(step())
        graphs.append(graph)
    with torch.no_grad():
        x.copy_(_matrix(700, 1024, "cuda", 8))
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    after = step()
    assert all(torch.equal(a, b) for r in kept for a, b in zip(after, r))
    ops.native.check_status()


def test_traced_programs_record_one_op():
    x, w = _matrix(6, 64, "cpu", 1, dtype=torch.float32).requires_grad_(True), _matrix(32, 64, "cpu", 2, dtype=torch.float32)
    (want,) = torch.autograd.grad(ops.fp8_linear(x, w).sum(), x)
    for backend in ("eager", "aot_eager"):
        f = torch.compile(lambda a: ops.fp8_linear(a, w).sum(), backend=backend, fullgraph=True)
        assert torch.allclose(torch.autograd.grad(f(x), x)[0], want)
    torch.library.opcheck(torch.ops.piper.fp8_linear.default, (x, w))
    with torch.no_grad():
        kept = ops.fp8_quantize(w, square=True)
        torch.library.opcheck(torch.ops.piper.fp8_linear_kept.default, (x.detach(), kept.data, 32))


@pytest.mark.parametrize("device", DEVICES)
def test_checkpointed_layers_recompute_what_they_keep(device):
    from torch.utils.checkpoint import checkpoint
    x, w = _matrix(40, 64, device, 1).requires_grad_(True), _matrix(32, 64, device, 2, std=0.1).requires_grad_(True)
    dy = _matrix(40, 32, device, 3)
    want = torch.autograd.grad(ops.fp8_linear(x, w), [x, w], dy)
    for reentrant in (False, True):
        y = checkpoint(lambda a, b: ops.fp8_linear(a, b), x, w, use_reentrant=reentrant)
        if reentrant:                     # this form wants backward()
            x.grad = w.grad = None
            y.backward(dy)
            got = (x.grad, w.grad)
        else:
            got = torch.autograd.grad(y, [x, w], dy)
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.gpu
def test_one_weight_in_two_calls_of_a_pass_and_two_buckets():
    """The same weight twice: both gradients in its bucket; and calls on two streams at once with buckets of their own."""
    w = _matrix(96, 256, "cuda", 2, std=0.1).requires_grad_(True)
    a, b = (_matrix(n, 256, "cuda", n).requires_grad_(True) for n in (130, 70))
    da, db = _matrix(130, 96, "cuda", 5), _matrix(70, 96, "cuda", 6)
    sink = torch.zeros(96, 256, device="cuda")
    ops.grad_sinks.register(w, sink)
    try:
        torch.autograd.grad([ops.fp8_linear(a, w), ops.fp8_linear(b, w)], [a, b, w], [da, db], allow_unused=True)
    finally:
        ops.grad_sinks.unregister(w)
    parts = [_rounded(d.t()) @ _rounded(x.t()).t() for d, x in ((da, a), (db, b))]
    size = sum(_rounded(d.t()).abs() @ _rounded(x.t()).t().abs() for d, x in ((da, a), (db, b)))
    assert bool(((sink.double().cpu() - sum(parts)).abs() <= 10 * 2.0 ** -22 * size).all())


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_of_the_gradients_raise(device):
    """Rounded operands have none; left out silently, a penalty on gradients would train nothing."""
    x, w = _matrix(40, 64, device, 1).requires_grad_(True), _matrix(32, 64, device, 2, std=0.1).requires_grad_(True)
    dy = _matrix(40, 32, device, 3)
    want = torch.autograd.grad(ops.fp8_linear(x, w), [x, w], dy)
    got = torch.autograd.grad(ops.fp8_linear(x, w), [x, w], dy, create_graph=True)
    assert all(torch.equal(a.detach(), b) and a.requires_grad and not b.requires_grad for a, b in zip(got, want))
    for g in got:
        with pytest.raises(RuntimeError, match="no derivative"):
            torch.autograd.grad(g.float().square().sum() + x.float().sum() + w.float().sum(), [x, w])
    only = torch.autograd.grad(ops.fp8_linear(x.detach(), w), w, dy, create_graph=True)[0]
    assert torch.equal(only.detach(), want[1])


@pytest.mark.parametrize("device", DEVICES)
def test_an_input_that_is_written_over_after_the_layer(device):
    """The backward pass has its own copy of it, in 8 bits."""
    x, w = _matrix(40, 64, device, 1), _matrix(32, 64, device, 2, std=0.1).requires_grad_(True)
    dy = _matrix(40, 32, device, 3)
    a = x.clone().requires_grad_(True)
    want = torch.autograd.grad(ops.fp8_linear(a * 1, w), [a, w], dy)
    h = a * 1
    y = ops.fp8_linear(h, w)
    h.add_(1)
    got = torch.autograd.grad([y, h], [a, w], [dy, torch.zeros_like(h)])
    assert all(torch.equal(p, q) for p, q in zip(want, got))
