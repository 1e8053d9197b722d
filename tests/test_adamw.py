"""AdamW over many tensors with moments in 32 and in 8 bits, against the formulas in 64 bits.

Tolerances.  A moment is two products and a sum with rounded constants, each within half a step (2^-24): 4 of those relative to
the sum of the addends' sizes (v has one product more).  A weight is its own product with a rounded constant and the update,
whose relative error is that of m, half that of v, and six more roundings (root, product, sum, quotient, rate, product).
An 8-bit moment is one of the two neighbours of the 32-bit one on its grid."""
import math

import pytest
import torch

from piper_b200 import ops
from piper_b200.ops.optim import BLOCK

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
EPS = 2.0 ** -24
SHAPES = [(1,), (255,), (256,), (257,), (3, 100), (64, 64), (5000,), (7, 11, 13), (0,), (2, 2048)]


def _tensors(dtype, grad_dtype, device, seed=0, shapes=SHAPES):
    g = torch.Generator().manual_seed(seed)
    params = [(torch.randn(s, generator=g) * 0.1).to(dtype).to(device) for s in shapes]
    grads = [(torch.randn(s, generator=g) * 10.0 ** -(i % 5)).to(grad_dtype).to(device) for i, s in enumerate(shapes)]
    return params, grads


HYPER = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


def _formula(w, m, v, g, step, lr, betas, eps, weight_decay, grad_scale=1.0):
    """(w, m, v) after a step and the sizes of what m and v are sums of, all in 64 bits."""
    b1, b2 = betas
    g = g.double().cpu() * grad_scale
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    upd = (m1 / (1 - b1 ** step)) / (torch.sqrt(v1 / (1 - b2 ** step)) + eps)
    return w * (1 - lr * weight_decay) - lr * upd, m1, v1, (b1 * m).abs() + ((1 - b1) * g).abs(), upd


def _parts(state, flat):
    return [flat[o:o + math.prod(s)].double().cpu().view(s) for o, s in zip(state.offsets, state.shapes)]


def _weights(params, state):
    return [w if p.dtype == torch.bfloat16 else p.double().cpu()
            for p, w in zip(params, _parts(state, state.master) if state.master is not None else params)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype,grad_dtype", [(torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                              (torch.float32, torch.float32), (torch.float32, torch.bfloat16)])
def test_steps_follow_the_formulas(dtype, grad_dtype, bits, device):
    params, _ = _tensors(dtype, grad_dtype, device)
    state = ops.AdamWState(params, bits=bits)
    for step in range(1, 5):
        _, grads = _tensors(dtype, grad_dtype, device, seed=step)
        m0, v0 = (_parts(state, t) for t in state.moments())
        w0 = _weights(params, state)
        ops.adamw_step(params, grads, state, grad_scale=0.5, **HYPER)
        m1, v1 = (_parts(state, t) for t in state.moments())
        w1 = _weights(params, state)
        assert state.steps == [step] * len(params)
        for i, g in enumerate(grads):
            w, m, v, m_size, upd = _formula(w0[i], m0[i], v0[i], g, step, grad_scale=0.5, **HYPER)
            m_tol, v_tol = 5 * EPS * m_size + 1e-44, 6 * EPS * v + 1e-44
            if bits == 32:
                assert bool(((m1[i] - m).abs() <= m_tol).all()) and bool(((v1[i] - v).abs() <= v_tol).all())
            else:
                for got, want, tol, least in ((m1[i], m, m_tol, 1.25 * 2.0 ** -16), (v1[i], v, v_tol, 1.25 * 2.0 ** -32)):
                    if got.numel():
                        pad = torch.zeros((got.numel() + BLOCK - 1) // BLOCK * BLOCK, dtype=torch.float64)
                        pad[:got.numel()] = want.reshape(-1).abs()
                        scale = pad.view(-1, BLOCK).amax(1).repeat_interleave(BLOCK)[:got.numel()].view(got.shape)
                        apart = torch.maximum(want.abs() / 8, scale * least) * (1 + 8 * EPS) + 2 * tol
                        assert bool(((got - want).abs() <= apart).all())
                        assert bool((got[want == 0] == 0).all())
                assert bool((v1[i][v > 0] > 0).all())
            ratio = m_tol / (m.abs() + 1e-300) + 12 * EPS
            w_tol = 4 * EPS * w0[i].abs() + HYPER["lr"] * upd.abs() * ratio + 2 * EPS * w.abs() + 1e-44
            assert bool(((w1[i] - w).abs() <= w_tol).all()), (i, float(((w1[i] - w).abs() / w_tol).max()))
            if dtype == torch.bfloat16:
                assert torch.equal(params[i].cpu(), w1[i].to(torch.bfloat16))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.gpu
def test_kernel_has_the_definitions_bits(bits):
    """Moments are rounded operation by operation, so the kernel's are those of plain tensor operations."""
    both = []
    for device in ("cpu", "cuda"):
        params, _ = _tensors(torch.bfloat16, torch.float32, device)
        state = ops.AdamWState(params, bits=bits)
        for step in range(1, 7):
            _, grads = _tensors(torch.bfloat16, torch.float32, device, seed=step)
            ops.adamw_step(params, grads, state, **HYPER)
        both.append(state)
    for name in ("m", "v", "m_scale", "v_scale"):
        a, b = (getattr(s, name) for s in both)
        assert (a is None and b is None) or torch.equal(a, b.cpu()), name
    assert all(torch.equal(a, b.cpu()) for a, b in zip(both[0].moments(), both[1].moments()))


@pytest.mark.parametrize("device", DEVICES)
def test_small_changes_arrive_on_average(device):
    """1,000 steps with a gradient that has dropped: v decays as it should although a step moves it by a hundredth of a code."""
    n = 1 << 14
    p = [torch.zeros(n, device=device)]
    state = ops.AdamWState(p, bits=8)
    g = torch.ones(n, device=device)
    g[::BLOCK] = 4.0                       # the block's scale does not fall with the rest
    state.set_moments(0 * g, g * g)
    small = torch.full((n,), 0.1, device=device)
    small[::BLOCK] = 4.0
    want = 1.0
    for _ in range(1000):
        ops.adamw_step(p, [small], state, lr=0.0, betas=(0.9, 0.999), weight_decay=0.0)
        want = 0.999 * want + 0.001 * 0.01
    rest = torch.arange(n, device=device) % BLOCK != 0
    m, v = state.moments()
    # a step's rounding has at most half a code (v / 16) of deviation, 1,000 of them are independent, 16,320 elements too
    assert abs(float(v[rest].mean()) - want) < 5 * 1000 ** 0.5 / 16 / 16320 ** 0.5 * want
    assert abs(float(m[rest].mean()) - 0.1) < 5 * 10 ** 0.5 / 16 / 16320 ** 0.5 * 0.1
    assert not state.v_scale.isnan().any()


@pytest.mark.parametrize("device", DEVICES)
def test_special_gradients(device):
    n = 3 * BLOCK
    for bits in (8, 32):
        p = [torch.ones(n, device=device)]
        state = ops.AdamWState(p, bits=bits)
        g = torch.zeros(n, device=device)
        ops.adamw_step(p, [g], state, lr=0.1, weight_decay=0.0)
        assert bool((p[0] == 1).all()) and not state.moments()[0].any() and not state.moments()[1].any()
        g[5], g[BLOCK] = 1e-20, 3e18          # squares below the normal numbers and near the largest
        ops.adamw_step(p, [g], state, lr=0.1, weight_decay=0.0)
        m, v = state.moments()
        assert bool(torch.isfinite(p[0]).all()) and bool((p[0][6:BLOCK] == 1).all()) and m[5] > 0 and v[BLOCK] > 1e33
        g[2 * BLOCK + 3] = float("nan")
        ops.adamw_step(p, [g], state, lr=0.1, weight_decay=0.0)
        m, v = state.moments()
        assert bool(torch.isnan(m[2 * BLOCK + 3])) and bool(torch.isnan(v[2 * BLOCK + 3]))
        assert int(torch.isnan(p[0]).sum()) == 1
        # with 8 bits the whole block has lost its scale; no other block has
        assert int(torch.isnan(m).sum()) == (BLOCK if bits == 8 else 1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("eps", [0.0, 1e-35, 1.0])
def test_eps_of_any_size(eps, device):
    p, state = [torch.ones(300, device=device)], None
    g = torch.full((300,), 1e-20, device=device)          # a square below the normal numbers
    g[100:200], g[200:] = 1.0, -1e10
    state = ops.AdamWState(p, bits=32)
    ops.adamw_step(p, [g], state, lr=0.1, eps=eps, weight_decay=0.0)
    w, _m, v, _size, upd = _formula(torch.ones(300).double(), torch.zeros(300).double(), torch.zeros(300).double(), g, 1, 0.1, (0.9, 0.999), eps, 0.0)
    # v of the first hundred is 1e-43, 71 of the smallest numbers: a 142nd of itself, half that in its root
    tol = torch.full((300,), 40 * EPS)
    tol[:100] = 1 / 142 + 1 / 70 if eps < 1.0 else 40 * EPS
    assert bool(((p[0].double().cpu() - w).abs() <= 0.1 * upd.abs() * tol + 2 * EPS).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("eps", [1e-35, 1e-28, 1e-20, 1e-18, 1e-16, 1e-14, 1e-12, 1e-10, 1e-8])
def test_vanishing_gradients_beside_any_eps(eps, device):
    """Squares below the normal numbers count beside an eps that is as small as their roots.  v is off by one of the smallest numbers, 2^-149, at
    most, and with it the root."""
    g = torch.tensor([1e-20, -1e-20, 1e-19, 1e-18, 3e-18, -3e-18, 4e-18, 1e-17, 1e-15, 1.0]).repeat_interleave(30)
    p = [torch.zeros(300, device=device)]
    state = ops.AdamWState(p, bits=32)
    w, m, v = (torch.zeros(300).double() for _ in range(3))
    for step in range(1, 4):
        before = p[0].double().cpu()
        ops.adamw_step(p, [g.to(device)], state, lr=1.0, eps=eps, weight_decay=0.0)
        w, m, v, _size, upd = _formula(w, m, v, g, step, 1.0, (0.9, 0.999), eps, 0.0)
        tol = 40 * EPS + 1 - torch.sqrt((1 - step * 2.0 ** -149 / v).clamp(min=0))
        assert bool(((before - p[0].double().cpu() - upd).abs() <= upd.abs() * tol + 2 * EPS * before.abs()).all()), step


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("large", [1e-3, 1.0, 1e5, 1e15])
def test_a_second_moment_above_0_stays_above_0(large, device):
    """However small beside the largest of its block: also where their quotient is below all numbers."""
    g = torch.full((2 * BLOCK,), 1.2e-21, device=device)         # v is 1e-45, the smallest number
    g[7] = large
    g[BLOCK + 3:BLOCK + 9] = 0.0
    p = [torch.zeros(2 * BLOCK, device=device)]
    state, wide = ops.AdamWState(p, bits=8), ops.AdamWState(p, bits=32)
    ops.adamw_step(p, [g], state)
    ops.adamw_step(p, [g], wide)
    assert torch.equal(state.v > 0, wide.v > 0) and int((state.v == 0).sum()) == 6
    state.set_moments(*wide.moments())
    assert torch.equal(state.v > 0, wide.v > 0)


@pytest.mark.parametrize("device", DEVICES)
def test_inference_tensors(device):
    with torch.inference_mode():
        p = [torch.ones(300, device=device)]
        state = ops.AdamWState(p, bits=8)
        ops.adamw_step(p, [torch.ones(300, device=device)], state, lr=0.1)
        assert bool((p[0] < 1).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
def test_missing_gradients_and_views(bits, device):
    base = torch.randn(4096 + 3, generator=torch.Generator().manual_seed(1)).to(device)
    views = [base[3:1003], base[1003:1004], base[1005:4099].view(2, -1)]       # no alignment but the type's
    alone = [v.clone() for v in views]
    grads = [torch.randn(v.shape, generator=torch.Generator().manual_seed(2)).to(device) for v in views]
    strided = [g.clone() if g.dim() == 1 else g.t().contiguous().t() for g in grads]
    before = base.clone()
    a, b = ops.AdamWState(views, bits=bits), ops.AdamWState(alone, bits=bits)
    for step in range(3):
        which = [None if step == 1 and i == 0 else g for i, g in enumerate(grads)]
        ops.adamw_step(views, which, a, **HYPER)
        ops.adamw_step(alone, [None if w is None else s for w, s in zip(which, strided)], b, **HYPER)
    assert a.steps == [2, 3, 3]
    assert all(torch.equal(x, y) for x, y in zip(views, alone)) and torch.equal(a.m, b.m) and torch.equal(a.v, b.v)
    assert torch.equal(base[:3], before[:3]) and base[1004] == before[1004]


@pytest.mark.parametrize("device", DEVICES)
def test_more_tensors_than_one_launch_takes(device):
    shapes = [(1 + 37 * i % 700,) for i in range(203)]
    params, grads = _tensors(torch.float32, torch.float32, device, shapes=shapes)
    want = [p.clone() for p in params]
    state = ops.AdamWState(params, bits=32)
    ops.adamw_step(params, grads, state, **HYPER)
    for p, w, g in zip(params, want, grads):
        one = ops.AdamWState([w], bits=32)
        ops.adamw_step([w], [g], one, **HYPER)
        assert torch.equal(p, w)


@pytest.mark.parametrize("device", DEVICES)
def test_states_are_saved_and_loaded(device):
    params, grads = _tensors(torch.bfloat16, torch.float32, device)
    state = ops.AdamWState(params, bits=8)
    for _ in range(2):
        ops.adamw_step(params, grads, state, **HYPER)
    saved = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in state.state_dict().items()}
    other = ops.AdamWState(params, bits=8)
    other.load_state_dict(saved)
    again = ops.AdamWState(params, bits=8)
    again.set_moments(*state.moments())                # values on the grid come back unchanged
    assert torch.equal(again.m, state.m) and torch.equal(again.v, state.v) and torch.equal(again.v_scale, state.v_scale)
    wide = ops.AdamWState(params, bits=32)
    wide.load_state_dict(saved)
    assert torch.equal(wide.m, state.moments()[0]) and wide.steps == state.steps
    narrow = ops.AdamWState(params, bits=8)
    narrow.load_state_dict(wide.state_dict())
    assert torch.equal(narrow.m, state.m) and torch.equal(narrow.master, state.master)
    twin = [p.clone() for p in params]
    ops.adamw_step(params, grads, state, **HYPER)
    ops.adamw_step(twin, grads, other, **HYPER)
    assert all(torch.equal(a, b) for a, b in zip(params, twin))


@pytest.mark.parametrize("device", DEVICES)
def test_moments_are_set_in_pieces(device, monkeypatch):
    """Pieces that end anywhere among the blocks give what one piece gives, short moments have zeros behind them."""
    from piper_b200.ops import optim
    params = [torch.zeros(n, device=device) for n in (1000, 5000, 3)]
    g = torch.Generator().manual_seed(1)
    states = []
    for piece in (1 << 20, 5 * BLOCK, BLOCK):
        monkeypatch.setattr(optim, "_PIECE", piece)
        state = ops.AdamWState(params, bits=8)
        g.manual_seed(1)
        m, v = (torch.randn(state.numel, generator=g).to(device) for _ in range(2))
        m, v = m * (torch.arange(state.numel, device=device) < 700), v.abs()
        state.set_moments(m, v)
        wide = ops.AdamWState(params, bits=32)
        wide.load_state_dict(state.state_dict())
        assert all(torch.equal(a, b) for a, b in zip(wide.moments(), state.moments()))
        narrow = ops.AdamWState(params, bits=8)
        narrow.load_state_dict(wide.state_dict())
        assert torch.equal(narrow.m, state.m) and torch.equal(narrow.v, state.v) and torch.equal(narrow.v_scale, state.v_scale)
        for bits in (8, 32):
            short = ops.AdamWState(params, bits=bits)
            short.set_moments(torch.ones_like(m), torch.ones_like(v))
            short.set_moments(m[:700], v[:700])
            a, b = short.moments()
            assert not a[700:].any() and not b[700:].any() and bool(a[:700].any())
        states.append(state)
    for s in states[1:]:
        assert torch.equal(s.m, states[0].m) and torch.equal(s.v, states[0].v) and torch.equal(s.m_scale, states[0].m_scale)
    for bad in ((m, v[:5]), (torch.zeros(state.numel + 1),) * 2, (m.view(2, -1), v.view(2, -1))):
        with pytest.raises(ValueError):
            state.set_moments(*bad)


@pytest.mark.gpu
def test_setting_moments_takes_little_memory():
    p = torch.zeros(64 << 20, device="cuda", dtype=torch.bfloat16)
    state = ops.AdamWState([p], bits=8)
    m, v = state.moments()
    m.normal_(), v.uniform_()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    state.set_moments(m, v)
    # a piece of 4 Mi elements at a time, a hundred bytes for each
    assert torch.cuda.max_memory_allocated() - before < (4 << 20) * 100
    a, b = state.moments()
    assert bool(((a - m).abs() <= m.abs() / 16 + state.m_scale.repeat_interleave(BLOCK) * 2.0 ** -16).all())
    assert bool(((b - v).abs() <= v / 16 + state.v_scale.repeat_interleave(BLOCK) * 2.0 ** -31).all())


@pytest.mark.parametrize("device", DEVICES)
def test_a_state_of_other_types_is_refused(device):
    """Same shapes, types in another order: the master copies would be those of other parameters.  A refused state changes nothing."""
    def tensors(*dtypes):
        return [torch.ones(300, dtype=t, device=device) for t in dtypes]

    f32, b16 = torch.float32, torch.bfloat16
    for bits in (8, 32):
        for source, target in (((f32, b16), (b16, f32)), ((f32, b16), (b16, b16)), ((b16, b16), (b16, f32)), ((b16, b16), (f32, f32)),
                               ((f32, f32), (b16, f32))):
            params = tensors(*target)
            other = ops.AdamWState(tensors(*source), bits=bits)
            state = ops.AdamWState(params, bits=40 - bits)
            ops.adamw_step(params, [torch.ones_like(p) for p in params], state)
            before = [t.clone() for t in (*state.moments(), *([] if state.master is None else [state.master]))]
            with pytest.raises(ValueError):
                state.load_state_dict(other.state_dict())
            after = [*state.moments(), *([] if state.master is None else [state.master])]
            assert all(torch.equal(x, y) for x, y in zip(before, after)) and state.steps == [1, 1]
            # a state without its types, as once saved
            old = {k: v for k, v in state.state_dict().items() if k != "dtypes"}
            if len(set(target)) == 1:
                state.load_state_dict(old)
            else:
                with pytest.raises(ValueError):
                    state.load_state_dict(old)
                state.load_state_dict(state.state_dict())
            cut = dict(state.state_dict(), m=state.m[:BLOCK], v=state.v[:BLOCK])
            with pytest.raises(ValueError):
                state.load_state_dict(cut)


def test_moments_of_eight_bits_take_two_bytes():
    p = [torch.zeros(1 << 16)]
    s = ops.AdamWState(p, bits=8)
    held = sum(t.numel() * t.element_size() for t in (s.m, s.v, s.m_scale, s.v_scale))
    assert held == (1 << 16) * 2 + (1 << 16) // BLOCK * 8


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    p = [torch.zeros(10, device=device), torch.zeros(4, 4, device=device)]
    with pytest.raises(ValueError):
        ops.AdamWState(p, bits=16)
    with pytest.raises(ValueError):
        ops.AdamWState([])
    with pytest.raises(ValueError):
        ops.AdamWState([p[0], p[0]])
    with pytest.raises(TypeError):
        ops.AdamWState([torch.zeros(4, dtype=torch.float16, device=device)])
    with pytest.raises(ValueError):
        ops.AdamWState([torch.zeros(4, 6, device=device).t()])
    state = ops.AdamWState(p)
    g = [torch.zeros_like(t) for t in p]
    for params, grads in ((p[:1], g[:1]), (p, g[:1]), (p, [g[0], g[0]]), (p, [g[1], g[1]]), ([p[1], p[0]], [g[1], g[0]]),
                          ([p[0].bfloat16(), p[1]], g)):
        with pytest.raises(ValueError):
            ops.adamw_step(params, grads, state)
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8), dict(weight_decay=-0.1),
                dict(lr=float("nan"))):
        with pytest.raises(ValueError):
            ops.adamw_step(p, g, state, **bad)
    assert state.steps == [0, 0]
    with pytest.raises(ValueError):
        state.load_state_dict(ops.AdamWState(p[:1]).state_dict())


@pytest.mark.parametrize("device", DEVICES)
def test_other_types_are_refused_on_either_device(device):
    p = [torch.ones(10, device=device), torch.ones(10, device=device, dtype=torch.bfloat16)]
    state = ops.AdamWState(p)
    g = [torch.ones(10, device=device) for _ in p]
    for params, grads in (([p[0].double(), p[1]], g), ([p[0].half(), p[1]], g), ([p[1], p[0]], g), (p, [g[0].double(), g[1]]),
                          (p, [g[0], g[1].half()]), (p, [g[0].long(), None])):
        with pytest.raises(ValueError):
            ops.adamw_step(params, grads, state)
    assert state.steps == [0, 0] and bool((p[0] == 1).all()) and bool((p[1] == 1).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
def test_parameters_that_share_memory_are_refused(bits, device):
    """Two of them would be stepped by one launch in no order; neighbours, and parameters without elements, are none of those."""
    room = torch.zeros(600, device=device)
    with pytest.raises(ValueError):
        ops.AdamWState([room[:300], room[299:]], bits=bits)
    with pytest.raises(ValueError):
        ops.AdamWState([room, room[5:9]], bits=bits)
    apart = [room[300:], room[:300], room[10:10]]
    state = ops.AdamWState(apart, bits=bits)
    g = [torch.ones_like(t) for t in apart]
    with pytest.raises(ValueError):
        ops.adamw_step([room[300:], room[1:301], room[10:10]], g, state)
    with pytest.raises(ValueError):
        ops.adamw_step([room[:300], room[:300], room[10:10]], g, state)
    with pytest.raises(ValueError):
        ops.adamw_step([torch.zeros(300, 2, device=device)[:, 0], room[:300], room[10:10]], g, state)
    assert state.steps == [0, 0, 0] and not room.any()
    ops.adamw_step(apart, g, state)
    assert state.steps == [1, 1, 1] and bool((room != 0).all())
    with pytest.raises(ValueError):
        state.set_step(-1)


@pytest.mark.parametrize("device", DEVICES)
def test_a_saved_tensor_that_was_stepped_is_noticed(device):
    w = torch.ones(8, device=device, requires_grad=True)
    state = ops.AdamWState([w])
    y = (w * w).sum()
    ops.adamw_step([w], [torch.ones(8, device=device)], state)
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()


@pytest.mark.gpu
def test_a_step_is_not_captured():
    p = [torch.zeros(256, device="cuda")]
    state = ops.AdamWState(p)
    g = [torch.ones(256, device="cuda")]
    ops.adamw_step(p, g, state)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            ops.adamw_step(p, g, state)
    torch.cuda.synchronize()
    ops.adamw_step(p, g, state)
    assert state.steps == [2]


@pytest.mark.gpu
def test_a_captured_step_is_refused_by_the_library():
    """It asks the stream of the parameters' device, whichever device is current where the step is called; also beside a capture that is
    another stream's alone."""
    p, g = [torch.zeros(256, device="cuda")], [torch.ones(256, device="cuda")]
    state = ops.AdamWState(p, bits=8)
    args = (p, g, state.m, state.v, state.m_scale, state.v_scale, state.master, state._table, 0, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        graph.capture_begin(capture_error_mode="thread_local")
        kept = torch.zeros(8, device="cuda")
        try:
            with pytest.raises(RuntimeError, match="captured"):
                ops.native.lib().adamw(*args)
            with torch.cuda.stream(torch.cuda.Stream()):
                ops.adamw_step(p, g, state)
        finally:
            graph.capture_end()
    torch.cuda.synchronize()
    assert state.steps == [1] and bool((p[0] < 0).all()) and kept.numel() == 8


@pytest.mark.gpu
def test_states_on_two_streams():
    results = []
    sets = [_tensors(torch.bfloat16, torch.float32, "cuda", seed=i) for i in range(2)]
    for streams in ([None, None], [torch.cuda.Stream(), torch.cuda.Stream()]):
        copies = [[p.clone() for p in s[0]] for s in sets]
        states = [ops.AdamWState(c, bits=8) for c in copies]
        torch.cuda.synchronize()
        for _ in range(3):
            for c, s, st, stream in zip(copies, sets, states, streams):
                with torch.cuda.stream(stream):
                    ops.adamw_step(c, s[1], st, **HYPER)
        torch.cuda.synchronize()
        results.append([t for c, s in zip(copies, states) for t in (*c, s.m, s.v)])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_bucket_with_eight_bit_moments(dtype):
    from piper_b200.runtime.storage import AdamConfig, ParamSlot, ParamStorage
    slots = [ParamSlot(0, "a.weight", (40, 30), dtype, True), ParamSlot(1, "b.weight", (70,), dtype, True)]
    cfg = AdamConfig(lr=1e-2, weight_decay=0.1, decoupled=True, state_bits=8)
    st = ParamStorage("k", slots, torch.device("cpu"), dtype, "local", 0, 1, None, cfg)
    want = [st.flat_params.clone()]
    state = ops.AdamWState(want, bits=8)
    for step in range(3):
        g = torch.randn(st.numel, generator=torch.Generator().manual_seed(step))
        st.flat_grads.copy_(g)
        st.step(0.25)
        ops.adamw_step(want, [g], state, lr=1e-2, betas=cfg.betas, eps=cfg.eps, weight_decay=0.1, grad_scale=0.25)
        assert torch.equal(st.flat_params, want[0]) and not st.flat_grads.any()
    m, v = st.moments()
    assert m.shape == (st.numel,) and bool((v >= 0).all())
    st.set_moments(m, v)
    assert torch.equal(st.moments()[0], m) and torch.equal(st.moments()[1], v)


@pytest.mark.parametrize("device", DEVICES)
def test_the_random_bits_of_a_state_that_continues_a_list(device):
    params, grads = _tensors(torch.float32, torch.float32, device, shapes=[(1000,)] * 4)
    params, grads = [params[0].clone() for _ in params], [grads[0]] * 4
    state = ops.AdamWState(params, bits=8)
    halves = [ops.AdamWState(params[:2], bits=8), ops.AdamWState(params[2:], bits=8, first=2)]
    for _ in range(2):
        copies = [p.clone() for p in params]
        ops.adamw_step(params, grads, state, **HYPER)
        for part, h in zip((slice(0, 2), slice(2, 4)), halves):
            ops.adamw_step(copies[part], grads[part], h, **HYPER)
        assert torch.equal(torch.cat([h.m for h in halves]), state.m) and torch.equal(torch.cat([h.v for h in halves]), state.v)
    codes = state.v.view(4, -1)
    assert all(not torch.equal(codes[i], codes[j]) for i in range(4) for j in range(i))
    last = ops.AdamWState(params[:1], bits=8, first=2 ** 32 - 1)
    ops.adamw_step(params[:1], grads[:1], last, **HYPER)
    for bad in (-1, 2 ** 32):
        with pytest.raises(ValueError):
            ops.AdamWState(params[:1], bits=8, first=bad)


def test_buckets_and_shards_round_by_bits_of_their_own():
    """Equal gradients of equal weights: buckets of other ordinals and shards of one bucket draw other bits, replicas the same."""
    from piper_b200.runtime.storage import AdamConfig, ParamSlot, ParamStorage
    cfg = AdamConfig(lr=1e-2, decoupled=True, state_bits=8)

    def codes(mode, rank, ordinal, ep=None):
        slot = ParamSlot(0, "a.gain", (4096,), torch.float32, True)
        if ep is not None:
            slot.ep_sharded, slot.full_shape, slot.ep_index, slot.ep_degree = True, (8192,), ep, 2
        st = ParamStorage("k", [slot], torch.device("cpu"), torch.float32, mode, rank, 2, None, cfg, ordinal=ordinal)
        st.step_count = 1
        n = st.state8.numel
        ops.adamw_step([torch.ones(n)], [torch.linspace(0.1, 1.0, 256).repeat(n // 256)], st.state8)
        return st.state8.m[:2048]

    one = codes("allreduce", 0, 7)
    assert torch.equal(one, codes("allreduce", 1, 7)) and not torch.equal(one, codes("allreduce", 0, 8))
    assert not torch.equal(codes("zero2", 0, 7), codes("zero2", 1, 7))
    assert torch.equal(codes("local", 0, 7, ep=1), codes("local", 1, 7, ep=1))
    assert not torch.equal(codes("local", 0, 7, ep=0), codes("local", 1, 7, ep=1))


def test_buckets_of_a_setup_have_ordinals():
    from piper_b200 import piper_setup
    from piper_b200.models.llama3 import LLAMA_CONFIGS, Transformer
    cfg = LLAMA_CONFIGS["tiny"]
    tok = torch.zeros(2, 64, dtype=torch.int64)
    schedule = [{"op": "place", "filter": {"PP": i}, "devices": [0]} for i in range(2)] + \
        [{"op": "split", "filter": {}, "dim_name": "MB", "num_microbatches": 2}]
    firsts = []
    for _ in range(2):
        actor = piper_setup(Transformer, (cfg, 64, 2), optim_fn=torch.optim.AdamW, optim_kwargs={"state_bits": 8}, example_inputs=[tok],
                            example_outputs=tok, model_dtype=torch.float32, const_attrs=Transformer.const_attrs(cfg, 64),
                            schedule_directives=schedule, device="cpu")
        firsts.append({k: b.storage.state8.first for k, b in actor.buckets.items() if b.storage is not None and b.storage.numel})
    assert firsts[0] == firsts[1] and len(firsts[0]) == 2 and len(set(firsts[0].values())) == 2


def test_state_bits_of_a_setup():
    from piper_b200.engine import _adam_config
    assert _adam_config(torch.optim.AdamW, {"state_bits": 8}).state_bits == 8
    assert _adam_config(torch.optim.AdamW, None).state_bits == 32
    for fn, bits in ((torch.optim.Adam, 8), (torch.optim.AdamW, 4)):
        with pytest.raises(ValueError):
            _adam_config(fn, {"state_bits": bits})
