"""A policy update on a packed batch: rotary positions, attention, log probabilities, the clipped loss within sequences and the
routers' balance losses together, in the bundled models."""
import pytest
import torch
import torch.utils.checkpoint

from piper_b200 import nn, ops
from piper_b200.ops import native

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
LENS = [130, 1, 77, 45]
T = sum(LENS) + 3
VOCAB = 512


def _model(kind, device, balance_coef=0.0, max_len=160):
    from piper_b200.models.llama3 import LlamaConfig, Transformer
    from piper_b200.models.qwen3 import PiperQwen3Model, Qwen3Config
    if kind == "llama":
        cfg = LlamaConfig(dim=256, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=VOCAB, ffn_hidden=256, rope_theta=10000.0)
        model = Transformer(cfg, max_len, 1)
    else:
        cfg = Qwen3Config(dim=256, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=64, vocab_size=VOCAB, num_experts=8, top_k=2,
                          moe_hidden=128, balance_coef=balance_coef)
        model = PiperQwen3Model(cfg, 1, max_len)
    g = torch.Generator().manual_seed(0)
    with torch.no_grad():
        for name, p in sorted(model.named_parameters()):
            p.copy_(torch.ones(p.shape) if p.dim() == 1 else torch.randn(p.shape, generator=g) * p.shape[-1] ** -0.5)
    model = model.to(device)
    if device == "cuda":
        model = model.to(torch.bfloat16)
    consts = type(model).const_attrs(cfg, max_len, device)
    model.rope_cos, model.rope_sin = consts["rope_cos"], consts["rope_sin"]
    return model


def _batch(device):
    g = torch.Generator().manual_seed(1)
    tokens = torch.randint(0, VOCAB, (1, T), generator=g)
    offsets = torch.tensor([0] + LENS).cumsum(0)
    return tokens.to(device), offsets, ops.pack_sequences(offsets, T, device=device)


@pytest.mark.parametrize("kind", ["llama", "qwen"])
def test_packed_sequences_are_sequences_by_themselves(kind):
    """On the CPU, in fp32: logits and gradients of a packed batch are those of its sequences one after the other."""
    model = _model(kind, "cpu")
    tokens, offsets, s = _batch("cpu")
    g = torch.Generator().manual_seed(2)
    up = torch.randn(T, VOCAB, generator=g)
    up[sum(LENS):] = 0
    out = model(tokens, s).view(T, VOCAB)
    names = [n for n, _ in model.named_parameters()]
    grads = torch.autograd.grad(out, list(model.parameters()), up)
    want, sums = [], [torch.zeros_like(p) for p in model.parameters()]
    for a, b in zip(offsets.tolist(), offsets.tolist()[1:]):
        o = model(tokens[:, a:b]).view(b - a, VOCAB)
        want.append(o.detach())
        for acc, d in zip(sums, torch.autograd.grad(o, list(model.parameters()), up[a:b])):
            acc += d
    want = torch.cat(want)
    # fp32 sums in another order: some 20 operations deep over at most 256 terms each, below 2^-24 x 20 x 256 of the largest
    depth = 2.0 ** -24 * 20 * 256
    assert float((out[:sum(LENS)].detach() - want).abs().max()) <= depth * float(want.abs().max())
    for n, a, b in zip(names, grads, sums):
        assert float((a - b).abs().max()) <= depth * float(b.abs().max()), n


def test_jitter_and_balance_loss_of_a_packed_batch_are_those_of_its_sequences():
    """The frozen router noise goes by a token's place in its sequence, and tokens behind the last sequence do not count."""
    from piper_b200.models.qwen3 import PiperQwen3Model, Qwen3Config
    cfg = Qwen3Config(dim=64, n_layers=1, n_heads=2, n_kv_heads=1, head_dim=32, vocab_size=VOCAB, num_experts=8, top_k=2, moe_hidden=32,
                      balance_coef=3.0, router_jitter_std=1.0)
    model = PiperQwen3Model(cfg, 1, 130)
    torch.manual_seed(0)
    with torch.no_grad():
        for p in model.parameters():
            p.copy_(torch.randn(p.shape) * 0.1)
    consts = PiperQwen3Model.const_attrs(cfg, 130)
    model.rope_cos, model.rope_sin, model.router_jitter = consts["rope_cos"], consts["rope_sin"], consts["router_jitter"].float()
    tokens, offsets, s = _batch("cpu")
    with torch.no_grad():
        out = model(tokens, s).view(T, VOCAB)
        for a, b in zip(offsets.tolist(), offsets.tolist()[1:]):
            alone = ops.pack_sequences(torch.tensor([0, b - a]), b - a)
            # fp32 sums in another order, as above
            want = model(tokens[:, a:b], alone).view(b - a, VOCAB)
            assert float((out[a:b] - want).abs().max()) <= 2.0 ** -24 * 20 * 256 * float(want.abs().max())

    def gate_gradient(toks):                     # of the balance loss alone
        model.zero_grad()
        (model(toks, s) * 0.0).sum().backward()
        return model.layers[0].moe.gate.weight.grad.clone()

    first = gate_gradient(tokens)
    other = tokens.clone()
    other[0, sum(LENS):] = (other[0, sum(LENS):] + 1) % VOCAB
    assert bool(first.any()) and torch.equal(first, gate_gradient(other))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["llama", "qwen"])
def test_logits_of_a_sequence_do_not_depend_on_the_others(kind, device):
    model = _model(kind, device)
    tokens, offsets, s = _batch(device)
    with torch.no_grad():
        first = model(tokens, s).view(T, VOCAB)
        other = tokens.clone()
        a, b = int(offsets[2]), int(offsets[3])
        other[0, a:b] = (other[0, a:b] + 1) % VOCAB
        second = model(other, s).view(T, VOCAB)
    end = int(offsets[-1])
    assert torch.equal(first[:a], second[:a]) and torch.equal(first[b:end], second[b:end])
    assert not torch.equal(first[a:b], second[a:b]) and bool(torch.isfinite(first[:end].float()).all())
    if device == "cuda":
        native.check_status()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["llama", "qwen"])
def test_a_policy_update(kind, device):
    """Forward, loss and backward; tokens without advantage and without KL term leave no gradient, and balance losses add theirs to
    the routers alone."""
    model = _model(kind, device)
    tokens, offsets, s = _batch(device)
    target = torch.roll(tokens, -1, 1).reshape(-1)
    g = torch.Generator().manual_seed(3)
    with torch.no_grad():
        old = ops.token_logprobs(model(tokens, s).view(T, VOCAB), target).logprob
    old = old + (torch.randn(T, generator=g) * 0.1).to(device)
    adv = torch.randn(T, generator=g).to(device)
    mask = torch.ones(T, dtype=torch.bool, device=device)
    mask[offsets[1:].to(device) - 1] = False              # the last token of a sequence predicts none

    def step(m, advantages, kl_coef):
        loss = nn.clipped_policy_loss(m(tokens, s), target, advantages, old, ref_logprob=old, mask=mask, sequences=s, kl_coef=kl_coef)
        m.zero_grad()
        loss.backward()
        return loss.detach(), {n: p.grad.clone() for n, p in m.named_parameters()}

    loss, grads = step(model, adv, 0.1)
    assert bool(torch.isfinite(loss)) and all(bool(torch.isfinite(d.float()).all()) for d in grads.values())
    assert all(bool(d.any()) for n, d in grads.items() if "gate" not in n)
    only = torch.zeros_like(adv)
    a, b = int(offsets[2]), int(offsets[3])
    only[a:b] = adv[a:b]
    _, grads = step(model, only, 0.0)
    table = grads["tok_embeddings.weight"]
    seen = torch.zeros(VOCAB, dtype=torch.bool, device=device)
    seen[tokens[0, a:b]] = True
    assert not bool(table[~seen].any()) and bool(table[tokens[0, a]].any())
    if kind == "qwen":
        zero, none = step(model, torch.zeros_like(adv), 0.0)
        assert float(zero) == 0 and not any(bool(d.any()) for d in none.values())
        balanced = _model(kind, device, balance_coef=0.5)
        zero, some = step(balanced, torch.zeros_like(adv), 0.0)
        assert float(zero) == 0 and bool(some["layers.1.moe.gate.weight"].any())
        assert not bool(some["output.weight"].any()) and not bool(some["layers.1.moe.experts.w2"].any())
    if device == "cuda":
        native.check_status()


@pytest.mark.parametrize("device", DEVICES)
def test_positions_that_the_tables_lack_are_nan(device):
    _tokens, offsets, s = _batch(device)
    cos, sin = ops.rope_tables(64, 100, 10000.0, device)
    c, d = nn.packed_rope(cos, sin, s)
    at = s.positions()
    assert bool(torch.isnan(c[at >= 100]).all()) and bool(torch.isnan(d[at >= 100]).all()) and int((at >= 100).sum()) == 30
    assert torch.equal(c[at < 100], cos[at[at < 100]]) and torch.equal(d[at < 100], sin[at[at < 100]])


@pytest.mark.parametrize("device", DEVICES)
def test_balance_losses_through_the_engine(device):
    """Two pipeline stages, two microbatches: every stage's routers get the gradient of their balance losses, the losses that come back
    are the model's own."""
    from piper_b200 import piper_exec_dag, piper_setup
    from piper_b200.models.qwen3 import PiperQwen3Model, Qwen3Config
    from piper_b200.runtime.storage import init_tensor

    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    cfg = Qwen3Config(dim=256, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=64, vocab_size=VOCAB, num_experts=8, top_k=2,
                      moe_hidden=128, balance_coef=1.5)
    g = torch.Generator().manual_seed(5)
    x, y = (torch.randint(0, VOCAB, (4, 128), generator=g) for _ in range(2))
    schedule = [{"op": "place", "filter": {"PP": i}, "devices": [0]} for i in range(2)] + \
        [{"op": "split", "filter": {}, "dim_name": "MB", "num_microbatches": 2}]
    actor = piper_setup(PiperQwen3Model, (cfg, 2, 128), optim_fn=torch.optim.AdamW, example_inputs=[x], example_outputs=y,
                        model_dtype=dtype, const_attrs=PiperQwen3Model.const_attrs(cfg, 128), schedule_directives=schedule,
                        device=device)
    actor.debug_keep_grads = True
    model = PiperQwen3Model(cfg, 2, 128).to(device).to(dtype)
    consts = PiperQwen3Model.const_attrs(cfg, 128, device)
    model.rope_cos, model.rope_sin = consts["rope_cos"], consts["rope_sin"]
    with torch.no_grad():
        for n, p in model.named_parameters():
            p.copy_(init_tensor(n, p.shape, dtype, torch.device(device)))
    losses = [float(v) for v in piper_exec_dag(nn.cross_entropy_loss)]
    got = {k: v.float() for k, v in actor.last_grads.items()}
    want = []
    for a, b in zip(x.to(device).split(2), y.to(device).split(2)):
        loss = nn.cross_entropy_loss(model(a), b)
        want.append(float(loss.detach()))
        loss.backward()
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -20
    # the same ops on the same microbatches: weight gradients of both summed in another order, two roundings of autograd's sum
    assert all(abs(a - b) <= 2.0 ** -20 * abs(b) for a, b in zip(losses, want)), (losses, want)
    for n, p in model.named_parameters():
        a, b = got[n], p.grad.float() / 2
        assert float((a - b).norm()) <= 3 * half * float(b.norm()) + 1e-8, n
    plain = PiperQwen3Model(Qwen3Config(**{**cfg.__dict__, "balance_coef": 0.0}), 2, 128).to(device).to(dtype)
    plain.load_state_dict(model.state_dict())
    plain.rope_cos, plain.rope_sin = model.rope_cos, model.rope_sin
    nn.cross_entropy_loss(plain(x.to(device)), y.to(device)).backward()
    for i in range(2):                           # both stages' routers differ from those without balance losses
        a, b = got[f"layers.{i}.moe.gate.weight"], plain.layers[i].moe.gate.weight.grad.float()
        assert float((a - b).norm()) > 0.05 * float(a.norm())
    if device == "cuda":
        native.check_status()


def test_full_graph_capture_records_the_ops():
    s = ops.pack_sequences(torch.tensor([0, 5, 14]), 16)
    g = torch.Generator().manual_seed(6)
    qkv, new, old, adv = (torch.randn(*shape, generator=g) for shape in ((16, 4 * 8), (16,), (16,), (16,)))
    logits = torch.randn(16, 4, generator=g)
    idx = torch.randint(0, 4, (16, 2), generator=g, dtype=torch.int32)

    def f(qkv, new, logits):
        out = ops.packed_attention(qkv, s, 2, 1, 8, 0.3).square().sum()
        loss = ops.clipped_policy_loss(new, old, adv, ref_logprob=old, sequences=s, kl_coef=0.1).loss
        return out + loss + ops.moe.moe_balance_loss(logits, idx).loss

    leaves = [t.requires_grad_(True) for t in (qkv, new, logits)]
    want = torch.autograd.grad(f(*leaves), leaves)
    # the graph of the forward pass, as the engine records it; a tracer of backward passes would need formulas that do not read tables
    compiled = torch.compile(f, backend="eager", fullgraph=True)
    for a, b in zip(torch.autograd.grad(compiled(*leaves), leaves), want):
        assert torch.allclose(a, b)


@pytest.mark.parametrize("device", DEVICES)
def test_under_recomputing_checkpoints(device):
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    s = ops.pack_sequences(torch.tensor([0, 70, 200]), 210, device=device)
    g = torch.Generator().manual_seed(7)
    qkv = torch.randn(210, 4 * 64, generator=g).to(dtype).to(device).requires_grad_(True)
    new, old, adv = (torch.randn(210, generator=g).to(device) for _ in range(3))
    new.requires_grad_(True)
    logits = torch.randn(210, 8, generator=g).to(dtype).to(device).requires_grad_(True)

    def block(qkv, new, logits):
        _w, idx, _c = ops.moe.moe_route(logits * 1.0, 2, True)
        out = ops.packed_attention(qkv * 1.0, s, 2, 1, 64, 0.125).float().sum()
        loss = ops.clipped_policy_loss(new * 1.0, old, adv, sequences=s).loss
        return out + loss + ops.moe.moe_balance_loss(logits * 1.0, idx).loss

    leaves = [qkv, new, logits]
    want = torch.autograd.grad(block(*leaves), leaves)
    for reentrant in (False, True):
        out = torch.utils.checkpoint.checkpoint(block, *leaves, use_reentrant=reentrant)
        for t in leaves:
            t.grad = None
        out.backward()
        assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("grouped", [False, True])
def test_ops_keep_to_their_schemas(grouped, device):
    """Schemas, fake bodies and registrations of the ops, as the dispatcher's own check sees them."""
    from piper_b200.ops import packed
    offsets = torch.tensor([0, 3, 9], dtype=torch.int32).to(device)
    tiles, own = packed.pack_table(offsets, 12, 3, grouped)
    g = torch.Generator().manual_seed(8)
    qkv, new, old, adv, logits = (torch.randn(*shape, generator=g).to(device) for shape in ((12, 256), (12,), (12,), (12,), (12, 4)))
    qkv = qkv.to(torch.bfloat16).requires_grad_(True)
    idx = torch.zeros(12, 2, dtype=torch.int32, device=device)
    weights, loss = (torch.ones(shape, device=device, requires_grad=True) for shape in ((3, 2), ()))
    calls = [(torch.ops.piper.packed_attention_fwd, (qkv, tiles, own if grouped else None, 1, 2, 2, 1, 64, 0.3, grouped)),
             (torch.ops.piper.clipped_policy_fwd, (new.requires_grad_(True), old, adv, old, adv > 0, None if grouped else tiles, 0.8, 1.2, 0.1)),
             (torch.ops.piper.moe_balance_fwd, (logits.requires_grad_(True), idx, adv > 0 if grouped else None)),
             (torch.ops.piper.moe_attach_loss, (weights, loss, 0.5))]
    if device == "cpu":                          # on a GPU rows of the table's memory that are not in use are not written
        calls.append((torch.ops.piper.pack_table, (offsets, 12, 3, grouped)))
    for op, args in calls:
        torch.library.opcheck(op.default, args, test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))


def _empty_for(offsets, tokens):
    """The layout that a GPU gives for offsets which do not rise from 0 to at most ``tokens``: their batch counts as empty."""
    from piper_b200.ops import packed
    s = ops.pack_sequences(torch.tensor([0, tokens]), tokens)
    return s._replace(offsets=torch.tensor(offsets, dtype=torch.int32), table=packed._table_ref([0, 0], tokens, 3))


BAD_OFFSETS = [[1000, 1100], [5, 300], [0, 300, 200], [0, 301], [0, -5, 3], [-40, 300]]


@pytest.mark.parametrize("offsets", BAD_OFFSETS)
def test_bad_offsets_look_up_nothing_out_of_range(offsets):
    """No token of such a batch belongs to a sequence; each has position 0, so all tables have a row for it."""
    s = _empty_for(offsets, 300)
    assert not bool(s.inside().any()) and not bool(s.positions().any())
    cos, sin = ops.rope_tables(64, 100, 10000.0, "cpu")
    c, d = nn.packed_rope(cos, sin, s)
    assert torch.equal(c, cos[:1].expand(300, -1)) and torch.equal(d, sin[:1].expand(300, -1))


@pytest.mark.parametrize("offsets", [[5, 300], [1000, 1100]])
def test_positions_below_zero_are_nan(offsets):
    """A table that calls tokens in front of the first offset its own: no row of the rotary tables is theirs, from the end neither."""
    s = ops.pack_sequences(torch.tensor([0, 300]), 300)._replace(offsets=torch.tensor(offsets, dtype=torch.int32))
    cos, sin = ops.rope_tables(64, 400, 10000.0, "cpu")
    c, d = nn.packed_rope(cos, sin, s)
    first = min(offsets[0], 300)
    assert bool(torch.isnan(c[:first]).all()) and bool(torch.isnan(d[:first]).all())
    assert torch.equal(c[first:], cos[:300 - first]) and torch.equal(d[first:], sin[:300 - first])


@pytest.mark.parametrize("kind", ["llama", "qwen"])
def test_a_model_takes_bad_offsets_as_an_empty_batch(kind):
    model = _model(kind, "cpu", balance_coef=0.5)
    if kind == "qwen":
        model.use_jitter, model.router_jitter = True, torch.randn(160, 8)
    tokens = torch.zeros(1, 300, dtype=torch.int64)
    for bad in (_empty_for([1000, 1100], 300),
                ops.pack_sequences(torch.tensor([0, 300]), 300)._replace(offsets=torch.tensor([1000, 1100], dtype=torch.int32))):
        assert model(tokens, bad).shape == (1, 300, VOCAB)


@pytest.mark.gpu
@pytest.mark.parametrize("offsets", BAD_OFFSETS)
def test_a_model_takes_bad_offsets_on_the_gpu_as_an_empty_batch(offsets):
    model = _model("qwen", "cuda", balance_coef=0.5)
    s = ops.pack_sequences(torch.tensor(offsets, device="cuda"), 300)
    assert not bool(s.inside().any()) and not bool(s.positions().any())
    tokens = torch.zeros(1, 300, dtype=torch.int64, device="cuda")
    logits = model(tokens, s)
    assert bool(torch.isfinite(logits.float()).all())
    with pytest.raises(native.PiperKernelError):
        native.check_status()
    native.check_status()


def test_the_engine_refuses_layouts_of_packed_batches():
    """Stages are traced without data and batches cut into microbatches by rows: a layout is refused by name in front of both."""
    from piper_b200 import piper_exec_dag, piper_setup
    from piper_b200.models.llama3 import LlamaConfig, Transformer
    cfg = LlamaConfig(dim=64, n_layers=2, n_heads=2, n_kv_heads=1, vocab_size=VOCAB, ffn_hidden=64, rope_theta=10000.0)
    tokens, _offsets, s = _batch("cpu")
    schedule = [{"op": "place", "filter": {"PP": 0}, "devices": [0]}, {"op": "split", "filter": {}, "dim_name": "MB", "num_microbatches": 1}]

    def setup(inputs):
        return piper_setup(Transformer, (cfg, T, 1), optim_fn=torch.optim.AdamW, example_inputs=inputs, example_outputs=tokens, device="cpu",
                           model_dtype=torch.float32, const_attrs=Transformer.const_attrs(cfg, T), schedule_directives=schedule)

    with pytest.raises(TypeError, match="packed batch"):
        setup([tokens, s])
    setup([tokens])
    with pytest.raises(TypeError, match="packed batch"):
        piper_exec_dag(nn.cross_entropy_loss, inputs=[tokens, s])
    assert len(piper_exec_dag(nn.cross_entropy_loss, inputs=[tokens])) == 1


@pytest.mark.gpu
def test_packed_sequences_are_sequences_by_themselves_on_the_gpu():
    """As on the CPU, in bf16: one by one, as batches of their own, the sequences give the same logits and sums of gradients, but for roundings.

    A layer rounds some 9 times on the way (norms, projections, rotations, attention, its probabilities, SwiGLU, sums) and twice as often
    on the way back, both passes do, and what a norm or an attention makes of an error is no larger relative to its size: of two layers
    and the head by norms 2 x 20 x 2^-8 forward, three times that for gradients.  Another position, neighbour or mask is off by its own size."""
    model = _model("llama", "cuda")
    tokens, offsets, s = _batch("cuda")
    up = torch.randn(T, VOCAB, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    up[sum(LENS):] = 0
    params = list(model.parameters())
    out = model(tokens, s).view(T, VOCAB)
    grads = torch.autograd.grad(out, params, up)
    sums = [torch.zeros_like(p, dtype=torch.float32) for p in params]
    bound = 2 * 20 * 2.0 ** -8
    for a, b in zip(offsets.tolist(), offsets.tolist()[1:]):
        o = model(tokens[:, a:b], ops.pack_sequences(torch.tensor([0, b - a]), b - a, device="cuda")).view(b - a, VOCAB)
        assert float((o - out[a:b]).float().norm()) <= bound * float(o.float().norm())
        for acc, d in zip(sums, torch.autograd.grad(o, params, up[a:b])):
            acc += d
    for (name, _p), got, want in zip(model.named_parameters(), grads, sums):
        assert float((got.float() - want).norm()) <= 3 * bound * float(want.norm()), name
    native.check_status()


def test_a_step_takes_its_inputs_from_an_iterator():
    from piper_b200 import piper_exec_dag, piper_setup
    from piper_b200.models.llama3 import LlamaConfig, Transformer
    cfg = LlamaConfig(dim=64, n_layers=1, n_heads=2, n_kv_heads=1, vocab_size=VOCAB, ffn_hidden=64, rope_theta=10000.0)
    tokens = torch.zeros(1, 128, dtype=torch.int64)
    schedule = [{"op": "place", "filter": {"PP": 0}, "devices": [0]}, {"op": "split", "filter": {}, "dim_name": "MB", "num_microbatches": 1}]
    piper_setup(Transformer, (cfg, 128, 1), optim_fn=torch.optim.AdamW, example_inputs=[tokens], example_outputs=tokens, device="cpu",
                model_dtype=torch.float32, const_attrs=Transformer.const_attrs(cfg, 128), schedule_directives=schedule)
    (first,) = piper_exec_dag(nn.cross_entropy_loss, inputs=iter([tokens + 1]))
    assert bool(torch.isfinite(torch.as_tensor(first)).all())
