"""A fine-tuning step through the engine: projections in 8 bits, a policy-gradient loss on token log probabilities with an
entropy term, AdamW with 8-bit moments; against the same model and ops stepped by hand.

Both sides run the same ops on the same microbatches.  They may differ where fp32 sums are added in another order: weight gradients
of two microbatches (in the bucket, or by autograd in the parameters' type)."""
import math

import pytest
import torch

from piper_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _schedule(stages):
    return [{"op": "place", "filter": {"PP": i}, "devices": [0]} for i in range(stages)] + \
        [{"op": "split", "filter": {}, "dim_name": "MB", "num_microbatches": 2}]


def _loss(output, tokens):
    from piper_b200.nn import policy_gradient_loss
    return policy_gradient_loss(output, tokens, entropy_coef=0.01, temperature=0.9)


@pytest.mark.parametrize("device", DEVICES)
def test_a_step_through_the_engine(device, tmp_path):
    from piper_b200 import piper_exec_dag, piper_setup
    from piper_b200.models.llama3 import LlamaConfig, Transformer
    from piper_b200.runtime.checkpoint import load_checkpoint, save_checkpoint
    from piper_b200.runtime.storage import init_tensor

    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    cfg = LlamaConfig(dim=256, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=1024, ffn_hidden=688, norm_eps=1e-6,
                      rope_theta=10000.0, max_seq_len=128, fp8=True)
    g = torch.Generator().manual_seed(0)
    x = torch.randint(0, cfg.vocab_size, (4, 128), generator=g)
    y = torch.randint(0, cfg.vocab_size, (4, 128), generator=g)
    y[:, :9] = -100                                   # the prompt
    hyper = {"lr": 1e-3, "weight_decay": 0.1, "betas": (0.9, 0.95)}

    def setup():
        actor = piper_setup(Transformer, (cfg, 128, 2), optim_fn=torch.optim.AdamW, optim_kwargs={**hyper, "state_bits": 8},
                            example_inputs=[x], example_outputs=y, model_dtype=dtype,
                            const_attrs=Transformer.const_attrs(cfg, 128), schedule_directives=_schedule(2), device=device)
        actor.debug_keep_grads = True
        return actor

    actor = setup()
    model = Transformer(cfg, 128, 2).to(device).to(dtype)         # the add at the stage boundary included
    consts = Transformer.const_attrs(cfg, 128, device)
    model.rope_cos, model.rope_sin = consts["rope_cos"], consts["rope_sin"]
    names = [n for n, _ in model.named_parameters()]
    with torch.no_grad():
        for n, p in model.named_parameters():
            p.copy_(init_tensor(n, p.shape, dtype, torch.device(device)))
    state = ops.AdamWState(list(model.parameters()), bits=8)
    for step in range(2):
        losses = [float(v) for v in piper_exec_dag(_loss)]
        got = {k: v.float() for k, v in actor.last_grads.items()}
        want = []
        for p in model.parameters():
            p.grad = None
        for a, b in zip(x.to(device).split(2), y.to(device).split(2)):
            loss = _loss(model(a), b)
            want.append(float(loss.detach()))
            loss.backward()
        half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -20
        for a, b in zip(losses, want):
            # the first step starts from the same weights; the second from weights whose gradients differ in their last digits
            assert abs(a - b) <= (2.0 ** -20 if step == 0 else 2.0 ** -6) * abs(b), (losses, want)
        if step == 0:
            for n, p in model.named_parameters():
                # the engine keeps the mean over the microbatches; two roundings of autograd's sum, and sums in another order
                a, b = got[n], p.grad.float() / 2
                assert float((a - b).norm()) <= 3 * half * float(b.norm()) + 1e-8, n
        ops.adamw_step(list(model.parameters()), [p.grad for p in model.parameters()], state, grad_scale=0.5, **hyper)
    assert names and all(b.storage.state8 is not None for b in actor.buckets.values() if b.storage is not None and b.storage.numel)
    if device == "cuda":
        ops.native.check_status()
    # a checkpoint holds decoded moments, and a resumed run continues with the same values
    save_checkpoint(actor, str(tmp_path), step=2, schedule=_schedule(2))
    before = {k: tuple(t.clone() for t in (*b.storage.moments(), b.storage.flat_params))
              for k, b in actor.buckets.items() if b.storage is not None and b.storage.numel}
    again = setup()
    assert load_checkpoint(again, str(tmp_path)) == 2
    for k, b in again.buckets.items():
        if k in before:
            st = b.storage
            assert all(torch.equal(a, c) for a, c in zip(before[k], (*st.moments(), st.flat_params)))
            assert st.step_count == 2
    assert [float(v) for v in piper_exec_dag(_loss)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("form", ["tuple", "dict"])
def test_advantages_through_the_engine(form, device):
    """What the loss takes beside the output comes in several tensors: each microbatch has its rows of tokens and advantages, and all of a
    tensor that has another number of rows."""
    from piper_b200 import piper_exec_dag, piper_setup
    from piper_b200.models.llama3 import LlamaConfig, Transformer
    from piper_b200.nn import policy_gradient_loss
    from piper_b200.runtime.storage import init_tensor

    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    cfg = LlamaConfig(dim=256, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=512, ffn_hidden=688, norm_eps=1e-6,
                      rope_theta=10000.0, max_seq_len=128)
    g = torch.Generator().manual_seed(4)
    x, y = (torch.randint(0, cfg.vocab_size, (4, 128), generator=g) for _ in range(2))
    adv, scale = torch.randn(4, 128, generator=g), torch.tensor([0.5, 2.0, 1.0])
    y[:, :9] = -100

    def loss_fn(out, labels):
        tokens, a, s = labels.values() if isinstance(labels, dict) else labels
        assert tokens.shape == a.shape == (2, 128) and s.shape == (3,) and a.device == s.device == out.device
        return policy_gradient_loss(out, tokens, a * s[0], entropy_coef=0.01)

    def pack(t, a):
        return {"tokens": t, "advantages": a, "scale": scale} if form == "dict" else (t, a, scale)

    actor = piper_setup(Transformer, (cfg, 128, 2), optim_fn=torch.optim.AdamW, optim_kwargs={"lr": 0.0, "state_bits": 8},
                        example_inputs=[x], example_outputs=pack(y, adv), model_dtype=dtype,
                        const_attrs=Transformer.const_attrs(cfg, 128), schedule_directives=_schedule(2), device=device)
    actor.debug_keep_grads = True
    model = Transformer(cfg, 128, 2).to(device).to(dtype)
    consts = Transformer.const_attrs(cfg, 128, device)
    model.rope_cos, model.rope_sin = consts["rope_cos"], consts["rope_sin"]
    with torch.no_grad():
        for n, p in model.named_parameters():
            p.copy_(init_tensor(n, p.shape, dtype, torch.device(device)))
    for labels in (None, pack(y.flip(0), -adv)):            # those of the setup, then those of the call
        losses = [float(v) for v in piper_exec_dag(loss_fn, labels=labels)]
        want = []
        for p in model.parameters():
            p.grad = None
        t, a = (y, adv) if labels is None else (y.flip(0), -adv)
        for xs, ts, s in zip(*(v.to(device).split(2) for v in (x, t, a))):
            loss = policy_gradient_loss(model(xs), ts, s * 0.5, entropy_coef=0.01)
            want.append(float(loss.detach()))
            loss.backward()
        half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -20
        # the same ops on the same rows; losses are sums of some 250 terms of the size of a log probability, 6
        assert len(losses) == 2 and all(abs(p - q) <= 2.0 ** -20 * 6 for p, q in zip(losses, want)), (losses, want)
        for n, p in model.named_parameters():
            got = actor.last_grads[n].float()
            assert float((got - p.grad.float() / 2).norm()) <= 3 * half * float(p.grad.float().norm()) + 1e-8, n


def test_which_labels_are_cut():
    import collections

    from piper_b200.runtime.actor import DagExecutor, _map_tensors

    class Executor:
        a = type("Actor", (), {"num_microbatches": 2})
        _microbatch = DagExecutor._microbatch
        cut = DagExecutor._microbatch_labels

    pair = collections.namedtuple("pair", "tokens advantages")
    t, w, own = torch.arange(8).view(4, 2), torch.ones(6), collections.OrderedDict(tokens=torch.arange(4))
    cut = Executor().cut
    assert torch.equal(cut(t, 1), t[2:]) and cut(None, 1) is None and cut(3, 0) == 3
    got = cut((torch.tensor(5), t, {"w": w, "t": [t, "name"]}, own), 1)
    assert got[0] == 5 and torch.equal(got[1], t[2:]) and got[2]["w"] is w and torch.equal(got[2]["t"][0], t[2:])
    assert got[2]["t"][1] == "name" and got[3] is own
    got = cut(pair(t, w), 0)
    assert type(got) is pair and torch.equal(got.tokens, t[:2]) and got.advantages is w
    assert cut((), 0) == () and _map_tensors(lambda x: x + 1, own) is own
    odd = torch.arange(3)
    assert cut((odd, odd), 0)[0] is odd                    # what is not divisible comes whole, as a single tensor does


@pytest.mark.parametrize("device", DEVICES)
def test_policy_gradient_loss(device):
    from piper_b200.nn import cross_entropy_loss, policy_gradient_loss
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(2, 5, 64, generator=g).to(device).requires_grad_(True)
    tokens = torch.randint(0, 64, (2, 5), generator=g).to(device)
    tokens[0, :2] = -100
    a, b = policy_gradient_loss(logits, tokens), torch.nn.functional.cross_entropy(logits.reshape(-1, 64), tokens.reshape(-1))
    da, db = (torch.autograd.grad(v, logits)[0] for v in (a, b))
    assert abs(float(a - b)) < 2.0 ** -20 * 10 and float((da - db).abs().max()) < 2.0 ** -20
    adv = torch.randn(2, 5, generator=g).to(device)
    z = logits.detach().double() / 0.7
    logp = torch.log_softmax(z, -1)
    on = tokens != -100
    lp = logp.gather(-1, tokens.clamp(min=0).unsqueeze(-1)).squeeze(-1)
    h = -(logp.exp() * logp).sum(-1)
    want = -((adv * lp + 0.2 * h) * on).sum() / on.sum()
    got = policy_gradient_loss(logits, tokens, adv, entropy_coef=0.2, temperature=0.7)
    assert abs(float(got) - float(want)) < 2.0 ** -20 * 20
    none = torch.full_like(tokens, -100)
    assert float(policy_gradient_loss(logits, none, entropy_coef=0.5)) == 0.0


@pytest.mark.parametrize("device", DEVICES)
def test_policy_gradient_loss_of_padding(device):
    """What stands at places that do not count changes nothing: neither logits nor advantages, for either kind of such tokens."""
    from piper_b200.nn import policy_gradient_loss
    g = torch.Generator().manual_seed(2)
    clean = torch.randn(3, 6, 72, generator=g)
    tokens = torch.randint(0, 72, (3, 6), generator=g)
    adv = torch.randn(3, 6, generator=g)
    tokens[0, 4:] = -100
    tokens[2, 3:] = 72
    pad = (tokens < 0) | (tokens >= 72)
    dirty = clean.clone()
    dirty[pad] = float("nan")
    results = []
    for logits, a in ((clean, adv), (dirty, torch.where(pad, float("nan"), adv))):
        x = logits.to(device).requires_grad_(True)
        loss = policy_gradient_loss(x, tokens.to(device), a.to(device), entropy_coef=0.3)
        results.append((loss.detach().cpu(), torch.autograd.grad(loss, x)[0].cpu()))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    only = clean[~pad].double()
    logp = torch.log_softmax(only, -1)
    want = -(adv[~pad] * logp.gather(-1, tokens[~pad].unsqueeze(-1)).squeeze(-1) - 0.3 * (logp.exp() * logp).sum(-1)).mean()
    assert abs(float(results[0][0]) - float(want)) < 2.0 ** -20 * 20


@pytest.mark.parametrize("device", DEVICES)
def test_policy_gradient_loss_of_a_masked_token_without_advantage(device):
    """Its log probability is -inf, but it is asked nothing: no loss and no gradient, as if it were not there (but counted)."""
    from piper_b200.nn import policy_gradient_loss
    g = torch.Generator().manual_seed(3)
    x = torch.randn(5, 40, generator=g)
    x[1, 7] = x[4, 0] = -math.inf
    x[3] = -math.inf
    tokens = torch.tensor([2, 7, -100, 5, 1])
    adv = torch.tensor([0.5, 0.0, 1.0, 0.0, 0.0])
    x = x.to(device).requires_grad_(True)
    for coef in (0.0, 0.25):
        loss = policy_gradient_loss(x, tokens.to(device), adv.to(device), entropy_coef=coef)
        (d,) = torch.autograd.grad(loss, x)
        logp = torch.log_softmax(x.detach().double().cpu(), -1)
        entropy = -torch.where(logp > -math.inf, logp.exp() * logp, 0).sum(-1)[[0, 1, 4]].sum()
        want = -(0.5 * logp[0, 2] + coef * entropy) / 4
        assert abs(float(loss.detach()) - float(want)) < 2.0 ** -20 * 20
        assert bool(torch.isfinite(d).all()) and not bool(d[2:4].any()) and bool(d[1].any()) == (coef > 0)
    # with an advantage it is what it is
    assert float(policy_gradient_loss(x, tokens.to(device), torch.ones(5, device=device))) == math.inf


def test_eight_bit_models_of_both_families():
    import dataclasses

    from piper_b200.models.llama3 import LLAMA_CONFIGS, Transformer
    from piper_b200.models.qwen3 import QWEN3_CONFIGS, PiperQwen3Model
    from piper_b200.nn import Linear
    llama = Transformer(dataclasses.replace(LLAMA_CONFIGS["tiny"], fp8=True), 128, 1)
    qwen = PiperQwen3Model(dataclasses.replace(QWEN3_CONFIGS["9M"], fp8=True, n_layers=2), 1, 128)
    for model in (llama, qwen):
        wide = [n for n, m in model.named_modules() if isinstance(m, Linear) and not m.fp8]
        assert all(n.endswith(("output", "gate")) for n in wide), wide
        assert any(isinstance(m, Linear) and m.fp8 for m in model.modules())
    x = Linear(32, 48, fp8=True)
    torch.nn.init.normal_(x.weight)
    a = torch.randn(3, 32)
    assert torch.equal(x(a), ops.fp8_linear(a, x.weight))


def _pipeline_worker(rank, world, schedule, stages, checkpointing):
    import dataclasses

    from piper_b200 import piper_exec_dag, piper_setup
    from piper_b200.models.llama3 import LLAMA_CONFIGS, Transformer

    cfg = dataclasses.replace(LLAMA_CONFIGS["tiny"], fp8=True)
    x, y = _tokens(cfg)
    actor = piper_setup(Transformer, (cfg, 64, stages), optim_fn=torch.optim.AdamW, optim_kwargs={"state_bits": 8, "lr": 1e-3},
                        example_inputs=[x], example_outputs=y, model_dtype=torch.float32,
                        const_attrs=Transformer.const_attrs(cfg, 64), schedule_directives=schedule, device="cpu",
                        activation_checkpointing=checkpointing)
    actor.debug_keep_grads = True
    losses = [float(v) for v in piper_exec_dag(_loss)]
    grads = dict(actor.last_grads)
    again = [float(v) for v in piper_exec_dag(_loss)]
    return {"losses": losses, "again": again, "grads": grads}


def _tokens(cfg):
    g = torch.Generator().manual_seed(3)
    tok = torch.randint(0, cfg.vocab_size, (4, 65), generator=g)
    return tok[:, :-1].contiguous(), tok[:, 1:].contiguous()


@pytest.mark.parametrize("kind,checkpointing", [("zerobubble", False), ("zerobubble", True), ("1f1b", False)])
def test_pipelines_of_two_ranks(kind, checkpointing, tmp_path):
    """The split backward pass defers the 8-bit weight gradients, recomputation keeps operands of its own; both sides round each
    microbatch by itself.  One sum in another order would take an element over a border between two codes, a sixteenth of it, and
    the next layer's rounding then more of them, up to the roundings' own size after a few layers: no small tolerance follows.  So
    the plain run adds in the ranks' order (one thread, the same stages); the loss's quarter is a power of two, which the scales
    pass on exactly, and gradients are the same but for the order in which four microbatches are added: 3 roundings, 2^-24 each,
    of sums that do not cancel to less than a hundredth of their terms' norm."""
    import dataclasses

    from piper_b200.compiler.builders import build_1f1b_schedule, build_zerobubble_schedule
    from piper_b200.models.llama3 import LLAMA_CONFIGS, Transformer
    from piper_b200.runtime.storage import materialize_module
    from tests.dist_utils import run_ranks

    order = build_zerobubble_schedule(2, 4) if kind == "zerobubble" else build_1f1b_schedule(2, 4)
    schedule = [{"op": "place", "filter": {"PP": i}, "devices": [i], "stream": "pp_stream"} for i in range(2)] + \
        [{"op": "split", "filter": {}, "dim_name": "MB", "num_microbatches": 4}] + list(order)
    results = run_ranks(2, _pipeline_worker, (schedule, 2, checkpointing), tmp_path)
    cfg = dataclasses.replace(LLAMA_CONFIGS["tiny"], fp8=True)
    model = Transformer(cfg, 64, 2)
    model.load_const_attrs()
    materialize_module(model)
    x, y = _tokens(cfg)
    want = []
    threads = torch.get_num_threads()
    torch.set_num_threads(1)
    try:
        for a, b in zip(x.split(1), y.split(1)):
            loss = _loss(model(a), b)
            (loss / 4).backward()
            want.append(float(loss.detach()))
    finally:
        torch.set_num_threads(threads)
    losses = [v for r in results for v in r["losses"]]
    assert len(losses) == 4 and all(abs(a - b) < 1e-6 * abs(b) for a, b in zip(losses, want)), (losses, want)
    grads = {k: v for r in results for k, v in r["grads"].items()}
    for n, p in model.named_parameters():
        assert float((grads[n] - p.grad).norm()) <= 2e-5 * float(p.grad.norm()), n
    assert sum(v for r in results for v in r["again"]) != sum(losses)          # the step was taken


def _replica_worker(rank, world, schedule, bits, directory):
    from piper_b200 import piper_exec_dag, piper_setup
    from piper_b200.models.llama3 import LLAMA_CONFIGS, Transformer
    from piper_b200.nn import cross_entropy_loss
    from piper_b200.runtime.checkpoint import load_checkpoint, save_checkpoint

    cfg = LLAMA_CONFIGS["tiny"]
    x, y = _tokens(cfg)
    mine = slice(2 * rank, 2 * rank + 2)
    actor = piper_setup(Transformer, (cfg, 64, 1), optim_fn=torch.optim.AdamW, optim_kwargs={"state_bits": bits, "lr": 1e-3},
                        example_inputs=[x[mine]], example_outputs=y[mine], model_dtype=torch.float32,
                        const_attrs=Transformer.const_attrs(cfg, 64), schedule_directives=schedule, device="cpu")

    def params():
        return {k: v.detach().clone() for k, v in actor.named_parameters().items()}

    before = params()
    piper_exec_dag(cross_entropy_loss)
    once = params()
    save_checkpoint(actor, directory, 1)
    piper_exec_dag(cross_entropy_loss)
    twice = params()
    load_checkpoint(actor, directory)
    piper_exec_dag(cross_entropy_loss)
    return {"before": before, "once": once, "twice": twice, "again": params()}


def _replicas(flags, bits, folder):
    from tests.dist_utils import run_ranks

    schedule = [{"op": "place", "filter": {"PP": 0}, "devices": [0, 1], "stream": "pp_stream"},
                {"op": "split", "filter": {}, "dim_name": "MB", "num_microbatches": 2},
                {"op": "replicate", "filter": {"PP": 0}, "devices": [0, 1], "gather_stream": "dp_stream",
                 "reduce_stream": "dp_stream", **flags}]
    return run_ranks(2, _replica_worker, (schedule, bits, str(folder / "saved")), folder)


@pytest.mark.parametrize("flags", [{}, {"shard_grads": True}, {"shard_params": True, "shard_grads": True}])
def test_replicas_with_eight_bit_moments(flags, tmp_path):
    """Every way to shard the optimizer: ranks agree to the bit, and steps from a checkpoint repeat to the bit.  The first step uses the
    moments as they are before they are rounded, so it is that of 32 bits on the same layout (another would add gradients in another
    order, and an update has the size of lr whatever its gradient's): the same operations but for a division by a square root's
    correction in place of a product, half a dozen roundings of an update of at most lr (1 + |w| / 10)."""
    one, other = _replicas(flags, 8, tmp_path)
    for when in ("once", "twice", "again"):
        assert one[when].keys() == other[when].keys()
        for k in one[when]:
            assert torch.equal(one[when][k], other[when][k]), (when, k)
    for k, w in one["before"].items():
        assert torch.equal(one["twice"][k], one["again"][k]), k
        assert not torch.equal(one["once"][k], w) and not torch.equal(one["twice"][k], one["once"][k]), k
    if not flags:
        folder = tmp_path / "wide"
        folder.mkdir()
        wide = _replicas(flags, 32, folder)[0]
        for k, w in one["before"].items():
            off = (one["once"][k] - wide["once"][k]).abs()
            assert bool((off <= 2.0 ** -23 * w.abs() + 8 * 2.0 ** -24 * 1e-3 * 1.1).all()), (k, float(off.max()))
