"""Operators of post-training on packed batches, as cases that can be timed and checked one by one.

``kind`` selects the operator:

* ``attention``  causal grouped-query attention over sequences of different lengths that lie one behind the other in one
                 batch of tokens (``ops.pack_sequences``, ``ops.packed_attention``), alone or with its gradient
* ``policy``     clipped policy loss with a KL term over the tokens of a packed batch, averaged over tokens or first within
                 every sequence, and its gradient (``ops.clipped_policy_loss``)
* ``balance``    balance loss of a router, tokens per expert and mean probabilities, alone or with the gradient of the router's
                 logits (``ops.moe.moe_balance_loss``)

Where ``own`` is false the operators run as elementary tensor operations in 32 bits, or 64 where sums are long.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
INF = float("inf")
CLIP_LOW, CLIP_HIGH = 0.2, 0.28
KL_COEF = 0.04


def listed() -> list:
    return [
        # one microbatch of conversations at the 8B configuration's heads, forward and backward: the largest
        {"name": "attention_8b_conversations", "kind": "attention", "T": 16384, "n": 12, "skew": 1.0, "behind": 0,
         "Hq": 32, "Hkv": 8, "hd": 128, "grad": True, "lens": 1},
        # one long document among many short ones at the 30B-A3B configuration's heads, padding behind them
        {"name": "attention_30b_long_short", "kind": "attention", "T": 8192, "n": 40, "skew": 1.6, "behind": 77,
         "Hq": 32, "Hkv": 4, "hd": 128, "grad": True, "lens": 4},
        # scoring packed replies with the 1B configuration's heads, forward only
        {"name": "attention_1b_score", "kind": "attention", "T": 6001, "n": 9, "skew": 0.7, "behind": 0,
         "Hq": 32, "Hkv": 8, "hd": 64, "grad": False, "lens": 3},
        # a few short sequences with the tiny configuration's heads: latency
        {"name": "attention_tiny", "kind": "attention", "T": 333, "n": 5, "skew": 0.8, "behind": 3,
         "Hq": 4, "Hkv": 4, "hd": 64, "grad": True, "lens": 5},
        # the update of a packed batch of replies: averaged within every reply first, with a reference model
        {"name": "policy_packed", "kind": "policy", "T": 65536, "n": 48, "skew": 0.8, "behind": 1000, "kl": True,
         "by_sequence": True, "lens": 6},
        # one microbatch of 4096 tokens, averaged over tokens, without a reference model
        {"name": "policy_tokens", "kind": "policy", "T": 4096, "n": 1, "skew": 0.0, "behind": 0, "kl": False,
         "by_sequence": False, "lens": 7},
        # one reply: latency
        {"name": "policy_one_reply", "kind": "policy", "T": 193, "n": 1, "skew": 0.0, "behind": 0, "kl": True,
         "by_sequence": True, "lens": 8},
        # a whole rollout at once, averaged over tokens
        {"name": "policy_rollout", "kind": "policy", "T": 500000, "n": 1, "skew": 0.0, "behind": 0, "kl": True,
         "by_sequence": False, "lens": 9},
        # router of the 30B-A3B configuration on a packed batch, with its gradient
        {"name": "balance_30b", "kind": "balance", "T": 16384, "E": 128, "k": 8, "dtype": "bf16", "masked": True, "grad": True},
        # router of the 9M configuration on one short sequence: latency
        {"name": "balance_9m", "kind": "balance", "T": 128, "E": 8, "k": 2, "dtype": "bf16", "masked": False, "grad": True},
        # a whole rollout at once, the router of the 9B configuration
        {"name": "balance_rollout", "kind": "balance", "T": 131072, "E": 64, "k": 8, "dtype": "bf16", "masked": False,
         "grad": True},
        # logits kept in fp32, an odd number of experts, a ragged batch
        {"name": "balance_odd", "kind": "balance", "T": 3001, "E": 60, "k": 4, "dtype": "fp32", "masked": True, "grad": True},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["attention", "attention", "policy", "balance"])
    lens = rng.randrange(1 << 30)
    if kind == "attention":
        Hq, Hkv, hd = rng.choice([(32, 8, 128), (32, 4, 128), (32, 8, 64), (4, 4, 64), (16, 4, 128), (4, 2, 64), (24, 8, 128),
                                  (64, 8, 128)])
        T = _log_int(rng, 1, 16384 * 32 // max(Hq, 32))
        n = _log_int(rng, 1, max(1, min(256, T)))
        # a drawn batch costs no more than the largest listed one, which has sequences of up to some 5000 tokens
        while (work_of_lengths(_lengths({"T": T, "n": n, "skew": 1.0, "behind": 0, "lens": lens})) * Hq * hd
               > work_of_lengths(_lengths(listed()[0])) * 32 * 128):
            T = T * 3 // 4
        return {"kind": kind, "T": T, "n": n, "skew": 1.0, "behind": rng.choice([0, 0, min(T, 5), min(T // 3, 200)]), "Hq": Hq,
                "Hkv": Hkv, "hd": hd, "grad": rng.random() < 0.7, "lens": lens}
    if kind == "policy":
        T = _log_int(rng, 1, 500000)
        return {"kind": kind, "T": T, "n": _log_int(rng, 1, max(1, min(512, T))), "skew": rng.choice([0.0, 0.8, 1.4]),
                "behind": rng.choice([0, 0, T // 10]), "kl": rng.random() < 0.6, "by_sequence": rng.random() < 0.6, "lens": lens}
    E = rng.choice([8, 32, 64, 128, 128, rng.randint(2, 256)])
    return {"kind": kind, "T": _log_int(rng, 1, 131072 * 64 // max(E, 64)), "E": E, "k": rng.randint(1, min(8, E)),
            "dtype": rng.choice(["bf16", "bf16", "fp32"]), "masked": rng.random() < 0.5, "grad": rng.random() < 0.7}


# ------------------------------------------------------------------ inputs
def _lengths(c: dict) -> list:
    """Lengths of the sequences of a packed batch, of spread exp(skew); some may be 0, ``behind`` tokens lie behind the last."""
    rng = random.Random(c["lens"])
    share = [math.exp(c["skew"] * rng.gauss(0, 1)) for _ in range(c["n"])]
    total, left = c["T"] - c["behind"], sum(share)
    out = [int(total * s / left) for s in share]
    out[share.index(max(share))] += total - sum(out)
    return out


def work_of_lengths(lens: list) -> int:
    """Pairs of a query and a key that it sees."""
    return sum(n * (n + 1) // 2 for n in lens)


def _starts(lens: list) -> list:
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _inputs(c: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rn(*shape, std=1.0, dtype=F32):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=F32) * std).to(dtype)

    def ru(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    T = c["T"]
    if c["kind"] == "attention":
        Hq, Hkv, hd = c["Hq"], c["Hkv"], c["hd"]
        qkv = rn(T, Hq + 2 * Hkv, hd)
        qkv[:, :Hq] *= 1.0 + 2.0 * ru(Hq, 1)                 # heads that look at much and at little
        qkv[:, Hq:Hq + Hkv] += rn(Hkv, hd, std=0.5)
        t = {"qkv": qkv.view(T, -1).to(BF16)}
        if c["grad"]:
            t["dout"] = rn(T, Hq * hd, std=1e-2, dtype=BF16)
        return t
    if c["kind"] == "policy":
        old = -torch.exp(rn(T, std=1.5) - 1.0)
        new = old + rn(T, std=0.15)
        far = ru(T) < 0.01
        new = torch.where(far, new + rn(T, std=1.5), new).clamp(max=-1e-6)
        adv, ref = rn(T), old + rn(T, std=0.3)
        mask = ru(T) < 0.7                                   # replies; prompts and padding are left out
        bad = ~mask & (ru(T) < 0.2)
        new, ref = torch.where(bad, -INF, new), torch.where(bad, float("nan"), ref)
        return {"new": new, "old": old, "adv": adv, "ref": ref if c["kl"] else None, "mask": mask,
                "dloss": torch.tensor(0.125, device="cuda")}
    E = c["E"]
    x = (rn(T, E, std=1.5) + rn(E, std=0.7)).to(BF16 if c["dtype"] == "bf16" else F32)
    idx = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :c["k"]].to(torch.int32).contiguous()
    return {"x": x, "idx": idx, "mask": ru(T) < 0.9 if c["masked"] else None, "dloss": torch.tensor(0.01, device="cuda")}


def prepare(case: dict, seed: int) -> dict:
    c = case
    s = {"case": c, **_inputs(c, seed)}
    if c["kind"] == "attention":
        s["qkv"].requires_grad_(c["grad"])
        s["lens"] = _lengths(c)
    elif c["kind"] == "policy":
        s["new"].requires_grad_(True)
        if c["by_sequence"]:
            s["lens"] = _lengths(c)
    else:
        s["x"].requires_grad_(c["grad"])
    if own and "lens" in s:
        from piper_b200 import ops
        s["sequences"] = ops.pack_sequences(torch.tensor(_starts(s["lens"])), c["T"], device="cuda")
    return s


# ------------------------------------------------------------------ plain forms, in 32 bits
def _plain_attention(s: dict):
    c = s["case"]
    T, Hq, Hkv, hd = c["T"], c["Hq"], c["Hkv"], c["hd"]
    G, scale = Hq // Hkv, hd ** -0.5
    x = s["qkv"].detach().float().view(T, Hq + 2 * Hkv, hd)
    out = torch.zeros(T, Hq, hd, device=x.device)
    if c["grad"]:
        do, dx = s["dout"].float().view(T, Hq, hd), torch.zeros_like(x)
    at = 0
    for n in s["lens"]:
        if n == 0:
            continue
        r = slice(at, at + n)
        at += n
        later = torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1)
        for h in range(Hkv):                                 # one group of query heads at a time
            q = x[r, h * G:(h + 1) * G].transpose(0, 1)
            k, v = x[r, Hq + h], x[r, Hq + Hkv + h]
            p = torch.matmul(q, k.t()) * scale
            p.masked_fill_(later, -INF)
            p = torch.exp(p - p.amax(2, keepdim=True))
            p = p / p.sum(2, keepdim=True)
            o = torch.matmul(p, v)
            out[r, h * G:(h + 1) * G] = o.transpose(0, 1)
            if c["grad"]:
                d = do[r, h * G:(h + 1) * G].transpose(0, 1)
                dx[r, Hq + Hkv + h] = torch.matmul(p.transpose(1, 2), d).sum(0)
                ds = p * (torch.matmul(d, v.t()) - (d * o).sum(2, keepdim=True))
                dx[r, h * G:(h + 1) * G] = torch.matmul(ds, k).transpose(0, 1) * scale
                dx[r, Hq + h] = torch.matmul(ds.transpose(1, 2), q).sum(0) * scale
    res = {"out": out.view(T, -1).to(BF16)}
    if c["grad"]:
        res["dqkv"] = dx.view(T, -1).to(BF16)
    return res


def _plain_policy(s: dict):
    c = s["case"]
    T, dev = c["T"], s["old"].device
    zero = torch.zeros((), dtype=F64, device=dev)
    on = s["mask"]
    if c["by_sequence"]:
        lens = torch.tensor(s["lens"], device=dev)
        of = torch.repeat_interleave(torch.arange(len(s["lens"]), device=dev), lens)
        of = torch.cat((of, torch.full((T - of.numel(),), len(s["lens"]), device=dev)))
        on = on & (of < len(s["lens"]))
        counts = torch.zeros(len(s["lens"]) + 1, dtype=F64, device=dev).index_add_(0, of, on.double())
        weight = 1.0 / (counts.clamp(min=1)[of] * (counts > 0).sum().clamp(min=1))
    else:
        weight = (1.0 / on.sum().clamp(min=1).double()).expand(T)
    weight = torch.where(on, weight, zero)
    diff = torch.where(on, s["new"].detach().double() - s["old"].double(), zero)
    ratio = torch.exp(diff)
    adv = torch.where(on, s["adv"].double(), zero)
    kept = -adv * ratio
    cut = -adv * ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
    loss, clipped = torch.maximum(kept, cut), (cut > kept) & on
    grad = torch.where(clipped, zero, kept)
    kl = torch.zeros(T, dtype=F64, device=dev)
    if c["kl"]:
        d = torch.where(on, s["ref"].double() - s["new"].detach().double(), zero)
        kl = torch.expm1(d) - d
        loss = loss + KL_COEF * kl
        grad = grad - KL_COEF * torch.expm1(d)
    n = on.sum().clamp(min=1)
    return {"loss": (weight * loss).sum().float(), "kl": (weight * kl).sum().float(),
            "clipped": (clipped.sum() / n.double()).float(), "dnew": (grad * weight * s["dloss"].double()).float()}


def _plain_balance(s: dict):
    c = s["case"]
    T, E, k = c["T"], c["E"], c["k"]
    x = s["x"].detach().float()
    on = torch.ones(T, dtype=torch.bool, device=x.device) if s["mask"] is None else s["mask"]
    e = torch.exp(x - x.amax(1, keepdim=True))
    p = e / e.sum(1, keepdim=True)
    n = on.sum().clamp(min=1).double()
    prob = torch.where(on.unsqueeze(1), p, torch.zeros_like(p)).sum(0, dtype=F64) / n
    counts = torch.zeros(E + 1, dtype=torch.int64, device=x.device)
    chosen = torch.where(on.unsqueeze(1), s["idx"].long(), E).reshape(-1)
    counts = counts.index_add_(0, chosen, torch.ones_like(chosen))[:E]
    f = counts.double() * (E / (n * k))
    out = {"loss": (f * prob).sum().float(), "counts": counts.to(torch.int32), "prob": prob.float()}
    if c["grad"]:
        f32 = (f * (s["dloss"].double() / n)).float()
        dx = p * (f32 - torch.matmul(p, f32).unsqueeze(1))
        out["dx"] = torch.where(on.unsqueeze(1), dx, torch.zeros_like(dx)).to(s["x"].dtype)
    return out


def run(s: dict):
    c = s["case"]
    kind = c["kind"]
    if not own:
        return {"attention": _plain_attention, "policy": _plain_policy, "balance": _plain_balance}[kind](s)
    from piper_b200 import ops
    if kind == "attention":
        out = ops.packed_attention(s["qkv"], s["sequences"], c["Hq"], c["Hkv"], c["hd"], c["hd"] ** -0.5)
        if not c["grad"]:
            return {"out": out}
        (d,) = torch.autograd.grad(out, s["qkv"], s["dout"])
        return {"out": out.detach(), "dqkv": d}
    if kind == "policy":
        r = ops.clipped_policy_loss(s["new"], s["old"], s["adv"], ref_logprob=s["ref"], mask=s["mask"],
                                    sequences=s.get("sequences"), clip=(CLIP_LOW, CLIP_HIGH), kl_coef=KL_COEF if c["kl"] else 0.0)
        (d,) = torch.autograd.grad(r.loss, s["new"], s["dloss"])
        return {"loss": r.loss.detach(), "kl": r.kl, "clipped": r.clipped, "dnew": d}
    r = ops.moe.moe_balance_loss(s["x"], s["idx"], mask=s["mask"])
    out = {"loss": r.loss.detach(), "counts": r.counts, "prob": r.prob}
    if c["grad"]:
        (out["dx"],) = torch.autograd.grad(r.loss, s["x"], s["dloss"])
    return out


# ------------------------------------------------------------------ the definition, in 64 bits
def _exact_attention(c: dict, t: dict):
    T, Hq, Hkv, hd = c["T"], c["Hq"], c["Hkv"], c["hd"]
    x = t["qkv"].double().view(T, Hq + 2 * Hkv, hd)
    out = torch.zeros(T, Hq, hd, dtype=F64, device=x.device)
    dx = torch.zeros_like(x) if c["grad"] else None
    starts = _starts(_lengths(c))
    rows = 2048                                              # queries at a time
    for a, b in zip(starts, starts[1:]):
        for h in range(Hq):
            kv = Hq + h // (Hq // Hkv)
            for i in range(a, b, rows):
                j = min(b, i + rows)
                q, k, v = x[i:j, h], x[a:j, kv], x[a:j, kv + Hkv]
                z = torch.einsum("qd,kd->qk", q, k) / math.sqrt(hd)
                seen = torch.arange(a, j, device=x.device).unsqueeze(0) <= torch.arange(i, j, device=x.device).unsqueeze(1)
                p = torch.softmax(torch.where(seen, z, -INF), 1)
                out[i:j, h] = p @ v
                if c["grad"]:
                    d = t["dout"][i:j].double().view(j - i, Hq, hd)[:, h]
                    dp = d @ v.t()
                    dz = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(hd)
                    dx[i:j, h] = dz @ k
                    dx[a:j, kv] += dz.t() @ q
                    dx[a:j, kv + Hkv] += p.t() @ d
    res = {"out": out.view(T, -1).float()}
    if c["grad"]:
        res["dqkv"] = dx.view(T, -1).float()
    return res


def _exact_policy(c: dict, t: dict):
    T = c["T"]
    on = t["mask"].clone()
    w = torch.zeros(T, dtype=F64, device="cuda")
    if c["by_sequence"]:
        starts = _starts(_lengths(c))
        on[starts[-1]:] = False
        parts = [(a, b, int(on[a:b].sum())) for a, b in zip(starts, starts[1:])]
        some = sum(m > 0 for _a, _b, m in parts)
        for a, b, m in parts:
            if m:
                w[a:b] = 1.0 / m / some
    else:
        w[:] = 1.0 / max(1, int(on.sum()))
    at = on.nonzero().squeeze(1)
    w = w[at]
    lp, adv = t["new"][at].double(), t["adv"][at].double()
    r = torch.exp(lp - t["old"][at].double())
    outside = torch.where(adv > 0, r > 1 + CLIP_HIGH, r < 1 - CLIP_LOW) & (adv != 0)
    lim = torch.where(adv > 0, 1 + CLIP_HIGH, 1 - CLIP_LOW).to(F64)
    each = -adv * torch.where(outside, lim, r)
    g = torch.where(outside, 0.0, -adv * r)
    kl = torch.zeros_like(each)
    if c["kl"]:
        u = t["ref"][at].double() - lp
        # e^u - 1 - u; its series where the terms cancel
        series = u * u * (0.5 + u * (1 / 6 + u * (1 / 24 + u * (1 / 120 + u / 720))))
        kl = torch.where(u.abs() < 1e-2, series, torch.exp(u) - 1 - u)
        each = each + KL_COEF * kl
        g = g + KL_COEF * (1 - torch.exp(u))
    dnew = torch.zeros(T, dtype=F64, device="cuda")
    dnew[at] = g * w * float(t["dloss"])
    return {"loss": (each * w).sum(), "kl": (kl * w).sum(), "clipped": outside.double().sum() / max(1, at.numel()),
            "dnew": dnew}


def _exact_balance(c: dict, t: dict):
    T, E, k = c["T"], c["E"], c["k"]
    at = torch.arange(T, device="cuda") if t["mask"] is None else t["mask"].nonzero().squeeze(1)
    p = torch.softmax(t["x"][at].double(), 1)
    n = max(1, at.numel())
    counts = torch.bincount(t["idx"][at].reshape(-1).long(), minlength=E)
    f, mean = counts.double() / (n * k), p.sum(0) / n
    out = {"loss": E * (f * mean).sum(), "counts": counts.to(torch.int32), "prob": mean}
    if c["grad"]:
        up = (E * float(t["dloss"]) / n * f).expand_as(p)    # gradient with respect to p
        dx = torch.zeros(T, E, dtype=F64, device="cuda")
        dx[at] = p * up - p * (p * up).sum(1, keepdim=True)
        out["dx"] = dx
    return out


def exact(case: dict, seed: int):
    t = _inputs(case, seed)
    return {"attention": _exact_attention, "policy": _exact_policy, "balance": _exact_balance}[case["kind"]](case, t)


def work(case: dict) -> dict:
    c = case
    T = c["T"]
    if c["kind"] == "attention":
        pairs = work_of_lengths(_lengths(c)) * c["Hq"]
        qkv, out = 2 * T * (c["Hq"] + 2 * c["Hkv"]) * c["hd"], 2 * T * c["Hq"] * c["hd"]
        # two products forward; five backward, one of them the scores again
        if c["grad"]:
            return {"bytes": 2 * qkv + 2 * out, "flops": 14 * pairs * c["hd"]}
        return {"bytes": qkv + out, "flops": 4 * pairs * c["hd"]}
    if c["kind"] == "policy":
        return {"bytes": T * (4 * 3 + 1 + (4 if c["kl"] else 0) + 4), "flops": T * (30 if c["kl"] else 15)}
    n, e = T * c["E"], 2 if c["dtype"] == "bf16" else 4
    small = 4 * T * c["k"] + 8 * c["E"] + (T if c["masked"] else 0)
    return {"bytes": n * e * (2 if c["grad"] else 1) + small, "flops": n * (12 if c["grad"] else 6)}
