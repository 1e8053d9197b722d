"""Operators of a fine-tuning step on few GPUs, as cases that can be timed and checked one by one.

``kind`` selects the operator:

* ``logprobs``  log probabilities of given tokens with the entropy and the most probable alternatives of their rows
                (``ops.token_logprobs``), with or without the gradient
* ``adamw``     one AdamW step over a list of tensors, moments held in 8 or in 32 bits (``ops.adamw_step``)
* ``fp8``       linear layer whose operands are rounded to e4m3 with a power-of-two scale for every 128 elements of the
                contraction (``ops.fp8_linear``), with its backward pass or with weights that were rounded before

Where ``own`` is false the operators run as elementary tensor operations in 32 bits.
"""
from __future__ import annotations

import math

import torch

own = False

BF16, F32 = torch.bfloat16, torch.float32
INF = float("inf")
GROUP = 128            # elements of a contraction that share a scale
BLOCK = 256            # elements of a tensor whose 8-bit moments share a scale
HYPER = {"lr": 3e-4, "betas": (0.9, 0.95), "eps": 1e-8, "weight_decay": 0.1}


def listed() -> list:
    return [
        # scoring sequences for a sampler's reply: the token's log probability and 20 alternatives, Llama vocabulary
        {"name": "logprobs_score_top20", "kind": "logprobs", "T": 1024, "V": 128256, "dtype": "bf16", "top": 20,
         "temperature": 1.0, "grad": False},
        # one microbatch of a policy update with an entropy bonus: forward and the gradient of all logits, the largest
        {"name": "logprobs_policy_train", "kind": "logprobs", "T": 4096, "V": 128256, "dtype": "bf16", "top": 0,
         "temperature": 1.0, "grad": True},
        # the last position of one sequence: a single row, latency
        {"name": "logprobs_one_row", "kind": "logprobs", "T": 1, "V": 128256, "dtype": "bf16", "top": 5,
         "temperature": 0.8, "grad": False},
        # upcast logits of an odd vocabulary, a ragged batch, alternatives that are trained too (distillation)
        {"name": "logprobs_odd_train", "kind": "logprobs", "T": 333, "V": 32003, "dtype": "fp32", "top": 3,
         "temperature": 0.7, "grad": True},
        # the update of one layer of the 8B configuration: fp32 gradient buckets, 8-bit moments, bf16 weights
        {"name": "adamw8_8b_layer", "kind": "adamw", "set": "layer", "dim": 4096, "qkv": 6144, "hidden": 14336, "layers": 1,
         "vocab": 0, "count": 0, "largest": 0, "bits": 8, "grads": "fp32", "params": "bf16"},
        # one layer of the 1B configuration with moments in 32 bits and bf16 gradients of plain autograd
        {"name": "adamw32_1b_layer", "kind": "adamw", "set": "layer", "dim": 2048, "qkv": 3584, "hidden": 8192, "layers": 1,
         "vocab": 0, "count": 0, "largest": 0, "bits": 32, "grads": "bf16", "params": "bf16"},
        # every tensor of the tiny configuration at once: latency and launches
        {"name": "adamw8_tiny_model", "kind": "adamw", "set": "layer", "dim": 256, "qkv": 768, "hidden": 688, "layers": 4,
         "vocab": 1024, "count": 0, "largest": 0, "bits": 8, "grads": "fp32", "params": "bf16"},
        # adapters, norms and odd matrices kept in fp32: many ragged tensors
        {"name": "adamw8_ragged", "kind": "adamw", "set": "ragged", "dim": 0, "qkv": 0, "hidden": 0, "layers": 0, "vocab": 0,
         "count": 56, "largest": 400001, "bits": 8, "grads": "bf16", "params": "fp32"},
        # gate and up projection of the 8B configuration on one microbatch: the largest product, with both gradients
        {"name": "fp8_8b_up_train", "kind": "fp8", "T": 4096, "K": 4096, "N": 28672, "mode": "train"},
        # down projection of the 1B configuration on a ragged number of tokens
        {"name": "fp8_1b_down_ragged", "kind": "fp8", "T": 1000, "K": 8192, "N": 2048, "mode": "train"},
        # gate and up projection of the tiny configuration: latency and launches
        {"name": "fp8_tiny_train", "kind": "fp8", "T": 512, "K": 256, "N": 1376, "mode": "train"},
        # scoring a few tokens with the 8B qkv projection, weights rounded once before
        {"name": "fp8_few_tokens", "kind": "fp8", "T": 24, "K": 4096, "N": 6144, "mode": "kept"},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["logprobs", "adamw", "fp8"])
    if kind == "logprobs":
        V = rng.choice([128256, 32000, 1024, 2048, _log_int(rng, 100, 128256), _log_int(rng, 1000, 40000)])
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        most = (4096 if dtype == "bf16" else 2048) * 128256 // V
        return {"kind": kind, "T": _log_int(rng, 1, min(8192, most)), "V": V, "dtype": dtype,
                "top": min(V, rng.choice([0, 0, 1, 5, 20, 32])), "temperature": rng.choice([1.0, 1.0, 0.6, 1.3]),
                "grad": rng.random() < 0.6}
    if kind == "adamw":
        bits, grads = rng.choice([8, 8, 32]), rng.choice(["fp32", "bf16"])
        params = rng.choice(["bf16", "bf16", "fp32"])
        c = {"kind": kind, "set": "layer", "dim": 0, "qkv": 0, "hidden": 0, "layers": 0, "vocab": 0, "count": 0,
             "largest": 0, "bits": bits, "grads": grads, "params": params}
        if rng.random() < 0.5:
            dim = rng.choice([256, 1024, 2048, 2560])
            return {**c, "dim": dim, "qkv": dim + 2 * 64 * rng.choice([2, 4, 8]), "hidden": 16 * _log_int(rng, 20, 512),
                    "layers": rng.choice([1, 1, 2]), "vocab": rng.choice([0, 0, 1024, 2048])}
        return {**c, "set": "ragged", "count": _log_int(rng, 1, 58), "largest": _log_int(rng, 50, 2000000)}
    T = _log_int(rng, 1, 4096)
    dim = rng.choice([256, 1024, 2048, 4096, 16 * _log_int(rng, 5, 160)])
    wide = rng.choice([1376, 1536, 6144, 8192, 14336, 16 * _log_int(rng, 5, 800)])
    K, N = (dim, wide) if rng.random() < 0.5 else (wide, dim)
    return {"kind": kind, "T": T, "K": K, "N": N, "mode": rng.choice(["train", "train", "kept"])}


# ------------------------------------------------------------------ inputs
def _shapes(c: dict) -> list:
    """The tensors of an update, in order."""
    if c["set"] == "layer":
        d, out = c["dim"], []
        if c["vocab"]:
            out.append((c["vocab"], d))
        for _ in range(c["layers"]):
            out += [(d,), (c["qkv"], d), (d, d), (d,), (2 * c["hidden"], d), (d, c["hidden"])]
        if c["vocab"]:
            out += [(d,), (c["vocab"], d)]
        return out
    # sizes spread over the logarithm, the largest first
    n, top = c["count"], c["largest"]
    return [(max(1, int(top ** (1.0 - 0.97 * i / max(1, n - 1)))),) if i % 2 else
            (max(1, int(top ** (1.0 - 0.97 * i / max(1, n - 1)))) // 7 + 1, 7) for i in range(n)]


def _offsets(shapes: list) -> tuple[list, int]:
    """Where each tensor's moments start, in whole blocks, and the length of all of them."""
    out, at = [], 0
    for s in shapes:
        out.append(at)
        at += (math.prod(s) + BLOCK - 1) // BLOCK * BLOCK
    return out, at


def _inputs(c: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rn(*shape, std=1.0, dtype=BF16):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=F32) * std).to(dtype)

    if c["kind"] == "logprobs":
        T, V, dtype = c["T"], c["V"], BF16 if c["dtype"] == "bf16" else F32
        x = rn(T, V, std=2.0, dtype=dtype)
        hot = torch.randint(0, V, (T, 8), generator=g, device="cuda")
        x.scatter_(1, hot, (torch.rand(T, 8, generator=g, device="cuda") * 8 + 6).to(dtype))
        if V > 1000:
            x[:, V - V // 100:] = -INF                      # ids that no token has
        tokens = hot[:, 0].clone()
        tokens[torch.rand(T, generator=g, device="cuda") < 0.05] = -100
        t = {"x": x, "tokens": tokens}
        if c["grad"]:
            t["dlp"], t["dH"] = rn(T, dtype=F32), rn(T, std=0.01, dtype=F32)
            t["dtop"] = rn(T, c["top"], std=0.1, dtype=F32)
        return t
    if c["kind"] == "adamw":
        shapes = _shapes(c)
        offsets, total = _offsets(shapes)
        t = {"p": [], "g": [], "step": 100}
        for s in shapes:
            scale = 10.0 ** float(torch.rand((), generator=g, device="cuda") * 2 - 4)
            t["p"].append(rn(*s, std=0.02, dtype=F32))
            t["g"].append(rn(*s, std=scale, dtype=F32 if c["grads"] == "fp32" else BF16))
        if c["bits"] == 8:
            t["m"] = torch.randint(0, 256, (total,), generator=g, device="cuda", dtype=torch.uint8)
            t["v"] = torch.randint(140, 256, (total,), generator=g, device="cuda", dtype=torch.uint8)
            t["ms"] = 10.0 ** (torch.rand(total // BLOCK, generator=g, device="cuda") * 2 - 4)
            t["vs"] = (t["ms"] * (1 + torch.rand(total // BLOCK, generator=g, device="cuda"))) ** 2
        else:
            t["m"] = rn(total, std=1e-3, dtype=F32)
            t["v"] = rn(total, std=2e-3, dtype=F32).square()
        return t
    T, K, N = c["T"], c["K"], c["N"]
    x = rn(T, K)
    x[:, torch.randint(0, K, (3,), generator=g, device="cuda")] *= 30      # channels that stand out
    t = {"x": x, "w": rn(N, K, std=K ** -0.5)}
    if c["mode"] == "train":
        t["dy"] = rn(T, N, std=1e-4)
    return t


def prepare(case: dict, seed: int) -> dict:
    c, t = case, _inputs(case, seed)
    s = {"case": c, **t}
    if c["kind"] == "logprobs":
        s["x"].requires_grad_(c["grad"])
    elif c["kind"] == "adamw":
        masters = s.pop("p")
        s["params"] = [p.to(BF16) for p in masters] if c["params"] == "bf16" else [p.clone() for p in masters]
        shapes = [tuple(p.shape) for p in masters]
        offsets, total = _offsets(shapes)
        if own:
            from piper_b200 import ops
            state = ops.AdamWState(s["params"], bits=c["bits"])
            state.set_step(s.pop("step"))
            state.m.copy_(s.pop("m"))
            state.v.copy_(s.pop("v"))
            if c["bits"] == 8:
                state.m_scale.copy_(s.pop("ms"))
                state.v_scale.copy_(s.pop("vs"))
            if c["params"] == "bf16":
                for o, p in zip(offsets, masters):
                    state.master[o:o + p.numel()].copy_(p.reshape(-1))
            s["state"] = state
        else:
            if c["params"] == "bf16":
                s["master"] = torch.zeros(total, dtype=F32, device="cuda")
                for o, p in zip(offsets, masters):
                    s["master"][o:o + p.numel()].copy_(p.reshape(-1))
            s["offsets"] = offsets
            live = torch.zeros(total, dtype=torch.bool, device="cuda")
            for o, p in zip(offsets, masters):
                live[o:o + p.numel()] = True
            s["live"] = live
    elif c["mode"] == "train":
        s["x"].requires_grad_(True)
        s["w"].requires_grad_(True)
    elif own:
        from piper_b200 import ops
        s["w"] = ops.fp8_quantize(s["w"], square=True)
    else:
        s["w"] = _fp8_values(s["w"].float(), True)
    return s


# ------------------------------------------------------------------ plain forms, in 32 bits
def _plain_logprobs(s: dict):
    c = s["case"]
    T, V, k = c["T"], c["V"], c["top"]
    tokens = s["tokens"]
    x = s["x"].detach().float()
    z = x / c["temperature"]
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    logp = z - top - torch.log(total)
    p = e / total
    plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
    entropy = -plogp.sum(1)
    counted = (tokens >= 0) & (tokens < V)
    at = tokens.clamp(0, V - 1).unsqueeze(1)
    lp = torch.where(counted, logp.gather(1, at).squeeze(1), torch.zeros((), device=x.device))
    ids = torch.empty(T, k, dtype=torch.int64, device=x.device)
    left = x
    for i in range(k):
        ids[:, i] = left.argmax(1)                       # the first of equal ones
        left = left.scatter(1, ids[:, i:i + 1], -INF)
    out = {"logprob": lp, "entropy": entropy, "top_logprob": logp.gather(1, ids), "top_id": ids}
    if c["grad"]:
        dlp = torch.where(counted, s["dlp"], torch.zeros_like(s["dlp"])).unsqueeze(1)
        dx = -p * (dlp + s["dtop"].sum(1, keepdim=True))
        dx.scatter_add_(1, at, dlp)
        dx.scatter_add_(1, ids, s["dtop"])
        dx -= s["dH"].unsqueeze(1) * (plogp + p * entropy.unsqueeze(1))
        out["dx"] = (dx / c["temperature"]).to(s["x"].dtype)
    return out


def _mix32(h: torch.Tensor) -> torch.Tensor:
    """32-bit integers, held in 64, to 32 bits that look random."""
    for shift, factor in ((16, 0x7FEB352D), (15, 0x846CA68B)):
        h = h ^ (h >> shift)
        h = (h * factor) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _random16(step: int, ordinal: int, n: int, device) -> tuple:
    seed = int(_mix32(torch.tensor((step * 0x9E3779B1 + ordinal * 0x85EBCA77) & 0xFFFFFFFF)))
    h = _mix32((torch.arange(n, device=device) + seed) & 0xFFFFFFFF)
    return h & 0xFFFF, h >> 16


def _decode(codes: torch.Tensor, scale: torch.Tensor, signed: bool) -> torch.Tensor:
    """The values of whole blocks: codes are the upper bits of a 32-bit number in [0, 1]."""
    c = codes.to(torch.int32)
    low = (c & 127) if signed else c
    x = torch.where(low > 0, (low + (889 if signed else 761)) << 20, torch.zeros_like(low)).view(F32)
    x = (x.view(-1, BLOCK) * scale.unsqueeze(1)).view(-1)
    return torch.where(c >= 128, -x, x) if signed else x


def _encode(x: torch.Tensor, r: torch.Tensor, signed: bool) -> tuple:
    """Codes and scales of whole blocks; r: 16 random bits for each element."""
    scale = x.view(-1, BLOCK).abs().amax(1)
    y = (x.abs().view(-1, BLOCK) / torch.where(scale > 0, scale, torch.ones_like(scale)).unsqueeze(1)).view(-1)
    base = 889 if signed else 761
    least = float(torch.tensor((base + 1) << 20, dtype=torch.int32).view(F32))
    codes = ((y.view(torch.int32) + (r << 4).to(torch.int32)) >> 20) - base
    small = (r.to(F32) * (least / 65536) < y) if signed else y > 0
    codes = torch.where(y < least, small.to(torch.int32), codes)
    if signed:
        codes = codes + 128 * (x < 0)
    return codes.to(torch.uint8), scale


def _plain_adamw(s: dict):
    c = s["case"]
    b1, b2 = HYPER["betas"]
    lr, eps, wd = HYPER["lr"], HYPER["eps"], HYPER["weight_decay"]
    s["step"] += 1
    step = s["step"]
    rate, root = lr / (1 - b1 ** step), 1 / math.sqrt(1 - b2 ** step)
    total = s["m"].numel()
    m_all, v_all = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
    for i, (p, g) in enumerate(zip(s["params"], s["g"])):
        n, o = p.numel(), s["offsets"][i]
        whole = (n + BLOCK - 1) // BLOCK * BLOCK
        part, blocks = slice(o, o + whole), slice(o // BLOCK, (o + whole) // BLOCK)
        live = s["live"][part]
        gf = torch.zeros(whole, device="cuda")
        gf[:n] = g.reshape(-1)
        if c["bits"] == 8:
            m = _decode(s["m"][part], s["ms"][blocks], True)
            v = _decode(s["v"][part], s["vs"][blocks], False)
        else:
            m, v = s["m"][part], s["v"][part]
        m = m * b1 + gf * (1 - b1)
        v = v * b2 + gf * (1 - b2) * gf
        m, v = torch.where(live, m, torch.zeros_like(m)), torch.where(live, v, torch.zeros_like(v))
        w = s["master"][o:o + n] if c["params"] == "bf16" else p.view(-1)
        upd = m[:n] / (torch.sqrt(v[:n]) * root + eps)
        w.copy_(w * (1 - lr * wd) - upd * rate)
        if c["params"] == "bf16":
            p.view(-1).copy_(w)
        if c["bits"] == 8:
            rm, rv = _random16(step, i, whole, "cuda")
            s["m"][part], s["ms"][blocks] = _encode(m, rm, True)
            s["v"][part], s["vs"][blocks] = _encode(v, rv, False)
            m_all[part] = _decode(s["m"][part], s["ms"][blocks], True)
            v_all[part] = _decode(s["v"][part], s["vs"][blocks], False)
        else:
            s["m"][part], s["v"][part] = m, v
            m_all[part], v_all[part] = m, v
    out = {"params": s["params"], "m": m_all, "v": v_all}
    if c["params"] == "bf16":
        out["master"] = s["master"]
    return out


def _fp8_values(x: torch.Tensor, square: bool) -> torch.Tensor:
    """x as e4m3 with a power-of-two scale for every 128 elements of a row, or for every 128 x 128."""
    rows, cols = x.shape
    h, w = GROUP if square else 1, GROUP
    pad = torch.zeros((rows + h - 1) // h * h, (cols + w - 1) // w * w, device=x.device)
    pad[:rows, :cols] = x
    tiles = pad.view(pad.shape[0] // h, h, pad.shape[1] // w, w)
    most = tiles.abs().amax((1, 3), keepdim=True)
    bits = most.view(torch.int32)
    field = torch.clamp((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).to(torch.int32), min=0)
    scale = torch.where(field > 0, field << 23, torch.full_like(field, 1 << 22)).view(F32)
    q = (tiles / scale).to(torch.float8_e4m3fn).float() * scale
    return q.view(pad.shape)[:rows, :cols]


def _plain_fp8(s: dict):
    c = s["case"]
    x = s["x"].detach().float()
    if c["mode"] == "kept":
        return {"y": (_fp8_values(x, False) @ s["w"].t()).to(BF16)}
    w, dy = _fp8_values(s["w"].detach().float(), True), s["dy"].float()
    return {"y": (_fp8_values(x, False) @ w.t()).to(BF16),
            "dx": (_fp8_values(dy, False) @ w).to(BF16),
            "dw": (_fp8_values(dy.t().contiguous(), False) @ _fp8_values(x.t().contiguous(), False).t()).to(BF16)}


def run(s: dict):
    c = s["case"]
    kind = c["kind"]
    if not own:
        return {"logprobs": _plain_logprobs, "adamw": _plain_adamw, "fp8": _plain_fp8}[kind](s)
    from piper_b200 import ops
    if kind == "logprobs":
        r = ops.token_logprobs(s["x"], s["tokens"], top=c["top"], temperature=c["temperature"])
        out = {"logprob": r.logprob.detach(), "entropy": r.entropy.detach(), "top_logprob": r.top_logprob.detach(),
               "top_id": r.top_id}
        if c["grad"]:
            outs, grads = [r.logprob, r.entropy], [s["dlp"], s["dH"]]
            if c["top"]:
                outs.append(r.top_logprob)
                grads.append(s["dtop"])
            (out["dx"],) = torch.autograd.grad(outs, s["x"], grads)
        return out
    if kind == "adamw":
        ops.adamw_step(s["params"], s["g"], s["state"], **HYPER)
        m, v = s["state"].moments()
        out = {"params": s["params"], "m": m, "v": v}
        if c["params"] == "bf16":
            out["master"] = s["state"].master
        return out
    y = ops.fp8_linear(s["x"], s["w"])
    if c["mode"] == "kept":
        return {"y": y}
    dx, dw = torch.autograd.grad(y, [s["x"], s["w"]], s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw}


# ------------------------------------------------------------------ the definition, in 64 bits
def _exact_logprobs(c: dict, t: dict):
    T, V, k, dev = c["T"], c["V"], c["top"], "cuda"
    lp, H = torch.zeros(T, dtype=torch.float64, device=dev), torch.zeros(T, dtype=torch.float64, device=dev)
    tl, ti = torch.zeros(T, k, dtype=torch.float64, device=dev), torch.zeros(T, k, dtype=torch.int64, device=dev)
    dx = torch.empty(T, V, dtype=F32, device=dev) if c["grad"] else None
    rows = max(1, (64 << 20) // V)
    for a in range(0, T, rows):
        b = min(T, a + rows)
        x64 = t["x"][a:b].double()
        z = x64 / c["temperature"]
        lsm = z - torch.logsumexp(z, 1, keepdim=True)
        p = lsm.exp()
        h = -torch.where(p > 0, p * lsm, 0.0).sum(1)
        y = t["tokens"][a:b]
        on = (y >= 0) & (y < V)
        yy = y.clamp(0, V - 1).unsqueeze(1)
        lp[a:b] = torch.where(on, lsm.gather(1, yy).squeeze(1), 0.0)
        H[a:b] = h
        if k:
            val, idx = torch.sort(x64, dim=1, descending=True, stable=True)
            ti[a:b] = idx[:, :k]
            tl[a:b] = lsm.gather(1, idx[:, :k])
            del val, idx
        if c["grad"]:
            up = torch.zeros_like(p)                       # gradient of the sum of all outputs with respect to log p
            up.scatter_add_(1, yy, torch.where(on, t["dlp"][a:b].double(), 0.0).unsqueeze(1))
            up.scatter_add_(1, ti[a:b], t["dtop"][a:b].double())
            d = up - p * up.sum(1, keepdim=True)
            d -= t["dH"][a:b].double().unsqueeze(1) * torch.where(p > 0, p * (lsm + h.unsqueeze(1)), 0.0)
            dx[a:b] = (d / c["temperature"]).float()
    out = {"logprob": lp, "entropy": H, "top_logprob": tl, "top_id": ti}
    if c["grad"]:
        out["dx"] = dx
    return out


def _power_of_two(e: torch.Tensor) -> torch.Tensor:
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_values(codes, scale, n, signed):
    """Eight bits to 64: sixteen (or 32) octaves of eight steps below the scale."""
    c = codes[:n].to(torch.int64)
    k = (c % 128 if signed else c) + (889 if signed else 761)
    x = (1 + (k % 8).double() / 8) * _power_of_two(k // 8 - 127)
    x = torch.where((c % 128 if signed else c) == 0, 0.0, x) * scale.double().repeat_interleave(BLOCK)[:n]
    return torch.where(c >= 128, -x, x) if signed else x


def _to_32(x: torch.Tensor) -> torch.Tensor:
    """A sum, product or quotient of 32-bit numbers, rounded as the definition has it."""
    return x.float().double()


def _exact_round(x, h, signed):
    """x on the grid of its block, the neighbour above taken with the probability of the distance."""
    n = x.numel()
    pad = torch.zeros((n + BLOCK - 1) // BLOCK * BLOCK, dtype=torch.float64, device=x.device)
    pad[:n] = x.abs()
    top = pad.view(-1, BLOCK).amax(1, keepdim=True)
    y = _to_32(pad.view(-1, BLOCK) / torch.where(top > 0, top, 1.0)).reshape(-1)[:n]
    least = 1.25 * 2.0 ** (-16 if signed else -32)
    e = torch.frexp(y).exponent - 1
    step = _power_of_two(e.clamp(min=-200) - 3)
    low = torch.floor(y / step) * step
    q = torch.where((y - low) / step + h.double() / 65536 >= 1, low + step, low)
    few = torch.where(h.double() / 65536 * least < y, least, 0.0) if signed else torch.where(y > 0, least, 0.0)
    q = torch.where(y < least, few, q)
    q = q * top.view(-1).repeat_interleave(BLOCK)[:n]
    return torch.where(x < 0, -q, q)


def _exact_adamw(c: dict, t: dict):
    shapes = _shapes(c)
    offsets, total = _offsets(shapes)
    b1, b2 = HYPER["betas"]
    step = t["step"] + 1
    params, m_all, v_all = [], torch.zeros(total, dtype=F32, device="cuda"), torch.zeros(total, dtype=F32, device="cuda")
    master = torch.zeros(total, dtype=F32, device="cuda")
    for i, s in enumerate(shapes):
        n, o = math.prod(s), offsets[i]
        w, g = t["p"][i].reshape(-1).double(), t["g"][i].reshape(-1).double()
        if c["bits"] == 8:
            q = slice(o // BLOCK, (o + n + BLOCK - 1) // BLOCK)
            m = _exact_values(t["m"][o:o + n], t["ms"][q], n, True)
            v = _exact_values(t["v"][o:o + n], t["vs"][q], n, False)
        else:
            m, v = t["m"][o:o + n].double(), t["v"][o:o + n].double()
        if c["bits"] == 8:
            # the moments are numbers of 32 bits, each operation rounded, before they are rounded to eight
            f1, f2, h1, h2 = torch.tensor([b1, b2, 1 - b1, 1 - b2], device="cuda").double()
            m = _to_32(_to_32(_to_32(m) * f1) + _to_32(g * h1))
            v = _to_32(_to_32(_to_32(v) * f2) + _to_32(_to_32(g * h2) * g))
        else:
            m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        w = w - HYPER["lr"] * (m / (1 - b1 ** step) / (torch.sqrt(v / (1 - b2 ** step)) + HYPER["eps"])
                               + HYPER["weight_decay"] * w)
        params.append(w.float().view(s))
        master[o:o + n] = w.float()
        if c["bits"] == 8:
            seed = (step * 0x9E3779B1 + i * 0x85EBCA77) % 2 ** 32

            def mix(h):
                h = h ^ (h >> 16)
                h = (h * 0x7FEB352D) % 2 ** 32
                h = h ^ (h >> 15)
                h = (h * 0x846CA68B) % 2 ** 32
                return h ^ (h >> 16)

            h = torch.arange(n, device="cuda") + mix(seed)
            # products of 32 by 31 bits stay below 2^63; the other factor goes in two halves
            h = h % 2 ** 32
            h = h ^ (h >> 16)
            h = (h * 0x7FEB352D) % 2 ** 32
            h = h ^ (h >> 15)
            h = ((h * 0x846C % 2 ** 16) * 65536 + h * 0xA68B) % 2 ** 32
            h = h ^ (h >> 16)
            m, v = _exact_round(m, h % 65536, True), _exact_round(v, h >> 16, False)
        m_all[o:o + n], v_all[o:o + n] = m.float(), v.float()
    out = {"params": params, "m": m_all, "v": v_all}
    if c["params"] == "bf16":
        out["master"] = master
    return out


def _exact_e4m3(x: torch.Tensor, square: bool) -> torch.Tensor:
    """x [rows, cols] in 64 bits on its e4m3 grid: four significant bits, none below 2^-9, ties to even."""
    rows, cols = x.shape
    h = GROUP if square else 1
    out = torch.empty_like(x)
    for j in range(0, cols, GROUP):
        part = x[:, j:j + GROUP]
        most = part.abs().amax(1)
        if square:
            most = torch.stack([b.amax() for b in most.split(h)]).repeat_interleave(h)[:rows]
        mant, e = torch.frexp(most / 448)                    # most = 448 * mant * 2^e, mant in [0.5, 1)
        e = torch.where(mant == 0.5, e - 1, e).clamp(min=-127)
        y = part / _power_of_two(e).unsqueeze(1)
        ulp = _power_of_two((torch.frexp(y).exponent - 1).clamp(min=-6) - 3)
        out[:, j:j + GROUP] = torch.round(y / ulp) * ulp * _power_of_two(e).unsqueeze(1)
    return out


def _exact_fp8(c: dict, t: dict):
    x, w = t["x"].double(), _exact_e4m3(t["w"].double(), True)
    out = {"y": (_exact_e4m3(x, False) @ w.t()).float()}
    if c["mode"] == "train":
        dy = t["dy"].double()
        out["dx"] = (_exact_e4m3(dy, False) @ w).float()
        out["dw"] = (_exact_e4m3(dy.t().contiguous(), False) @ _exact_e4m3(x.t().contiguous(), False).t()).float()
    return out


def exact(case: dict, seed: int):
    t = _inputs(case, seed)
    return {"logprobs": _exact_logprobs, "adamw": _exact_adamw, "fp8": _exact_fp8}[case["kind"]](case, t)


def work(case: dict) -> dict:
    c = case
    if c["kind"] == "logprobs":
        T, V, e = c["T"], c["V"], 2 if c["dtype"] == "bf16" else 4
        n = T * V
        small = T * (8 + 8 + c["top"] * 12)
        if not c["grad"]:
            return {"bytes": n * e + small, "flops": 5 * n}
        return {"bytes": 3 * n * e + 2 * small, "flops": 12 * n}
    if c["kind"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(c))
        grad, state = 4 if c["grads"] == "fp32" else 2, c["bits"] // 8
        # gradient, weights in and out (a master copy beside bf16 ones), both moments in and out, in 32 bits besides if held in 8
        per = grad + 8 + (2 if c["params"] == "bf16" else 0) + 4 * state + (8 if c["bits"] == 8 else 0)
        return {"bytes": n * per, "flops": 15 * n}
    T, K, N = c["T"], c["K"], c["N"]
    if c["mode"] == "kept":
        return {"bytes": 2 * T * K + N * K + N * K // 128 + 2 * T * N, "flops": 2 * T * N * K}
    # x, w, dy in, y, dx, dw out; three products
    return {"bytes": 2 * (2 * T * K + 2 * N * K + 2 * T * N), "flops": 6 * T * N * K}
