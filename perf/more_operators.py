"""Rotary positions, the paged cache behind them in 16 and in 4 bits, and tokens' log probabilities, as measurable cases.

Operators of gomlx_hip.ops, over the types, head layouts and lengths they take:

  rope      rope: rotary positions of one or several axes; its gradient is the inverse rotation
  append    kv_append_rope (bits 16): new tokens' keys, rotated on the way, and values into the
            pages of a cache, their queries rotated beside them; kv4_append_rope (bits 4): into a
            cache of 4-bit values (returned as the values it holds, by kv4_read)
  paged4    sdpa_paged_kv4: one new token a sequence over the pages of a 4-bit cache
  logprobs  token_logprobs: log probability of each row's token, entropy, log-sum-exp and the
            most probable tokens
  lp_grad   token_logprobs_grad: the gradient of the logits

`own` False: their plain form, elementary torch operations in float32 (angles in float64)
rounded once at the end.  `own` True: the framework's entry points.  `exact` evaluates a
case in float64.

The 4-bit cache: a byte holds values 2 i (low half) and 2 i + 1 of a head's row as E2M1 codes,
sign and one of MAGNITUDES; 32 consecutive values share a scale 2^(byte - 127).
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
GROUP = 32


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # The queries of a training batch at the benchmark's attention size.
        {"name": "rope_train", "op": "rope", "B": 4, "H": 16, "S": 2048, "D": 128, "R": 128, "axes": 1, "pairs": "half",
         "inverse": False, "dtype": "bf16"},
        # The gradient through the rotation of a clip's tokens, positions in time, height and width.
        {"name": "rope_video_grad", "op": "rope", "B": 2, "H": 12, "S": 4500, "D": 64, "R": 64, "axes": 3,
         "pairs": "neighbours", "inverse": True, "dtype": "f32"},
        # A decoding step's new token of 16 sequences, pages of 64 tokens.
        {"name": "append_step", "op": "append", "bits": 16, "B": 16, "S": 1, "H": 32, "Hkv": 8, "D": 128, "R": 128,
         "axes": 1, "pairs": "half", "page": 64, "cap": 4096, "layout": "token", "dtype": "bf16"},
        # A batch of prompts with pictures among their tokens, of many lengths, pages of 16.
        {"name": "append_prompt", "op": "append", "bits": 16, "B": 8, "S": 1024, "H": 32, "Hkv": 8, "D": 128, "R": 128,
         "axes": 3, "pairs": "half", "page": 16, "cap": 2048, "layout": "head", "dtype": "f16"},
        # A decoding step into 4 bits, short conversations, half of each head rotated.
        {"name": "append4_step", "op": "append", "bits": 4, "B": 16, "S": 1, "H": 32, "Hkv": 8, "D": 128, "R": 64,
         "axes": 1, "pairs": "neighbours", "page": 64, "cap": 256, "layout": "head", "dtype": "f16"},
        # A batch of prompts of many lengths into 4 bits.
        {"name": "append4_prompt", "op": "append", "bits": 4, "B": 8, "S": 1024, "H": 32, "Hkv": 8, "D": 128, "R": 128,
         "axes": 1, "pairs": "half", "page": 64, "cap": 1280, "layout": "head", "dtype": "bf16"},
        # A decoding step of a large batch whose 16-bit cache would be four times the memory.
        {"name": "paged4_batch", "op": "paged4", "B": 64, "H": 32, "Hkv": 8, "D": 128, "page": 64, "cap": 8192, "W": 0,
         "sinks": 0, "ragged": True, "layout": "head", "dtype": "bf16"},
        # A decoding step of one very long conversation.
        {"name": "paged4_single", "op": "paged4", "B": 1, "H": 32, "Hkv": 8, "D": 128, "page": 64, "cap": 131072, "W": 0,
         "sinks": 0, "ragged": False, "layout": "head", "dtype": "f16"},
        # A decoding step's answers with their twenty most probable alternatives.
        {"name": "logprobs_step", "op": "logprobs", "N": 16, "V": 131072, "padded": False, "top": 20, "scale": 1.0,
         "dtype": "bf16"},
        # Scoring the tokens of whole sequences.
        {"name": "logprobs_score", "op": "logprobs", "N": 4096, "V": 131072, "padded": False, "top": 5, "scale": 1.0,
         "dtype": "bf16"},
        # Training's gradient at the benchmark's vocabulary, with an entropy term.
        {"name": "lp_grad_train", "op": "lp_grad", "N": 8192, "V": 32000, "padded": False, "entropy": True, "scale": 1.0,
         "dtype": "bf16"},
        # The gradient of a small float32 batch at an odd vocabulary and a temperature.
        {"name": "lp_grad_ragged", "op": "lp_grad", "N": 256, "V": 32003, "padded": False, "entropy": False, "scale": 1.25,
         "dtype": "f32"},
    ]


def _size(rng, lo, hi, step=1):
    """A size in [lo, hi], spread over the logarithm; a multiple of `step`."""
    v = math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))
    return min(hi, max(lo, int(round(v / step)) * step))


def _heads(rng):
    Hkv = rng.choice([1, 2, 3, 4, 8])
    return Hkv * rng.choice([1, 1, 2, 4, 8]), Hkv


def draw(rng):
    op = rng.choice(["rope", "append", "append", "paged4", "paged4", "logprobs", "logprobs", "lp_grad"])
    dt = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("logprobs", "lp_grad"):
        V = _size(rng, 17, 160000)
        N = _size(rng, 1, min(8192, (1 << 28) // V))
        c = {"op": op, "N": N, "V": V, "padded": rng.random() < 0.3, "scale": rng.choice([1.0, 1.0, 0.7, 1.6]), "dtype": dt}
        return {**c, "top": rng.choice([0, 1, 5, 20, 32])} if op == "logprobs" else {**c, "entropy": rng.random() < 0.5}
    H, Hkv = _heads(rng)
    layout = rng.choice(["token", "head"])
    page = rng.choice([16, 16, 32, 64, 64, 128, 8, 20])
    if op == "paged4":
        D = rng.choice([64, 128, 128, 96, 32, 256])
        cap = _size(rng, 16, 65536)
        B = _size(rng, 1, max(1, min(128, (1 << 28) // (cap * Hkv * D))))
        return {"op": op, "B": B, "H": H, "Hkv": Hkv, "D": D, "page": page, "cap": cap,
                "W": rng.choice([0, 0, _size(rng, 16, 4096)]), "sinks": rng.choice([0, 4, 4, 40]),
                "ragged": rng.random() < 0.6, "layout": layout, "dtype": dt}
    bits = rng.choice([16, 4]) if op == "append" else 0
    D = rng.choice([64, 128, 128, 96, 256] if bits == 4 else [64, 128, 128, 80, 96, 36, 256])
    axes = rng.choice([1, 1, 2, 3])
    R = rng.choice([D, D, D // 4 * 2])
    c = {"op": op, "H": H, "D": D, "R": R, "axes": axes, "pairs": rng.choice(["half", "half", "neighbours"]), "dtype": dt}
    if op == "rope":
        S = _size(rng, 1, 8192)
        return {**c, "B": _size(rng, 1, max(1, min(32, (1 << 24) // (S * H * D)))), "S": S, "inverse": rng.random() < 0.5}
    S = rng.choice([1, _size(rng, 2, 1024)])
    return {**c, "bits": bits, "B": _size(rng, 1, max(1, min(64, 8192 // S))), "S": S, "Hkv": Hkv, "page": page,
            "cap": S + _size(rng, 16, 256), "layout": layout}


def _spread(B, most):
    """B lengths from most / B to most, none of them sorted."""
    return [max(1, most * (1 + (5 * b + B - 1) % B) // B - b % 2) if math.gcd(5, B) == 1 else max(1, most * (b + 1) // B)
            for b in range(B)]


def _lens(c):
    """The sequences' lengths (paged4), or how many of their tokens are real (append)."""
    if c["op"] == "append":
        return _spread(c["B"], c["S"])
    return _spread(c["B"], c["cap"]) if c["ragged"] else [max(1, c["cap"] - 3 * b) for b in range(c["B"])]


def _sections(c):
    """How many pairs each axis of positions turns."""
    half = c["R"] // 2
    first = half if c["axes"] == 1 else half // 4
    rest = (half - first) // max(1, c["axes"] - 1)
    return [half] if c["axes"] == 1 else [half - rest * (c["axes"] - 1)] + [rest] * (c["axes"] - 1)


def work(case):
    c = case
    es = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "rope":
        return {"bytes": 2 * c["B"] * c["H"] * c["S"] * c["D"] * es + 4 * c["axes"] * c["B"] * c["S"], "flops": 0}
    if c["op"] == "append":
        new = sum(_lens(c)) * c["Hkv"]
        held = c["D"] * es if c["bits"] == 16 else c["D"] // 2 + c["D"] // GROUP
        read = 0
        if c["bits"] == 4:  # the cache's values
            read = 2 * c["B"] * c["cap"] * c["Hkv"] * (held + 2 * c["D"])
        return {"bytes": 2 * c["B"] * c["S"] * c["H"] * c["D"] * es + 2 * new * (c["D"] * es + held) + read, "flops": 0}
    if c["op"] == "paged4":
        seen = 0
        for n in _lens(c):
            first = max(0, n - (c["W"] or n))
            seen += n - first + min(c["sinks"], first)
        return {"bytes": 2 * seen * c["Hkv"] * (c["D"] // 2 + c["D"] // GROUP) + 2 * c["B"] * c["H"] * c["D"] * es,
                "flops": 4 * seen * c["H"] * c["D"]}
    n = c["N"] * c["V"]
    if c["op"] == "logprobs":
        return {"bytes": n * es + c["N"] * (16 + 8 * c["top"]), "flops": 4 * n}
    return {"bytes": 2 * n * es + 16 * c["N"], "flops": 4 * n}


# ---------------------------------------------------------------- the inputs
def _pool(c, g, dt):
    """A cache's storage and the pages of its sequences, one permutation shared out."""
    per = -(-c["cap"] // c["page"])
    pages = c["B"] * per + 3

    def rows(width, t):
        shape = (pages, c["page"], c["Hkv"], width) if c["layout"] == "token" else (pages, c["Hkv"], c["page"], width)
        x = torch.empty(shape, device=DEV, dtype=t)
        return x.transpose(1, 2) if c["layout"] == "token" else x

    table = torch.randperm(pages, generator=g, device=DEV)[: c["B"] * per].view(c["B"], per).to(torch.int32)
    if c["op"] == "append" and c["bits"] == 16:
        return [rows(c["D"], dt) for _ in range(2)], table
    wide = 4 * -(-c["D"] // 128)  # bytes of a row's scales: whole words
    return [(rows(c["D"] // 2, torch.uint8), rows(wide, torch.uint8)) for _ in range(2)], table


def prepare(case, seed):
    c = case
    dt = TORCH[c["dtype"]]
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=g, device=DEV, dtype=dt)  # noqa: E731
    s = {"case": c, "work": {}}  # workspaces, which a program keeps beside its tensors
    if c["op"] in ("logprobs", "lp_grad"):
        N, V = c["N"], c["V"]
        wide = -(-V // 64) * 64 if c["padded"] else V
        s["logits"] = rand(N, wide).mul_(2.5)[:, :V]
        s["ids"] = torch.randint(0, V, (N,), generator=g, device=DEV, dtype=torch.int32)
        best = torch.arange(0, N, 2, device=DEV)  # every other token is a likely one
        s["logits"][best, s["ids"][best].long()] += 9
        if c["op"] == "lp_grad":
            s["d_logp"] = torch.randn((N,), generator=g, device=DEV)
            s["d_entropy"] = torch.randn((N,), generator=g, device=DEV) * 0.1 if c["entropy"] else None
            _, s["entropy"], s["lse"], _, _ = _logprobs_plain({**s, "case": {**c, "top": 0}})
        return s
    if c["op"] == "paged4":
        s["lens"] = torch.tensor(_lens(c), dtype=torch.int32, device=DEV)
        s["scale"] = 1.0 / math.sqrt(c["D"])
        s["q"] = rand(c["B"], c["H"], c["D"])
        (s["k_cache"], s["v_cache"]), s["table"] = _pool(c, g, dt)
        for codes, scales in (s["k_cache"], s["v_cache"]):
            for p in range(0, codes.shape[0], 512):  # values of many sizes, in the types' plain rounding
                x = torch.randn((*codes[p : p + 512].shape[:3], c["D"]), generator=g, device=DEV)
                codes[p : p + 512], scales[p : p + 512, ..., : c["D"] // GROUP] = _encode(x)
        return s
    s["freqs"] = (10000.0 ** (-torch.arange(0, c["R"], 2, dtype=torch.float64) / c["R"])).float().to(DEV)
    s["sections"] = _sections(c)
    s["axis"] = torch.repeat_interleave(torch.arange(c["axes"]), torch.tensor(s["sections"])).to(DEV)
    # Projections' outputs: [B, S, heads, D] in memory, looked at head by head.
    if c["op"] == "rope":
        s["x"] = rand(c["B"], c["S"], c["H"], c["D"]).transpose(1, 2)
        s["positions"] = torch.randint(0, 131072, (c["axes"], c["B"], c["S"]), generator=g, device=DEV, dtype=torch.int32)
        return s
    s["lens"] = torch.tensor(_lens(c), dtype=torch.int32, device=DEV)
    qkv = rand(c["B"], c["S"], c["H"] + 2 * c["Hkv"], c["D"]).transpose(1, 2)
    s["q"], s["k"], s["v"] = qkv.split([c["H"], c["Hkv"], c["Hkv"]], 1)
    s["starts"] = torch.randint(0, c["cap"] - c["S"] + 1, (c["B"],), generator=g, device=DEV, dtype=torch.int32)
    s["positions"] = None
    if c["axes"] > 1:
        s["positions"] = torch.randint(0, 4096, (c["axes"], c["B"], c["S"]), generator=g, device=DEV, dtype=torch.int32)
    caches, s["table"] = _pool(c, g, dt)
    for cache in caches:
        if c["bits"] == 16:
            cache.copy_(torch.randn(cache.shape, generator=g, device=DEV, dtype=dt))
        else:
            x = torch.randn((*cache[0].shape[:3], c["D"]), generator=g, device=DEV)
            codes, scales = _encode(x)
            cache[0].copy_(codes)
            cache[1].zero_()[..., : c["D"] // GROUP] = scales
    s["k_cache"], s["v_cache"] = caches
    return s


# ---------------------------------------------------------------- the plain forms
def _power(e):
    """2^e in float32 of whole numbers e."""
    return (e.to(torch.int32) + 127 << 23).view(torch.float32)


def _encode(x):
    """(codes, scales) of float32 values whose last axis is a whole number of groups."""
    x = x.unflatten(-1, (-1, GROUP))
    most, e = torch.frexp(x.abs().amax(-1, keepdim=True))
    e = torch.where(most <= 0.75, e - 3, e - 2).clamp(-126, 125)  # most 2^e <= 6 2^(e - 3) where most <= 3/4
    e = torch.where(most > 0, e, torch.full_like(e, -126))
    x = x * _power(-e)
    a = x.abs()
    code = sum(((a > lo) if i % 2 == 0 else (a >= lo)).to(torch.uint8)
               for i, lo in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)))  # the middles; ties to the even code
    code = (code | torch.signbit(x).to(torch.uint8) << 3).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, (e.squeeze(-1) + 127).to(torch.uint8)


def _decode(codes, scales, D):
    """The float32 values of rows of a 4-bit cache."""
    table = torch.tensor([*MAGNITUDES, *(-m for m in MAGNITUDES)], device=DEV)
    x = table[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()].unflatten(-1, (-1, GROUP))
    return (x * _power(scales[..., : D // GROUP, None].int() - 127)).flatten(-2)


def _turn(s, x, positions, inverse=False):
    """x [B, heads, S, D], rotated, in float32."""
    c = s["case"]
    R = c["R"]
    a = positions[s["axis"]].permute(1, 2, 0).double() * s["freqs"].double()  # [B, S, R / 2]
    cos, sin = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]
    sin = -sin if inverse else sin
    x = x.float()
    if c["pairs"] == "half":
        u, v = x[..., : R // 2], x[..., R // 2 : R]
        y = torch.cat((u * cos - v * sin, u * sin + v * cos), -1)
    else:
        u, v = x[..., 0:R:2], x[..., 1:R:2]
        y = torch.stack((u * cos - v * sin, u * sin + v * cos), -1).flatten(-2)
    return torch.cat((y, x[..., R:]), -1)


def _rope_plain(s):
    return _turn(s, s["x"], s["positions"], s["case"]["inverse"]).to(s["x"].dtype)


def _append_plain(s):
    c = s["case"]
    # Tokens that are not real write their sequence's first token once more.
    i = torch.arange(c["S"], device=DEV)[None, :].expand(c["B"], -1)
    positions = s["positions"] if s["positions"] is not None else (s["starts"][:, None] + i)[None]
    q = _turn(s, s["q"], positions).to(s["q"].dtype)
    k, v = _turn(s, s["k"], positions), s["v"].float()
    i = torch.where(i < s["lens"][:, None], i, torch.zeros_like(i))
    pos = s["starts"][:, None] + i
    page = s["table"].gather(1, (pos // c["page"]).long()).long()
    at = (pos % c["page"]).long()
    b = torch.arange(c["B"], device=DEV)[:, None]
    k, v = k[b, :, i], v[b, :, i]
    if c["bits"] == 16:
        s["k_cache"][page, :, at] = k.to(s["k"].dtype)
        s["v_cache"][page, :, at] = v.to(s["v"].dtype)
        return q, s["k_cache"], s["v_cache"]
    (kc, ks), (vc, vs) = s["k_cache"], s["v_cache"]
    n = c["D"] // GROUP
    kc[page, :, at], ks[..., :n][page, :, at] = _encode(k)
    vc[page, :, at], vs[..., :n][page, :, at] = _encode(v)
    held = lambda t: t[s["table"].long()].transpose(1, 2).flatten(2, 3)[:, :, : c["cap"]]  # noqa: E731
    return q, _decode(held(kc), held(ks), c["D"]).bfloat16(), _decode(held(vc), held(vs), c["D"]).bfloat16()


def _paged4_plain(s):
    c = s["case"]
    G = c["H"] // c["Hkv"]
    held = lambda t: t[s["table"].long()].transpose(1, 2).flatten(2, 3)  # noqa: E731
    key = torch.arange(s["table"].shape[1] * c["page"], device=DEV)[None, :]
    n = s["lens"][:, None]
    see = (key < n) & ((key >= n - (c["W"] or c["cap"])) | (key < c["sinks"]))
    k = _decode(held(s["k_cache"][0]), held(s["k_cache"][1]), c["D"])
    x = torch.matmul(s["q"].float().view(c["B"], c["Hkv"], G, c["D"]), k.transpose(-1, -2)) * s["scale"]
    del k
    x.masked_fill_(~see[:, None, None], -math.inf)
    x = (x - x.amax(-1, keepdim=True)).exp_()
    v = _decode(held(s["v_cache"][0]), held(s["v_cache"][1]), c["D"])
    o = torch.matmul(x, v) / x.sum(-1, keepdim=True)
    return o.view(c["B"], c["H"], c["D"]).to(s["q"].dtype)


def _logprobs_plain(s):
    c = s["case"]
    x = s["logits"].float()
    t = x * c["scale"]
    m = t.amax(-1, keepdim=True)
    t = t - m
    e = t.exp()
    total = e.sum(-1)
    log = total.log()
    entropy = log - (e * t).sum(-1) / total
    logp = t.gather(1, s["ids"].long()[:, None])[:, 0] - log
    lse = m[:, 0] + log
    if not c["top"]:
        return logp, entropy, lse, None, None
    # Float order as integer order (-0 as 0), equal logits by their index.
    bits = (x + 0.0).view(torch.int32)
    key = (bits ^ (bits >> 31 & 0x7FFFFFFF)).long() << 32 | torch.arange(c["V"] - 1, -1, -1, device=DEV)
    at = c["V"] - 1 - (torch.topk(key, min(c["top"], c["V"]), -1).values & 0xFFFFFFFF)
    return logp, entropy, lse, t.gather(1, at) - log[:, None], at.to(torch.int32)


def _lp_grad_plain(s):
    c = s["case"]
    t = s["logits"].float() * c["scale"] - s["lse"][:, None]
    p = t.exp()
    d = p * -s["d_logp"][:, None]
    if s["d_entropy"] is not None:
        d -= s["d_entropy"][:, None] * p * (t + s["entropy"][:, None])
    d[torch.arange(c["N"], device=DEV), s["ids"].long()] += s["d_logp"]
    return (d * c["scale"]).to(s["logits"].dtype)


# ---------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(state, op)
    return {"rope": _rope_plain, "append": _append_plain, "paged4": _paged4_plain, "logprobs": _logprobs_plain,
            "lp_grad": _lp_grad_plain}[op](state)


def _run_own(s, op):
    path = os.path.join(os.getcwd(), "go-darwinml_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from gomlx_hip import ops
    c, w = s["case"], s["work"]
    if op == "rope":
        return ops.rope(s["x"], s["positions"], s["freqs"], s["sections"], interleaved=c["pairs"] != "half",
                        inverse=c["inverse"])
    if op == "append":
        args = dict(counts=s["lens"], positions=s["positions"], sections=s["sections"], interleaved=c["pairs"] != "half")
        if c["bits"] == 16:
            q = ops.kv_append_rope(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["starts"], s["freqs"],
                                   **args)
            return q, s["k_cache"], s["v_cache"]
        q = ops.kv4_append_rope(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["starts"], s["freqs"],
                                **args)
        return (q, *ops.kv4_read(s["k_cache"], s["v_cache"], s["table"], c["cap"], dtype=torch.bfloat16))
    if op == "paged4":
        if "ws" not in w:
            w["ws"] = ops.sdpa_paged_kv4_workspace(s["q"], s["k_cache"], s["table"])
        return ops.sdpa_paged_kv4(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["scale"], window=c["W"],
                                  sinks=c["sinks"], workspace=w["ws"])
    if op == "logprobs":
        if "ws" not in w:
            w["ws"] = ops.token_logprobs_workspace(s["logits"], min(c["top"], c["V"]))
        return ops.token_logprobs(s["logits"], s["ids"], top=min(c["top"], c["V"]), scale=c["scale"], workspace=w["ws"])
    return ops.token_logprobs_grad(s["logits"], s["ids"], s["lse"], s["d_logp"], entropy=s["entropy"],
                                   d_entropy=s["d_entropy"], scale=c["scale"])


# ---------------------------------------------------------------- the definition in 64 bits
def _rotated(c, x, pos, freqs):
    """x [S, D] in float64 at pos [axes, S]: as multiplication by complex numbers."""
    half, first = c["R"] // 2, 0
    y = x.double().clone()
    u, v = (y[:, :half], y[:, half : c["R"]]) if c["pairs"] == "half" else (y[:, 0 : c["R"] : 2], y[:, 1 : c["R"] : 2])
    z = torch.complex(u.contiguous(), v.contiguous())
    for a, n in enumerate(_sections(c)):
        angle = torch.outer(pos[a].double(), freqs[first : first + n].double())
        z[:, first : first + n] *= torch.polar(torch.ones_like(angle), -angle if c.get("inverse") else angle)
        first += n
    u.copy_(z.real)
    v.copy_(z.imag)
    return y


def _nearest(x):
    """The values that a 4-bit cache holds for rows x, in float64: by distance to each of them."""
    g = x.double().reshape(-1, GROUP)
    most = g.abs().amax(1, keepdim=True)
    steps = torch.tensor([2.0 ** n for n in range(-126, 126)], dtype=torch.float64, device=DEV)
    unit = steps[(most > 6 * steps[:-1]).sum(1, keepdim=True)]  # the first that six times it reaches
    order = (0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0)  # the even codes first: they win ties
    away = torch.stack([(g.abs() / unit - m).abs() for m in order])
    pick = torch.tensor(order, dtype=torch.float64, device=DEV)[away.argmin(0)]
    # (argmin takes any of equal distances: those of ties are put right.)
    for lo, hi, even in ((0, 0.5, 0), (0.5, 1, 1), (1, 1.5, 1), (1.5, 2, 2), (2, 3, 2), (3, 4, 4), (4, 6, 4)):
        pick = torch.where(g.abs() / unit == (lo + hi) / 2, torch.full_like(pick, float(even)), pick)
    return (pick * unit * torch.where(g < 0, -1.0, 1.0)).reshape(x.shape)


def _values(cache, D):
    """A 4-bit cache's values in float64, [pages, Hkv, page, D]."""
    codes, scales = cache
    sizes = torch.tensor(MAGNITUDES, dtype=torch.float64, device=DEV)
    y = torch.empty((*codes.shape[:3], D), dtype=torch.float64, device=DEV)
    for half, code in ((0, codes % 16), (1, codes // 16)):
        y[..., half::2] = sizes[(code % 8).long()] * (1 - 2.0 * (code >= 8))
    steps = torch.tensor([2.0 ** (n - 127) for n in range(255)], dtype=torch.float64, device=DEV)
    y *= steps[scales[..., : D // GROUP].long()].repeat_interleave(GROUP, -1)
    return y


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["op"] == "rope":
        y = torch.empty(s["x"].shape, dtype=torch.float64, device=DEV)
        for b in range(c["B"]):
            for h in range(c["H"]):
                y[b, h] = _rotated(c, s["x"][b, h], s["positions"][:, b], s["freqs"])
        return y
    if c["op"] == "append":
        if c["bits"] == 16:
            kc, vc = s["k_cache"].double(), s["v_cache"].double()
        else:
            kc, vc = _values(s["k_cache"], c["D"]), _values(s["v_cache"], c["D"])
        q = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
        starts, lens = s["starts"].tolist(), _lens(c)
        for b in range(c["B"]):
            at = torch.arange(starts[b], starts[b] + c["S"], device=DEV)
            pos = at[None] if s["positions"] is None else s["positions"][:, b]
            for h in range(c["H"]):
                q[b, h] = _rotated(c, s["q"][b, h], pos, s["freqs"])
            n = lens[b]
            page, row = s["table"][b].long()[at[:n] // c["page"]], at[:n] % c["page"]
            for h in range(c["Hkv"]):
                k, v = _rotated(c, s["k"][b, h, :n], pos[:, :n], s["freqs"]), s["v"][b, h, :n].double()
                kc[page, h, row], vc[page, h, row] = (k, v) if c["bits"] == 16 else (_nearest(k), _nearest(v))
        if c["bits"] == 4:
            kc, vc = (t[s["table"].long()].transpose(1, 2).flatten(2, 3)[:, :, : c["cap"]] for t in (kc, vc))
        return q, kc, vc
    if c["op"] == "paged4":
        out = torch.empty(c["B"], c["H"], c["D"], dtype=torch.float64, device=DEV)
        for b, n in enumerate(_lens(c)):
            rows = torch.arange(n, device=DEV)
            rows = rows[(rows < c["sinks"]) | (rows >= n - c["W"])] if c["W"] else rows
            page, at = s["table"][b].long()[rows // c["page"]], rows % c["page"]
            k, v = (_values([t[page, :, at][None] for t in cache], c["D"])[0] for cache in (s["k_cache"], s["v_cache"]))
            for h in range(c["H"]):
                p = torch.softmax(torch.mv(k[:, h * c["Hkv"] // c["H"]], s["q"][b, h].double()) * s["scale"], 0)
                out[b, h] = torch.mv(v[:, h * c["Hkv"] // c["H"]].T, p)
        return out
    got = []
    for n in range(0, c["N"], 256):
        x = s["logits"][n : n + 256].double()
        lp = torch.log_softmax(x * c["scale"], -1)
        ids = s["ids"][n : n + 256].long()[:, None]
        if c["op"] == "lp_grad":
            # The gradient for the log-sum-exp and the entropy that the call is given.
            lp = x * c["scale"] - s["lse"][n : n + 256].double()[:, None]
            hit = torch.zeros_like(lp).scatter_(1, ids, 1.0)
            d = s["d_logp"][n : n + 256].double()[:, None] * (hit - lp.exp())
            if c["entropy"]:
                d -= s["d_entropy"][n : n + 256].double()[:, None] * lp.exp() * (lp + s["entropy"][n : n + 256].double()[:, None])
            got.append(d * c["scale"])
            continue
        k = min(c["top"], c["V"])
        row = [lp.gather(1, ids)[:, 0], -(lp.exp() * lp).sum(-1), torch.logsumexp(x * c["scale"], -1), None, None]
        if k:
            least = torch.topk(x, k, -1).values[:, -1]
            at = []
            for r in range(x.shape[0]):  # the few that are in question, by index, then by a stable order
                few = torch.nonzero(x[r] >= least[r])[:, 0]
                at.append(few[torch.sort(x[r][few], descending=True, stable=True).indices[:k]])
            row[4] = torch.stack(at)
            row[3] = lp.gather(1, row[4])
            row[4] = row[4].to(torch.int32)
        got.append(row)
    if c["op"] == "lp_grad":
        return torch.cat(got)
    return tuple(None if t[0] is None else torch.cat(t) for t in zip(*got))
