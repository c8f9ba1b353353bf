"""Sliding-window attention with sinks, its gradient, and the paged key-value cache, as measurable cases.

Four operators of gomlx_hip.ops, over the types, head layouts and lengths they take:

  window    sdpa_window: causal attention whose queries see the last `window` keys
            and the first `sinks` ones (prompts and training's forward pass)
  grad      sdpa_window_grad: dq, dk, dv of it, from its output and log-sum-exp
  append    kv_append: new tokens' keys and values into the pages of a cache
  paged     sdpa_paged: one new token a sequence over its pages

`own` False: their plain form, elementary torch operations in float32 rounded once at
the end.  `own` True: the framework's entry points.  `exact` evaluates a case in
float64, head by head.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # A prompt chunk of one short conversation continued in float32, at a ragged
        # head dim: the smallest call.
        {"name": "window_chunk", "op": "window", "B": 1, "H": 8, "Hkv": 2, "Sq": 37, "Sk": 164, "D": 80, "W": 48,
         "sinks": 2, "padded": False, "dtype": "f32"},
        # A training batch's forward pass at the benchmark's attention size.
        {"name": "window_train", "op": "window", "B": 4, "H": 16, "Hkv": 16, "Sq": 2048, "Sk": 2048, "D": 128,
         "W": 512, "sinks": 4, "padded": False, "dtype": "bf16"},
        # Prefill of one long prompt with grouped-query heads.
        {"name": "window_prompt", "op": "window", "B": 1, "H": 32, "Hkv": 8, "Sq": 8192, "Sk": 8192, "D": 128,
         "W": 2048, "sinks": 4, "padded": False, "dtype": "bf16"},
        # A padded batch of sequences of many lengths, heads of 64.
        {"name": "window_padded", "op": "window", "B": 8, "H": 12, "Hkv": 12, "Sq": 1000, "Sk": 1000, "D": 64,
         "W": 128, "sinks": 1, "padded": True, "dtype": "f16"},
        # The gradient of the training batch.
        {"name": "grad_train", "op": "grad", "B": 4, "H": 16, "Hkv": 16, "Sq": 2048, "Sk": 2048, "D": 128, "W": 512,
         "sinks": 4, "padded": False, "dtype": "bf16"},
        # The gradient over one long sequence, shared kv heads.
        {"name": "grad_long", "op": "grad", "B": 1, "H": 32, "Hkv": 8, "Sq": 4096, "Sk": 4096, "D": 128, "W": 1024,
         "sinks": 4, "padded": False, "dtype": "bf16"},
        # The gradient of the padded batch.
        {"name": "grad_padded", "op": "grad", "B": 8, "H": 12, "Hkv": 12, "Sq": 1000, "Sk": 1000, "D": 64, "W": 128,
         "sinks": 1, "padded": True, "dtype": "f16"},
        # A decoding step's new token of 16 sequences, pages of 64 tokens.
        {"name": "append_step", "op": "append", "B": 16, "S": 1, "Hkv": 8, "D": 128, "page": 64, "cap": 4096,
         "layout": "token", "dtype": "bf16"},
        # A batch of prompts of many lengths behind what their caches hold, pages of 16.
        {"name": "append_prompt", "op": "append", "B": 8, "S": 1024, "Hkv": 8, "D": 128, "page": 16, "cap": 2048,
         "layout": "head", "dtype": "bf16"},
        # A decoding step over long caches of about one length (the benchmark's decoding size).
        {"name": "paged_batch", "op": "paged", "B": 8, "H": 32, "Hkv": 8, "D": 128, "page": 64, "cap": 8192, "W": 0,
         "sinks": 0, "ragged": False, "layout": "token", "dtype": "bf16"},
        # A decoding step of one very long conversation.
        {"name": "paged_single", "op": "paged", "B": 1, "H": 32, "Hkv": 8, "D": 128, "page": 64, "cap": 65536, "W": 0,
         "sinks": 0, "ragged": False, "layout": "head", "dtype": "bf16"},
        # A serving batch of sequences from a few tokens to the whole cache, with a window and sinks.
        {"name": "paged_window", "op": "paged", "B": 64, "H": 32, "Hkv": 8, "D": 128, "page": 16, "cap": 4096,
         "W": 1024, "sinks": 4, "ragged": True, "layout": "token", "dtype": "f16"},
    ]


def _size(rng, lo, hi, step=1):
    """A size in [lo, hi], spread over the logarithm; a multiple of `step`."""
    v = math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))
    return min(hi, max(lo, int(round(v / step)) * step))


def _heads(rng):
    Hkv = rng.choice([1, 2, 3, 4, 8])
    return Hkv * rng.choice([1, 1, 2, 4, 8]), Hkv


def draw(rng):
    op = rng.choice(["window", "window", "grad", "grad", "append", "paged", "paged"])
    dt = rng.choice(["bf16", "bf16", "f16", "f32"])
    H, Hkv = _heads(rng)
    if op in ("window", "grad"):
        D = rng.choice([64, 128, 128, 80, 96, 40] + ([256] if dt != "f32" else []))
        most = 1 << (35 if dt == "f32" or op == "grad" else 37)
        S = _size(rng, 16, min(8192, math.isqrt(most // (H * D))), rng.choice([1, 1, 64]))
        Sk, Sq = S, S
        if rng.random() < 0.25:
            Sq = _size(rng, 1, S)
        B = _size(rng, 1, max(1, min(16, most // (H * Sq * Sk * D))))
        return {"op": op, "B": B, "H": H, "Hkv": Hkv, "Sq": Sq, "Sk": Sk, "D": D,
                "W": rng.choice([0, _size(rng, 1, S), _size(rng, 16, 1024)]),
                "sinks": rng.choice([0, 1, 4, 4, 16, 70]), "padded": rng.random() < 0.4, "dtype": dt}
    D = rng.choice([64, 128, 128, 80, 96] + ([256] if dt != "f32" else []))
    page = rng.choice([16, 16, 32, 64, 64, 128, 8, 20])
    layout = rng.choice(["token", "head"])
    if op == "append":
        S = rng.choice([1, _size(rng, 2, 1024)])
        cap = S + _size(rng, 16, 1024)
        return {"op": op, "B": _size(rng, 1, max(1, min(64, 8192 // S))), "S": S, "Hkv": Hkv, "D": D, "page": page,
                "cap": cap, "layout": layout, "dtype": dt}
    cap = _size(rng, 16, 32768)
    B = _size(rng, 1, max(1, min(64, (1 << 26) // (cap * Hkv * D * (2 if dt == "f32" else 1)))))
    return {"op": op, "B": B, "H": H, "Hkv": Hkv, "D": D, "page": page, "cap": cap,
            "W": rng.choice([0, 0, _size(rng, 16, 4096)]), "sinks": rng.choice([0, 4, 4, 40]),
            "ragged": rng.random() < 0.6, "layout": layout, "dtype": dt}


def _spread(B, most):
    """B lengths from most / B to most, none of them sorted."""
    return [max(1, most * (1 + (5 * b + B - 1) % B) // B - b % 2) if math.gcd(5, B) == 1 else max(1, most * (b + 1) // B)
            for b in range(B)]


def _lens(c):
    """The sequences' lengths: what a case's masks and works go by."""
    if c["op"] in ("window", "grad"):
        return [max(1, n) for n in _spread(c["B"], c["Sk"])] if c["padded"] else [c["Sk"]] * c["B"]
    if c["op"] == "paged":
        return _spread(c["B"], c["cap"]) if c["ragged"] else [max(1, c["cap"] - 3 * b) for b in range(c["B"])]
    return _spread(c["B"], c["S"])  # append: how many tokens of each sequence are real


def _pairs(c):
    """(query, key) pairs a head of the whole batch looks at."""
    W = c["W"] or c["Sk"]
    n = 0
    for length in _lens(c):
        for p in range(c["Sk"] - c["Sq"], length):
            first = max(0, p + 1 - W)
            n += p + 1 - first + min(c["sinks"], first)
    return n


def work(case):
    c = case
    es = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "append":
        return {"bytes": 4 * sum(_lens(c)) * c["Hkv"] * c["D"] * es, "flops": 0}
    if c["op"] == "paged":
        seen = 0
        for n in _lens(c):
            first = max(0, n - (c["W"] or n))
            seen += n - first + min(c["sinks"], first)
        return {"bytes": (2 * seen * c["Hkv"] + 2 * c["B"] * c["H"]) * c["D"] * es, "flops": 4 * seen * c["H"] * c["D"]}
    q = c["B"] * c["H"] * c["Sq"] * c["D"]
    kv = c["B"] * c["Hkv"] * c["Sk"] * c["D"]
    rows = c["B"] * c["H"] * c["Sq"]
    if c["op"] == "window":
        return {"bytes": (2 * q + 2 * kv) * es + rows * 4, "flops": 4 * _pairs(c) * c["H"] * c["D"]}
    return {"bytes": (4 * q + 4 * kv) * es + rows * 4, "flops": 10 * _pairs(c) * c["H"] * c["D"]}


# ---------------------------------------------------------------- the inputs
def _pool(c, g, dt):
    """The pages of a cache, one permutation of them shared out to the sequences."""
    per = -(-c["cap"] // c["page"])
    pages = c["B"] * per + 3
    caches = []
    for _ in range(2):
        shape = (pages, c["page"], c["Hkv"], c["D"]) if c["layout"] == "token" else (pages, c["Hkv"], c["page"], c["D"])
        t = torch.randn(shape, generator=g, device=DEV, dtype=dt)
        caches.append(t.transpose(1, 2) if c["layout"] == "token" else t)
    table = torch.randperm(pages, generator=g, device=DEV)[: c["B"] * per].view(c["B"], per).to(torch.int32)
    return caches[0], caches[1], table


def prepare(case, seed):
    c = case
    dt = TORCH[c["dtype"]]
    g = torch.Generator(device=DEV).manual_seed(seed)
    lens = torch.tensor(_lens(c), dtype=torch.int32, device=DEV)
    rand = lambda *shape: torch.randn(shape, generator=g, device=DEV, dtype=dt)  # noqa: E731
    s = {"case": c, "lens": lens, "scale": 1.0 / math.sqrt(c["D"])}
    if c["op"] in ("window", "grad"):
        # Projections' outputs: [B, S, H, D] in memory, looked at head by head.
        s["q"] = rand(c["B"], c["Sq"], c["H"], c["D"]).transpose(1, 2)
        s["k"] = rand(c["B"], c["Sk"], c["Hkv"], c["D"]).transpose(1, 2)
        s["v"] = rand(c["B"], c["Sk"], c["Hkv"], c["D"]).transpose(1, 2)
        if c["op"] == "grad":
            s["do"] = rand(c["B"], c["Sq"], c["H"], c["D"]).transpose(1, 2)
            s["o"], s["lse"] = _window_plain(s)
            s["o"] = s["o"].transpose(1, 2).contiguous().transpose(1, 2)
    else:
        s["k_cache"], s["v_cache"], s["table"] = _pool(c, g, dt)
        if c["op"] == "paged":
            s["q"] = rand(c["B"], c["H"], c["D"])
        else:
            s["k"] = rand(c["B"], c["S"], c["Hkv"], c["D"]).transpose(1, 2)
            s["v"] = rand(c["B"], c["S"], c["Hkv"], c["D"]).transpose(1, 2)
            s["starts"] = torch.randint(0, c["cap"] - c["S"] + 1, (c["B"],), generator=g, device=DEV, dtype=torch.int32)
    s["work"] = {}  # workspaces, which a program keeps beside its tensors
    return s


# ---------------------------------------------------------------- the plain forms
def _visible(s):
    """[B, 1, 1, Sq, Sk]: the keys each query sees."""
    c = s["case"]
    pos = torch.arange(c["Sk"] - c["Sq"], c["Sk"], device=DEV)[:, None]
    key = torch.arange(c["Sk"], device=DEV)[None, :]
    see = (key <= pos) & ((key > pos - (c["W"] or c["Sk"])) | (key < c["sinks"]))
    return (see[None] & (pos < s["lens"][:, None, None]))[:, None, None]


def _grouped(s, name):
    """Query-side tensors as [B, Hkv, G, Sq, D], key-side ones as [B, Hkv, 1, Sk, D], in float32."""
    c, t = s["case"], s[name]
    if t.shape[1] == c["H"] and name not in ("k", "v"):
        return t.float().reshape(c["B"], c["Hkv"], c["H"] // c["Hkv"], c["Sq"], c["D"])
    return t.float()[:, :, None]


def _window_plain(s):
    c = s["case"]
    x = torch.matmul(_grouped(s, "q"), _grouped(s, "k").transpose(-1, -2)).mul_(s["scale"])
    x.masked_fill_(~_visible(s), -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    x = x.sub_(m).exp_()
    l = x.sum(-1, keepdim=True)
    o = torch.matmul(x, _grouped(s, "v")) / torch.where(l > 0, l, torch.ones_like(l))
    lse = (m + torch.log(l)).reshape(c["B"], c["H"], c["Sq"])
    return o.reshape(c["B"], c["H"], c["Sq"], c["D"]).to(s["q"].dtype), lse


def _grad_plain(s):
    c = s["case"]
    q, k, v, do, o = (_grouped(s, n) for n in ("q", "k", "v", "do", "o"))
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(s["scale"]).sub_(s["lse"].reshape(q.shape[:-1])[..., None]).exp_()
    p = p.masked_fill_(~_visible(s), 0.0)
    dv = torch.matmul(p.transpose(-1, -2), do).sum(2)
    d = torch.matmul(do, v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(s["scale"])
    dk = torch.matmul(d.transpose(-1, -2), q).sum(2)
    dq = torch.matmul(d, k).reshape(c["B"], c["H"], c["Sq"], c["D"])
    dt = s["q"].dtype
    return dq.to(dt), dk.to(dt), dv.to(dt)


def _append_plain(s):
    c = s["case"]
    # Tokens that are not real write their sequence's first token once more.
    i = torch.arange(c["S"], device=DEV)[None, :].expand(c["B"], -1)
    i = torch.where(i < s["lens"][:, None], i, torch.zeros_like(i))
    pos = s["starts"][:, None] + i
    page = s["table"].gather(1, (pos // c["page"]).long()).long()
    at = (pos % c["page"]).long()
    b = torch.arange(c["B"], device=DEV)[:, None]
    s["k_cache"][page, :, at] = s["k"][b, :, i]
    s["v_cache"][page, :, at] = s["v"][b, :, i]
    return s["k_cache"], s["v_cache"]


def _paged_plain(s):
    c = s["case"]
    G = c["H"] // c["Hkv"]
    k, v = (t[s["table"].long()].float().transpose(1, 2).reshape(c["B"], c["Hkv"], -1, c["D"]) for t in (s["k_cache"], s["v_cache"]))
    q = s["q"].float().view(c["B"], c["Hkv"], G, c["D"])
    key = torch.arange(k.shape[2], device=DEV)[None, :]
    n = s["lens"][:, None]
    see = (key < n) & ((key >= n - (c["W"] or c["cap"])) | (key < c["sinks"]))
    x = (torch.matmul(q, k.transpose(-1, -2)) * s["scale"]).masked_fill_(~see[:, None, None], -math.inf)
    x = (x - x.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(x, v) / x.sum(-1, keepdim=True)
    return o.view(c["B"], c["H"], c["D"]).to(s["q"].dtype)


# ---------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(state, op)
    return {"window": _window_plain, "grad": _grad_plain, "append": _append_plain, "paged": _paged_plain}[op](state)


def _run_own(s, op):
    path = os.path.join(os.getcwd(), "go-darwinml_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from gomlx_hip import ops
    c, w = s["case"], s["work"]
    if op == "window":
        return ops.sdpa_window(s["q"], s["k"], s["v"], s["scale"], c["W"], c["sinks"], q_start=c["Sk"] - c["Sq"],
                               lens=s["lens"] if c["padded"] else None, with_lse=True)
    if op == "grad":
        if "ws" not in w:
            w["ws"] = ops.sdpa_window_grad_workspace(s["q"], s["k"], c["W"], c["sinks"], q_start=c["Sk"] - c["Sq"])
        return ops.sdpa_window_grad(s["do"], s["q"], s["k"], s["v"], s["o"], s["lse"], s["scale"], c["W"], c["sinks"],
                                    q_start=c["Sk"] - c["Sq"], lens=s["lens"] if c["padded"] else None,
                                    workspace=w["ws"])
    if op == "append":
        ops.kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["starts"], counts=s["lens"])
        return s["k_cache"], s["v_cache"]
    if "ws" not in w:
        w["ws"] = ops.sdpa_paged_workspace(s["q"], s["k_cache"], s["table"])
    return ops.sdpa_paged(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["scale"], window=c["W"],
                          sinks=c["sinks"], workspace=w["ws"])


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    """A head at a time, each sequence cut to its length, by softmax's definition."""
    c = case
    s = prepare(c, seed)
    scale = 1.0 / math.sqrt(c["D"])
    lens = _lens(c)
    if c["op"] == "append":
        k_cache, v_cache = s["k_cache"].clone(), s["v_cache"].clone()
        table, starts = s["table"].tolist(), s["starts"].tolist()
        for b in range(c["B"]):
            for i in range(lens[b]):
                page, at = table[b][(starts[b] + i) // c["page"]], (starts[b] + i) % c["page"]
                k_cache[page, :, at] = s["k"][b, :, i]
                v_cache[page, :, at] = s["v"][b, :, i]
        return k_cache, v_cache
    G = c["H"] // c["Hkv"]
    if c["op"] == "paged":
        out = torch.empty(c["B"], c["H"], c["D"], dtype=torch.float64, device=DEV)
        for b, n in enumerate(lens):
            rows = torch.arange(n, device=DEV)
            rows = rows[(rows < c["sinks"]) | (rows >= n - c["W"])] if c["W"] else rows
            page = s["table"][b].long()[rows // c["page"]]
            k = s["k_cache"][page, :, rows % c["page"]].double()
            v = s["v_cache"][page, :, rows % c["page"]].double()
            for h in range(c["H"]):
                w = torch.softmax(torch.mv(k[:, h // G], s["q"][b, h].double()) * scale, 0)
                out[b, h] = torch.mv(v[:, h // G].T, w)
        return out
    first = c["Sk"] - c["Sq"]
    shape = (c["B"], c["H"], c["Sq"])
    like = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=DEV)  # noqa: E731
    o, lse = like(s["q"]), torch.full(shape, -math.inf, dtype=torch.float64, device=DEV)
    dq, dk, dv = like(s["q"]), like(s["k"]), like(s["v"])
    far = torch.arange(c["Sk"], device=DEV)
    for b, n in enumerate(lens):
        if n <= first:
            continue
        gap = torch.arange(first, n, device=DEV)[:, None] - far[:n]
        hidden = (gap < 0) | ((gap >= c["W"]) & (far[:n] >= c["sinks"])) if c["W"] else gap < 0
        for h in range(c["H"]):
            q = s["q"][b, h, : n - first].double()
            k, v = s["k"][b, h // G, :n].double(), s["v"][b, h // G, :n].double()
            x = (q @ k.T * scale).masked_fill(hidden, -math.inf)
            if c["op"] == "window":
                lse[b, h, : n - first] = torch.logsumexp(x, 1)
                o[b, h, : n - first] = torch.softmax(x, 1) @ v
                continue
            p = torch.exp(x - s["lse"][b, h, : n - first].double()[:, None])
            g = s["do"][b, h, : n - first].double()
            t = p * (g @ v.T - (g * s["o"][b, h, : n - first].double()).sum(1, keepdim=True)) * scale
            dq[b, h, : n - first] = t @ k
            dk[b, h // G, :n] += t.T @ q
            dv[b, h // G, :n] += p.T @ g
    return (o, lse) if c["op"] == "window" else (dq, dk, dv)
