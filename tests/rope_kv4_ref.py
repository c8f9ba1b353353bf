"""Rotary positions, the 4-bit cache's values and tokens' log probabilities in float64, with the
bounds that their rounding errors obey.  u = finfo(type).eps / 2 (a rounding is off by at most u
relative to the value), F = 2^-24 (fp32), a = 2^-25 (half a step of f16's subnormals).

* rotation: cos and sin are rounded to fp32 (F each; before that they are off by less than 2^-40
  for positions up to 2^20), two products and their sum round once each:
    3.1 F (|x cos| + |y sin|) + 2^-40 (|x| + |y|), then the output's u
* log-sum-exp of n logits x = scale * logit with largest m, by lanes that add at most `adds`
  terms each and are joined in 8 more steps: a product with log2 e is off by 2 F |x|, the
  multiply-add by F |x - m|, a base-2 exponential by 2^-23, a sum by F for each addition:
    el = (adds + 40) F + 4 F max |x| + F E|x - m|, over p, and 2 F |lse| for the result;
  the entropy is the same sum with terms weighted by |x - m|, which E|x - m| (at most log n +
  the entropy) bounds beside the rounding:
    eh = el (2 + E|x - m|) + 4 F (entropy + log n)
* gradient p (A + B t) + [v = id] C, t = x - lse: t is off by F |t|, the exponent by 2 F |t|, p by
  2^-23 and both, A by 2 F of its terms, the products and sums by F each:
    p (|A'| + |B t|) F (4 |t| + 12) + 4 F |C| + 2^-126 (|A'| + |B t|), then the output's u"""
import math

import torch

F = 2.0 ** -24
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def units(dt):
    return (0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2), (2.0 ** -25 if dt == torch.float16 else 0.0)


def rotate(x, positions, freqs, sections=None, interleaved=False, inverse=False):
    """(turned, bound) of x [B, H, S, D] in float64; positions [axes, B, S] or [B, S]."""
    dt = x.dtype
    u, a = units(dt)
    positions = positions[None] if positions.dim() == 2 else positions
    half = freqs.shape[0]
    sections = [half] if sections is None else sections
    angle = torch.empty((*positions.shape[1:], half), dtype=torch.float64, device=x.device)
    at = 0
    for axis, n in enumerate(sections):
        angle[..., at:at + n] = positions[axis].double()[..., None] * freqs[at:at + n].double()
        at += n
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    s = -s if inverse else s
    y = x.double().clone()
    bound = u * y.abs() * 0
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    p, q = x.double()[..., first], x.double()[..., second]
    y[..., first], y[..., second] = p * c - q * s, p * s + q * c
    far = 2.0 ** -40 * (p.abs() + q.abs())
    bound[..., first] = 3.1 * F * ((p * c).abs() + (q * s).abs()) + far
    bound[..., second] = 3.1 * F * ((p * s).abs() + (q * c).abs()) + far
    turned = torch.arange(x.shape[-1], device=x.device) < 2 * half
    return y, bound + (u * (y.abs() + bound) + a) * turned


# ---------------------------------------------------------------- 4 bits
def encode(x):
    """(codes [..., D], scale bytes [..., D / 32]) by definition: the least power of two of which
    32 values are at most 6, the nearest of the eight sizes, ties to the even code."""
    g = x.double().unflatten(-1, (-1, 32))
    most = g.abs().amax(-1, keepdim=True)
    finite = torch.isfinite(g).all(-1, keepdim=True)
    steps = torch.tensor([2.0 ** n for n in range(-126, 126)], dtype=torch.float64, device=x.device)
    scale = (most > 6 * steps[:-1]).sum(-1, keepdim=True)
    y = g.abs() / steps[scale]
    sizes = torch.tensor(MAGNITUDES, dtype=torch.float64, device=x.device)
    code = torch.zeros_like(y, dtype=torch.long)
    for i in range(7):
        mid = (sizes[i] + sizes[i + 1]) / 2
        code = torch.where((y > mid) | ((y == mid) & (i % 2 == 1)), i + 1, code)
    code = code + 8 * torch.signbit(g).long()
    return code.flatten(-2), torch.where(finite, scale + 1, 255).squeeze(-1)


def decode(codes, scales, D):
    """float64 values of codes [..., D / 2] and scales [..., bytes]."""
    sizes = torch.tensor([*MAGNITUDES, *(-m for m in MAGNITUDES)], dtype=torch.float64, device=codes.device)
    x = sizes[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()].unflatten(-1, (-1, 32))
    steps = torch.tensor([2.0 ** (n - 127) for n in range(255)] + [math.nan], dtype=torch.float64, device=codes.device)
    return (x * steps[scales[..., :D // 32].long()][..., None]).flatten(-2)


# ---------------------------------------------------------------- log probabilities
def f32(scale):
    """A scale as the entry points take it."""
    return torch.tensor(scale, dtype=torch.float32).item()


def logprobs(logits, ids, scale, adds):
    """((logp, bound), (entropy, bound), (lse, bound)) of rows without NaN and +infinity."""
    x = logits.double() * f32(scale)
    V = x.shape[1]
    m = x.amax(1, keepdim=True)
    lse = torch.logsumexp(x, 1)
    none = m[:, 0] == -torch.inf
    p = torch.where(x == -torch.inf, 0.0, torch.exp(x - torch.where(none, 0.0, lse)[:, None]))
    far = torch.where(x == -torch.inf, 0.0, m - x)
    lp = torch.where(x == -torch.inf, 0.0, x - lse[:, None])
    H = -(p * torch.where(p > 0, lp, 0.0)).sum(1)
    mean = (p * far).sum(1)
    big = torch.where(x == -torch.inf, 0.0, x.abs()).amax(1)
    el = (adds + 40) * F + 4 * F * big + F * mean
    there = (ids >= 0) & (ids < V)
    at = ids.long().clamp(0, V - 1)[:, None]
    logp = torch.where(there, torch.where(none, -torch.inf, (x - lse[:, None]).gather(1, at)[:, 0]), 0.0)
    bl = el + 2 * F * lse.abs().nan_to_num(posinf=0.0)
    return (logp, (el + 4 * F * logp.abs().nan_to_num(posinf=0.0)) * there), \
        (H, el * (2 + mean) + 4 * F * (H + math.log(V))), (lse, bl)


def top(logits, k):
    """Indices of the k largest logits of a row: by value, then by index; NaN above all."""
    out = []
    for row in logits.double().tolist():
        key = [(0, 0.0) if v != v else (1, -v) for v in row]
        out.append(sorted(range(len(row)), key=lambda i: (key[i], i))[:k])
    return torch.tensor(out, dtype=torch.int32).view(len(out), k)


def gradient(logits, ids, lse, entropy, d_logp, d_entropy, scale):
    """(d_logits, bound) from the given lse and entropy."""
    u, a = units(logits.dtype)
    V, scale = logits.shape[1], f32(scale)
    x = logits.double() * scale
    none = (lse == -torch.inf)[:, None]
    t = torch.where(none | (x == -torch.inf), -300.0, x - lse.double()[:, None])
    p = torch.where(none | (x == -torch.inf), 0.0, torch.exp(t))
    there = ((ids >= 0) & (ids < V))[:, None]
    g = torch.where(there, d_logp.double()[:, None], 0.0) if d_logp is not None else torch.zeros_like(t[:, :1])
    h = d_entropy.double()[:, None] if d_entropy is not None else torch.zeros_like(g)
    H = entropy.double()[:, None] if entropy is not None else torch.zeros_like(g)
    hit = torch.zeros_like(t).scatter_(1, ids.long().clamp(0, V - 1)[:, None], 1.0) * there
    hit = torch.where(none, 0.0, hit)
    d = scale * (g * (hit - p) - h * p * (t + H))
    size = scale * (g.abs() + (h * H).abs() + (h * t).abs())
    bound = p * size * F * (4 * t.abs() + 12) + 4 * F * scale * g.abs() * hit + 2.0 ** -126 * size
    bound = bound + F * d.abs()
    return d, bound + u * (d.abs() + bound) + a
