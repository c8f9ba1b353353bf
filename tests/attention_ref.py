"""Sliding-window attention with sinks in float64, with the bound that each output's
rounding error obeys.  Shared by the tests of the windowed and the paged attention.

With u = finfo(type).eps / 2 (a rounding is off by at most u relative to the value), f =
2^-24 (fp32) and, for f16, a = 2^-25 (half a step of its subnormals):

* a score of D fp32 products and sums, scaled, is off by at most es = (D + 4) f max(scale
  sum |q| |k|) and its exponent by as much again in the multiply-add and the base-2
  exponential's argument (|s| <= max scale sum |q| |k|, log-sum-exp likewise): a weight
  is off by e = 4 es + 2^-20 relative (the 2^-20: exp2, sum of n weights and the division);
* o = sum p v: p is rounded once (16-bit types), o once:
    (u + e) sum p |v| + u |o|   (+ a sum |v| + a: f16's small weights, off by a while the largest is 1)
* dv = sum p do: (u + e) sum p |do| + u |dv|  (+ 2^-8 a sum |do| + a)
* dS = p (dP - delta): dP and delta are D fp32 products each, off by ed = (D + 4) f (sum |do| |v| + sum |do| |o|);
  with t = (u + e) |dS| + p ed (+ a / scale):  dq: scale sum t |k| + u |dq| (+ a), dk: scale sum t |q| + u |dk| (+ a)

* fp32's own smallest normal value z = 2^-126: the base-2 exponential flushes a weight
  below it to zero, and so may the products and sums, so a weight is off by z more, dS by
  z (|dP| + |delta| + 1), and each of an output's n terms and the output itself by z.

Each sum of n terms in fp32 adds n f of the sum of magnitudes.  fp32 outputs: u = f."""
import torch

F = 2.0 ** -24
Z = 2.0 ** -126


def visible(B, Sq, Sk, q_start, window, sinks, lens=None, device="cpu"):
    """[B, 1, Sq, Sk]: which keys a query sees."""
    pos = torch.arange(q_start, q_start + Sq, device=device)[:, None]
    key = torch.arange(Sk, device=device)[None, :]
    see = (key <= pos) & ((key > pos - (window or Sk + 1)) | (key < sinks))
    n = torch.full((B,), Sk, device=device) if lens is None else lens.to(device).long().clamp(0, Sk)
    return (see[None] & (pos < n[:, None, None]) & (key < n[:, None, None]))[:, None]


def _units(dt):
    u = torch.finfo(dt).eps / 2
    return u, 2.0 ** -25 if dt == torch.float16 else 0.0


def _expand(k, H):
    return k.repeat_interleave(H // k.shape[1], 1)


def _fold(x, Hkv):
    return x.view(x.shape[0], Hkv, -1, *x.shape[2:]).sum(2)


def forward(q, k, v, scale, see):
    """(o, lse, bound of o, bound of lse) in float64; values at padding must be finite."""
    dt, D = q.dtype, q.shape[3]
    u, a = _units(dt)
    q, k, v = q.double(), _expand(k.double(), q.shape[1]), _expand(v.double(), q.shape[1])
    x = (q @ k.mT * scale).masked_fill(~see, -torch.inf)
    lse = torch.logsumexp(x, -1)
    p = torch.exp(x - torch.where(lse == -torch.inf, 0.0, lse)[..., None])
    o = p @ v
    size = (q.abs() @ k.abs().mT * scale).masked_fill(~see, 0).amax() if see.any() else torch.zeros((), device=q.device)
    n = see.shape[-1]
    e = 4 * (D + 4) * F * size + 2.0 ** -20 + n * F
    r = 0.0 if dt == torch.float32 else u
    bo = (r + e) * (p @ v.abs()) + u * o.abs() + a * (see.double() @ v.abs() + 1)
    bo = bo + Z * (see.double() @ (v.abs() + 1) + 1)
    return o, lse, bo, e + 4 * F * lse.abs().nan_to_num(posinf=0.0)


def gradient(do, q, k, v, o, lse, scale, see):
    """((dq, bound), (dk, bound), (dv, bound)) in float64, from the given o and lse."""
    dt, H, Hkv, D = q.dtype, q.shape[1], k.shape[1], q.shape[3]
    u, a = _units(dt)
    do, q, o = do.double(), q.double(), o.double()
    k, v = _expand(k.double(), H), _expand(v.double(), H)
    lse = lse.double()
    x = (q @ k.mT * scale).masked_fill(~see, -torch.inf)
    p = torch.exp(x - torch.where(lse == -torch.inf, 0.0, lse)[..., None])
    ds = p * (do @ v.mT - (do * o).sum(-1, keepdim=True))
    size = (q.abs() @ k.abs().mT * scale).masked_fill(~see, 0).amax() + lse.abs().nan_to_num(posinf=0.0).amax()
    n = max(see.shape[-2:]) * (H // Hkv)
    e = 4 * (D + 4) * F * size + 2.0 ** -20 + n * F
    ed = (D + 4) * F * (do.abs() @ v.abs().mT + (do * o).abs().sum(-1, keepdim=True))
    r = 0.0 if dt == torch.float32 else u
    t = (r + e) * ds.abs() + p * ed + (a / scale) * see
    t = t + Z * ((do @ v.mT).abs() + (do * o).sum(-1, keepdim=True).abs() + 1) * see
    dq, dk, dv = ds @ k * scale, _fold(ds.mT @ q * scale, Hkv), _fold(p.mT @ do, Hkv)
    bq = scale * (t @ k.abs()) + u * dq.abs() + a + Z * (n + 1)
    bk = _fold(scale * (t.mT @ q.abs()), Hkv) + u * dk.abs() + a + Z * (n + 1)
    bv = _fold((r + e) * (p.mT @ do.abs()) + (a * 2.0 ** -8 + Z) * (see.double().mT @ do.abs()), Hkv)
    bv = bv + u * dv.abs() + a + Z * (n + 1)
    return (dq, bq), (dk, bk), (dv, bv)


def within(got, ref, bound, what=""):
    """Whether every value lies within its bound (or is the same infinity)."""
    got = got.double()
    bad = ~((got - ref).abs() <= bound) & ~(got == ref)
    if bad.any():
        i = tuple(int(j) for j in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off, first at {i}: "
                             f"{got[i].item()} for {ref[i].item()}, bound {bound[i].item()}")
