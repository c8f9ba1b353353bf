"""The windowed attention's gradient in f16 for gradients d_out of any size (a mean loss
gives small ones, loss scaling large ones), against float64.

Bounds as in attention_ref.py, but for the rounding of dS = p (dP - delta) and p to f16: each
value is off by half a step, u relative, or, where it is small, by an absolute part that must
stay far below the largest: 2^-31 of the largest |dS| of its query (dq) or key (dk), as if
that one were raised to 2^6 at least before subnormals' half a step, 2^-25, is taken; and 2^-40
for p.  The outputs are rounded once: u relative or 2^-25."""
import pytest
import torch

import attention_ref as ref
from attention_ref import F, Z
from gomlx_hip import ops

pytestmark = pytest.mark.gpu

U, A = 2.0 ** -11, 2.0 ** -25


def _fold(x, Hkv):
    return x.view(x.shape[0], Hkv, -1, *x.shape[2:]).sum(2)


def gradient(do, q, k, v, o, lse, scale, see):
    """((dq, bound), (dk, bound), (dv, bound)) in float64."""
    H, Hkv, D = q.shape[1], k.shape[1], q.shape[3]
    do, q, o, lse = do.double(), q.double(), o.double(), lse.double()
    k, v = (t.double().repeat_interleave(H // Hkv, 1) for t in (k, v))
    x = (q @ k.mT * scale).masked_fill(~see, -torch.inf)
    p = torch.exp(x - torch.where(lse == -torch.inf, 0.0, lse)[..., None])
    ds = p * (do @ v.mT - (do * o).sum(-1, keepdim=True))
    size = (q.abs() @ k.abs().mT * scale).masked_fill(~see, 0).amax() + lse.abs().nan_to_num(posinf=0.0).amax()
    n = max(see.shape[-2:]) * (H // Hkv)
    e = 4 * (D + 4) * F * size + 2.0 ** -20 + n * F
    ed = (D + 4) * F * (do.abs() @ v.abs().mT + (do * o).abs().sum(-1, keepdim=True))
    t = (U + e) * ds.abs() + p * ed + Z * see
    tq = t + 2.0 ** -31 * ds.abs().amax(-1, keepdim=True) * see
    # (A kv head's sums run over all the heads that share it.)
    most = ds.abs().amax(-2, keepdim=True).view(ds.shape[0], Hkv, -1, 1, ds.shape[-1]).amax(2)
    tk = t + 2.0 ** -31 * most.repeat_interleave(H // Hkv, 1) * see
    dq, dk, dv = ds @ k * scale, _fold(ds.mT @ q * scale, Hkv), _fold(p.mT @ do, Hkv)
    bq = scale * (tq @ k.abs()) + U * dq.abs() + A
    bk = _fold(scale * (tk.mT @ q.abs()), Hkv) + U * dk.abs() + A
    bv = _fold((U + e) * (p.mT @ do.abs()) + 2.0 ** -40 * (see.double().mT @ do.abs()), Hkv) + U * dv.abs() + A
    return (dq, bq), (dk, bk), (dv, bv)


CASES = [  # (B, H, Hkv, Sq, Sk, q_start, window, sinks, lens)
    (1, 2, 2, 600, 600, 0, 500, 0, None),
    (1, 4, 1, 300, 2100, 1800, 0, 0, None),             # chunks of queries, long lists of keys
    (2, 4, 2, 700, 700, 0, 40, 4, (700, 333)),          # sinks in workgroups of their own
    (4, 64, 16, 257, 257, 0, 200, 4, None),             # grids of many workgroups
    (1, 2, 1, 64, 64, 0, 3, 0, None),                   # large weights
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("size", [2.0 ** -14, 2.0 ** -10, 2.0 ** -6, 1.0, 2.0 ** 10])
def test_gradients_of_any_size(cuda, case, D, size):
    """d_out and, with it, dS from the smallest to the largest; q small and k large (so that
    dq lies inside f16's range) and the other way round."""
    B, H, Hkv, Sq, Sk, start, window, sinks, lens = case
    print(case, D, size, flush=True)
    g = torch.Generator(device=cuda).manual_seed(Sq + D)
    lens = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=cuda)
    see = ref.visible(B, Sq, Sk, start, window, sinks, lens, cuda)
    big = size if size > 1 else 1.0
    for f in (8.0, 1 / 8):
        q = (torch.randn((B, H, Sq, D), generator=g, device=cuda) / f / big).half()
        k = (torch.randn((B, Hkv, Sk, D), generator=g, device=cuda) * f / big).half()
        v = (torch.randn((B, Hkv, Sk, D), generator=g, device=cuda) * (128 if size > 1 else 1)).half()
        do = (torch.randn((B, H, Sq, D), generator=g, device=cuda) * size).half()
        scale = D ** -0.5
        o, lse = ops.sdpa_window(q, k, v, scale, window, sinks, q_start=start, lens=lens, with_lse=True)
        got = ops.sdpa_window_grad(do, q, k, v, o, lse, scale, window, sinks, q_start=start, lens=lens)
        for name, x, (want, bound) in zip(("dq", "dk", "dv"), got, gradient(do, q, k, v, o, lse, scale, see)):
            ref.within(x, want, bound, f"{name} at {f}")


def test_growing_along_the_sequence(cuda):
    """d_out that grows by 2^20 along the queries and values along the keys: the sums' scale
    has to fall again and again, and what came before keeps its bits."""
    B, H, S, D = 1, 4, 1000, 128
    g = torch.Generator(device=cuda).manual_seed(3)
    q, k, v, do = (torch.randn((B, H, S, D), generator=g, device=cuda) for _ in range(4))
    grow = torch.exp2(torch.linspace(-12, 8, S, device=cuda))[:, None]
    for a, b in ((grow, 1.0), (grow.flip(0), 1.0), (1.0, grow), (1.0, grow.flip(0))):
        q2, k2, v2, do2 = q.half(), (k / 16).half(), (v * b).half(), (do * a).half()
        see = ref.visible(B, S, S, 0, 300, 2, device=cuda)
        o, lse = ops.sdpa_window(q2, k2, v2, 0.09, 300, 2, with_lse=True)
        got = ops.sdpa_window_grad(do2, q2, k2, v2, o, lse, 0.09, 300, 2)
        for name, x, (want, bound) in zip(("dq", "dk", "dv"), got, gradient(do2, q2, k2, v2, o, lse, 0.09, see)):
            ref.within(x, want, bound, name)
