"""Windowed and paged attention in f16 where one key (a sink with a value near zero) takes
nearly all of the softmax: the other weights are small, and the output is theirs alone.

A weight is raised by 2^7 before it is rounded to f16, so it is off by half a step, u relative,
or by 2^-25 / 2^7 = 2^-32 of the largest; the fp32 parts as in attention_ref.py."""
import pytest
import torch

import attention_ref as ref
from attention_ref import F, Z
from gomlx_hip import ops

pytestmark = pytest.mark.gpu

U, A = 2.0 ** -11, 2.0 ** -25


def forward(q, k, v, scale, see):
    """(o, its bound) in float64."""
    D = q.shape[3]
    q = q.double()
    k, v = (t.double().repeat_interleave(q.shape[1] // t.shape[1], 1) for t in (k, v))
    x = (q @ k.mT * scale).masked_fill(~see, -torch.inf)
    p = torch.softmax(x, -1)
    o = p @ v
    size = (q.abs() @ k.abs().mT * scale).masked_fill(~see, 0).amax()
    e = 4 * (D + 4) * F * size + 2.0 ** -20 + see.shape[-1] * F
    small = 2.0 ** -32 * p.amax(-1, keepdim=True) + Z
    return o, (U + e) * (p @ v.abs()) + U * o.abs() + A + small * (see.double() @ v.abs())


def _operands(cuda, B, H, Hkv, Sq, Sk, D, gap):
    """Scores of a sink, key 0, that lie `gap` above the others' in base 2."""
    g = torch.Generator(device=cuda).manual_seed(D + Sk)
    q = torch.randn((B, H, Sq, D), generator=g, device=cuda) / 4
    k = torch.randn((B, Hkv, Sk, D), generator=g, device=cuda)
    v = torch.randn((B, Hkv, Sk, D), generator=g, device=cuda) * 1024
    q[..., 0], k[..., 0], k[:, :, 0, 0], v[:, :, 0] = 8.0, 0.0, gap * 0.6931 / (8 * D ** -0.5), 0.0
    return q.half(), k.half(), v.half()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("gap", [6, 14, 20])
@pytest.mark.parametrize("H,Hkv,Sq,Sk", [(2, 1, 40, 300), (64, 16, 257, 257), (32, 32, 1024, 1024)])
def test_window(cuda, D, gap, H, Hkv, Sq, Sk):
    q, k, v = _operands(cuda, 2, H, Hkv, Sq, Sk, D, gap)
    see = ref.visible(2, Sq, Sk, Sk - Sq, 100, 2, device=cuda)
    got, lse = ops.sdpa_window(q, k, v, D ** -0.5, 100, 2, with_lse=True)
    o, bound = forward(q, k, v, D ** -0.5, see)
    ref.within(got, o, bound, "o")
    _, want, _, bl = ref.forward(q, k, v, D ** -0.5, see)
    ref.within(lse, want, bl, "lse")


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("gap", [6, 14, 20])
@pytest.mark.parametrize("split", [False, True])
def test_paged(cuda, D, gap, split):
    B, H, Hkv, n, page = 2, 8, 2, 1600, 16
    q, k, v = _operands(cuda, B, H, Hkv, 1, n, D, gap)
    kc, vc = (t.transpose(1, 2).reshape(B * n // page, page, Hkv, D).transpose(1, 2) for t in (k, v))
    table = torch.arange(B * n // page, dtype=torch.int32, device=cuda).view(B, -1)
    lens = torch.full((B,), n, dtype=torch.int32, device=cuda)
    got = ops.sdpa_paged(q[:, :, 0], kc, vc, table, lens, D ** -0.5, 900, 2, split=split)
    o, bound = forward(q, k, v, D ** -0.5, ref.visible(B, 1, n, n - 1, 900, 2, device=cuda))
    ref.within(got[:, :, None], o, bound, "o")
