"""Strides of axes of one entry, which address nothing: any that is not negative will do, and
the values are those of ordinary strides."""
import pytest
import torch

from gomlx_hip import ops

pytestmark = pytest.mark.gpu


def _odd(t):
    """The same values, axes of one entry (but the head dim) at a stride of 13 or 2^40 + 5."""
    st = [s if n != 1 or i == t.dim() - 1 else (13, (1 << 40) + 5)[i % 2] for i, (n, s) in enumerate(zip(t.shape, t.stride()))]
    return t.as_strided(t.shape, st)


def _rand(cuda, shape, dt, seed=0):
    return torch.randn(shape, generator=torch.Generator(device=cuda).manual_seed(seed), device=cuda).to(dt)


@pytest.mark.parametrize("dt,D", [(torch.bfloat16, 128), (torch.float16, 40), (torch.float32, 64)])
@pytest.mark.parametrize("B,H,Hkv,Sq,Sk", [(1, 1, 1, 1, 1), (1, 4, 1, 1, 90), (1, 1, 1, 70, 70), (3, 2, 1, 1, 1), (1, 4, 2, 1, 33)])
def test_window(cuda, dt, D, B, H, Hkv, Sq, Sk):
    q, do = (_rand(cuda, (B, H, Sq, D), dt, i) for i in range(2))
    k, v = (_rand(cuda, (B, Hkv, Sk, D), dt, 2 + i) for i in range(2))
    o, lse = ops.sdpa_window(q, k, v, 0.2, 30, 2, with_lse=True)
    want = ops.sdpa_window_grad(do, q, k, v, o, lse, 0.2, 30, 2)
    o2, lse2 = _odd(torch.zeros_like(o)), torch.zeros_like(lse)
    ops.sdpa_window(_odd(q), _odd(k), _odd(v), 0.2, 30, 2, out=o2, lse=lse2)
    assert torch.equal(o2, o) and torch.equal(lse2, lse)
    outs = [_odd(torch.zeros_like(t)) for t in want]
    ops.sdpa_window_grad(_odd(do), _odd(q), _odd(k), _odd(v), o2, lse2, 0.2, 30, 2, outs=outs)
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("dt,D", [(torch.bfloat16, 128), (torch.float32, 36)])
@pytest.mark.parametrize("B,H,Hkv,S,pages,page,per", [(1, 1, 1, 1, 1, 1, 1), (1, 4, 1, 5, 6, 16, 4), (2, 2, 2, 1, 9, 1, 3),
                                                      (1, 2, 2, 20, 1, 64, 1), (3, 1, 1, 1, 700, 16, 200)])
def test_paged(cuda, dt, D, B, H, Hkv, S, pages, page, per):
    kc, vc = (_rand(cuda, (pages, Hkv, page, D), dt, i) for i in range(2))
    k, v = (_rand(cuda, (B, Hkv, S, D), dt, 2 + i) for i in range(2))
    q = _rand(cuda, (B, H, D), dt, 5)
    table = torch.arange(B * per, dtype=torch.int32, device=cuda).view(B, per) % pages
    starts = torch.zeros(B, dtype=torch.int32, device=cuda)
    k2, v2 = _odd(kc.clone()), _odd(vc.clone())
    ops.kv_append(k, v, kc, vc, table, starts)
    ops.kv_append(_odd(k), _odd(v), k2, v2, table, starts)
    assert torch.equal(k2, kc) and torch.equal(v2, vc)
    lens = torch.full((B,), per * page, dtype=torch.int32, device=cuda)
    want = ops.sdpa_paged(q, kc, vc, table, lens, 0.2)
    out = _odd(torch.zeros_like(q))
    ops.sdpa_paged(_odd(q), k2, v2, table, lens, 0.2, out=out)
    assert torch.equal(out, want)
