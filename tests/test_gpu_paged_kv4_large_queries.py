"""Decoding over 4 bits with fp32 queries up to the type's largest values: above the largest bf16, their
first bf16 part must not round to infinity."""
import pytest
import torch

from gomlx_hip import ops
from test_gpu_kv4 import cache4, table_of
from test_gpu_paged_kv4 import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("split", [False, True])
def test_queries_above_the_largest_bf16(cuda, D, split):
    """One value of a row, with keys of 0, 1/2 and 1 of both signs, so that products and sums are
    finite; times 2^-126 the scores are of order 4."""
    B, H, Hkv, page, per = 2, 8, 2, 16, 40
    pages, table = table_of(cuda, B, per)
    kc, vc = cache4(cuda, pages, page, Hkv, D, "head")
    sizes = torch.tensor([0, 1, 2, 8, 9, 10], dtype=torch.uint8, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    lo, hi = (sizes[torch.randint(0, 6, kc[0].shape, generator=g, device=cuda)] for _ in range(2))
    kc[0].copy_(lo | hi << 4)
    kc[1].fill_(127)
    most = torch.finfo(torch.float32).max
    q = torch.zeros((B, H, D), device=cuda)
    for h, value in enumerate((most, -most, 3.4e38, -3.4e38, 3.397e38, 3.389e38, 1.0, most)):
        q[:, h, 5 * h] = value
    lens = torch.tensor([per * page - 3, 77], dtype=torch.int32, device=cuda)
    got = ops.sdpa_paged_kv4(q, kc, vc, table, lens, 2.0 ** -126, split=split)
    assert got.isfinite().all()
    check(q, kc, vc, table, lens, 2.0 ** -126, 0, 0, got)
    # Infinite and NaN queries stay what they are, in their own rows.
    q2 = q.clone()
    q2[0, 1, 3], q2[1, 4, 0] = float("inf"), float("nan")
    bad = ops.sdpa_paged_kv4(q2, kc, vc, table, lens, 2.0 ** -126, split=split)
    assert bad[0, 1].isnan().all() and bad[1, 4].isnan().all()
    bad[0, 1], bad[1, 4] = got[0, 1], got[1, 4]
    assert torch.equal(bad, got)
