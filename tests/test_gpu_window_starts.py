"""The windowed attention's gradient for queries that begin inside a tile, without sinks and
with finite windows, in grids whose lists of tiles are dealt out in chunks."""
import pytest
import torch

from test_gpu_window_attention import check, lens_of, run_both, tensors

pytestmark = pytest.mark.gpu

CASES = [  # (B, H, Hkv, Sq, Sk, q_start, window, sinks, lens)
    (1, 4, 1, 200, 201, 1, 3, 0, None),
    (1, 8, 2, 200, 300, 100, 50, 0, None),
    (2, 4, 4, 1615, 1621, 6, 302, 0, None),
    (1, 2, 2, 130, 146, 16, 34, 0, None),
    (1, 4, 1, 257, 288, 31, 33, 0, None),
    (2, 4, 1, 100, 190, 63, 2, 0, (190, 101)),
    (1, 3, 3, 33, 127, 94, 66, 0, None),
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dt,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64), (torch.bfloat16, 256)])
def test_queries_begin_inside_a_tile(cuda, case, dt, D):
    print(case, dt, D, flush=True)
    q, k, v, do = tensors(cuda, case, dt, D)
    scale = D ** -0.5
    check(cuda, case, q, k, v, do, scale, *run_both(q, k, v, do, scale, case, lens_of(cuda, case)))
