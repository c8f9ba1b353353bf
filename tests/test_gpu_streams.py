"""Calls on a stream that is not torch's current one, with outputs and workspaces of their
own: memory that the current stream freed with work still queued on it is not handed to
them, and what they returned, once freed, is not handed out while the current stream still
reads it."""
import pytest
import torch

from gomlx_hip import ops

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _rand(cuda, *shape, dt=BF16, seed=0):
    return torch.randn(shape, generator=torch.Generator(device=cuda).manual_seed(seed), device=cuda).to(dt)


def _window(cuda):
    q, k, v = (_rand(cuda, 2, 8, 300, 128, seed=i) for i in range(3))
    return lambda s: ops.sdpa_window(q, k, v, 0.09, 100, 4, with_lse=True, stream=s)


def _grad(cuda):
    q, k, v, do = (_rand(cuda, 2, 8, 300, 128, seed=i) for i in range(4))
    o, lse = ops.sdpa_window(q, k, v, 0.09, 100, 4, with_lse=True)
    return lambda s: ops.sdpa_window_grad(do, q, k, v, o, lse, 0.09, 100, 4, stream=s)


def _paged(cuda):
    kc, vc = _rand(cuda, 200, 8, 16, 128, seed=1), _rand(cuda, 200, 8, 16, 128, seed=2)
    table = torch.arange(200, dtype=torch.int32, device=cuda).view(2, 100)
    lens = torch.tensor([1600, 901], dtype=torch.int32, device=cuda)
    q = _rand(cuda, 2, 32, 128)
    return lambda s: (ops.sdpa_paged(q, kc, vc, table, lens, 0.09, stream=s),)


def _sdpa(cuda):
    q, k, v = _rand(cuda, 1, 8, 1, 128), _rand(cuda, 1, 8, 4096, 128, seed=1), _rand(cuda, 1, 8, 4096, 128, seed=2)
    assert ops.sdpa_workspace(q, 8, 4096, False) is not None
    return lambda s: (ops.sdpa(q, k, v, 0.09, False, stream=s),)


def _gemm(cuda):
    a, b = _rand(cuda, 64, 8192), _rand(cuda, 8192, 512, seed=1)
    assert ops.gemm_workspace(BF16, BF16, 1, 64, 512, 8192, cuda) is not None
    return lambda s: (ops.gemm(a, b, stream=s), *ops.gemm_grouped(a, [b, b], stream=s))


def _rows(cuda):
    x, t = _rand(cuda, 4096, 1000), _rand(cuda, 500, 512)
    ids = torch.arange(300, dtype=torch.int32, device=cuda)
    return lambda s: (ops.softmax(x, stream=s), ops.rmsnorm(x, stream=s), ops.layernorm(x, stream=s),
                      ops.softmax_axis(x, 0, stream=s), ops.gather_rows(t, ids, stream=s), ops.argminmax(x, 1, stream=s),
                      ops.iota((700, 30), 0, stream=s), ops.scale_mask_softmax(x.view(8, 512, 1000), 0.5, False, stream=s),
                      ops.scale_mask_softmax_ex(x.view(2, 4, 512, 1000), 0.5, True, stream=s))


def _queue(x):
    """Some milliseconds of work on the current stream."""
    y = x
    for _ in range(8):
        y = y @ x
    return y


@pytest.mark.parametrize("make", [_window, _grad, _paged, _sdpa, _gemm, _rows])
@pytest.mark.parametrize("handle", ["own", "default"])
def test_memory_follows_the_call(cuda, make, handle):
    print(make.__name__, handle, flush=True)
    call = make(cuda)
    want = call(None)
    big = _rand(cuda, 8192, 8192)
    s, other = torch.cuda.Stream(), torch.cuda.Stream()
    raw = s.cuda_stream if handle == "own" else 0
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        call(None)  # memory of the call's sizes, with the current stream
        torch.cuda.synchronize()
        for _ in range(3):
            # Freed here while writes to it are queued.
            _queue(big)
            freed = [t.fill_(1) for t in call(None)] + [torch.full((1 << n,), -1, dtype=torch.int8, device=cuda)
                                                        for n in range(12, 25)]
            mine = {t.data_ptr() for t in freed}
            del freed
            got = call(raw)
            assert not mine & {t.data_ptr() for t in got}
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            # Read here by queued work, freed, and asked for again there.
            _queue(big)
            read = [t.clone() for t in got]
            mine = {t.data_ptr() for t in got}
            del got
            got = call(raw)
            assert not mine & {t.data_ptr() for t in got}
            for t in got:
                t.record_stream(s if raw else torch.cuda.default_stream())
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(read, want))
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            del got, read
