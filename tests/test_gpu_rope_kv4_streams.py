"""Rotary positions, the 4-bit cache and log probabilities on a stream that is not torch's current
one, with outputs and workspaces of their own (as test_gpu_streams.py), and captured together
as a step of a server, replayed beside eager calls."""
import pytest
import torch

import test_gpu_streams
from gomlx_hip import ops
from test_gpu_kv4 import cache4, freqs_of, rand, table_of

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _rope(cuda):
    x, freqs = rand(cuda, 2, 8, 300, 128, seed=1), freqs_of(64, cuda)
    pos = torch.randint(0, 10000, (2, 300), device=cuda, dtype=torch.int32)
    return lambda s: (ops.rope(x, pos, freqs, stream=s), ops.rope(x, pos, freqs, interleaved=True, inverse=True, stream=s))


def _append(cuda):
    pages, table = table_of(cuda, 2, 20)
    q, k, v = rand(cuda, 2, 8, 300, 128, seed=1), rand(cuda, 2, 2, 300, 128, seed=2), rand(cuda, 2, 2, 300, 128, seed=3)
    kc, vc = (torch.zeros(pages, 2, 16, 128, dtype=q.dtype, device=cuda) for _ in range(2))
    k4, v4 = (ops.kv4_cache(pages, 16, 2, 128, cuda) for _ in range(2))
    starts, freqs = torch.tensor([3, 15], dtype=torch.int32, device=cuda), freqs_of(64, cuda)
    return lambda s: (ops.kv_append_rope(q, k, v, kc, vc, table, starts, freqs, stream=s),
                      ops.kv4_append_rope(q, k, v, k4, v4, table, starts, freqs, stream=s),
                      *ops.kv4_read(k4, v4, table, 310, starts, stream=s))


def _paged4(cuda):
    pages, table = table_of(cuda, 2, 100)
    kc, vc = cache4(cuda, pages, 16, 8, 128, "head")
    lens = torch.tensor([1600, 901], dtype=torch.int32, device=cuda)
    q = rand(cuda, 2, 32, 128)
    assert ops.sdpa_paged_kv4_workspace(q, kc, table) is not None
    return lambda s: (ops.sdpa_paged_kv4(q, kc, vc, table, lens, 0.09, stream=s),)


def _logprobs(cuda):
    x = rand(cuda, 9, 50001, dt=F32, seed=1)
    ids = torch.arange(9, dtype=torch.int32, device=cuda)
    g = torch.ones(9, device=cuda)
    assert ops.token_logprobs_workspace(x, 5) is not None
    _, entropy, lse, _, _ = ops.token_logprobs(x, ids)
    return lambda s: (*ops.token_logprobs(x, ids, top=5, stream=s), ops.token_logprobs_grad(x, ids, lse, g, entropy, g, stream=s))


@pytest.mark.parametrize("make", [_rope, _append, _paged4, _logprobs])
@pytest.mark.parametrize("handle", ["own", "default"])
def test_memory_follows_the_call(cuda, make, handle):
    test_gpu_streams.test_memory_follows_the_call(cuda, make, handle)


def test_two_streams_at_once(cuda):
    """Calls on two streams, each with its own outputs and workspace, give what they give alone."""
    calls = [make(cuda) for make in (_rope, _paged4, _logprobs)]
    want = [call(None) for call in calls]
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append([call(None) for call in calls])
    torch.cuda.synchronize()
    for each in got:
        for outs, wants in zip(each, want):
            assert all(torch.equal(a, b) for a, b in zip(outs, wants))


def test_a_captured_step(cuda):
    """One step of a server captured whole (rotation and append into 4 bits, decoding attention, log
    probabilities of the tokens picked), replayed as the sequences grow, beside eager calls on the
    same cache: every replay gives what the eager step gives."""
    B, H, Hkv, D, V, per = 5, 16, 2, 128, 20000, 60
    pages, table = table_of(cuda, B, per)
    k4, v4 = cache4(cuda, pages, 16, Hkv, D, "head")
    head, freqs = rand(cuda, H * D, V, seed=5), freqs_of(D // 2, cuda)
    at = torch.tensor([0, 7, 500, 901, 63], dtype=torch.int32, device=cuda)
    qkv = rand(cuda, B, H + 2 * Hkv, 1, D, seed=6)
    q, k, v = qkv.split([H, Hkv, Hkv], 1)

    def step(starts, lens):
        turned = ops.kv4_append_rope(q, k, v, k4, v4, table, starts, freqs)
        o = ops.sdpa_paged_kv4(turned[:, :, 0], k4, v4, table, lens, 0.09, 512, 4)
        logits = ops.gemm(o.view(B, H * D), head)
        return o, *ops.token_logprobs(logits, ops.argminmax(logits, 1), top=3)

    lens = at + 1
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(at, lens)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step(at, lens)
    for i in range(4):
        qkv.copy_(rand(cuda, B, H + 2 * Hkv, 1, D, seed=7 + i))
        g.replay()
        got = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, step(at, lens)))
        torch.cuda.synchronize()
        at += 1
        lens += 1
