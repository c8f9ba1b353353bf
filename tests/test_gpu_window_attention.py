"""Sliding-window attention with sinks and its gradient (ghip_sdpa_window_fwd / _bwd)
against float64, value by value within the rounding bounds of attention_ref.py."""
import pytest
import torch

import attention_ref as ref
from gomlx_hip import ops
from gomlx_hip._lib import BackendError

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [(BF16, 128), (BF16, 64), (F16, 128), (F16, 40), (BF16, 80), (BF16, 256), (F16, 200), (F32, 64), (F32, 100),
         (F32, 128), (F32, 4)]

CASES = [  # (B, H, Hkv, Sq, Sk, q_start, window, sinks, lens)
    (1, 1, 1, 1, 1, 0, 1, 0, None),
    (1, 2, 2, 130, 130, 0, 1, 0, None),           # a window of the query's own key: o = v
    (2, 2, 2, 257, 257, 0, 64, 4, None),          # windows of whole tiles
    (1, 2, 1, 300, 300, 0, 65, 1, None),
    (1, 2, 1, 300, 300, 0, 63, 64, None),         # sinks end with a tile
    (1, 1, 1, 333, 333, 0, 30, 65, None),         # sinks of two tiles, a gap behind them
    (1, 3, 3, 200, 200, 0, 0, 0, None),           # no bound: causal
    (1, 2, 2, 190, 190, 0, 500, 7, None),         # a window longer than the keys
    (1, 4, 1, 37, 300, 263, 48, 2, None),         # a prompt's last chunk
    (1, 2, 2, 37, 300, 100, 90, 70, None),        # a chunk in the middle, keys behind it
    (2, 8, 2, 1, 700, 699, 100, 4, None),         # a single token
    (5, 4, 2, 150, 150, 0, 40, 3, (150, 1, 0, 64, 65)),
    (4, 2, 2, 70, 200, 130, 50, 4, (200, 130, 131, 7)),   # chunk rows past the length, whole chunks of padding
    (3, 2, 1, 129, 129, 0, 0, 0, (1000, -3, 128)),        # lengths out of range are clamped
    (1, 6, 2, 600, 600, 0, 200, 130, None),       # sinks across the key blocks of the gradient
    (1, 2, 1, 1100, 1100, 0, 256, 4, None),
    # grids of many workgroups
    (2, 64, 16, 257, 257, 0, 64, 4, None),
    (4, 64, 64, 130, 200, 70, 50, 4, (200, 130, 131, 7)),
    (1, 64, 8, 600, 600, 0, 200, 130, None),
    (2, 48, 48, 400, 400, 0, 0, 0, (400, 333)),
]


def tensors(cuda, case, dt, D, seed=0):
    B, H, Hkv, Sq, Sk = case[:5]
    g = torch.Generator(device=cuda).manual_seed(1000 + seed + Sq + 7 * Sk + D)
    q, do = (torch.randn((B, H, Sq, D), generator=g, device=cuda).to(dt) for _ in range(2))
    k, v = (torch.randn((B, Hkv, Sk, D), generator=g, device=cuda).to(dt) for _ in range(2))
    return q, k, v, do


def lens_of(cuda, case):
    return None if case[8] is None else torch.tensor(case[8], dtype=torch.int32, device=cuda)


def run_both(q, k, v, do, scale, case, lens):
    _, _, _, _, _, start, window, sinks, _ = case
    o, lse = ops.sdpa_window(q, k, v, scale, window, sinks, q_start=start, lens=lens, with_lse=True)
    return o, lse, ops.sdpa_window_grad(do, q, k, v, o, lse, scale, window, sinks, q_start=start, lens=lens)


def check(cuda, case, q, k, v, do, scale, o, lse, grads):
    B, H, Hkv, Sq, Sk, start, window, sinks, _ = case
    see = ref.visible(B, Sq, Sk, start, window, sinks, lens_of(cuda, case), cuda)
    eo, elser, bo, bl = ref.forward(q, k, v, scale, see)
    ref.within(o, eo, bo, "o")
    ref.within(lse, elser, bl, "lse")
    for name, got, (want, bound) in zip(("dq", "dk", "dv"), grads, ref.gradient(do, q, k, v, o, lse, scale, see)):
        ref.within(got, want, bound, name)


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dt,D", TYPES)
def test_window_attention_and_gradient(cuda, case, dt, D):
    print(case, dt, D, flush=True)
    q, k, v, do = tensors(cuda, case, dt, D)
    scale = D ** -0.5
    check(cuda, case, q, k, v, do, scale, *run_both(q, k, v, do, scale, case, lens_of(cuda, case)))


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F32, 64), (BF16, 96)])
def test_strides(cuda, dt, D):
    """[B, S, H, D] storage, rows wider than the head dim, and a kv head all heads share
    through a stride of 0."""
    case = (2, 4, 2, 150, 150, 0, 50, 3, None)
    q, k, v, do = tensors(cuda, case, dt, D)
    scale = D ** -0.5
    bshd = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, do)]
    wide = [torch.cat([t, torch.full_like(t, float("nan"))], 3)[..., :D] for t in (q, k, v, do)]
    want = run_both(q, k, v, do, scale, case, None)
    for ts in (bshd, wide):
        got = run_both(*ts, scale, case, None)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert all(torch.equal(a, b) for a, b in zip(got[2], want[2]))
    k1, v1 = k[:, :1].contiguous(), v[:, :1].contiguous()
    kx, vx = k1.expand(-1, 2, -1, -1), v1.expand(-1, 2, -1, -1)
    got = run_both(q, kx, vx, do, scale, case, None)
    check(cuda, case, q, kx, vx, do, scale, *got)
    # outputs in the caller's [B, S, H, D] storage
    outs = [torch.empty_like(t) for t in (bshd[0], bshd[1], bshd[2])]
    o = torch.empty_like(bshd[0])
    lse = torch.empty(q.shape[:3], device=cuda)
    ops.sdpa_window(q, k, v, scale, 50, 3, q_start=0, out=o, lse=lse)
    ops.sdpa_window_grad(do, q, k, v, o, lse, scale, 50, 3, q_start=0, outs=outs)
    assert torch.equal(o, want[0]) and all(torch.equal(a, b) for a, b in zip(outs, want[2]))


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F32, 64), (F16, 256)])
@pytest.mark.parametrize("fill", [float("nan"), float("inf"), None])
def test_padding_reaches_nothing(cuda, dt, D, fill):
    """Rows of q, k, v, o, d_out past a length: NaN, infinities, the type's lowest value."""
    case = (4, 4, 2, 140, 140, 0, 33, 2, (140, 65, 0, 3))
    q, k, v, do = tensors(cuda, case, dt, D)
    scale, lens = D ** -0.5, lens_of(cuda, case)
    fill = torch.finfo(dt).min if fill is None else fill
    want = run_both(q, k, v, do, scale, case, lens)
    q2, k2, v2, do2, o2 = (t.clone() for t in (q, k, v, do, want[0]))
    for b, n in enumerate(case[8]):
        for t in (q2, k2, v2, do2, o2):
            t[b, :, n:] = fill
    o, lse = ops.sdpa_window(q2, k2, v2, scale, 33, 2, q_start=0, lens=lens, with_lse=True)
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    got = ops.sdpa_window_grad(do2, q2, k2, v2, o2, lse, scale, 33, 2, q_start=0, lens=lens)
    assert all(torch.equal(a, b) for a, b in zip(got, want[2]))
    for b, n in enumerate(case[8]):
        assert not o[b, :, n:].any() and torch.isneginf(lse[b, :, n:]).all()
        assert not got[0][b, :, n:].any() and not got[1][b, :, n:].any() and not got[2][b, :, n:].any()


def test_large_scores(cuda):
    """Scores of thousands, falling and rising along the keys: the running maximum moves
    at every tile, or never."""
    case = (1, 2, 2, 256, 256, 0, 100, 4, None)
    for sign in (1.0, -1.0):
        q, k, v, do = tensors(cuda, case, F32, 64)
        q = q.abs() * 4
        k = k.abs() * torch.linspace(0.1, 20, 256, device=cuda)[:, None] * sign
        check(cuda, case, q, k, v, do, 1.0, *run_both(q, k, v, do, 1.0, case, None))


def test_differences(cuda):
    """The gradient against central differences of the forward kernel in float32, summed
    in float64.  With h = 2^-6 the differences' own error is h^2 / 6 of a third derivative
    of the size of the first (4e-5) and the forward's rounding over 2 h (2^-20 / 2^-5 =
    3e-5) times the root of the number of outputs: 1e-3 of the gradient's norm holds both."""
    case = (1, 4, 2, 70, 70, 0, 20, 3, None)
    q, k, v, do = tensors(cuda, case, F32, 64)
    scale, h = 0.125, 2.0 ** -6
    _, _, grads = run_both(q, k, v, do, scale, case, None)

    def loss(*ts):
        return (ops.sdpa_window(*ts, scale, 20, 3, q_start=0).double() * do.double()).sum()

    for i, g in enumerate(grads):
        for seed in range(3):
            d = torch.randn(g.shape, generator=torch.Generator(device=cuda).manual_seed(seed), device=cuda)
            up, down = [q, k, v], [q, k, v]
            up[i], down[i] = up[i] + h * d, down[i] - h * d
            diff = (loss(*up) - loss(*down)) / (2 * h)
            assert abs(diff - (g.double() * d.double()).sum()) <= 1e-3 * g.double().norm()


def test_same_bits_and_streams_and_graph(cuda):
    """Twice the same bits; another stream; captured forward and backward replayed with
    new inputs between eager calls."""
    case = (2, 8, 2, 300, 300, 0, 100, 4, (300, 211))
    q, k, v, do = tensors(cuda, case, BF16, 128)
    scale, lens = 128 ** -0.5, lens_of(cuda, case)
    a, b = run_both(q, k, v, do, scale, case, lens), run_both(q, k, v, do, scale, case, lens)
    flat = lambda r: (r[0], r[1], *r[2])  # noqa: E731
    assert all(torch.equal(x, y) for x, y in zip(flat(a), flat(b)))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c = run_both(q, k, v, do, scale, case, lens)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, y) for x, y in zip(flat(a), flat(c)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run_both(q, k, v, do, scale, case, lens)
    for seed in range(3):
        for t, n in zip((q, k, v, do), tensors(cuda, case, BF16, 128, seed=50 + seed)):
            t.copy_(n)
        graph.replay()
        got = [t.clone() for t in flat(out)]
        torch.cuda.synchronize()
        want = run_both(q, k, v, do, scale, case, lens)
        assert all(torch.equal(x, y) for x, y in zip(got, flat(want)))


@pytest.mark.parametrize("G", [1, 3])
@pytest.mark.parametrize("sinks", [1, 33, 64, 128, 129])
def test_many_sinks(cuda, sinks, G):
    """The gradient's ways of summing sinks' keys: chunks in one to four blocks of 32, and
    beyond 128 sinks whole lists; sequences whose queries end before, inside and behind the
    windows of the sinks' blocks."""
    for lens in (None, (700, 90, 300)):
        case = (3, 2 * G, 2, 700, 700, 0, 40, sinks, lens)
        q, k, v, do = tensors(cuda, case, BF16, 64, seed=sinks)
        check(cuda, case, q, k, v, do, 0.125, *run_both(q, k, v, do, 0.125, case, lens_of(cuda, case)))


def test_a_stream_of_the_callers(cuda):
    """`stream` given as a handle while torch's current stream is another: the workspace
    stays the call's until that stream is done with it."""
    case = (2, 8, 2, 300, 300, 0, 100, 4, None)
    q, k, v, do = tensors(cuda, case, BF16, 128)
    o, lse, want = run_both(q, k, v, do, 0.09, case, None)
    s = torch.cuda.Stream()
    outs = [torch.empty_like(t) for t in want]
    torch.cuda.synchronize()
    for _ in range(5):
        for t in outs:
            t.zero_()
        torch.cuda.synchronize()
        ops.sdpa_window_grad(do, q, k, v, o, lse, 0.09, 100, 4, q_start=0, outs=outs, stream=s.cuda_stream)
        junk = [torch.full((1 << 20,), float("nan"), device=cuda) for _ in range(8)]
        s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        del junk


def test_rows_far_apart(cuda):
    """A slice of K and V over more than 4 GiB: 64-bit offsets."""
    Sk, D, step = 34000, 128, 1 << 16
    store = torch.zeros(Sk * step, dtype=BF16, device=cuda)  # 4.4 GB
    g = torch.Generator(device=cuda).manual_seed(3)
    k = store.as_strided((1, 1, Sk, D), (0, 0, step, 1))
    v = store.as_strided((1, 1, Sk, D), (0, 0, step, 1), 1024)
    k.copy_(torch.randn(k.shape, generator=g, device=cuda))
    v.copy_(torch.randn(v.shape, generator=g, device=cuda))
    q, do = (torch.randn((1, 2, 130, D), generator=g, device=cuda).to(BF16) for _ in range(2))
    case = (1, 2, 1, 130, Sk, Sk - 130, 1000, 5, None)
    got = run_both(q, k, v, do, 0.1, case, None)
    want = run_both(q, k.contiguous(), v.contiguous(), do, 0.1, case, None)
    assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[2], want[2]))
    check(cuda, case, q, k, v, do, 0.1, *got)


def test_unbounded_window_is_causal_attention(cuda):
    """window 0 is ghip_sdpa_fwd's causal attention (both within their bound of float64)."""
    case = (2, 4, 2, 333, 333, 0, 0, 0, None)
    q, k, v, _ = tensors(cuda, case, BF16, 128)
    see = ref.visible(2, 333, 333, 0, 0, 0, device=cuda)
    want, _, bound, _ = ref.forward(q, k, v, 0.09, see)
    ref.within(ops.sdpa_window(q, k, v, 0.09, q_start=0), want, bound, "window")
    # its running sum takes the rounded weights: one more rounding of each
    ref.within(ops.sdpa(q, k, v, 0.09, True), want, 2 * bound, "sdpa")


def test_empty(cuda):
    q = torch.empty((0, 2, 5, 64), dtype=BF16, device=cuda)
    k = torch.empty((0, 2, 5, 64), dtype=BF16, device=cuda)
    assert ops.sdpa_window(q, k, k, 0.1).shape == (0, 2, 5, 64)
    q = torch.empty((2, 2, 0, 64), dtype=BF16, device=cuda)
    k = torch.randn((2, 2, 5, 64), device=cuda).to(BF16)
    o, lse = ops.sdpa_window(q, k, k, 0.1, with_lse=True)
    assert o.shape == (2, 2, 0, 64) and lse.shape == (2, 2, 0)
    _, dk, dv = ops.sdpa_window_grad(q, q, k, k, q, lse, 0.1)
    assert not dk.any() and not dv.any()


def test_refusals_on_the_device(cuda):
    q = torch.randn((1, 2, 8, 64), device=cuda).to(BF16)
    with pytest.raises(ValueError, match="is needed"):
        ops.sdpa_window(q, q[:, :, :, :32], q, 0.1)
    with pytest.raises(ValueError, match="is needed"):
        ops.sdpa_window(q, q.float(), q.float(), 0.1)
    with pytest.raises(ValueError, match="head dim must be contiguous"):
        ops.sdpa_window(q, q.transpose(2, 3).contiguous().transpose(2, 3), q, 0.1)
    with pytest.raises(ValueError, match="device"):
        ops.sdpa_window(q, q.cpu(), q, 0.1)
    with pytest.raises(ValueError, match="lens"):
        ops.sdpa_window(q, q, q, 0.1, lens=torch.ones(1, device=cuda, dtype=torch.int64))
    with pytest.raises(BackendError, match="aligned"):
        ops.sdpa_window(torch.randn(1 * 2 * 8 * 64 + 4, device=cuda).to(BF16)[4:].view(1, 2, 8, 64), q, q, 0.1)
    with pytest.raises(BackendError, match="outside"):
        ops.sdpa_window(q, q, q, 0.1, q_start=1)
    lse = torch.zeros((1, 2, 8), device=cuda)
    with pytest.raises(BackendError, match="workspace of"):
        ops.sdpa_window_grad(q, q, q, q, q, lse, 0.1, workspace=torch.empty(16, dtype=torch.uint8, device=cuda))
    with pytest.raises(ValueError, match="workspace must be contiguous"):
        ops.sdpa_window_grad(q, q, q, q, q, lse, 0.1,
                             workspace=torch.empty(1, dtype=torch.uint8, device=cuda).expand(1 << 20))
