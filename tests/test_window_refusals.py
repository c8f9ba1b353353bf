"""What the windowed and the paged attention refuse, decided on the host before any HIP
call (no GPU), and the float64 reference of their tests against differences."""
import ctypes

import pytest
import torch

import attention_ref as ref
from gomlx_hip import _lib

I3 = ctypes.c_int64 * 3
BF16, F16, F32 = _lib.DT_BFLOAT16, _lib.DT_FLOAT16, _lib.DT_FLOAT32
PTR = 1 << 20  # never dereferenced: every call here is refused


def window(dt=BF16, B=1, H=4, Hkv=2, Sq=8, Sk=8, D=64, q_start=0, window=0, sinks=0, scale=1.0, q=PTR, o=PTR, st=None):
    s = I3(*(st or (H * Sk * D, Sk * D, D)))
    _lib.call("ghip_sdpa_window_fwd", dt, q, PTR, PTR, o, None, B, H, Hkv, Sq, Sk, D, s, s, s, s, q_start, window, sinks,
              None, scale, None)


def grad(dt=BF16, D=64, ws=PTR, nbytes=1 << 20, lse=PTR, dq=PTR):
    s = I3(4096, 512, D)
    _lib.call("ghip_sdpa_window_bwd", dt, PTR, PTR, PTR, PTR, PTR, lse, dq, PTR, PTR, 1, 4, 2, 8, 8, D, s, s, s, s, s, s,
              s, s, 0, 0, 0, None, 1.0, ws, nbytes, None)


def paged(dt=BF16, B=1, H=4, Hkv=2, D=64, pages=4, size=16, per=2, window=0, sinks=0, scale=1.0, q=PTR, st=None, ws=None,
          nbytes=0, ts=2):
    s = I3(*(st or (Hkv * size * D, size * D, D)))
    _lib.call("ghip_sdpa_paged", dt, q, PTR, PTR, PTR, B, H, Hkv, D, pages, size, per, PTR, ts, PTR, I3(H * D, D), s, s,
              I3(H * D, D), window, sinks, scale, ws, nbytes, None)


def append(es=2, B=1, S=2, Hkv=2, D=64, pages=4, size=16, per=2, k=PTR, st=None, ts=2):
    s = I3(*(st or (4096, 64, 64)))
    _lib.call("ghip_kv_append", es, k, PTR, PTR, PTR, B, S, Hkv, D, pages, size, per, PTR, ts, PTR, None, s, s, s, s, None)


REFUSED = [
    (window, dict(H=3), 1, "multiple of num_kv_heads"), (window, dict(B=-1), 1, "bad sizes"),
    (window, dict(D=0), 1, "bad sizes"), (window, dict(q_start=1), 1, "outside"), (window, dict(Sq=9), 1, "outside"),
    (window, dict(q_start=-1), 1, "outside"), (window, dict(window=-1), 1, "negative"),
    (window, dict(sinks=-1), 1, "negative"), (window, dict(scale=0.0), 1, "scale"),
    (window, dict(scale=float("nan")), 1, "scale"), (window, dict(scale=float("inf")), 1, "scale"),
    (window, dict(dt=_lib.DT_FLOAT64), 2, "needs float32"), (window, dict(D=60), 2, "head dim"),
    (window, dict(D=264), 2, "head dim"), (window, dict(dt=F32, D=132), 2, "head dim"),
    (window, dict(dt=F32, D=66), 2, "head dim"), (window, dict(q=None), 1, "q is null"),
    (window, dict(q=PTR + 8), 2, "aligned"), (window, dict(o=PTR + 4), 2, "aligned"),
    (window, dict(st=(-512, 64, 64)), 2, "strides"), (window, dict(st=(512, 64, 68)), 2, "strides"),
    (window, dict(st=(512, 64, 1 << 24)), 2, "below 32 MiB"), (window, dict(st=(512, 64, 1 << 58)), 2, "below 32 MiB"),
    (window, dict(B=1 << 16, H=256, Sq=1, Sk=1), 2, "too large"),  # 2^32 threads
    (window, dict(Sq=1, Sk=(1 << 29) + 8, st=(64, 64, 64)), 2, "too large"),
    (window, dict(B=1 << 40, H=1 << 40, Hkv=1), 2, "too large"),
    (grad, dict(D=300), 2, "head dim"), (grad, dict(ws=None), 1, "workspace of"), (grad, dict(nbytes=100), 1, "workspace of"),
    (grad, dict(ws=PTR + 8), 1, "workspace must be"), (grad, dict(lse=None), 1, "lse is null"),
    (grad, dict(dq=None), 1, "dq is null"), (grad, dict(dq=PTR + 2), 2, "dq must be"),
    (paged, dict(H=3), 1, "multiple of num_kv_heads"), (paged, dict(size=0), 1, "bad sizes"),
    (paged, dict(pages=0), 1, "without pages"), (paged, dict(per=0), 1, "without pages"),
    (paged, dict(window=-2), 1, "negative"), (paged, dict(scale=-1.0), 1, "scale"), (paged, dict(D=12), 2, "head dim"),
    (paged, dict(dt=_lib.DT_INT8), 2, "needs float32"), (paged, dict(q=None), 1, "null"),
    (paged, dict(q=PTR + 2), 2, "16-byte aligned"), (paged, dict(st=(2048, 1024, 68)), 2, "16-byte aligned"),
    (paged, dict(st=(-2048, 1024, 64)), 2, "16-byte aligned"), (paged, dict(ts=-1), 1, "table stride"),
    (paged, dict(size=1 << 20, per=1 << 20), 2, "at most"),
    (paged, dict(size=64, per=1024, ws=PTR, nbytes=64), 1, "workspace of"),
    (paged, dict(size=64, per=1024, ws=PTR + 8, nbytes=1 << 30), 1, "workspace must be"),
    (append, dict(es=3), 2, "elements of"), (append, dict(S=-1), 1, "bad sizes"), (append, dict(k=None), 1, "null"),
    (append, dict(pages=0), 1, "without pages"), (append, dict(k=PTR + 1), 1, "aligned"),
    (append, dict(st=(-1, 64, 64)), 2, "negative strides"), (append, dict(ts=-2), 1, "table stride"),
    (paged, dict(B=1 << 14, H=1 << 10), 2, "fewer than 2\\^24 heads"),
    (append, dict(S=1 << 20, Hkv=64, D=1024), 2, "too large"), (append, dict(B=70000), 2, "too large"), (append, dict(size=1 << 20, per=1 << 20), 2, "too large"),
]


@pytest.mark.parametrize("fn,kw,code,words", REFUSED)
def test_refused(fn, kw, code, words):
    with pytest.raises(_lib.BackendError, match=words) as e:
        fn(**kw)
    assert e.value.code == code


def test_gradient_grids():
    """More workgroups than a launch holds, of either kernel, and a list of tiles past 32
    bits: refused, not wrapped around."""
    s = I3(0, 0, 64)
    for B, H, Hkv, Sq, Sk in ((1 << 16, 256, 256, 1, 1), (1 << 10, 64, 64, 1, 1 << 14), (1, 1 << 22, 1, 1 << 15, 1 << 15)):
        with pytest.raises(_lib.BackendError, match="too large") as e:
            _lib.call("ghip_sdpa_window_bwd", BF16, *[PTR] * 9, B, H, Hkv, Sq, Sk, 64, *[s] * 8, 0, 0, 0, None, 1.0, PTR,
                      1 << 50, None)
        assert e.value.code == 2
    assert _lib.load().ghip_sdpa_window_bwd_workspace_bytes(BF16, 1, 1 << 24, 1, 1 << 15, 1 << 15, 64, 0, 1, 4) == 0


def test_nothing_to_do():
    """Empty batches and prompts return before any pointer is looked at."""
    window(B=0, q=None)
    window(Sq=0, q=None)
    paged(B=0, q=None)
    append(S=0, k=None)
    assert _lib.load().ghip_sdpa_window_bwd_workspace_bytes(BF16, 0, 4, 2, 8, 8, 64, 0, 0, 0) == 0
    assert _lib.load().ghip_sdpa_window_bwd_workspace_bytes(BF16, 1, 4, 3, 8, 8, 64, 0, 0, 0) == 0
    assert _lib.load().ghip_sdpa_paged_workspace_bytes(BF16, 0, 4, 2, 64, 16, 100) == 0


def test_workspace_policy():
    """Paged decoding splits caches of more than 4 tiles a sequence (of 8 KiB a kv head: 32
    tokens of 128 16-bit values), or 12 with 512 (sequence, kv head, 16 heads) units; the
    gradient's workspace holds the rows' two statistics and, where sinks' keys or few
    workgroups are shared out, fp32 shares of at most half of q's bytes a block of sinks."""
    ws = _lib.load().ghip_sdpa_paged_workspace_bytes
    assert ws(BF16, 16, 32, 8, 128, 16, 8) == 0 and ws(BF16, 16, 32, 8, 128, 16, 9) == 2 * 1024 * 4 * 129 * 4
    assert ws(F16, 64, 32, 8, 128, 64, 6) == 0 and ws(F16, 64, 32, 8, 128, 64, 7) > 0
    assert ws(BF16, 1, 40, 2, 64, 16, 16) == 0 and ws(BF16, 1, 40, 2, 64, 16, 17) == 2 * 1024 * 16 * 65 * 4
    assert ws(F32, 1, 8, 8, 128, 16, 4) == 0 and ws(F32, 1, 8, 8, 128, 16, 5) == 2 * 1024 * 129 * 4
    gw = _lib.load().ghip_sdpa_window_bwd_workspace_bytes
    assert gw(BF16, 4, 16, 16, 2048, 2048, 128, 0, 512, 0) == 2 * 4 * 16 * 2048 * 4
    rows = 2 * 4 * 16 * 2048 * 4
    assert 0 < gw(BF16, 4, 16, 16, 2048, 2048, 128, 0, 512, 4) - rows <= 4 * 16 * 2048 * 128
    assert gw(BF16, 4, 16, 16, 2048, 2048, 128, 0, 512, 300) == rows  # many sinks: no shares
    assert gw(BF16, 4, 16, 16, 2048, 2048, 128, 0, 0, 4) == rows      # no window: nothing lies beyond it
    assert gw(BF16, 1, 2, 1, 512, 512, 128, 0, 0, 0) > 2 * 2 * 512 * 4  # 8 workgroups: chunks
    for sizes in ((0, 5), (1, 1), (0, 0), (1, 700), (3, 3)):  # no or few queries
        for window, sinks in ((0, 0), (1, 1), (0, 4), (7, 0), (3, 500)):
            assert gw(F16, 1, 4, 2, *sizes, 64, 0, window, sinks) >= 2 * 4 * sizes[0] * 4


def test_reference_gradient_against_differences():
    """attention_ref's formula in float64 against central differences of its forward: with
    h = 2^-16 their own error is about h^2 plus 2^-52 / h, below 1e-8 of values of order 1."""
    torch.manual_seed(0)
    q, do = (torch.randn(2, 4, 9, 6, dtype=torch.float64) for _ in range(2))
    k, v = (torch.randn(2, 2, 12, 6, dtype=torch.float64) for _ in range(2))
    see = ref.visible(2, 9, 12, 2, 4, 2, torch.tensor([12, 7]))
    o, lse, _, _ = ref.forward(q, k, v, 0.4, see)
    grads = ref.gradient(do, q, k, v, o, lse, 0.4, see)
    h = 2.0 ** -16
    for i, (g, _) in enumerate(grads):
        for seed in range(3):
            d = torch.randn(g.shape, dtype=torch.float64, generator=torch.Generator().manual_seed(seed))
            up, down = [q, k, v], [q, k, v]
            up[i], down[i] = up[i] + h * d, down[i] - h * d
            diff = sum(s * (ref.forward(*t, 0.4, see)[0] * do).sum() for s, t in ((1, up), (-1, down))) / (2 * h)
            assert abs(diff - (g * d).sum()) < 1e-7


def test_reference_sees():
    """visible() row by row."""
    see = ref.visible(1, 4, 6, 2, 2, 1)[0, 0].int().tolist()
    assert see == [[1, 1, 1, 0, 0, 0], [1, 0, 1, 1, 0, 0], [1, 0, 0, 1, 1, 0], [1, 0, 0, 0, 1, 1]]
    assert not ref.visible(1, 4, 6, 2, 2, 1, torch.tensor([2])).any()
