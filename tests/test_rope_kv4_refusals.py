"""What rotary positions, the 4-bit cache and the log probabilities refuse, decided on the host
before any HIP call (no GPU), and their float64 references against differences and by hand."""
import ctypes

import pytest
import torch

import rope_kv4_ref as ref
from gomlx_hip import _lib, ops

I3 = ctypes.c_int64 * 3
BF16, F16, F32 = _lib.DT_BFLOAT16, _lib.DT_FLOAT16, _lib.DT_FLOAT32
PTR = 1 << 20  # never dereferenced: every call here is refused


def plan(R=64, axes=1, sections=(32, 0, 0, 0), positions=PTR, freqs=PTR, steps=(0, 8, 1), interleaved=0):
    return _lib.Rope(positions, *steps, axes, *sections, freqs, R, interleaved)


def rope(dt=BF16, B=1, H=4, S=8, D=64, x=PTR, st=None, r=None, **kw):
    s = I3(*(st or (H * S * D, S * D, D)))
    _lib.call("ghip_rope", dt, x, PTR, B, H, S, D, s, s, r or plan(**kw), 0, None)


def append(dt=BF16, B=1, H=4, Hkv=2, S=2, D=64, pages=4, size=16, per=2, q=PTR, k=PTR, st=None, ts=2, r="plan", starts=PTR, **kw):
    s = I3(*(st or (4096, 64, 64)))
    _lib.call("ghip_kv_append_rope", dt, q, PTR, k, PTR, PTR, PTR, B, H, Hkv, S, D, pages, size, per, PTR, ts, starts, None,
              s, s, s, s, s, s, plan(**kw) if r == "plan" else r, None)


def cache(codes=PTR, scales=PTR, cst=(1 << 12, 512, 32), sst=(64, 64, 4)):
    return _lib.Kv4(codes, scales, *cst, *sst)


def append4(dt=BF16, B=1, H=4, Hkv=2, S=2, D=64, pages=4, size=16, per=2, k=PTR, ts=2, kc=None, vc=None, **kw):
    s = I3(4096, 64, 64)
    _lib.call("ghip_kv4_append_rope", dt, PTR, PTR, k, PTR, kc or cache(), vc or cache(), B, H, Hkv, S, D, pages, size, per,
              PTR, ts, PTR, None, s, s, s, s, plan(**kw), None)


def read4(dt=BF16, B=1, Hkv=2, S=20, D=64, pages=4, size=16, per=2, k=PTR, ts=2, kc=None, st=(4096, 64, 64)):
    s = I3(*st)
    _lib.call("ghip_kv4_read", dt, kc or cache(), cache(), k, PTR, B, Hkv, S, D, pages, size, per, PTR, ts, None, s, s, None)


def paged4(dt=BF16, B=1, H=4, Hkv=2, D=64, pages=4, size=16, per=2, window=0, sinks=0, scale=1.0, q=PTR, kc=None, vc=None,
           ws=None, nbytes=0, ts=2, qst=(256, 64, 0)):
    _lib.call("ghip_sdpa_paged_kv4", dt, q, kc or cache(), vc or cache(), PTR, B, H, Hkv, D, pages, size, per, PTR, ts, PTR,
              I3(*qst), I3(256, 64, 0), window, sinks, scale, ws, nbytes, None)


def logprobs(dt=BF16, N=4, V=100, top=5, scale=1.0, x=PTR, step=100, ids=PTR, logp=PTR, tl=PTR, ws=None, nbytes=0):
    _lib.call("ghip_token_logprobs", dt, x, step, ids, N, V, top, scale, logp, PTR, PTR, tl, PTR, ws, nbytes, None)


def lp_grad(dt=BF16, N=4, V=100, scale=1.0, x=PTR, step=100, lse=PTR, entropy=PTR, d_logp=PTR, d_entropy=PTR, d=PTR, dstep=100):
    _lib.call("ghip_token_logprobs_grad", dt, x, step, PTR, lse, entropy, d_logp, d_entropy, N, V, scale, d, dstep, None)


REFUSED = [
    (rope, dict(dt=_lib.DT_FLOAT64), 2, "needs float32"), (rope, dict(B=-1), 1, "bad sizes"), (rope, dict(D=0), 1, "bad sizes"),
    (rope, dict(D=258), 2, "at most 256"), (rope, dict(R=66, sections=(33, 0, 0, 0)), 1, "rotary_dim"),
    (rope, dict(R=31), 1, "rotary_dim"), (rope, dict(R=-2), 1, "rotary_dim"), (rope, dict(axes=0), 1, "axes"),
    (rope, dict(axes=5), 1, "axes"), (rope, dict(axes=2, sections=(20, 10, 0, 0)), 1, "sections hold 30 pairs"),
    (rope, dict(axes=2, sections=(40, -8, 0, 0)), 1, "negative section"), (rope, dict(freqs=None), 1, "freqs"),
    (rope, dict(positions=None), 1, "positions are needed"), (rope, dict(steps=(0, -8, 1)), 2, "negative strides"),
    (rope, dict(x=None), 1, "null"), (rope, dict(x=PTR + 1), 1, "aligned to elements"),
    (rope, dict(st=(512, -64, 64)), 2, "negative strides"), (rope, dict(st=(512, 1 << 60, 64)), 2, "negative strides"),
    (rope, dict(B=1 << 20, S=1 << 20), 2, "too large"), (rope, dict(S=1 << 30, H=1 << 20), 2, "too large"),
    (append, dict(Hkv=0), 1, "bad sizes"), (append, dict(size=0), 1, "bad sizes"), (append, dict(pages=0), 1, "without pages"),
    (append, dict(ts=-1), 1, "table stride"), (append, dict(q=None), 1, "null"), (append, dict(k=None), 1, "null"),
    (append, dict(starts=None), 1, "null"), (append, dict(positions=None, axes=2, sections=(16, 16, 0, 0)), 1, "positions are"),
    (append, dict(size=1 << 20, per=1 << 20), 2, "too large"), (append, dict(dt=_lib.DT_INT8), 2, "needs float32"),
    (append, dict(R=128, sections=(64, 0, 0, 0)), 1, "rotary_dim"), (append, dict(k=PTR + 1), 1, "aligned to elements"),
    (append4, dict(D=72), 2, "multiple of 32"), (append4, dict(D=288), 2, "at most 256"),
    (append4, dict(kc=cache(codes=None)), 1, "null"), (append4, dict(vc=cache(scales=None)), 1, "null"),
    (append4, dict(kc=cache(codes=PTR + 4)), 2, "16-byte aligned"), (append4, dict(vc=cache(scales=PTR + 2)), 2, "4-byte aligned"),
    (append4, dict(kc=cache(cst=(4096, 512, 40))), 2, "whole 16 bytes"), (append4, dict(kc=cache(sst=(64, 64, 3))), 2, "whole 4"),
    (append4, dict(kc=cache(cst=(-4096, 512, 32))), 2, "non-negative"), (append4, dict(k=PTR + 1), 1, "aligned to elements"),
    (read4, dict(S=33), 1, "33 tokens where a sequence's pages hold 32"), (read4, dict(k=PTR + 8), 2, "16-byte aligned"),
    (read4, dict(st=(4096, 64, 68)), 2, "16-byte aligned"), (read4, dict(D=48), 2, "multiple of 32"),
    (read4, dict(k=None), 1, "null"), (read4, dict(B=70000), 2, "too large"), (read4, dict(kc=cache(codes=None)), 1, "null"),
    (paged4, dict(H=3), 1, "multiple of num_kv_heads"), (paged4, dict(size=0), 1, "bad sizes"),
    (paged4, dict(pages=0), 1, "without pages"), (paged4, dict(window=-2), 1, "negative"), (paged4, dict(scale=-1.0), 1, "scale"),
    (paged4, dict(scale=float("nan")), 1, "scale"), (paged4, dict(D=48), 2, "multiple of 32"), (paged4, dict(D=288), 2, "multiple of 32"),
    (paged4, dict(dt=_lib.DT_INT8), 2, "needs float32"), (paged4, dict(q=None), 1, "null"), (paged4, dict(q=PTR + 2), 2, "q must be"),
    (paged4, dict(qst=(256, 68, 0)), 2, "q must be"), (paged4, dict(kc=cache(cst=(4096, 512, 24))), 2, "codes must be"),
    (paged4, dict(vc=cache(scales=PTR + 1)), 2, "codes must be"), (paged4, dict(kc=cache(scales=None)), 1, "null"),
    (paged4, dict(ts=-1), 1, "table stride"), (paged4, dict(size=1 << 20, per=1 << 20), 2, "at most"),
    (paged4, dict(B=1 << 14, H=1 << 10), 2, "fewer than 2\\^24 heads"),
    (paged4, dict(kc=cache(cst=(1 << 32, 512, 32))), 2, "4 GiB"), (paged4, dict(vc=cache(cst=(4096, 512, 1 << 33))), 2, "4 GiB"),
    (paged4, dict(vc=cache(sst=(1 << 32, 64, 4))), 2, "4 GiB"), (paged4, dict(kc=cache(sst=(64, 64, 1 << 32))), 2, "4 GiB"),
    (read4, dict(Hkv=65536), 2, "too large"), (read4, dict(S=1 << 31, size=1 << 20, per=1 << 10), 2, "too large"),
    (paged4, dict(size=64, per=1024, ws=PTR, nbytes=64), 1, "workspace of"),
    (paged4, dict(size=64, per=1024, ws=PTR + 8, nbytes=1 << 30), 1, "workspace must be"),
    (logprobs, dict(dt=_lib.DT_FLOAT64), 2, "needs float32"), (logprobs, dict(V=0), 1, "bad sizes"), (logprobs, dict(N=-1), 1, "bad sizes"),
    (logprobs, dict(scale=0.0), 1, "scale"), (logprobs, dict(scale=float("inf")), 1, "scale"), (logprobs, dict(top=33), 1, "top 33"),
    (logprobs, dict(top=-1), 1, "top -1"), (logprobs, dict(V=4), 1, "top 5"), (logprobs, dict(x=None), 1, "null"),
    (logprobs, dict(ids=None), 1, "null"), (logprobs, dict(logp=None), 1, "null"), (logprobs, dict(tl=None), 1, "null"),
    (logprobs, dict(x=PTR + 1), 1, "aligned to elements"), (logprobs, dict(step=-100), 2, "row stride"),
    (logprobs, dict(N=1 << 24), 2, "fewer than 2\\^24 rows"), (logprobs, dict(V=(1 << 30) + 1), 2, "fewer than"),
    (logprobs, dict(N=1, V=1 << 20, ws=PTR, nbytes=64), 1, "workspace of"),
    (logprobs, dict(N=1, V=1 << 20, ws=PTR + 8, nbytes=1 << 30), 1, "workspace must be"),
    (lp_grad, dict(d_logp=None, d_entropy=None), 1, "null"), (lp_grad, dict(entropy=None), 1, "null"), (lp_grad, dict(lse=None), 1, "null"),
    (lp_grad, dict(d=None), 1, "null"), (lp_grad, dict(dstep=99), 1, "overlap"), (lp_grad, dict(scale=-1.0), 1, "scale"),
    (lp_grad, dict(d=PTR + 1), 1, "aligned to elements"), (lp_grad, dict(N=(1 << 24) - 1, V=1 << 20, dstep=1 << 20), 2, "too large"),
]


@pytest.mark.parametrize("fn,kw,code,words", REFUSED)
def test_refused(fn, kw, code, words):
    with pytest.raises(_lib.BackendError, match=words) as e:
        fn(**kw)
    assert e.value.code == code


def test_nothing_to_do():
    """Empty batches return before any pointer is looked at."""
    rope(B=0, x=None)
    rope(S=0, x=None)
    append(S=0, k=None)
    append4(B=0, k=None)
    read4(S=0, k=None)
    paged4(B=0, q=None)
    logprobs(N=0, x=None)
    lp_grad(N=0, x=None)


def test_workspaces():
    L = _lib.load()
    ws = L.ghip_token_logprobs_workspace_bytes
    assert ws(BF16, 16, 131072, 20) == 16 * 16 * (16 + 160) and ws(F32, 1, 131072, 0) == 32 * 16
    assert ws(BF16, 1024, 131072, 20) == 0 and ws(BF16, 1, 2000, 5) == 0 and ws(BF16, 1, 131072, 33) == 0
    assert ws(BF16, 1, 1 << 30, 1) == 64 * 24 and ws(BF16, 0, 131072, 1) == 0
    ws = L.ghip_sdpa_paged_kv4_workspace_bytes
    assert ws(16, 32, 8, 128, 64, 6) == 0 and ws(16, 32, 8, 128, 64, 7) == 2 * 2048 * 4 * 129 * 4 + 16 * 8 * 8
    assert ws(64, 32, 8, 128, 64, 12) == 0 and ws(64, 32, 8, 128, 64, 13) > 0
    assert ws(128, 32, 8, 128, 64, 24) == 0 and ws(128, 32, 8, 128, 64, 25) > 0
    assert ws(0, 32, 8, 128, 64, 100) == 0 and ws(1, 8, 8, 256, 64, 100) == 2 * 1024 * 257 * 4 + 8 * 8


def test_host_tensors_are_refused():
    x = torch.zeros(1, 2, 3, 64)
    with pytest.raises(ValueError, match="device tensors"):
        ops.rope(x, torch.zeros(1, 3, dtype=torch.int32), torch.zeros(32))
    with pytest.raises(ValueError, match="device tensors"):
        ops.token_logprobs(torch.zeros(2, 10), torch.zeros(2, dtype=torch.int32))


def test_reference_rotation():
    """By hand: a quarter turn; lengths stay; the inverse undoes; and the gradient of a sum
    of outputs is the inverse rotation, against differences (exact for a linear map but for
    2^-52 / h of values of order 1)."""
    x = torch.tensor([[[[1.0, 2.0, 3.0, 4.0, 5.0]]]], dtype=torch.float64)
    pos, freqs = torch.tensor([[2]], dtype=torch.int32), torch.tensor([torch.pi / 4, 0.0])
    y, _ = ref.rotate(x, pos, freqs)
    assert torch.allclose(y, torch.tensor([-3.0, 2.0, 1.0, 4.0, 5.0], dtype=torch.float64), atol=1e-6)
    y, _ = ref.rotate(x, pos, freqs, interleaved=True)
    assert torch.allclose(y, torch.tensor([-2.0, 1.0, 3.0, 4.0, 5.0], dtype=torch.float64), atol=1e-6)
    torch.manual_seed(0)
    x, d, w = (torch.randn(2, 3, 4, 10, dtype=torch.float64) for _ in range(3))
    pos, freqs = torch.randint(-50, 50, (2, 2, 4), dtype=torch.int32), torch.rand(4)
    for inter in (False, True):
        turned = lambda t: ref.rotate(t, pos, freqs, [1, 3], inter)[0]  # noqa: E731
        assert torch.allclose(ref.rotate(turned(x), pos, freqs, [1, 3], inter, inverse=True)[0], x, atol=1e-12)
        grad = ref.rotate(w, pos, freqs, [1, 3], inter, inverse=True)[0]
        h = 2.0 ** -10
        diff = ((turned(x + h * d) - turned(x - h * d)) * w).sum() / (2 * h)
        assert abs(diff - (grad * d).sum()) < 1e-10


def test_reference_codes():
    """Every code and every tie by hand."""
    x = torch.zeros(32)
    x[:16] = torch.tensor([0, 0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.75, -0.0, 0.74, 2.51, -5.1, 4.9])
    codes, scales = ref.encode(x)
    assert scales.tolist() == [127]
    assert codes[:16].tolist() == [0, 0, 1, 2, 2, 4, 4, 6, 6, 7, 10, 8, 1, 5, 15, 6]
    for most, byte in ((6.0, 127), (6.01, 128), (3.0, 126), (12.0, 128), (2.0 ** -130, 1), (0.0, 1), (3e38, 252), (float("inf"), 255)):
        x = torch.zeros(32)
        x[3] = -most
        assert ref.encode(x)[1].tolist() == [byte]
    packed = torch.tensor([[0x21, 0xF8] + [0] * 14], dtype=torch.uint8)
    assert ref.decode(packed, torch.tensor([[128]], dtype=torch.uint8), 32)[0, :4].tolist() == [1.0, 2.0, 0.0, -12.0]
    assert ref.decode(packed, torch.tensor([[255]], dtype=torch.uint8), 32).isnan().all()


def test_reference_logprob_gradient():
    """The gradient's formula against central differences of logp and entropy: h = 2^-16, their
    own error about h^2 plus 2^-52 / h."""
    torch.manual_seed(0)
    x = torch.randn(5, 13, dtype=torch.float64) * 2
    x[1, 3] = -torch.inf
    ids = torch.tensor([0, 12, 5, -100, 13], dtype=torch.int32)
    g, h = torch.randn(5, dtype=torch.float64), torch.randn(5, dtype=torch.float64)
    there = (ids >= 0) & (ids < 13)

    def value(t):
        (logp, _), (H, _), _ = ref.logprobs(t, ids, 0.7, 0)
        return (torch.where(there, logp, 0.0) * g + H * h).sum()

    (_, _), (H, _), (lse, _) = ref.logprobs(x, ids, 0.7, 0)
    d, _ = ref.gradient(x, ids, lse, H, g, h, 0.7)
    step = 2.0 ** -16
    for seed in range(4):
        w = torch.randn(x.shape, dtype=torch.float64, generator=torch.Generator().manual_seed(seed))
        diff = (value(x + step * w) - value(x - step * w)) / (2 * step)
        assert abs(diff - (d * w).sum()) < 1e-7
    assert not d[1, 3].any()
