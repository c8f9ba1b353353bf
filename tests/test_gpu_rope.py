"""Rotary positions against float64 within rope_kv4_ref.py's bounds: types, pairings, axes,
partial rotations, odd sizes, strides, far positions, in place, the gradient."""
import pytest
import torch

import attention_ref
import rope_kv4_ref as ref
from gomlx_hip import ops
from gomlx_hip._lib import BackendError

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def rand(cuda, *shape, dt=BF16, seed=0):
    return torch.randn(shape, generator=torch.Generator(device=cuda).manual_seed(seed), device=cuda).to(dt)


def freqs_of(half, cuda):
    return (10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))).float().to(cuda)


def positions_of(cuda, axes, B, S, most=131072, seed=1):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return torch.randint(-most // 8, most, (axes, B, S), generator=g, device=cuda, dtype=torch.int32)


CASES = [  # (B, H, S, D, rotary_dim, sections)
    (1, 1, 1, 2, 2, None), (1, 1, 1, 128, 128, None), (2, 3, 5, 64, 64, None), (1, 32, 7, 128, 64, None),
    (3, 2, 33, 80, 40, None), (2, 5, 17, 36, 18, None), (1, 2, 9, 7, 6, None), (1, 2, 9, 255, 254, None),
    (2, 4, 100, 128, 128, (16, 24, 24)), (1, 3, 41, 256, 256, (64, 64)), (2, 2, 30, 96, 96, (0, 48)),
    (1, 2, 30, 64, 64, (8, 8, 8, 8)), (4, 16, 700, 128, 128, None), (1, 300, 3, 64, 32, None), (2, 8, 3, 64, 2, None),
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_rope(cuda, case, dt):
    B, H, S, D, R, sections = case
    x = rand(cuda, B, H, S, D, dt=dt)
    pos, freqs = positions_of(cuda, len(sections or (1,)), B, S), freqs_of(R // 2, cuda)
    for inter in (False, True):
        for inverse in (False, True):
            got = ops.rope(x, pos, freqs, sections, interleaved=inter, inverse=inverse)
            want, bound = ref.rotate(x, pos, freqs, sections, inter, inverse)
            attention_ref.within(got, want, bound, f"{inter} {inverse}")
            assert torch.equal(got[..., R:], x[..., R:])
            y = x.clone()
            assert ops.rope(y, pos, freqs, sections, interleaved=inter, inverse=inverse, out=y) is y
            assert torch.equal(y, got)


@pytest.mark.parametrize("dt", [BF16, F32])
def test_strides(cuda, dt):
    """Slices of a fused projection, [B, S, H, D] storage, unaligned rows, a broadcast input,
    positions shared by the batch; outputs of another layout leave what lies between alone."""
    B, H, S, D = 2, 3, 11, 64
    freqs = freqs_of(32, cuda)
    pos = positions_of(cuda, 1, 1, S)[0].expand(B, S)
    want = None
    qkv = rand(cuda, B, S, 5 * H, D, dt=dt)
    odd = torch.zeros((B, H, S, D + 1), dtype=dt, device=cuda)
    odd[..., 1:] = qkv.transpose(1, 2)[:, H:2 * H]
    for x in (qkv.transpose(1, 2)[:, H:2 * H], qkv.transpose(1, 2)[:, H:2 * H].contiguous(), odd[..., 1:]):
        for room in (torch.full((B, S, H, D + 8), 7.0, dtype=dt, device=cuda), torch.full((B, S, H, D + 3), 7.0, dtype=dt, device=cuda)):
            out = room.transpose(1, 2)[..., :D]
            ops.rope(x, pos, freqs, out=out)
            want = out.clone() if want is None else want
            assert torch.equal(out, want) and (room[..., D:] == 7.0).all()
    attention_ref.within(want, *ref.rotate(qkv.transpose(1, 2)[:, H:2 * H], pos, freqs))
    one = rand(cuda, 1, 1, S, D, dt=dt)
    assert torch.equal(ops.rope(one.expand(B, H, S, D), pos, freqs), ops.rope(one, pos[:1], freqs).expand(B, H, S, D))


def test_far_positions(cuda):
    """Angles up to 2^31: the products are exact to 64 bits on both sides, the turns that are
    taken off cost 2^-52 of the angle each: 2^-20 at most."""
    x = rand(cuda, 1, 2, 6, 64, dt=F32)
    pos = torch.tensor([[0, -2 ** 31, 2 ** 31 - 1, 10 ** 9, -12345678, 1 << 24]], dtype=torch.int32, device=cuda)
    freqs = freqs_of(32, cuda)
    want, bound = ref.rotate(x, pos, freqs)
    attention_ref.within(ops.rope(x, pos, freqs), want, bound + 2.0 ** -20 * x.double().abs().amax())


@pytest.mark.parametrize("inter", [False, True])
def test_gradient(cuda, inter):
    """The inverse rotation of a gradient is the gradient: <rope(x), w> = <x, rope(w, inverse)>, and
    against differences along random directions (the map is linear)."""
    x, w = rand(cuda, 2, 4, 50, 80, dt=F32), rand(cuda, 2, 4, 50, 80, dt=F32, seed=3)
    pos, freqs = positions_of(cuda, 2, 2, 50), freqs_of(24, cuda)
    turn = lambda t, **kw: ops.rope(t, pos, freqs, (10, 14), interleaved=inter, **kw).double()  # noqa: E731
    grad = turn(w, inverse=True)
    # Both sums have terms off by 3.1 F (|x c| + |y s|) at most, so by 5 F |x| |w|.
    size = (x.double().abs().sum() * w.double().abs().amax()) * 10 * ref.F
    assert abs((turn(x) * w).sum() - (x * grad).sum()) <= size
    d = rand(cuda, 2, 4, 50, 80, dt=F32, seed=4)
    diff = ((turn(x + d) - turn(x - d)) * w).sum() / 2
    assert abs(diff - (grad * d).sum()) <= 4 * size


def test_replayed(cuda):
    x, pos, freqs = rand(cuda, 2, 4, 30, 128), positions_of(cuda, 1, 2, 30)[0], freqs_of(64, cuda)
    ops.rope(x, pos, freqs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.rope(x, pos, freqs)
    for i in range(3):
        x.mul_(0.5).add_(0.1)
        pos.add_(7)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.rope(x, pos, freqs))


def test_refusals_on_the_device(cuda):
    x, pos, freqs = rand(cuda, 2, 4, 30, 64), positions_of(cuda, 1, 2, 30)[0], freqs_of(32, cuda)
    with pytest.raises(ValueError, match="freqs"):
        ops.rope(x, pos, freqs.double())
    with pytest.raises(ValueError, match="freqs"):
        ops.rope(x, pos, freqs.repeat(2)[::2])
    with pytest.raises(ValueError, match="positions"):
        ops.rope(x, pos.long(), freqs)
    with pytest.raises(ValueError, match="positions"):
        ops.rope(x, pos[:1], freqs)
    with pytest.raises(ValueError, match="sections"):
        ops.rope(x, pos, freqs, (16, 16))
    with pytest.raises(ValueError, match="out"):
        ops.rope(x, pos, freqs, out=x[:1])
    with pytest.raises(ValueError, match="head dim must be contiguous"):
        ops.rope(x.transpose(2, 3).contiguous().transpose(2, 3), pos, freqs)
    with pytest.raises(BackendError, match="rotary_dim"):
        ops.rope(x, pos, freqs_of(33, cuda))
    assert ops.rope(x[:, :, :0], pos[:, :0], freqs).shape == (2, 4, 0, 64)


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("D,R", [(64, 64), (80, 40), (36, 36), (20, 8), (12, 4)])
def test_every_width(cuda, dt, D, R):
    """Rows and outputs that begin 0, 1, 2, 4 and 8 elements into their memory, at strides of as many
    more than D: the same bits however many elements a thread takes, nothing else written."""
    B, H, S = 2, 3, 5
    x, pos, freqs = rand(cuda, B, H, S, D, dt=dt), positions_of(cuda, 1, B, S), freqs_of(R // 2, cuda)
    for inter in (False, True):
        want, bound = ref.rotate(x, pos, freqs, None, inter)
        first = None
        for a in (0, 1, 2, 4, 8):
            for b in (0, 1, 2, 4, 8):
                source, room = (torch.full((B * H * S * (D + n) + n,), 7.0, dtype=dt, device=cuda) for n in (a, b))
                rows = source[a:].view(B, H, S, D + a)[..., :D]
                rows.copy_(x)
                out = room[b:].view(B, H, S, D + b)[..., :D]
                ops.rope(rows, pos, freqs, interleaved=inter, out=out)
                first = out.clone() if first is None else first
                assert torch.equal(out, first), (a, b)
                assert (room[:b] == 7.0).all() and (room[b:].view(B, H, S, D + b)[..., D:] == 7.0).all()
        attention_ref.within(first, want, bound)
