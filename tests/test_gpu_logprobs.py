"""Log probabilities of given tokens, entropy, the largest logits and the gradient, against
rope_kv4_ref.py: types, odd vocabularies, strides, shared rows, masked, constant, sorted and
NaN rows, ids that are no token."""
import pytest
import torch

import attention_ref
import rope_kv4_ref as ref
from gomlx_hip import ops

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def logits_of(cuda, N, V, dt, seed=0, wide=None):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = (torch.randn((N, wide or V), generator=g, device=cuda) * 2.5).to(dt)
    ids = torch.randint(0, V, (N,), generator=g, device=cuda, dtype=torch.int32)
    return x[:, :V], ids


def adds_of(V, es, split):
    """Additions of a lane and of the joins."""
    waves = 1 if V * es <= 8192 else 4
    return V // (64 * waves) + 80


def check(x, ids, top, scale=1.0, split=True):
    got = ops.token_logprobs(x, ids, top=top, scale=scale, split=split)
    for what, g, (want, bound) in zip(("logp", "entropy", "lse"), got, ref.logprobs(x, ids, scale, adds_of(x.shape[1], x.element_size(), split))):
        attention_ref.within(g, want, bound, what)
    if not top:
        assert got[3] is None and got[4] is None
        return got
    best = ref.top(x.cpu(), top)
    assert torch.equal(got[4].cpu(), best)
    for i in range(0, top, max(1, top // 3)):  # each is that token's own log probability
        assert torch.equal(got[3][:, i], ops.token_logprobs(x, got[4][:, i].contiguous(), scale=scale, split=split)[0])
    return got


SIZES = [(1, 1), (3, 2), (5, 7), (2, 17), (7, 63), (4, 64), (3, 500), (2, 1000), (3, 2047), (1, 2049), (2, 4099), (9, 8200),
         (1, 32003), (2, 50001), (1, 131072), (600, 5000), (300, 9001), (1, 300007)]


@pytest.mark.parametrize("N,V", SIZES)
@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_logprobs(cuda, N, V, dt):
    x, ids = logits_of(cuda, N, V, dt)
    some = slice(0, 12)  # (the reference of the largest is a loop)
    print(N, V, dt, flush=True)
    for top in (0, 1, 5, 32):
        for split in (True, False):
            k = min(top, V)
            got = ops.token_logprobs(x, ids, top=k, scale=0.7, split=split)
            for what, g, (want, bound) in zip(("logp", "entropy", "lse"), got, ref.logprobs(x, ids, 0.7, adds_of(V, x.element_size(), split))):
                attention_ref.within(g, want, bound, what)
            if k:
                assert torch.equal(got[4][some].cpu(), ref.top(x[some].cpu(), k))
    check(x[some], ids[some], min(6, V))


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("V", [61, 1500, 8003, 40001])
def test_strides_and_alignment(cuda, dt, V):
    """Rows of a padded vocabulary, rows that begin at any element, one row for all."""
    for wide in (V, V + 1, V + 3, -(-V // 64) * 64 + 64):
        x, ids = logits_of(cuda, 5, V, dt, wide=wide)
        check(x, ids, 5)
    x, ids = logits_of(cuda, 1, V, dt)
    got = ops.token_logprobs(x.expand(5, V), ids.expand(5).contiguous(), top=3)
    assert all(torch.equal(t, t[:1].expand_as(t)) for t in got)


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("V", [300, 3001, 60001])
@pytest.mark.parametrize("split", [True, False])
def test_ties_and_orders(cuda, dt, V, split):
    """Constant rows, few values, rising and falling rows, zeros of both signs, one peak, the
    type's lowest value as a mask: the lowest index wins."""
    at = torch.arange(V, device=cuda)
    x = torch.zeros((8, V), device=cuda)
    x[0], x[1], x[2] = 3.0, (at * 7 % 5).float(), at.float() / V * 30
    x[3], x[4] = -x[2], torch.where(at % 2 == 0, -0.0, 0.0)
    x[5, V - 1] = 50.0
    x[6] = torch.finfo(dt).min
    x[6, V // 2] = 1.0
    x[7] = (at % 64).float()
    x = x.to(dt)
    ids = torch.tensor([0, 1, 2, 3, 4, V - 1, V // 2, 0], dtype=torch.int32, device=cuda)
    for top in (1, 20, 32):
        check(x, ids, top, split=split)


@pytest.mark.parametrize("V", [100, 3000, 50000])
@pytest.mark.parametrize("split", [True, False])
def test_masked_rows(cuda, V, split):
    """Tokens of -infinity: all but one, all but two far apart, all, a given one."""
    x, ids = logits_of(cuda, 6, V, F32)
    inf = float("inf")
    x[0], x[1], x[2] = -inf, -inf, -inf
    x[0, V - 2], x[1, 0], x[1, V - 1] = 2.0, 1.0, 1.0
    x[3, ids[3].item()] = -inf
    x[4, 1:] = -inf
    ids[0], ids[1], ids[2], ids[4] = V - 2, 3, 1, 0
    got = check(x, ids, 7, split=split)
    assert got[0][0] == 0 and got[1][0] == 0 and got[0][1] == -inf and got[0][3] == -inf
    assert got[2][2] == -inf and got[1][2] == 0 and got[0][2] == -inf
    assert (got[3][2] == -inf).all() and got[4][2].tolist() == list(range(7))
    d = ops.token_logprobs_grad(x, ids, got[2], torch.ones(6, device=cuda), got[1], torch.ones(6, device=cuda))
    want, bound = ref.gradient(x, ids, got[2], got[1], torch.ones(6, device=cuda), torch.ones(6, device=cuda), 1.0)
    keep = [0, 1, 2, 4, 5]  # (row 3 is given a token that cannot be: its gradient is of -infinity)
    attention_ref.within(d[keep], want[keep], bound[keep])
    assert not d[2].any()


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("V", [100, 3000, 50000])
@pytest.mark.parametrize("split", [True, False])
def test_rows_with_nan(cuda, dt, V, split):
    """A NaN or +infinity: NaN for its row, the largest as ever with NaN above all, and no other
    row touched."""
    x, ids = logits_of(cuda, 7, V, dt)
    clean = ops.token_logprobs(x, ids, top=9, split=split)
    x[1, V - 1] = x[3, 0] = x[3, V // 2] = float("nan")
    x[4, 17], x[5, 20], x[5, 21] = float("inf"), float("inf"), -float("inf")
    got = ops.token_logprobs(x, ids, top=9, split=split)
    assert torch.equal(got[4].cpu(), ref.top(x.cpu(), 9))
    for t, c in zip(got, clean):
        assert torch.equal(t[[0, 2, 6]], c[[0, 2, 6]])
    for t in got[:4]:
        assert t[[1, 3, 4, 5]].isnan().all()


def test_ids_that_are_no_token(cuda):
    x, _ = logits_of(cuda, 5, 5000, BF16)
    ids = torch.tensor([-1, -100, 5000, 2 ** 31 - 1, 7], dtype=torch.int32, device=cuda)
    logp, H, lse, _, _ = check(x, ids, 3)
    assert not logp[:4].any() and logp[4] != 0
    g = torch.randn(5, device=cuda)
    d = ops.token_logprobs_grad(x, ids, lse, g)
    assert not d[:4].any()
    attention_ref.within(d, *ref.gradient(x, ids, lse, None, g, None, 1.0))
    d = ops.token_logprobs_grad(x, ids, lse, g, H, g)
    attention_ref.within(d, *ref.gradient(x, ids, lse, H, g, g, 1.0))


@pytest.mark.parametrize("N,V", [(1, 1), (3, 2), (5, 7), (7, 63), (3, 500), (2, 2048), (3, 2049), (5, 8200), (2, 32003), (1, 131072), (70, 1000)])
@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_gradient(cuda, N, V, dt):
    x, ids = logits_of(cuda, N, V, dt)
    g = torch.randn(N, generator=torch.Generator(device=cuda).manual_seed(1), device=cuda)
    _, H, lse, _, _ = ops.token_logprobs(x, ids, scale=0.8)
    for dl, de in ((g, None), (None, g), (g, g * 0.3)):
        d = ops.token_logprobs_grad(x, ids, lse, dl, H if de is not None else None, de, scale=0.8)
        attention_ref.within(d, *ref.gradient(x, ids, lse, H if de is not None else None, dl, de, 0.8))
        for wide in (V + 1, V + 8):  # rows apart, of another alignment; what lies between stays
            room = torch.full((N, wide), 5.0, dtype=dt, device=cuda)
            ops.token_logprobs_grad(x, ids, lse, dl, H if de is not None else None, de, scale=0.8, out=room[:, :V])
            assert torch.equal(room[:, :V], d) and (room[:, V:] == 5.0).all()
        y = x.clone()
        assert ops.token_logprobs_grad(y, ids, lse, dl, H if de is not None else None, de, scale=0.8, out=y) is y
        assert torch.equal(y, d)


def test_gradient_against_differences(cuda):
    """Central differences of the operator's own fp32 outputs along random directions: with step
    2^-6 their error is about its square times third derivatives (below 1), and the outputs'
    own 2^-20 over it."""
    x, ids = logits_of(cuda, 4, 300, F32)
    g, h = torch.randn(4, device=cuda), torch.randn(4, device=cuda)
    _, H, lse, _, _ = ops.token_logprobs(x, ids)
    d = ops.token_logprobs_grad(x, ids, lse, g, H, h).double()

    def value(t):
        logp, e, _, _, _ = ops.token_logprobs(t, ids)
        return (logp.double() * g + e.double() * h).sum()

    for seed in range(3):
        w = torch.randn(x.shape, generator=torch.Generator(device=cuda).manual_seed(seed), device=cuda)
        w /= w.norm()
        step = 2.0 ** -6
        diff = (value(x + step * w) - value(x - step * w)) / (2 * step)
        assert abs(diff - (d * w).sum()) < 2.0 ** -10


def test_rows_of_a_large_matrix(cuda):
    """More than 2^32 bytes of logits: the last rows as the same rows alone."""
    N, V = 17000, 131072 + 8
    x = torch.zeros((N, V), dtype=BF16, device=cuda)
    last, ids = logits_of(cuda, 3, V, BF16)
    x[-3:] = last
    all_ids = torch.zeros(N, dtype=torch.int32, device=cuda)
    all_ids[-3:] = ids
    got = ops.token_logprobs(x, all_ids, top=3)
    want = ops.token_logprobs(last, ids, top=3, split=False)
    assert all(torch.equal(a[-3:], b) for a, b in zip(got, want))
    g = torch.ones(N, device=cuda)
    d = ops.token_logprobs_grad(x, all_ids, got[2], g, out=x)
    assert torch.equal(d[-3:], ops.token_logprobs_grad(last, ids, want[2], g[:3]))
    del x, d, got


def test_replayed(cuda):
    """Captured forward and backward that share a workspace with another captured call, replayed with
    eager work between, while an eager call's outputs live."""
    a, ids = logits_of(cuda, 4, 40000, BF16)
    b, jds = logits_of(cuda, 2, 90000, BF16, seed=2)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=cuda)
    g = torch.randn(4, device=cuda)
    eager = ops.token_logprobs(a, ids, top=5)
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        out = ops.token_logprobs(a, ids, top=5, workspace=ws)
        d = ops.token_logprobs_grad(a, ids, out[2], g, out[1], g)
    with torch.cuda.graph(second):
        other = ops.token_logprobs(b, jds, top=8, workspace=ws)
    kept = [t.clone() for t in eager]
    for i in range(3):
        a.add_(0.5 * i).mul_(1.01)
        b.mul_(0.9)
        first.replay()
        second.replay()
        torch.cuda.synchronize()
        want = ops.token_logprobs(a, ids, top=5)
        assert all(torch.equal(x, y) for x, y in zip(out, want))
        assert torch.equal(d, ops.token_logprobs_grad(a, ids, want[2], g, want[1], g))
        assert all(torch.equal(x, y) for x, y in zip(other, ops.token_logprobs(b, jds, top=8)))
        assert all(torch.equal(x, y) for x, y in zip(eager, kept))


@pytest.mark.parametrize("handle", ["own", 0])
def test_a_stream_of_the_callers(cuda, handle):
    x, ids = logits_of(cuda, 4, 60000, BF16)
    want = ops.token_logprobs(x, ids, top=5)
    s, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        for _ in range(4):
            got = ops.token_logprobs(x, ids, top=5, stream=s.cuda_stream if handle == "own" else handle)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals_on_the_device(cuda):
    x, ids = logits_of(cuda, 4, 100, BF16)
    f = torch.zeros(4, device=cuda)
    with pytest.raises(ValueError, match="ids"):
        ops.token_logprobs(x, ids.long())
    with pytest.raises(ValueError, match="ids"):
        ops.token_logprobs(x, ids[:2])
    with pytest.raises(ValueError, match="contiguous"):
        ops.token_logprobs(x.t(), torch.zeros(100, dtype=torch.int32, device=cuda))
    with pytest.raises(ValueError, match="logits"):
        ops.token_logprobs(x[0], ids)
    with pytest.raises(ValueError, match="five outputs"):
        ops.token_logprobs(x, ids, top=3, outs=(f, f, f, None, None))
    with pytest.raises(ValueError, match="output 0"):
        ops.token_logprobs(x, ids, outs=(f[:2], f, f, None, None))
    with pytest.raises(ValueError, match="d_logp or d_entropy"):
        ops.token_logprobs_grad(x, ids, f, None)
    with pytest.raises(ValueError, match="d_logp or d_entropy"):
        ops.token_logprobs_grad(x, ids, f, f, d_entropy=f)
    with pytest.raises(ValueError, match="lse"):
        ops.token_logprobs_grad(x, ids, f.double(), f)
    with pytest.raises(ValueError, match="out"):
        ops.token_logprobs_grad(x, ids, f, f, out=x[:2])
    assert ops.token_logprobs(x[:0], ids[:0], top=2)[4].shape == (0, 2)


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("V", [300, 3001, 60001])
@pytest.mark.parametrize("split", [True, False])
def test_large_numbers_as_masks(cuda, dt, V, split):
    """Rows of nothing but one large number, up to the type's lowest and largest, are even, as any
    constant row (exponents of 0, a sum of V ones, exact below 2^24; its logarithm in base 2 and
    the product with ln 2 are within 4 roundings); beside a lower one the largest has all of the
    weight, and so has an ordinary one beside a large mask."""
    low, high = torch.finfo(dt).min, torch.finfo(dt).max
    fills = [low, high, -1e5, -1e10, -1e30, 3e20]
    x = torch.empty((len(fills) + 2, V), device=cuda, dtype=dt)
    for r, fill in enumerate(fills):
        x[r] = fill
    x[6], x[7] = low, -1e20
    x[6, V // 3], x[7, V - 1] = high, 2.0
    ids = torch.tensor([V - 1, 0, 1, V // 2, 5, 7, V // 3, V - 1], dtype=torch.int32, device=cuda)
    logp, entropy, lse, top_logps, top_ids = ops.token_logprobs(x, ids, top=2, split=split)
    even = torch.log(torch.tensor([V] * len(fills) + [1, 1], dtype=torch.float64))
    near = 4 * 2.0 ** -24 * even
    assert ((entropy.cpu().double() - even).abs() <= near).all()
    assert ((logp.cpu().double() + even).abs() <= near).all()
    assert ((top_logps[:, 0].cpu().double() + even).abs() <= near).all()
    assert top_ids[:, 0].tolist() == [0] * len(fills) + [V // 3, V - 1]
    most = x.double().amax(1).cpu()
    assert ((lse.cpu().double() - (most + even)).abs() <= 4 * 2.0 ** -24 * (most.abs() + even)).all()


@pytest.mark.parametrize("split", [True, False])
@pytest.mark.parametrize("V", [600011, 1100003])
def test_long_rows(cuda, V, split):
    """Slices of several runs, and more runs than a lane has maxima apart: random, few values,
    rising and falling rows, one token left, two equal tokens at the ends, a constant."""
    at = torch.arange(V, device=cuda)
    x, ids = logits_of(cuda, 7, V, BF16)
    x[1] = (at * 7 % 5).to(BF16)
    x[2], x[3] = (at.float() / V * 30).to(BF16), (at.float() / V * -30).to(BF16)
    x[4], x[5], x[6] = -float("inf"), torch.finfo(BF16).min, -1.5
    x[4, V // 2], x[5, 0], x[5, V - 1] = 1.0, 1.0, 1.0
    ids[4], ids[5] = V // 2, V - 1
    for top in (0, 1, 32):
        check(x, ids, top, split=split)
        check(x[:1], ids[:1], top, split=split)
