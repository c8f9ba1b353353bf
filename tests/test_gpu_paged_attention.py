"""The paged key-value cache: kv_append against torch indexing (bit for bit) and
sdpa_paged against float64 within the rounding bounds of attention_ref.py (the joined
shares are fp32: what joining adds is in the bound's fp32 part)."""
import pytest
import torch

import attention_ref as ref
from gomlx_hip import ops
from gomlx_hip._lib import BackendError

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [(BF16, 128), (F16, 64), (BF16, 80), (F16, 256), (F32, 128), (F32, 64), (F32, 36), (BF16, 8)]


def cache(cuda, B, Hkv, D, page, per, dt, layout="token", seed=0, spare=2):
    """(k_cache, v_cache) viewed as [pages, Hkv, page, D] and a table of shuffled pages."""
    g = torch.Generator(device=cuda).manual_seed(seed + B + 3 * page + D)
    pages = B * per + spare
    shape = (pages, page, Hkv, D) if layout == "token" else (pages, Hkv, page, D)
    kv = [torch.randn(shape, generator=g, device=cuda).to(dt) for _ in range(2)]
    if layout == "token":
        kv = [t.transpose(1, 2) for t in kv]
    table = torch.randperm(pages, generator=g, device=cuda)[: B * per].view(B, per).to(torch.int32)
    return kv[0], kv[1], table


def dense(c, table, b, n):
    """[1, Hkv, n, D]: a sequence's first n tokens."""
    t = c[table[b].long().clamp(0, c.shape[0] - 1)]
    return t.transpose(1, 2).reshape(-1, c.shape[1], c.shape[3])[:n].transpose(0, 1)[None]


def check(q, kc, vc, table, lens, scale, window, sinks, got, hidden=None):
    cap = table.shape[1] * kc.shape[2]
    for b, n in enumerate(lens.tolist()):
        n = min(max(n, 0), cap)
        if n == 0:
            assert not got[b].any()
            continue
        k, v = dense(kc, table, b, n), dense(vc, table, b, n)
        see = ref.visible(1, 1, n, n - 1, window, sinks, device=q.device)
        if hidden is not None:
            see = see & ~hidden[b, :n]
        # what is not seen is not used, whatever it holds
        k, v = (torch.where(see[0, 0, 0][:, None], t, torch.zeros_like(t)) for t in (k, v))
        o, _, bound, _ = ref.forward(q[b][None, :, None], k, v, scale, see)
        ref.within(got[b][None, :, None], o, bound, f"sequence {b} of {n}")


CASES = [  # (B, H, Hkv, page, per, lens, window, sinks)
    (1, 1, 1, 16, 1, (1,), 0, 0),
    (3, 4, 4, 16, 8, (0, 128, 77), 0, 0),              # an empty sequence, a full one
    (6, 8, 2, 16, 20, (1, 15, 16, 17, 64, 319), 0, 0),
    (2, 8, 1, 64, 40, (2560, 2001), 0, 0),             # many tiles: units split over workers
    (1, 32, 8, 32, 300, (9600,), 0, 0),
    (4, 8, 2, 16, 64, (1024, 1000, 100, 3), 100, 4),   # a window with sinks, a gap and none
    (3, 2, 2, 16, 64, (1024, 513, 40), 33, 0),
    (3, 4, 2, 16, 64, (1024, 700, 90), 16, 90),        # sinks of several tiles
    (2, 40, 2, 16, 16, (256, 130), 0, 0),              # 20 heads a kv head: two units
    (2, 33, 1, 8, 40, (320, 33), 64, 2),               # pages of 8
    (2, 4, 2, 20, 30, (600, 411), 100, 5),             # pages that end inside a tile
    (2, 4, 2, 1, 90, (90, 61), 0, 0),                  # pages of one token
    (2, 4, 2, 7, 90, (1000, -5), 0, 0),                # lengths out of range are clamped
    (70, 4, 2, 16, 12, tuple((37 * i) % 193 for i in range(70)), 50, 3),  # more sequences than a wave has lanes
    (130, 2, 1, 16, 2, tuple(i % 33 for i in range(130)), 0, 0),
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dt,D", TYPES)
def test_paged_attention(cuda, case, dt, D):
    B, H, Hkv, page, per, lens, window, sinks = case
    print(case, dt, D, flush=True)
    for layout in ("token", "head"):
        kc, vc, table = cache(cuda, B, Hkv, D, page, per, dt, layout)
        q = torch.randn((B, H, D), generator=torch.Generator(device=cuda).manual_seed(5), device=cuda).to(dt)
        n = torch.tensor(lens, dtype=torch.int32, device=cuda)
        for split in (False, True):
            got = ops.sdpa_paged(q, kc, vc, table, n, D ** -0.5, window, sinks, split=split)
            check(q, kc, vc, table, n, D ** -0.5, window, sinks, got)


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F32, 128), (BF16, 80)])
@pytest.mark.parametrize("page", [16, 20])
@pytest.mark.parametrize("split", [False, True])
def test_unseen_rows_reach_nothing(cuda, dt, D, page, split):
    """NaN and infinities in every row that is not seen: behind the length, before the
    window, on no sequence's page; table entries behind the length name no page."""
    B, H, Hkv, per, window, sinks = 3, 8, 2, 60, 70, 3
    kc, vc, table = cache(cuda, B, Hkv, D, page, per, dt)
    lens = torch.tensor([per * page - 9, 333, 50], dtype=torch.int32, device=cuda)
    q = torch.randn((B, H, D), device=cuda).to(dt)
    want = ops.sdpa_paged(q, kc, vc, table, lens, 0.1, window, sinks, split=split)
    check(q, kc, vc, table, lens, 0.1, window, sinks, want)
    for fill in (float("nan"), float("inf"), torch.finfo(dt).min):
        k2, v2 = torch.full_like(kc, fill), torch.full_like(vc, fill)
        t2 = table.clone()
        for b, n in enumerate(lens.tolist()):
            j = torch.arange(n, device=cuda)
            j = j[(j >= n - window) | (j < sinks)]
            pg = table[b].long()[j // page]
            k2[pg, :, j % page], v2[pg, :, j % page] = kc[pg, :, j % page], vc[pg, :, j % page]
            t2[b, (n + page - 1) // page:] = 2 ** 31 - 1 if b else -1
        got = ops.sdpa_paged(q, k2, v2, t2, lens, 0.1, window, sinks, split=split)
        assert torch.equal(got, want)


@pytest.mark.parametrize("split", [False, True])
def test_bad_pages_are_not_seen(cuda, split):
    B, H, Hkv, D, page, per = 2, 4, 2, 128, 16, 40
    kc, vc, table = cache(cuda, B, Hkv, D, page, per, BF16)
    lens = torch.tensor([640, 500], dtype=torch.int32, device=cuda)
    table[0, 3], table[0, 39], table[1, 0], table[1, 5] = -1, kc.shape[0], -2 ** 31, 2 ** 31 - 1
    hidden = torch.zeros((B, per * page), dtype=torch.bool, device=cuda)
    for b in range(B):
        bad = (table[b] < 0) | (table[b] >= kc.shape[0])
        hidden[b] = bad.repeat_interleave(page)
    q = torch.randn((B, H, D), device=cuda).to(BF16)
    got = ops.sdpa_paged(q, kc, vc, table, lens, 0.1, split=split)
    check(q, kc, vc, table, lens, 0.1, 0, 0, got, hidden)
    table[:] = -1
    assert not ops.sdpa_paged(q, kc, vc, table, lens, 0.1, split=split).any()


def test_query_and_output_strides(cuda):
    B, H, Hkv, D = 3, 8, 2, 64
    kc, vc, table = cache(cuda, B, Hkv, D, 16, 30, F16)
    lens = torch.tensor([480, 100, 7], dtype=torch.int32, device=cuda)
    qkv = torch.randn((B, H + 2 * Hkv, D), device=cuda).to(F16)
    q = qkv[:, :H]  # a slice of a fused projection
    want = ops.sdpa_paged(q.contiguous(), kc, vc, table, lens, 0.1)
    out = torch.zeros((H, B, D), dtype=F16, device=cuda)
    ops.sdpa_paged(q, kc, vc, table, lens, 0.1, out=out.transpose(0, 1))
    assert torch.equal(out.transpose(0, 1), want)
    # a table that is a slice of a wider one, a cache with a head of rows between heads
    wide = torch.full((B, 50), -7, dtype=torch.int32, device=cuda)
    wide[:, 10:40] = table
    k3 = torch.stack([kc, kc], 2).flatten(1, 2)[:, ::2]
    assert torch.equal(ops.sdpa_paged(q, k3, vc, wide[:, 10:40], lens, 0.1), want)


def test_offsets_past_32_bits(cuda):
    """A cache of more than 4 GiB (K and V in one), its last pages used."""
    pages, Hkv, page, D = 70000, 2, 64, 128
    store = torch.zeros((2, pages, Hkv, page, D), dtype=BF16, device=cuda)  # 2 x 2.3 GB
    kc, vc = store[0], store[1]
    lens = torch.tensor([200, 129], dtype=torch.int32, device=cuda)
    table = torch.tensor([[69999, 3, 69998, 34000], [35001, 69997, 1, 2]], dtype=torch.int32, device=cuda)
    k, v = (torch.randn((2, Hkv, 200, D), device=cuda).to(BF16) for _ in range(2))
    # pages twice as far apart: offsets up to 9 GB from the caches' base
    far = torch.zeros((pages, 2, Hkv, page, D), dtype=BF16, device=cuda)
    kf, vf = far[:, 0], far[:, 1]
    zero = torch.zeros(2, dtype=torch.int32, device=cuda)
    q = torch.randn((2, 8, D), device=cuda).to(BF16)
    for a, b in ((kc, vc), (kf, vf)):
        ops.kv_append(k, v, a, b, table, zero, counts=lens)
        got = ops.sdpa_paged(q, a, b, table, lens, 0.1)
        for s in range(2):
            n = int(lens[s])
            assert torch.equal(dense(a, table, s, n)[0], k[s, :, :n])
        check(q, a, b, table, lens, 0.1, 0, 0, got)


# ---------------------------------------------------------------- append
def append_ref(k, v, kc, vc, table, starts, counts):
    page = kc.shape[2]
    for b in range(k.shape[0]):
        for i in range(min(k.shape[2], k.shape[2] if counts is None else int(counts[b]))):
            pos = int(starts[b]) + i
            if not 0 <= pos < table.shape[1] * page:
                continue
            pg = int(table[b, pos // page])
            if 0 <= pg < kc.shape[0]:
                kc[pg, :, pos % page], vc[pg, :, pos % page] = k[b, :, i], v[b, :, i]


APPENDS = [  # (B, S, Hkv, D, page, per, starts, counts, dtype)
    (1, 1, 1, 128, 16, 1, (0,), None, BF16),
    (4, 1, 8, 128, 64, 4, (0, 63, 64, 255), None, BF16),
    (3, 40, 2, 64, 16, 6, (0, 17, 56), (40, 3, 0), F16),
    (3, 9, 3, 80, 20, 3, (-4, 55, 60), None, BF16),        # before the first token, past the last page
    (2, 33, 2, 36, 7, 9, (0, 30), (50, -1), F32),          # counts out of range
    (2, 6, 2, 5, 4, 4, (3, 1), None, BF16),                # rows of 10 bytes
    (2, 6, 1, 3, 4, 4, (3, 1), None, torch.int8),
    (2, 6, 1, 3, 4, 4, (3, 1), None, torch.float64),
    (2, 300, 4, 256, 32, 12, (11, 64), (300, 299), BF16),
]


@pytest.mark.parametrize("case", APPENDS)
@pytest.mark.parametrize("layout", ["token", "head"])
def test_append(cuda, case, layout):
    B, S, Hkv, D, page, per, starts, counts, dt = case
    print(case, layout, flush=True)
    kc, vc, table = cache(cuda, B, Hkv, D, page, per, torch.float32, layout)
    kc, vc = kc.mul(50).to(dt), vc.mul(50).to(dt)
    if B > 1:
        table[0, -1] = -3
        table[1, 0] = kc.shape[0]
    k, v = (torch.randn((B, S, Hkv, D), device=cuda).mul(50).to(dt).transpose(1, 2) for _ in range(2))
    st = torch.tensor(starts, dtype=torch.int32, device=cuda)
    ct = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=cuda)
    k2, v2 = kc.clone(), vc.clone()
    append_ref(k, v, k2, v2, table, st, ct)
    ops.kv_append(k, v, kc, vc, table, st, ct)
    assert torch.equal(kc, k2) and torch.equal(vc, v2)
    # other storage of the new tokens: the same rows
    kc2, vc2 = torch.zeros_like(kc), torch.zeros_like(vc)
    ops.kv_append(k.contiguous(), v.contiguous(), kc2, vc2, table, st, ct)
    kc3, vc3 = torch.zeros_like(kc), torch.zeros_like(vc)
    append_ref(k, v, kc3, vc3, table, st, ct)
    assert torch.equal(kc2, kc3) and torch.equal(vc2, vc3)


def test_append_unaligned(cuda):
    """Rows that start at odd elements."""
    kc, vc, table = cache(cuda, 2, 2, 64, 16, 3, BF16)
    store = torch.randn((2, 2, 5, 67), device=cuda).to(BF16)
    k = store[..., 3:]
    st = torch.tensor([0, 14], dtype=torch.int32, device=cuda)
    k2, v2 = kc.clone(), vc.clone()
    append_ref(k, k, k2, v2, table, st, None)
    ops.kv_append(k, k, kc, vc, table, st)
    assert torch.equal(kc, k2) and torch.equal(vc, v2)


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("dt,D,H,Hkv", [(BF16, 128, 8, 2), (F16, 64, 4, 4), (F32, 64, 4, 2)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
def test_prompt_then_decoding(cuda, dt, D, H, Hkv, window, sinks):
    """Prompts of several lengths through the windowed attention and into the pages, then
    tokens one by one: every step's output is the whole sequence's row in float64."""
    B, S, steps, page, per = 3, 70, 20, 16, 6
    lens = torch.tensor([70, 41, 1], dtype=torch.int32, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(9)
    total = S + steps
    q = torch.randn((B, H, total, D), generator=g, device=cuda).to(dt)
    k, v = (torch.randn((B, Hkv, total, D), generator=g, device=cuda).to(dt) for _ in range(2))
    kc, vc, table = cache(cuda, B, Hkv, D, page, per, dt)
    scale = D ** -0.5
    out = ops.sdpa_window(q[:, :, :S], k[:, :, :S], v[:, :, :S], scale, window, sinks, q_start=0, lens=lens)
    ops.kv_append(k[:, :, :S], v[:, :, :S], kc, vc, table, torch.zeros_like(lens), counts=lens)
    see = ref.visible(B, total, total, 0, window, sinks, device=cuda)
    want, _, bound, _ = ref.forward(q, k, v, scale, see)
    for b, n in enumerate(lens.tolist()):
        ref.within(out[b, :, :n], want[b, :, :n], bound[b, :, :n], "prompt")
    at = lens.clone()
    rows = torch.arange(B, device=cuda)
    ws = ops.sdpa_paged_workspace(q[:, :, 0], kc, table)
    for _ in range(steps):
        i = at.long()
        ops.kv_append(k[rows, :, i][:, :, None], v[rows, :, i][:, :, None], kc, vc, table, at)
        at += 1
        got = ops.sdpa_paged(q[rows, :, i].contiguous(), kc, vc, table, at, scale, window, sinks, workspace=ws)
        ref.within(got, want[rows, :, i], bound[rows, :, i], "decoding")


def test_captured_steps_share_a_workspace(cuda):
    """Two captured decoding steps (append, then attention) with one workspace, replayed
    in turn with eager work between, against eager calls."""
    B, H, Hkv, D, page, per = 4, 8, 2, 128, 16, 80
    kc, vc, table = cache(cuda, B, Hkv, D, page, per, BF16)
    q = torch.randn((2, B, H, D), device=cuda).to(BF16)
    k, v = (torch.randn((2, B, Hkv, 1, D), device=cuda).to(BF16) for _ in range(2))
    lens = torch.tensor([[1000, 30, 500, 1], [1280, 31, 77, 640]], dtype=torch.int32, device=cuda)
    ws = torch.empty(1 << 24, dtype=torch.uint8, device=cuda)
    graphs, outs = [], []
    for i in range(2):
        starts = (lens[i] - 1).contiguous()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            ops.kv_append(k[i], v[i], kc, vc, table, starts)
            outs.append(ops.sdpa_paged(q[i], kc, vc, table, lens[i], 0.1, 300, 4, workspace=ws))
        graphs.append((gr, starts))
    k2, v2 = kc.clone(), vc.clone()
    for turn in range(3):
        q.add_(0.25 * (turn + 1))
        k.mul_(-0.5)
        got = []
        for (gr, _), o in zip(graphs, outs):
            gr.replay()
            got.append(o.clone())
        torch.cuda.synchronize()
        for i in range(2):
            ops.kv_append(k[i], v[i], k2, v2, table, graphs[i][1])
            assert torch.equal(got[i], ops.sdpa_paged(q[i], k2, v2, table, lens[i], 0.1, 300, 4))
        assert torch.equal(kc, k2) and torch.equal(vc, v2)


def test_same_bits_on_another_stream(cuda):
    kc, vc, table = cache(cuda, 3, 2, 128, 16, 200, F16)
    lens = torch.tensor([3200, 1700, 64], dtype=torch.int32, device=cuda)
    q = torch.randn((3, 8, 128), device=cuda).to(F16)
    want = ops.sdpa_paged(q, kc, vc, table, lens, 0.1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.sdpa_paged(q, kc, vc, table, lens, 0.1)
    s.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("handle", ["own", 0])
def test_a_stream_of_the_callers(cuda, handle):
    """`stream` as a handle (0: the default stream) while torch's current stream is another;
    the workspace stays the call's until that stream is done with it."""
    kc, vc, table = cache(cuda, 4, 2, 64, 16, 40, BF16)
    q = torch.randn((4, 8, 64), device=cuda).to(BF16)
    lens = torch.tensor([640, 3, 0, 500], dtype=torch.int32, device=cuda)
    want = ops.sdpa_paged(q, kc, vc, table, lens, 0.1)
    s, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        for _ in range(5):
            got = torch.zeros_like(want)
            torch.cuda.synchronize()
            ops.sdpa_paged(q, kc, vc, table, lens, 0.1, out=got, stream=s.cuda_stream if handle == "own" else handle)
            junk = [torch.full((1 << 20,), float("nan"), device=cuda) for _ in range(8)]
            torch.cuda.synchronize()
            assert torch.equal(got, want)
            del junk


def test_refusals_on_the_device(cuda):
    kc, vc, table = cache(cuda, 2, 2, 64, 16, 3, BF16)
    q = torch.randn((2, 4, 64), device=cuda).to(BF16)
    lens = torch.tensor([3, 4], dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError, match="block_table"):
        ops.sdpa_paged(q, kc, vc, table.long(), lens, 0.1)
    with pytest.raises(ValueError, match="block_table"):
        ops.sdpa_paged(q, kc, vc, table[:1], lens, 0.1)
    with pytest.raises(ValueError, match="lens"):
        ops.sdpa_paged(q, kc, vc, table, lens.long(), 0.1)
    with pytest.raises(ValueError, match="v_cache"):
        ops.sdpa_paged(q, kc, vc[:2], table, lens, 0.1)
    with pytest.raises(ValueError, match="k_cache"):
        ops.sdpa_paged(q.half(), kc, vc, table, lens, 0.1)
    with pytest.raises(ValueError, match="workspace must be contiguous"):
        ops.sdpa_paged(q, kc, vc, table, lens, 0.1,
                       workspace=torch.empty(1, dtype=torch.uint8, device=cuda).expand(1 << 20))
    with pytest.raises(BackendError, match="multiple of num_kv_heads"):
        ops.sdpa_paged(q[:, :3], kc, vc, table, lens, 0.1)
    k = torch.randn((2, 2, 1, 64), device=cuda)
    with pytest.raises(ValueError, match="k_cache"):
        ops.kv_append(k, k, kc, vc, table, lens)
    with pytest.raises(ValueError, match="starts"):
        ops.kv_append(k.to(BF16), k.to(BF16), kc, vc, table, lens[:1])
    assert ops.sdpa_paged(q[:0], kc, vc, table[:0], lens[:0], 0.1).shape == (0, 4, 64)
