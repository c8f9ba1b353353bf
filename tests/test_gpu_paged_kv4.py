"""Decoding attention over a 4-bit cache against float64 on the values that it holds, within
attention_ref.py's bounds (the weights keep 16 bits and more, so they are wider than needed)."""
import pytest
import torch

import attention_ref
import rope_kv4_ref as ref
from gomlx_hip import ops
from test_gpu_kv4 import cache4, freqs_of, rand, table_of

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [(BF16, 128), (F16, 64), (BF16, 96), (F16, 256), (F32, 128), (F32, 256), (F32, 32), (BF16, 32), (BF16, 256), (F16, 160)]


def held(c, table, b, n, D):
    """[1, Hkv, n, D]: the values of a sequence's first n tokens, in float64."""
    t = ref.decode(*c, D)[table[b].long().clamp(0, c[0].shape[0] - 1)]
    return t.transpose(1, 2).reshape(-1, t.shape[1], D)[:n].transpose(0, 1)[None]


def check(q, kc, vc, table, lens, scale, window, sinks, got, hidden=None):
    D, cap = q.shape[2], table.shape[1] * kc[0].shape[2]
    for b, n in enumerate(lens.tolist()):
        n = min(max(n, 0), cap)
        if n == 0:
            assert not got[b].any()
            continue
        k, v = held(kc, table, b, n, D), held(vc, table, b, n, D)
        see = attention_ref.visible(1, 1, n, n - 1, window, sinks, device=q.device)
        if hidden is not None:
            see = see & ~hidden[b, :n]
        k, v = (torch.where(see[0, 0, 0][:, None], t, torch.zeros_like(t)) for t in (k, v))
        o, _, bound, _ = attention_ref.forward(q[b][None, :, None], k, v, scale, see)
        attention_ref.within(got[b][None, :, None], o, bound, f"sequence {b} of {n}")


CASES = [  # (B, H, Hkv, page, per, lens, window, sinks)
    (1, 1, 1, 16, 1, (1,), 0, 0),
    (3, 4, 4, 16, 8, (0, 128, 77), 0, 0),              # an empty sequence, a full one
    (6, 8, 2, 16, 25, (1, 63, 64, 65, 128, 399), 0, 0),
    (2, 8, 1, 64, 40, (2560, 2001), 0, 0),             # many tiles: units split over workers
    (1, 32, 8, 32, 300, (9600,), 0, 0),
    (4, 8, 2, 16, 64, (1024, 1000, 100, 3), 100, 4),   # a window with sinks, a gap and none
    (3, 2, 2, 16, 64, (1024, 513, 40), 33, 0),
    (3, 4, 2, 16, 64, (1024, 700, 90), 16, 90),        # sinks of several tiles
    (2, 40, 2, 16, 32, (512, 130), 0, 0),              # 20 heads a kv head: two units
    (2, 33, 1, 8, 80, (640, 33), 64, 2),               # pages of 8
    (2, 4, 2, 20, 30, (600, 411), 100, 5),             # pages that end inside a tile
    (2, 4, 2, 1, 90, (90, 61), 0, 0),                  # pages of one token
    (2, 4, 2, 7, 90, (1000, -5), 0, 0),                # lengths out of range are clamped
    (70, 4, 2, 16, 30, tuple((67 * i) % 481 for i in range(70)), 50, 3),  # more sequences than a wave has lanes
    (130, 2, 1, 16, 2, tuple(i % 33 for i in range(130)), 0, 0),
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dt,D", TYPES)
def test_attention(cuda, case, dt, D):
    B, H, Hkv, page, per, lens, window, sinks = case
    print(case, dt, D, flush=True)
    pages, table = table_of(cuda, B, per)
    q = rand(cuda, B, H, D, dt=dt, seed=9)
    n = torch.tensor(lens, dtype=torch.int32, device=cuda)
    for layout in ("token", "head"):
        kc, vc = cache4(cuda, pages, page, Hkv, D, layout)
        for split in (False, True):
            got = ops.sdpa_paged_kv4(q, kc, vc, table, n, D ** -0.5, window, sinks, split=split)
            check(q, kc, vc, table, n, D ** -0.5, window, sinks, got)


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 96), (F32, 32), (BF16, 160)])
@pytest.mark.parametrize("split", [False, True])
def test_unseen_rows_reach_nothing(cuda, dt, D, split):
    """Scales of 255 (NaN) in every row that is not seen and in the bytes of seen rows that belong
    to no value; table entries behind the length name no page."""
    B, H, Hkv, page, per, window, sinks = 3, 8, 2, 20, 60, 70, 3
    pages, table = table_of(cuda, B, per)
    kc, vc = cache4(cuda, pages, page, Hkv, D, "token")
    lens = torch.tensor([per * page - 9, 333, 50], dtype=torch.int32, device=cuda)
    q = rand(cuda, B, H, D, dt=dt)
    want = ops.sdpa_paged_kv4(q, kc, vc, table, lens, 0.1, window, sinks, split=split)
    check(q, kc, vc, table, lens, 0.1, window, sinks, want)
    k2, v2 = ([torch.full_like(t, 255) for t in c] for c in (kc, vc))
    t2 = table.clone()
    for b, n in enumerate(lens.tolist()):
        j = torch.arange(n, device=cuda)
        j = j[(j >= n - window) | (j < sinks)]
        pg = table[b].long()[j // page]
        for c, c2 in ((kc, k2), (vc, v2)):
            c2[0][pg, :, j % page] = c[0][pg, :, j % page]
            c2[1][..., :D // 32][pg, :, j % page] = c[1][..., :D // 32][pg, :, j % page]
        t2[b, (n + page - 1) // page:] = 2 ** 31 - 1 if b else -1
    assert torch.equal(ops.sdpa_paged_kv4(q, k2, v2, t2, lens, 0.1, window, sinks, split=split), want)
    # A NaN that is seen reaches its own sequence's kv head, no other.
    b, j = 1, 332
    k2[1][int(table[b, j // page]), 1, j % page, 0] = 255
    got = ops.sdpa_paged_kv4(q, k2, v2, t2, lens, 0.1, window, sinks, split=split)
    assert got[1, 4:].isnan().all() and torch.equal(got[1, :4], want[1, :4]) and torch.equal(got[[0, 2]], want[[0, 2]])


@pytest.mark.parametrize("split", [False, True])
def test_bad_pages_are_not_seen(cuda, split):
    B, H, Hkv, D, page, per = 2, 4, 2, 128, 16, 40
    pages, table = table_of(cuda, B, per)
    kc, vc = cache4(cuda, pages, page, Hkv, D, "head")
    lens = torch.tensor([640, 500], dtype=torch.int32, device=cuda)
    table[0, 3], table[0, 39], table[1, 0], table[1, 5] = -1, pages, -2 ** 31, 2 ** 31 - 1
    hidden = torch.stack([((t < 0) | (t >= pages)).repeat_interleave(page) for t in table])
    q = rand(cuda, B, H, D)
    got = ops.sdpa_paged_kv4(q, kc, vc, table, lens, 0.1, split=split)
    check(q, kc, vc, table, lens, 0.1, 0, 0, got, hidden)
    table[:] = -1
    assert not ops.sdpa_paged_kv4(q, kc, vc, table, lens, 0.1, split=split).any()


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_values_of_every_size(cuda, dt):
    """Values up to 2^100 and down to 2^-100 in one cache: sums in fp32 of exact values, whatever
    the queries' type (f16 holds neither)."""
    B, H, Hkv, D, page, per = 1, 4, 1, 64, 16, 20
    pages, table = table_of(cuda, B, per)
    kc, vc = cache4(cuda, pages, page, Hkv, D, "head")
    for byte, c in ((227, vc), (27, vc), (20, kc)):
        for t in (c[1],):
            t.fill_(byte)
        q = rand(cuda, B, H, D, dt=dt)
        lens = torch.tensor([320], dtype=torch.int32, device=cuda)
        got = ops.sdpa_paged_kv4(q.float(), kc, vc, table, lens, 0.1)
        check(q.float(), kc, vc, table, lens, 0.1, 0, 0, got)
        if dt != F16:
            check(q, kc, vc, table, lens, 0.1, 0, 0, ops.sdpa_paged_kv4(q, kc, vc, table, lens, 0.1))


def test_query_and_output_strides(cuda):
    B, H, Hkv, D = 3, 8, 2, 64
    pages, table = table_of(cuda, B, 30)
    kc, vc = cache4(cuda, pages, 16, Hkv, D, "token")
    lens = torch.tensor([480, 100, 7], dtype=torch.int32, device=cuda)
    q = rand(cuda, B, H + 4, D, dt=F16)[:, :H]  # a slice of a fused projection
    want = ops.sdpa_paged_kv4(q.contiguous(), kc, vc, table, lens, 0.1)
    out = torch.zeros((H, B, D), dtype=F16, device=cuda)
    ops.sdpa_paged_kv4(q, kc, vc, table, lens, 0.1, out=out.transpose(0, 1))
    assert torch.equal(out.transpose(0, 1), want)
    wide = torch.full((B, 50), -7, dtype=torch.int32, device=cuda)
    wide[:, 10:40] = table
    assert torch.equal(ops.sdpa_paged_kv4(q, kc, vc, wide[:, 10:40], lens, 0.1), want)


def test_offsets_past_32_bits(cuda):
    """Codes of more than 4 GiB: the pages at both ends."""
    Hkv, D, page = 8, 128, 64
    pages = (9 << 30) // 2 // (Hkv * page * 64)
    codes = torch.zeros((pages, Hkv, page, 64), dtype=torch.uint8, device=cuda)
    scales = torch.full((pages, Hkv, page, 4), 127, dtype=torch.uint8, device=cuda)
    table = torch.tensor([[pages - 1, 0, pages - 2, 1, pages // 2, pages - 3]], dtype=torch.int32, device=cuda)
    lens = torch.tensor([6 * page], dtype=torch.int32, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(0)
    for p in table[0].tolist():
        codes[p] = torch.randint(0, 256, codes[p].shape, generator=g, device=cuda, dtype=torch.uint8)
    c = (codes, scales)
    q = rand(cuda, 1, 32, D)
    few = table[0].long()
    small = (codes[few].contiguous(), scales[few].contiguous())
    order = torch.arange(6, dtype=torch.int32, device=cuda)[None]
    for split in (False, True):
        assert torch.equal(ops.sdpa_paged_kv4(q, c, c, table, lens, 0.1, split=split),
                           ops.sdpa_paged_kv4(q, small, small, order, lens, 0.1, split=split))
    k = rand(cuda, 1, Hkv, 1, D)
    at = torch.tensor([5], dtype=torch.int32, device=cuda)
    for cache, t in ((c, table), (small, order)):
        ops.kv4_append_rope(None, k, k, cache, cache, t, at, freqs_of(64, cuda))
    assert torch.equal(codes[pages - 1], small[0][0]) and torch.equal(scales[pages - 1], small[1][0])
    assert all(torch.equal(a, b) for a, b in zip(ops.kv4_read(c, c, table, 300), ops.kv4_read(small, small, order, 300)))


def test_captured_calls_share_a_workspace(cuda):
    B, H, Hkv, D, page, per = 4, 8, 2, 128, 16, 80
    pages, table = table_of(cuda, B, per)
    kc, vc = cache4(cuda, pages, page, Hkv, D, "head")
    q = rand(cuda, 2, B, H, D)
    lens = torch.tensor([[1000, 30, 500, 1], [1280, 31, 77, 640]], dtype=torch.int32, device=cuda)
    ws = ops.sdpa_paged_kv4_workspace(q[0], kc, table)
    ops.sdpa_paged_kv4(q[0], kc, vc, table, lens[0], 0.1, workspace=ws)
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, ops.sdpa_paged_kv4(q[i], kc, vc, table, lens[i], 0.1, 300, 4, workspace=ws)))
    for turn in range(3):
        q.add_(0.25 * (turn + 1))
        lens.sub_(turn).clamp_(min=0)
        got = []
        for g, o in graphs:
            g.replay()
            got.append(o.clone())
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(got[i], ops.sdpa_paged_kv4(q[i], kc, vc, table, lens[i], 0.1, 300, 4))


def test_a_serving_step(cuda):
    """Prompts, a later chunk and tokens one by one with every operator in its place: rotation and
    append into 4 bits, windowed attention over the tokens read back, decoding attention, log
    probabilities of the answers; each step against float64 on the values that the cache holds."""
    B, H, Hkv, D, page, per, V = 3, 8, 2, 64, 16, 12, 1000
    dt, scale, sections = BF16, D ** -0.5, (8, 12, 12)
    pages, table = table_of(cuda, B, per)
    kc, vc = ops.kv4_cache(pages, page, Hkv, D, cuda), ops.kv4_cache(pages, page, Hkv, D, cuda)
    freqs, head = freqs_of(32, cuda), rand(cuda, V, H * D, dt=dt, seed=3)
    at = torch.zeros(B, dtype=torch.int32, device=cuda)
    new = torch.tensor([70, 41, 1], dtype=torch.int32, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(4)
    for chunk in range(2):  # a prompt with pictures, then a second chunk behind it
        qkv = rand(cuda, B, 70, H + 2 * Hkv, D, seed=20 + chunk).transpose(1, 2)
        q, k, v = qkv.split([H, Hkv, Hkv], 1)
        pos = torch.randint(0, 100, (3, B, 70), generator=g, device=cuda, dtype=torch.int32)
        ops.kv4_append_rope(q, k, v, kc, vc, table, at, freqs, counts=new, positions=pos, sections=sections, q_out=q)
        attention_ref.within(q[0, :, :5], *(t[0, :, :5] for t in ref.rotate(rand(cuda, B, 70, H + 2 * Hkv, D, seed=20 + chunk).transpose(1, 2)[:, :H], pos, freqs, sections)))
        at += new
        keys, values = ops.kv4_read(kc, vc, table, int(at.max()), lens=at)
        for b, n in enumerate(at.tolist()):  # (chunks of different lengths: a sequence at a time)
            first = n - int(new[b])
            args = q[b:b + 1, :, :n - first], keys[b:b + 1, :, :n], values[b:b + 1, :, :n]
            got = ops.sdpa_window(*args, scale, q_start=first)
            see = attention_ref.visible(1, n - first, n, first, 0, 0, device=cuda)
            k64, v64 = held(kc, table, b, n, D), held(vc, table, b, n, D)
            o, _, bound, _ = attention_ref.forward(args[0], k64, v64, scale, see)
            attention_ref.within(got, o, bound, "prompt")
    ws = None
    for step in range(5):
        qkv = rand(cuda, B, 1, H + 2 * Hkv, D, seed=40 + step).transpose(1, 2)
        q, k, v = qkv.split([H, Hkv, Hkv], 1)
        q = ops.kv4_append_rope(q, k, v, kc, vc, table, at, freqs)
        at += 1
        ws = ops.sdpa_paged_kv4_workspace(q[:, :, 0], kc, table) if ws is None else ws
        o = ops.sdpa_paged_kv4(q[:, :, 0], kc, vc, table, at, scale, workspace=ws)
        check(q[:, :, 0], kc, vc, table, at, scale, 0, 0, o)
        logits = ops.gemm(o.reshape(B, H * D), head.t())
        ids = ops.argminmax(logits, 1)
        logp, H_, lse, lp, best = ops.token_logprobs(logits, ids, top=4)
        wants = ref.logprobs(logits, ids, 1.0, 64)
        for got, (want, bound) in zip((logp, H_, lse), wants):
            attention_ref.within(got, want, bound, "log probabilities")
        assert torch.equal(best[:, 0], ids) and torch.equal(lp[:, 0], logp)
        assert torch.equal(best.cpu(), ref.top(logits.cpu(), 4))
