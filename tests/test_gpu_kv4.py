"""The appends that rotate, into 16 and into 4 bits, and the way back: against rope_kv4_ref.py,
codes bit for bit where nothing turns; bad pages, counts, rows that stay as they were."""
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


def table_of(cuda, B, per, spare=3, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    pages = B * per + spare
    return pages, torch.randperm(pages, generator=g, device=cuda)[:B * per].view(B, per).to(torch.int32)


def cache16(cuda, pages, page, Hkv, D, dt, layout, seed=5):
    shape = (pages, page, Hkv, D) if layout == "token" else (pages, Hkv, page, D)
    c = [rand(cuda, *shape, dt=dt, seed=seed + i) for i in range(2)]
    return [t.transpose(1, 2) if layout == "token" else t for t in c]


def cache4(cuda, pages, page, Hkv, D, layout, seed=5):
    """Two caches of random bytes: codes and scales of the middle sizes."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    wide = (D + 127) // 128 * 4
    made = []
    for _ in range(2):
        pair = []
        for width, lo, hi in ((D // 2, 0, 256), (wide, 120, 132)):
            shape = (pages, page, Hkv, width) if layout == "token" else (pages, Hkv, page, width)
            t = torch.randint(lo, hi, shape, generator=g, device=cuda, dtype=torch.uint8)
            pair.append(t.transpose(1, 2) if layout == "token" else t)
        made.append(tuple(pair))
    return made


def rows_of(table, starts, counts, S, page, pages):
    """(b, i, page, row) of every token that is appended."""
    out = []
    for b, n in enumerate(counts):
        for i in range(min(S, max(n, 0))):
            pos = starts[b] + i
            if 0 <= pos < table.shape[1] * page:
                pg = int(table[b, pos // page])
                if 0 <= pg < pages:
                    out.append((b, i, pg, pos % page))
    return out


CASES = [  # (B, S, H, Hkv, D, R, page, per, starts, counts, sections)
    (1, 1, 8, 2, 64, 64, 16, 2, (3,), None, None),
    (3, 1, 4, 4, 128, 128, 16, 3, (0, 47, 15), None, None),
    (2, 40, 8, 2, 128, 64, 16, 6, (0, 56), (40, 33), None),
    (2, 9, 0, 3, 96, 96, 20, 2, (11, 31), (0, 9), None),
    (4, 7, 3, 1, 32, 32, 8, 4, (-3, 28, 5, 0), (7, 7, 12, -1), (6, 10)),
    (1, 300, 32, 8, 256, 256, 64, 5, (17,), None, (32, 48, 48)),
    (2, 50, 4, 2, 64, 30, 16, 4, (1, 2), (50, 50), None),
]


def operands(cuda, case, dt, inter):
    B, S, H, Hkv, D, R, page, per, starts, counts, sections = case
    pages, table = table_of(cuda, B, per)
    qkv = rand(cuda, B, S, H + 2 * Hkv, D, dt=dt).transpose(1, 2)
    q, k, v = qkv.split([H, Hkv, Hkv], 1)
    freqs = freqs_of(R // 2, cuda)
    st = torch.tensor(starts, dtype=torch.int32, device=cuda)
    n = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=cuda)
    axes = len(sections or (1,))
    g = torch.Generator(device=cuda).manual_seed(2)
    pos = torch.randint(0, 5000, (axes, B, S), generator=g, device=cuda, dtype=torch.int32) if sections else None
    at = pos if sections else (st[:, None] + torch.arange(S, device=cuda, dtype=torch.int32))[None]
    rows = rows_of(table.cpu(), starts, counts or (S,) * B, S, page, pages)
    kw = dict(counts=n, positions=pos, sections=sections, interleaved=inter)
    return pages, table, (q if H else None, k, v), freqs, st, at, rows, kw


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dt,layout,inter", [(BF16, "token", False), (F16, "head", True), (F32, "token", True), (BF16, "head", True)])
def test_append16(cuda, case, dt, layout, inter):
    B, S, H, Hkv, D, R, page, per, starts, counts, sections = case
    pages, table, (q, k, v), freqs, st, at, rows, kw = operands(cuda, case, dt, inter)
    kc, vc = cache16(cuda, pages, page, Hkv, D, dt, layout)
    k0, v0 = kc.clone(), vc.clone()
    got = ops.kv_append_rope(q, k, v, kc, vc, table, st, freqs, **kw)
    if q is None:
        assert got is None
    else:
        attention_ref.within(got, *ref.rotate(q, at, freqs, sections, inter), "q")
        assert torch.equal(got, ops.rope(q, at.to(torch.int32), freqs, sections, interleaved=inter))
    turned = ops.rope(k, at.to(torch.int32), freqs, sections, interleaved=inter)  # (tested against float64)
    for b, i, pg, r in rows:
        k0[pg, :, r], v0[pg, :, r] = turned[b, :, i], v[b, :, i]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)
    # Nothing turned: kv_append, bit for bit.
    ops.kv_append_rope(None, k, v, kc, vc, table, st, None, counts=kw["counts"])
    ops.kv_append(k, v, k0, v0, table, st, counts=kw["counts"])
    assert torch.equal(kc, k0) and torch.equal(vc, v0)


def unpack(codes):
    return torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dt,layout,inter", [(BF16, "token", False), (F16, "head", True), (F32, "token", True), (BF16, "head", True)])
def test_append4(cuda, case, dt, layout, inter):
    """Nothing turned: codes and scales by definition.  Turned: each value within half a step of
    what it should be and the rotation's own error, the scale right but for that error."""
    B, S, H, Hkv, D, R, page, per, starts, counts, sections = case
    pages, table, (q, k, v), freqs, st, at, rows, kw = operands(cuda, case, dt, inter)
    for turns in (False, True):
        kc, vc = cache4(cuda, pages, page, Hkv, D, layout)
        before = [t.clone() for t in (*kc, *vc)]
        got = ops.kv4_append_rope(q, k, v, kc, vc, table, st, freqs if turns else None, **(kw if turns else dict(counts=kw["counts"])))
        if q is not None:
            assert torch.equal(got, ops.rope(q, at.to(torch.int32), freqs, sections, interleaved=inter) if turns else q)
        n = D // 32
        codes, scales = ref.encode(v)
        want = ref.encode(k) if not turns else None
        turned, bound = ref.rotate(k.float(), at, freqs, sections, inter)
        for b, i, pg, r in rows:
            assert torch.equal(unpack(vc[0][pg, :, r]), codes[b, :, i]) and torch.equal(vc[1][pg, :, r, :n].long(), scales[b, :, i])
            if not turns:
                assert torch.equal(unpack(kc[0][pg, :, r]), want[0][b, :, i])
                assert torch.equal(kc[1][pg, :, r, :n].long(), want[1][b, :, i])
                continue
            x, e = turned[b, :, i], bound[b, :, i]
            held = ref.decode(kc[0][pg, :, r], kc[1][pg, :, r], D)
            unit = 2.0 ** (kc[1][pg, :, r, :n].double() - 127)
            most = x.abs().unflatten(-1, (-1, 32)).amax(-1)
            slack = e.unflatten(-1, (-1, 32)).amax(-1)
            assert (most <= 6 * unit + slack).all() and (most >= 3 * unit - slack).all()
            step = unit.repeat_interleave(32, -1)
            size = x.abs() / step
            half = torch.where(size < 2, 0.25, torch.where(size < 4, 0.5, 1.0))
            assert ((held - x).abs() <= half * step + e).all()
        # Rows of other tokens, and the bytes of a row's scales that hold none, stay as they were.
        for t, t0 in zip((*kc, *vc), before):
            keep = torch.ones(t.shape[:3], dtype=torch.bool, device=cuda)
            for b, i, pg, r in rows:
                keep[pg, :, r] = False
            assert torch.equal(t[keep], t0[keep])
            if t.shape[3] != D // 2:
                assert torch.equal(t[..., n:], t0[..., n:])


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_append4_of_every_size(cuda, dt):
    """Ties, zeros of both signs, the types' smallest and largest values, NaN and infinities (of
    their 32 values alone), bit for bit."""
    x = torch.zeros((1, 1, 40, 64), dtype=F32)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    for i in range(20):
        x[0, 0, i, :8] = ties * 2.0 ** (i - 10)
        x[0, 0, i, 8:16] = -ties * 2.0 ** (i - 10) * (1 + 2.0 ** -7)
        x[0, 0, i, 32:40] = torch.rand(8, generator=torch.Generator().manual_seed(i)) * 2.0 ** (i - 10)
    fi = torch.finfo(dt)
    x[0, 0, 20, 0], x[0, 0, 21, 0], x[0, 0, 22, 0], x[0, 0, 23, 5] = fi.max, fi.min, fi.tiny, -fi.smallest_normal
    x[0, 0, 24, 33], x[0, 0, 25, 1], x[0, 0, 26, 31], x[0, 0, 27, 32] = float("nan"), float("inf"), -float("inf"), -float("nan")
    x[0, 0, 24:28, 2], x[0, 0, 28, :] = 1.0, -0.0
    x = x.to(dt).to(cuda)
    pages, table = table_of(cuda, 1, 3)
    kc, vc = cache4(cuda, pages, 16, 1, 64, "head")
    ops.kv4_append_rope(None, x, x, kc, vc, table, torch.zeros(1, dtype=torch.int32, device=cuda), None)
    codes, scales = ref.encode(x)
    pg, row = table[0].long()[torch.arange(40, device=cuda) // 16], torch.arange(40, device=cuda) % 16
    for c in (kc, vc):
        assert torch.equal(c[1][pg, :, row, :2].long(), scales[0].transpose(0, 1))
        got = unpack(c[0][pg, :, row]).unflatten(-1, (2, 32))
        fine = (scales[0].transpose(0, 1) != 255)[..., None]
        want = codes[0].transpose(0, 1).unflatten(-1, (2, 32))
        assert torch.equal(torch.where(fine, got, 0), torch.where(fine, want, 0))
    k, v = ops.kv4_read(kc, vc, table, 40, dtype=F32)
    assert torch.equal(k.isnan(), (scales == 255).repeat_interleave(32, -1))
    assert torch.equal(k.nan_to_num(), v.nan_to_num())


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("D,page,layout", [(32, 16, "head"), (64, 20, "token"), (96, 8, "head"), (128, 64, "token"), (256, 16, "token")])
def test_read(cuda, dt, D, page, layout):
    """The values, exactly; zeros past a length, on no page; any tokens' count; strided outputs."""
    B, Hkv, per = 3, 2, 4
    pages, table = table_of(cuda, B, per)
    kc, vc = cache4(cuda, pages, page, Hkv, D, layout)
    table[1, 1], table[2, 0] = -1, pages
    S = per * page - 3
    lens = torch.tensor([S, S + 50, 5], dtype=torch.int32, device=cuda)
    for n in (None, lens):
        out = torch.full((B, S, 2 * Hkv, D), 3.0, dtype=dt, device=cuda).transpose(1, 2)
        got = ops.kv4_read(kc, vc, table, S, lens=n, dtype=dt)
        ops.kv4_read(kc, vc, table, S, lens=n, outs=(out[:, :Hkv], out[:, Hkv:]))
        for c, t, o in ((kc, got[0], out[:, :Hkv]), (vc, got[1], out[:, Hkv:])):
            x = ref.decode(*c, D)[table.long().clamp(0, pages - 1)].transpose(1, 2).flatten(2, 3)[:, :, :S].clone()
            for b in range(B):
                bad = ((table[b] < 0) | (table[b] >= pages)).repeat_interleave(page)[:S]
                x[b, :, bad] = 0
                if n is not None:
                    x[b, :, int(n[b]):] = 0
            assert torch.equal(t.double(), x) and torch.equal(o, t)


def test_bad_pages(cuda):
    """Tokens on pages out of range are skipped; the queries are turned all the same."""
    B, S, H, Hkv, D, page, per = 2, 40, 4, 2, 64, 16, 3
    pages, table = table_of(cuda, B, per)
    table[0, 1], table[1, 0], table[1, 2] = -1, pages, 2 ** 31 - 1
    q, k = rand(cuda, B, H, S, D), rand(cuda, B, Hkv, S, D, seed=1)
    freqs, st = freqs_of(32, cuda), torch.zeros(2, dtype=torch.int32, device=cuda)
    rows = rows_of(table.cpu(), (0, 0), (S, S), S, page, pages)
    pos = torch.arange(S, dtype=torch.int32, device=cuda).expand(B, S)
    turned = ops.rope(k, pos, freqs)
    kc, vc = cache16(cuda, pages, page, Hkv, D, BF16, "token")
    k0, v0 = kc.clone(), vc.clone()
    assert torch.equal(ops.kv_append_rope(q, k, k, kc, vc, table, st, freqs), ops.rope(q, pos, freqs))
    k4, v4 = cache4(cuda, pages, page, Hkv, D, "head")
    b4 = [t.clone() for t in (*k4, *v4)]
    assert torch.equal(ops.kv4_append_rope(q, k, k, k4, v4, table, st, freqs), ops.rope(q, pos, freqs))
    keep = torch.ones((pages, Hkv, page), dtype=torch.bool, device=cuda)
    for b, i, pg, r in rows:
        k0[pg, :, r], v0[pg, :, r] = turned[b, :, i], k[b, :, i]
        keep[pg, :, r] = False
    assert torch.equal(kc, k0) and torch.equal(vc, v0)
    assert all(torch.equal(t[keep], t0[keep]) for t, t0 in zip((*k4, *v4), b4))


def test_odd_alignment(cuda):
    """Rows at any whole element (no 16-byte vectors), in both caches, as aligned ones."""
    B, S, H, Hkv, D, page, per = 2, 5, 3, 2, 64, 8, 2
    pages, table = table_of(cuda, B, per)
    freqs, st = freqs_of(32, cuda), torch.tensor([2, 9], dtype=torch.int32, device=cuda)
    x = rand(cuda, B, H + 2 * Hkv, S, D)
    odd = torch.zeros((B, H + 2 * Hkv, S, D + 1), dtype=BF16, device=cuda)[..., 1:]
    odd.copy_(x)
    got = []
    for t in (x, odd):
        q, k, v = t.split([H, Hkv, Hkv], 1)
        kc, vc = cache16(cuda, pages, page, Hkv, D, BF16, "head")
        k4, v4 = cache4(cuda, pages, page, Hkv, D, "head")
        got.append([ops.kv_append_rope(q, k, v, kc, vc, table, st, freqs), kc, vc,
                    ops.kv4_append_rope(q, k, v, k4, v4, table, st, freqs), *k4, *v4])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_in_place_and_replayed(cuda):
    """The queries turned where they lie, in a captured step replayed with eager work between."""
    B, H, Hkv, D, page, per = 4, 8, 2, 128, 16, 4
    pages, table = table_of(cuda, B, per)
    freqs, st = freqs_of(64, cuda), torch.tensor([0, 17, 40, 63], dtype=torch.int32, device=cuda)
    qkv = rand(cuda, B, 1, H + 2 * Hkv, D).transpose(1, 2)
    q, k, v = qkv.split([H, Hkv, Hkv], 1)
    k4, v4 = cache4(cuda, pages, page, Hkv, D, "head")
    k5, v5 = ([t.clone() for t in c] for c in (k4, v4))
    ops.kv4_append_rope(None, k, v, k5, v5, table, st, freqs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.kv4_append_rope(q, k, v, k4, v4, table, st, freqs, q_out=q)
        read = ops.kv4_read(k4, v4, table, 64)
    for i in range(3):
        qkv.copy_(rand(cuda, B, 1, H + 2 * Hkv, D, seed=10 + i).transpose(1, 2))
        want = ops.kv4_append_rope(q.clone(), k, v, k5, v5, table, st, freqs)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(q, want) and all(torch.equal(a, b) for a, b in zip((*k4, *v4), (*k5, *v5)))
        assert all(torch.equal(a, b) for a, b in zip(read, ops.kv4_read(k5, v5, table, 64)))
        st.copy_((st + 1) % 64)


def test_refusals_on_the_device(cuda):
    pages, table = table_of(cuda, 2, 3)
    kc, vc = cache4(cuda, pages, 16, 2, 64, "head")
    k = rand(cuda, 2, 2, 1, 64)
    st, freqs = torch.zeros(2, dtype=torch.int32, device=cuda), freqs_of(32, cuda)
    with pytest.raises(ValueError, match="codes"):
        ops.kv4_append_rope(None, k, k, kc, (vc[0][:2], vc[1]), table, st, freqs)
    with pytest.raises(ValueError, match="scales"):
        ops.kv4_append_rope(None, k, k, (kc[0], kc[1][..., :2]), vc, table, st, freqs)
    with pytest.raises(ValueError, match="starts"):
        ops.kv4_append_rope(None, k, k, kc, vc, table, st.long(), freqs)
    with pytest.raises(ValueError, match="go with freqs"):
        ops.kv4_append_rope(None, k, k, kc, vc, table, st, None, positions=st[:, None])
    with pytest.raises(ValueError, match="q_out goes with q"):
        ops.kv4_append_rope(None, k, k, kc, vc, table, st, freqs, q_out=k)
    with pytest.raises(ValueError, match="block_table"):
        ops.kv4_read(kc, vc, table.long(), 10)
    with pytest.raises(BackendError, match="49 tokens"):
        ops.kv4_read(kc, vc, table, 49)
    with pytest.raises(ValueError, match="q"):
        ops.kv_append_rope(k.float(), k, k, *cache16(cuda, pages, 16, 2, 64, BF16, "head"), table, st, freqs)
    assert ops.kv4_read(kc, vc, table, 0)[0].shape == (2, 2, 0, 64)
