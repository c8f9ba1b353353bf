"""Appends of prompts, whose workgroups take several tokens and several rows a slot: workgroups
that hold tokens of two sequences, appended ones beside others, tokens on bad pages, and a last
one that is not full.  Bit for bit against the rotation alone (tested against float64), and,
into 4 bits, against the codes of what it turns.

The rotation is of fp32 values, products and sums rounded one by one, so the fp32 rotation of the
widened keys is what the codes are taken of."""
import pytest
import torch

import attention_ref
import rope_kv4_ref as ref
from gomlx_hip import ops

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32

CASES = [  # (B, S, H, Hkv, D, rotary_dim): tokens of a workgroup, in bf16, into 16 / 4 bits
    (7, 1171, 8, 2, 64, 64),      # 10 / 16
    (7, 1171, 32, 8, 128, 128),   # 2 / 3
    (9, 5003, 1, 1, 32, 32),      # 16 / 16
    (7, 2411, 0, 2, 64, 32),      # 16 / 16, no queries
    (2, 3001, 24, 4, 96, 24),     # 1 / 1, a quarter turned, its queries into 4 bits shared by two workgroups
    (31, 67, 4, 4, 256, 256),     # 2 / 2
]


def tokens_of(table, starts, counts, S, page, pages):
    """(b, i, page, row) of the tokens that are appended, as index vectors."""
    B, per = table.shape
    i = torch.arange(S, device=table.device)[None].expand(B, S)
    pos = starts.long()[:, None] + i
    inside = (i < counts.long()[:, None]) & (pos >= 0) & (pos < per * page)
    at = pos.clamp(0, per * page - 1)
    pg = table.long().gather(1, at // page)
    b, i = torch.nonzero(inside & (pg >= 0) & (pg < pages), as_tuple=True)
    return b, i, pg[b, i], (at % page)[b, i]


def setup(cuda, case, dt, seed):
    B, S, H, Hkv, D, R = case
    g = torch.Generator(device=cuda).manual_seed(seed)
    page = 20
    per = -(-S // page) + 2
    pages = B * per + 3
    table = torch.randperm(pages, generator=g, device=cuda)[:B * per].view(B, per).to(torch.int32)
    table[0, 1], table[B - 1, 3], table[B // 2, 2] = -1, pages, 2 ** 31 - 1
    x = torch.randn((B, S, H + 2 * Hkv, D), generator=g, device=cuda).to(dt).transpose(1, 2)
    q, k, v = x.split([H, Hkv, Hkv], 1)
    starts = torch.randint(-3, 3 * page, (B,), generator=g, device=cuda, dtype=torch.int32)
    counts = torch.randint(S // 2, S + 9, (B,), generator=g, device=cuda, dtype=torch.int32)
    counts[B // 2] = 0
    freqs = (10000.0 ** (-torch.arange(R // 2, dtype=torch.float64) / (R // 2))).float().to(cuda)
    pos = starts[:, None] + torch.arange(S, device=cuda, dtype=torch.int32)
    at = tokens_of(table, starts, counts, S, page, pages)
    return (pages, Hkv, page), table, (q if H else None, k, v), starts, counts, freqs, pos, at


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dt,inter", [(BF16, False), (F16, True), (F32, False)])
def test_prompts_into_16_bits(cuda, case, dt, inter):
    print(case, dt, flush=True)
    D = case[4]
    shape, table, (q, k, v), starts, counts, freqs, pos, (b, i, pg, row) = setup(cuda, case, dt, 1)
    kc, vc = (torch.full((*shape, D), f, dtype=dt, device=cuda) for f in (3.0, 4.0))
    k0, v0 = kc.clone(), vc.clone()
    got = ops.kv_append_rope(q, k, v, kc, vc, table, starts, freqs, counts=counts, interleaved=inter)
    if q is not None:
        assert torch.equal(got, ops.rope(q, pos, freqs, interleaved=inter))
    turned = ops.rope(k, pos, freqs, interleaved=inter)
    attention_ref.within(turned, *ref.rotate(k, pos, freqs, None, inter))
    k0[pg, :, row], v0[pg, :, row] = turned[b, :, i], v[b, :, i]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dt,inter", [(BF16, False), (F16, True), (F32, False)])
def test_prompts_into_4_bits(cuda, case, dt, inter):
    print(case, dt, flush=True)
    D = case[4]
    shape, table, (q, k, v), starts, counts, freqs, pos, (b, i, pg, row) = setup(cuda, case, dt, 2)
    g = torch.Generator(device=cuda).manual_seed(3)
    wide = (D + 127) // 128 * 4
    caches = [tuple(torch.randint(0, 256, (*shape, w), generator=g, device=cuda, dtype=torch.uint8) for w in (D // 2, wide))
              for _ in range(2)]
    want = [[t.clone() for t in c] for c in caches]
    got = ops.kv4_append_rope(q, k, v, *caches, table, starts, freqs, counts=counts, interleaved=inter)
    if q is not None:
        assert torch.equal(got, ops.rope(q, pos, freqs, interleaved=inter))
    for (codes0, scales0), x in zip(want, (ops.rope(k.float(), pos, freqs, interleaved=inter), v)):
        codes, scales = ref.encode(x)
        packed = (codes[..., 0::2] | codes[..., 1::2] << 4).to(torch.uint8)
        codes0[pg, :, row], scales0[pg, :, row, :D // 32] = packed[b, :, i], scales[b, :, i].to(torch.uint8)
    for c, c0 in zip(caches, want):
        assert torch.equal(c[0], c0[0]) and torch.equal(c[1], c0[1])


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_many_rows(cuda, dt):
    """Rotation alone with three rows a slot, of tokens that a workgroup's number does not divide."""
    B, H, S, D = 2, 16, 8999, 128
    x = torch.randn((B, S, H, D), generator=torch.Generator(device=cuda).manual_seed(4), device=cuda).to(dt).transpose(1, 2)
    freqs = (10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)).float().to(cuda)
    pos = torch.randint(0, 100000, (B, S), generator=torch.Generator(device=cuda).manual_seed(5), device=cuda, dtype=torch.int32)
    got = ops.rope(x, pos, freqs)
    attention_ref.within(got, *ref.rotate(x, pos, freqs))
    y = x.clone(memory_format=torch.preserve_format)
    ops.rope(y, pos, freqs, out=y)
    assert torch.equal(y, got)
