"""Log probabilities of more long rows than workgroups stay on the card, so each takes several one
after the other: odd vocabularies (no two rows of a workgroup begin alike), every type, with rows
of every kind among them.  Each row against float64, the largest against a stable sort."""
import pytest
import torch

import attention_ref
import rope_kv4_ref as ref
from gomlx_hip import ops

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INF = float("inf")


def largest(x, k):
    """Indices of the k largest logits of each row: by value (NaN above all), then by index."""
    key = torch.where(x.isnan(), torch.inf, x.double()).unsqueeze(0)
    # (A NaN is above +infinity: sorted by that second, which a stable sort keeps.)
    order = torch.sort(key[0], dim=1, descending=True, stable=True)[1]
    nan = x.isnan().gather(1, order)
    order = order.gather(1, torch.sort(nan.to(torch.uint8), dim=1, descending=True, stable=True)[1])
    return order[:, :k].to(torch.int32)


def rows_of_every_kind(x, ids, seed):
    """Puts rows of other kinds at random places of x, and returns (rows with a NaN or +infinity,
    rows whose ids are a token of -infinity)."""
    N, V = x.shape
    g = torch.Generator(device=x.device).manual_seed(seed)
    kind = torch.randint(0, 40, (N,), generator=g, device=x.device)
    at = torch.arange(V, device=x.device)
    low = torch.finfo(x.dtype).min
    x[kind == 0] = -INF
    x[kind == 1] = low
    x[kind == 2] = 1.5
    x[kind == 3] = (at * 7 % 5).to(x.dtype)
    x[kind == 4] = (at.float() / V * 30).to(x.dtype)
    x[kind == 5] = (at.float() / V * -30).to(x.dtype)
    m = torch.zeros_like(x, dtype=torch.bool)
    m[:, : V - V // 10] = (kind == 6)[:, None]
    x[m] = -INF
    x[(kind == 7).nonzero(as_tuple=True)[0], V - 1] = float("nan")
    n = (kind == 8).nonzero(as_tuple=True)[0]
    x[n, 0], x[n, V // 2] = INF, float("nan")
    n = (kind == 9).nonzero(as_tuple=True)[0]
    x[n[:, None], torch.arange(V // 3, V // 3 + 50, device=x.device)] = INF
    x[kind == 10] = float("nan")
    n = (kind == 11).nonzero(as_tuple=True)[0]
    x[n] = -INF
    x[n, ids[n].long()] = 2.0
    return (kind >= 7) & (kind <= 10)


def adds_of(V, es):
    """Additions of a lane and of the joins; a wave alone takes the rows of nothing but a mask."""
    return V // 64 + 80


def check(x, ids, bad, top, scale, **kw):
    got = ops.token_logprobs(x, ids, top=top, scale=scale, **kw)
    fine = ~bad
    assert all(t[bad].isnan().all() for t in got[:3])
    for lo in range(0, x.shape[0], 512):
        part = torch.arange(lo, min(lo + 512, x.shape[0]), device=x.device)
        part = part[fine[part]]
        for what, g, (want, bound) in zip(("logp", "entropy", "lse"), got, ref.logprobs(x[part], ids[part], scale, adds_of(x.shape[1], x.element_size()))):
            attention_ref.within(g[part], want, bound, what)
    if not top:
        return got
    for lo in range(0, x.shape[0], 512):
        assert torch.equal(got[4][lo:lo + 512], largest(x[lo:lo + 512], top))
    assert got[3][bad].isnan().all()
    for i in (0, top - 1):  # each is that token's own log probability
        own = ops.token_logprobs(x, got[4][:, i].contiguous(), scale=scale, **kw)[0]
        assert torch.equal(got[3][fine, i], own[fine])
    return got


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("N,V", [(2999, 9001), (1777, 40003)])
def test_rows_one_after_the_other(cuda, N, V, dt):
    print(N, V, dt, flush=True)
    g = torch.Generator(device=cuda).manual_seed(N)
    x = (torch.randn((N, V), generator=g, device=cuda) * 2.5).to(dt)
    ids = torch.randint(0, V, (N,), generator=g, device=cuda, dtype=torch.int32)
    bad = rows_of_every_kind(x, ids, 1)
    for top in (0, 5, 32):
        check(x, ids, bad, top, 0.7)


def test_many_turns(cuda):
    """More than 32 rows a workgroup, so those without usual sums are noted in several words."""
    N, V = 90001, 8201
    g = torch.Generator(device=cuda).manual_seed(N)
    x = torch.randn((N, V), generator=g, device=cuda, dtype=BF16)
    ids = torch.randint(0, V, (N,), generator=g, device=cuda, dtype=torch.int32)
    check(x, ids, rows_of_every_kind(x, ids, 4), 5, 0.7)


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("N,V", [(700, 333), (500, 2001), (300, 5003)])
def test_rows_of_one_run(cuda, N, V, dt):
    """The same rows where one workgroup, or one wave, holds a row."""
    g = torch.Generator(device=cuda).manual_seed(N)
    x = (torch.randn((N, V), generator=g, device=cuda) * 2.5).to(dt)
    ids = torch.randint(0, V, (N,), generator=g, device=cuda, dtype=torch.int32)
    bad = rows_of_every_kind(x, ids, 2)
    for top in (0, 5, 32):
        for split in (True, False):
            check(x, ids, bad, top, 0.7, split=split)


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("N,V", [(120, 32003), (40, 131072), (70, 300007)])
def test_rows_in_slices(cuda, N, V, dt):
    """The same rows, each shared by several workgroups."""
    g = torch.Generator(device=cuda).manual_seed(N)
    x = (torch.randn((N, V), generator=g, device=cuda) * 2.5).to(dt)
    ids = torch.randint(0, V, (N,), generator=g, device=cuda, dtype=torch.int32)
    bad = rows_of_every_kind(x, ids, 3)
    for top in (0, 5, 32):
        check(x, ids, bad, top, 0.7)
        check(x, ids, bad, top, 0.7, split=False)


def least_time(call):
    """The shortest of some replays of a captured call, after one."""
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    times = []
    for _ in range(6):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        graph.replay()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b))
    return min(times[1:])


@pytest.mark.parametrize("fill", [-INF, torch.finfo(BF16).min, float("nan")])
@pytest.mark.parametrize("N,every", [(16, 16), (2600, 8)])
def test_padding_costs_no_multiple(cuda, fill, N, every):
    """A finished sequence in a step, padded rows in a batch, a row gone wrong: such a row is read twice
    more at most, by as many waves as an ordinary one, so the call takes 1.5 to 4 times the ordinary
    rows' time (with one wave a row that read its logits one by one, once more for each of the
    largest beside a NaN, 12 to 200 times)."""
    V = 131072
    x = (torch.randn((N, V), generator=torch.Generator(device=cuda).manual_seed(0), device=cuda) * 2.5).to(BF16)
    ids = torch.zeros(N, dtype=torch.int32, device=cuda)
    ws = ops.token_logprobs_workspace(x, 20)
    plain = least_time(lambda: ops.token_logprobs(x, ids, top=20, workspace=ws, split=ws is not None))
    if fill != fill:
        x[3::every, V // 2] = fill
    else:
        x[3::every] = fill
    padded = least_time(lambda: ops.token_logprobs(x, ids, top=20, workspace=ws, split=ws is not None))
    print(f"{plain * 1e3:.1f} us, padded {padded * 1e3:.1f} us", flush=True)
    assert padded < 8 * plain
