"""Log probabilities against 64 bits within bounds that follow each path's own
additions (logprob_bounds.py), and rows whose mass lies at the seams between
pieces, trips, blocks, tiles and parts, where a lost value shows whole."""
import math

import pytest
import torch

import har_cuda
from logprob_bounds import bounded64, head_chain, walk_chain
from score_util import check_logprobs, product, quantize64
from test_gpu_logprobs import DT, given, head_of, head_score, score, unstored

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = har_cuda.Context(0)
    yield c
    c.close()


def special(x):
    """All equal; rising and falling by 100, so that references move; the same in
    steps; one value far above the rest, first and last."""
    T, V = x.shape
    ramp = torch.linspace(0.0, 100.0, V)
    rows = [torch.zeros(V), ramp, ramp.flip(0), (ramp / 7).floor() * 7, torch.full((V,), -20.0), torch.full((V,), -20.0)]
    rows[4][0] = rows[5][V - 1] = 0.0
    for t, r in enumerate(rows[:T]):
        x[t] = r
    return x


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,V,k", [(6, 131072, 5), (8, 50021, 20), (37, 131072, 1), (150, 98303, 0), (300, 50021, 3),
                                   (700, 8191, 5), (1300, 40009, 2), (600, 262145, 4)])
def test_rows_within_the_bounds(ctx, dtype, T, V, k):
    x = torch.randn(T, V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(T + V)) * 2.5
    x[:6] = special(torch.empty(6, V)).cuda()
    x = x.to(DT[dtype])
    tok = given(T, T, V, 2)
    got = score(ctx, x, tok, k)
    rows = sorted(set(range(6)) | {T // 2, T - 1})
    check_logprobs({n: v[rows] for n, v in got.items()}, bounded64(x[rows], tok[rows], k, walk_chain(V, x.element_size())),
                   (dtype, T, V))


@pytest.mark.parametrize("T,V,K,k", [(8, 65536, 64, 3), (60, 131071, 48, 5), (203, 50021, 96, 3), (130, 600001, 16, 1),
                                     (257, 290001, 40, 24), (1100, 30011, 64, 0), (2100, 50001, 32, 5)])
def test_head_within_the_bounds(ctx, T, V, K, k):
    w, q, s = head_of(ctx, 71, V, K)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(T)).cuda()
    x[2] = 0.0                                       # all logits equal
    tok = given(72, T, V, 1)
    got = head_score(ctx, w, x, tok, k)
    ctx.synchronize()
    rows = sorted({0, 1, 2, T // 2, T - 1})
    logits = product(*quantize64(x[rows]), q, s, torch.float32)
    chain = head_chain(T, V) if unstored(T, V, k) else walk_chain(V, 4)
    check_logprobs({n: v[rows] for n, v in got.items()}, bounded64(logits, tok[rows], k, chain), (T, V, K))


def seams(V, *sizes):
    """Positions p so that p, p + 1 lie on either side of multiples of these sizes:
    the first, one in the middle, the last; and the row's own ends."""
    at = {0, V - 2}
    for n in sizes:
        last = (V - 2) // n
        at |= {n * i - 1 for i in (1, max(1, last // 2), last) if 0 < n * i < V - 1}
    return sorted(at)


@pytest.mark.parametrize("dtype,pad", [("f32", 0), ("f32", 1), ("f16", 3), ("bf16", 0)])
@pytest.mark.parametrize("V", [5000, 131072])
@pytest.mark.parametrize("together", [True, False])
def test_mass_at_the_seams(ctx, dtype, pad, V, together):
    """Two equal values carry a row: pieces of 16 bytes, 4 of them a thread, trips
    of 128 and 256 threads, 1 to 16 blocks a row."""
    n = 16 // DT[dtype].itemsize
    pieces = -(-V // n)
    sizes = [n, 32 * n, 128 * n, 256 * n, 512 * n, 1024 * n] + [-(-pieces // c) * n for c in (2, 4, 8, 16)]
    at = seams(V, *sizes)
    x = torch.full((len(at), V + pad), -25.0)
    for t, p in enumerate(at):
        x[t, p:p + 2] = 3.0
    x = x.to(DT[dtype]).cuda()[:, :V]
    tok = torch.tensor([[p, p + 1] for p in at], dtype=torch.int32).cuda()
    calls = [slice(None)] if together else [slice(t, t + 1) for t in range(len(at))]
    for r in calls:
        got = score(ctx, x[r], tok[r], 2)
        check_logprobs(got, bounded64(x[r], tok[r], 2, walk_chain(V, x.element_size())), (dtype, V, r))
        assert torch.equal(got["ids"], tok[r])
        assert float((got["logprobs"] + math.log(2)).abs().max()) < 1e-4  # e^-28 V: 1e-7


@pytest.mark.parametrize("T", [40, 130, 300])
def test_mass_at_the_seams_of_the_head(ctx, T):
    """Each hidden state picks two neighbouring vocabulary rows: 32 columns a read,
    128 a half, 256 a tile, the tiles of a part, the last, partial tile."""
    V, k = 420_001, 2
    vt = -(-V // 256)
    at = seams(V, 32, 128, 256, 37 * 256, 74 * 256, vt // 2 * 256) + [(vt - 1) * 256 - 1, (vt - 1) * 256, V - 34]
    K = 64
    assert len(at) <= K and unstored(T, V, k) == (T > 64)
    q = torch.zeros(V, K, dtype=torch.int8)
    for j, p in enumerate(at):
        q[p:p + 2, j] = 127
    q, s = q.cuda(), torch.full((V,), 25.0 / 127 ** 2, device="cuda")
    w = ctx.wrap_i8(q, s)
    x = torch.zeros(T, K)
    col = torch.arange(T) % len(at)
    x[torch.arange(T), col] = 127.0
    tok = torch.tensor(at, dtype=torch.int32)[col].unsqueeze(1) + torch.tensor([0, 1], dtype=torch.int32)
    x, tok = x.cuda(), tok.cuda()
    got = head_score(ctx, w, x, tok, k)
    ctx.synchronize()
    assert torch.equal(got["ids"], tok)
    # V values 25 below two equal ones: log p = -log(2 + (V - 2) e^-25)
    lp = -math.log(2.0 + (V - 2) * math.exp(-25.0))
    rows = list(range(0, T, max(1, T // 40)))
    logits = product(*quantize64(x[rows]), q, s, torch.float32)
    chain = head_chain(T, V) if unstored(T, V, k) else walk_chain(V, 4)
    ref = bounded64(logits, tok[rows], k, chain)
    check_logprobs({n: v[rows] for n, v in got.items()}, ref, T)
    assert float((got["logprobs"].double() - lp).abs().max()) < max(ref["tol_z"]) + 25 * 2.0 ** -22


def test_stored_and_unstored_logits_agree_within_the_bounds(ctx):
    T, V, K, k = 300, 290001, 96, 20
    assert unstored(T, V, k)
    w, q, s = head_of(ctx, 73, V, K)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(74)).cuda()
    tok = given(75, T, V, 1)
    many, few = head_score(ctx, w, x, tok, k), head_score(ctx, w, x[100:164], tok[100:164], k)
    ctx.synchronize()
    assert torch.equal(many["ids"][100:164], few["ids"])
    rows = [100, 163]
    logits = product(*quantize64(x[rows]), q, s, torch.float32)
    for chain, got, first in ((head_chain(T, V), many, 0), (walk_chain(V, 4), few, 100)):
        check_logprobs({n: v[[r - first for r in rows]] for n, v in got.items()}, bounded64(logits, tok[rows], k, chain), first)
