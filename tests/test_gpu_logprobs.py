"""Log probabilities of given tokens, entropy and top alternatives against the
definition in 64 bits, from logits and straight from hidden states."""
import math
import threading

import pytest
import torch

import har_cuda
from score_util import check_logprobs, logprobs64, product, quantize64

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ctx():
    c = har_cuda.Context(0)
    yield c
    c.close()


def outputs(T, G, k):
    f = dict(dtype=torch.float32, device="cuda")
    return {"logprobs": torch.full((T, G), 5.0, **f), "entropy": torch.full((T,), 5.0, **f),
            "ids": torch.full((T, k), 5, dtype=torch.int32, device="cuda"), "top": torch.full((T, k), 5.0, **f)}


def score(ctx, logits, tokens, k):
    o = outputs(logits.shape[0], tokens.shape[1], k)
    ctx.token_logprobs(logits, tokens, o["logprobs"], o["entropy"], o["ids"], o["top"])
    ctx.synchronize()
    return o


def given(seed, T, V, G):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, V, (T, G), generator=g, dtype=torch.int32).cuda()


def logits_of(seed, T, V, dtype, pad=0, std=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, V + pad, generator=g) * std).to(DT[dtype]).cuda()[:, :V]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,V,G,k,pad", [(1, 1, 1, 1, 0), (1, 2, 2, 5, 0), (3, 31, 1, 32, 1), (2, 33, 0, 3, 0),
                                         (5, 257, 3, 20, 2), (1, 1000, 1, 0, 0), (4, 4099, 1, 20, 0),
                                         (1, 50021, 1, 20, 0), (2, 50021, 2, 32, 3), (160, 700, 1, 5, 1),
                                         (400, 1203, 1, 2, 0), (1, 131072, 1, 20, 0), (3, 131072, 1, 1, 8),
                                         (40, 16384, 1, 8, 0)])
def test_rows(ctx, dtype, T, V, G, k, pad):
    x = logits_of(T + V + k, T, V, dtype, pad)
    tok = given(V, T, V, G)
    check_logprobs(score(ctx, x, tok, k), logprobs64(x, tok, k), (dtype, T, V))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [40, 5000, 70001])
def test_masks_and_values_that_are_not_numbers(ctx, dtype, V):
    """-inf masks; a row of nothing else; one token left; the type's lowest
    value; +inf and NaN; ties between far apart ids; an outlier; +0 and -0."""
    x = logits_of(V, 11, V, dtype)
    low = torch.finfo(DT[dtype]).min
    x[0, 1:] = -math.inf
    x[1] = -math.inf
    x[2] = -math.inf
    x[2, V - 1] = 3.0
    x[3] = low
    x[4, V // 2:] = low
    x[5, 7] = math.inf
    x[6, V - 2] = math.nan
    x[7] = 1.5
    x[8] = 0.0
    x[8, ::2] = -0.0
    x[9, 5] = 60000.0
    x[10, ::3] = -math.inf
    tok = torch.stack([torch.arange(11) % V, torch.full((11,), V - 1), torch.full((11,), -1)], 1).int().cuda()
    check_logprobs(score(ctx, x, tok, 20), logprobs64(x, tok, 20), (dtype, V))


@pytest.mark.parametrize("T", [1, 20, 300])
def test_orders_that_insert_every_value(ctx, T):
    """Ascending and descending rows, few distinct values: the candidate lists
    turn over as often as they can."""
    V = 9001
    up = torch.arange(V, dtype=torch.float32) * 1e-3
    x = torch.stack([up, up.flip(0), (torch.arange(V) % 3).float(), torch.where(torch.arange(V) > V - 30, 1.0, 0.0)])
    x = x.repeat((T + 3) // 4, 1)[:T].cuda()
    tok = given(1, T, V, 1)
    n = min(T, 8)
    got = score(ctx, x, tok, 32)
    ref = logprobs64(x[:n], tok[:n], 32)
    check_logprobs({k: v[:n] for k, v in got.items()}, ref, T)
    for i in range(n, T):
        assert torch.equal(got["ids"][i], got["ids"][i % 4]) and torch.equal(got["top"][i], got["top"][i % 4])


def test_tokens_outside_the_vocabulary(ctx):
    x = logits_of(3, 2, 100, "f32")
    for bad in (100, -2, 2 ** 31 - 1, -2 ** 31):
        tok = torch.tensor([[4, -1], [bad, 7]], dtype=torch.int32, device="cuda")
        o = outputs(2, 2, 3)
        ctx.token_logprobs(x, tok, o["logprobs"], o["entropy"], o["ids"], o["top"])
        with pytest.raises(har_cuda.HarCudaError) as e:
            ctx.synchronize()
        assert e.value.status == har_cuda.ERR_DEVICE
        check_logprobs(o, logprobs64(x, tok, 3))
    ctx.synchronize()                          # the error word was read and cleared


def test_outputs_left_out(ctx):
    x, tok = logits_of(4, 6, 999, "bf16"), given(4, 6, 999, 2)
    full = score(ctx, x, tok, 5)
    for keep in ("logprobs", "entropy", "ids", "top"):
        o = outputs(6, 2, 5)
        a = {n: (v if n == keep else None) for n, v in o.items()}
        ctx.token_logprobs(x, tok if keep == "logprobs" else None, a["logprobs"], a["entropy"], a["ids"], a["top"])
        assert torch.equal(o[keep], full[keep]), keep
    ctx.token_logprobs(x)                      # nothing asked for


def test_no_rows_and_repeated_rows(ctx):
    o = outputs(0, 1, 2)
    ctx.token_logprobs(torch.empty(0, 9, device="cuda"), torch.empty(0, 1, dtype=torch.int32, device="cuda"),
                       o["logprobs"], o["entropy"], o["ids"], o["top"])
    x = logits_of(5, 1, 777, "f16")
    tok = given(6, 7, 777, 1)
    ref = logprobs64(x.expand(7, 777), tok, 4)
    check_logprobs(score(ctx, x.expand(7, 777), tok, 4), ref)


def test_results_do_not_change_from_call_to_call(ctx):
    x, tok = logits_of(8, 3, 40000, "f32"), given(9, 3, 40000, 1)
    a = score(ctx, x, tok, 20)
    for _ in range(5):
        b = score(ctx, x, tok, 20)
        assert all(torch.equal(a[n], b[n]) for n in a)


def test_refusals(ctx):
    x, tok = logits_of(10, 4, 50, "f32"), given(11, 4, 50, 2)
    o = outputs(4, 2, 3)

    def refused(status, *a, **k):
        with pytest.raises(har_cuda.HarCudaError) as e:
            ctx.token_logprobs(*a, **k)
        assert e.value.status == status, e.value

    refused(har_cuda.ERR_ARG, x.double(), tok, o["logprobs"])
    refused(har_cuda.ERR_ARG, x.cpu(), tok, o["logprobs"])
    refused(har_cuda.ERR_ARG, x, tok.long(), o["logprobs"])
    refused(har_cuda.ERR_ARG, x, None, o["logprobs"])
    refused(har_cuda.ERR_GEOMETRY, x, tok[:3], o["logprobs"])
    refused(har_cuda.ERR_GEOMETRY, x, tok, o["logprobs"][:, :1])
    refused(har_cuda.ERR_GEOMETRY, x, tok, o["logprobs"], o["entropy"][:3])
    refused(har_cuda.ERR_GEOMETRY, x, None, None, None, o["ids"], o["top"][:, :2])
    refused(har_cuda.ERR_GEOMETRY, x, None, None, None, torch.empty(4, 33, dtype=torch.int32, device="cuda"))
    refused(har_cuda.ERR_GEOMETRY, x[0], tok, o["logprobs"])
    refused(har_cuda.ERR_ARG, x.t().contiguous().t(), tok, o["logprobs"])
    refused(har_cuda.ERR_GEOMETRY, torch.empty(4, 0, device="cuda"), None, None, o["entropy"])


# ---- from hidden states -----------------------------------------------------------------


def head_of(ctx, seed, V, K):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-127, 128, (V, (K + 15) // 16 * 16), generator=g, dtype=torch.int8).cuda()[:, :K]
    s = ((torch.rand(V, generator=g) + 0.5) * 2.5 / (73 * math.sqrt(K))).cuda()
    return ctx.wrap_i8(q, s), q, s


def head_score(ctx, w, x, tok, k, **kw):
    o = outputs(x.shape[0], tok.shape[1], k)
    ctx.i8_head_logprobs(w, x, tok, o["logprobs"], o["entropy"], o["ids"], o["top"], **kw)
    return o


@pytest.mark.parametrize("T,V,K,G,k,dtype", [(1, 1, 16, 1, 1, "f32"), (1, 300, 64, 1, 20, "f32"), (2, 33, 17, 2, 32, "f16"),
                                             (3, 2000, 256, 1, 5, "bf16"), (8, 5003, 2048, 1, 20, "f32"),
                                             (17, 1025, 100, 0, 3, "f32"), (40, 3001, 333, 3, 0, "bf16"),
                                             (130, 1500, 128, 1, 5, "f32"), (203, 2777, 199, 2, 32, "f16"),
                                             (300, 513, 512, 1, 1, "f32"), (129, 9000, 64, 1, 20, "f32")])
def test_head(ctx, T, V, K, G, k, dtype):
    """The logits are those of i8_linear bit for bit, so alternatives and ties
    are theirs."""
    g = torch.Generator().manual_seed(T * V)
    x = torch.randn(T, K + 3, generator=g).to(DT[dtype]).cuda()[:, :K]
    w, q, s = head_of(ctx, V, V, K)
    tok = given(T, T, V, G)
    if T > 2 and G:
        tok[1] = -1
    logits = product(*quantize64(x), q, s, torch.float32)
    got = head_score(ctx, w, x, tok, k)
    ctx.synchronize()
    check_logprobs(got, logprobs64(logits, tok, k), (T, V, K))


@pytest.mark.parametrize("T", [1, 6, 150])
def test_head_ties_and_rows_that_are_not_numbers(ctx, T):
    """Equal rows of the head tie; a zero row of x ties everywhere; a NaN in x
    makes its row NaN and no other."""
    V, K = 1300, 96
    w, q, s = head_of(ctx, 5, V, K)
    q[1::7], s[1::7] = q[0].clone(), s[0].clone()
    g = torch.Generator().manual_seed(6)
    x = torch.randn(T, K, generator=g).cuda()
    if T > 3:
        x[2] = 0.0
        x[3, 5] = math.nan
    tok = given(7, T, V, 1)
    logits = product(*quantize64(x), q, s, torch.float32)
    got = head_score(ctx, w, x, tok, 32)
    ctx.synchronize()
    check_logprobs(got, logprobs64(logits, tok, 32), T)


@pytest.mark.parametrize("T", [1, 9, 140])
def test_head_tokens_outside_the_vocabulary(ctx, T):
    w, q, s = head_of(ctx, 8, 400, 64)
    x = torch.randn(T, 64, generator=torch.Generator().manual_seed(9)).cuda()
    tok = torch.full((T, 2), 3, dtype=torch.int32, device="cuda")
    tok[0, 1], tok[T - 1, 0] = 400, -5
    got = head_score(ctx, w, x, tok, 4)
    with pytest.raises(har_cuda.HarCudaError) as e:
        ctx.synchronize()
    assert e.value.status == har_cuda.ERR_DEVICE
    check_logprobs(got, logprobs64(product(*quantize64(x), q, s, torch.float32), tok, 4), T)


@pytest.mark.parametrize("T", [1, 5, 200])
def test_head_captured_and_replayed(ctx, T):
    V, K = 1111, 160
    w, q, s = head_of(ctx, 12, V, K)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(13)).cuda()
    tok = given(14, T, V, 1)
    need = w.head_workspace(T, 1, 7)
    work = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
    o = outputs(T, 1, 7)
    args = (w, x, tok, o["logprobs"], o["entropy"], o["ids"], o["top"])
    ctx.i8_head_logprobs(*args, workspace=work)
    torch.cuda.synchronize()
    g, side, refused = torch.cuda.CUDAGraph(), torch.cuda.Stream(), False
    try:
        with torch.cuda.stream(side):
            g.capture_begin()
            ctx.bind_torch_stream()
            try:
                ctx.i8_head_logprobs(*args)
            except har_cuda.HarCudaError as e:
                refused = e.status == har_cuda.ERR_ARG
            ctx.i8_head_logprobs(*args, workspace=work)
            g.capture_end()
    finally:
        ctx.bind_torch_stream()
    assert refused == bool(need)
    x.mul_(-1.5)
    g.replay()
    torch.cuda.synchronize()
    check_logprobs(o, logprobs64(product(*quantize64(x), q, s, torch.float32), tok, 7), T)


def test_head_refusals(ctx):
    w, _, _ = head_of(ctx, 15, 64, 32)
    x, tok = torch.randn(4, 32, device="cuda"), given(1, 4, 64, 1)
    o = outputs(4, 1, 2)
    args = (tok, o["logprobs"], o["entropy"], o["ids"], o["top"])

    def refused(status, *a, **k):
        with pytest.raises(har_cuda.HarCudaError) as e:
            ctx.i8_head_logprobs(*a, **k)
        assert e.value.status == status, e.value

    refused(har_cuda.ERR_GEOMETRY, w, x[:, :31], *args)
    refused(har_cuda.ERR_ARG, w, x.long(), *args)
    refused(har_cuda.ERR_GEOMETRY, w, x, tok[:3], *args[1:])
    refused(har_cuda.ERR_ARG, w, x, None, *args[1:])
    refused(har_cuda.ERR_ARG, w, x, *args, workspace=torch.empty(1, dtype=torch.uint8, device="cuda"))
    assert w.head_workspace(-1, 1, 1) == -1 and w.head_workspace(4, 1, 33) == -1


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_rows_of_a_few_values_that_are_not_numbers(ctx, dtype):
    """Rows shorter than a warp's first trip with NaN among them: filling must
    not take an element's place."""
    for V in (1, 3, 9, 40):
        x = logits_of(V, 4, V, dtype, pad=1)
        x[0] = math.nan
        x[1, 0] = math.nan
        x[2] = -math.inf
        x[2, V // 2] = math.nan
        tok = given(1, 4, V, 1)
        check_logprobs(score(ctx, x, tok, 32), logprobs64(x, tok, 32), (dtype, V))


@pytest.mark.parametrize("dtype,T,V,k", [("f32", 600, 300001, 20), ("f32", 1200, 98001, 5), ("f16", 1200, 190001, 32),
                                         ("bf16", 20000, 131072, 3)])
def test_long_rows_and_large_matrices(ctx, dtype, T, V, k):
    """Rows that are searched in several parts, and offsets past 2^31 (the last:
    2.6e9 logits): rows checked one by one, from both ends."""
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.empty(T, V, dtype=DT[dtype], device="cuda")
    for t in range(0, T, 500):
        x[t:t + 500] = torch.randn(min(500, T - t), V, device="cuda", generator=g) * 2.5
    x[1, : V - 40] = -math.inf
    x[T - 2] = x[T - 2].sort().values          # ascending: every part is better than the last
    x[T - 1] = 1.25
    tok = given(2, T, V, 1)
    got = score(ctx, x, tok, k)
    rows = [0, 1, T // 2, T - 2, T - 1]
    check_logprobs({n: v[rows] for n, v in got.items()}, logprobs64(x[rows], tok[rows], k), (dtype, T, V))


@pytest.mark.parametrize("T,V,K,k", [(200, 1, 16, 1), (200, 33, 48, 32), (140, 300, 80, 32), (300, 257, 640, 24),
                                     (1000, 600, 64, 5)])
def test_head_of_few_rows(ctx, T, V, K, k):
    """More alternatives than vocabulary, tiles that end early, more rows than a
    tile; the logits stay in the workspace."""
    w, q, s = head_of(ctx, V, V, K)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(V)).cuda()
    tok = given(3, T, V, 2)
    got = head_score(ctx, w, x, tok, k)
    ctx.synchronize()
    check_logprobs(got, logprobs64(product(*quantize64(x), q, s, torch.float32), tok, k), (T, V))


def test_head_of_many_rows(ctx):
    """Many rows over a small vocabulary; the logits stay in the workspace."""
    T, V, K, k = 9001, 700, 64, 6
    w, q, s = head_of(ctx, 4, V, K)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(5)).cuda()
    tok = given(6, T, V, 1)
    got = head_score(ctx, w, x, tok, k)
    ctx.synchronize()
    rows = list(range(0, 3)) + list(range(2900, 3300)) + list(range(T - 500, T))
    ref = logprobs64(product(*quantize64(x[rows]), q, s, torch.float32), tok[rows], k)
    check_logprobs({n: v[rows] for n, v in got.items()}, ref, T)


@pytest.mark.parametrize("T", [3, 200])
def test_head_scales_that_are_not_numbers(ctx, T):
    """Channels whose scale is NaN or overflows: NaN and infinite logits make
    every value NaN, and the ids still stand in order."""
    V, K = 300, 32
    w, q, s = head_of(ctx, 6, V, K)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(7)).cuda()
    tok = given(8, T, V, 1)
    for bad in ("nan", "big"):
        s2 = s.clone()
        if bad == "nan":
            s2[5:290] = math.nan
        else:
            s2[3:295] = 3e38
        wb = ctx.wrap_i8(q, s2)
        got = head_score(ctx, wb, x, tok, 32)
        ctx.synchronize()
        check_logprobs(got, logprobs64(product(*quantize64(x), q, s2, torch.float32), tok, 32), (bad, T))


# ---- from hidden states, where the logits are not stored ------------------------------
#
# More than 64 tokens and more than 12 MB of logits, times the alternatives: the
# product's epilogue keeps the sums and the lists.  A sample of rows is checked:
# both ends, the joints between tiles of 128 and 256 tokens, and the special ones.


def unstored(T, V, k):
    return T > 64 and 4 * T * V > (max(k, 8) if k else 1) * 12 * 2 ** 20


def sample_rows(T):
    near = [0, 1, 2, 3, 4, 5, 127, 128, 129, 255, 256, 257, 511, 512, T // 2, T - 2, T - 1]
    return sorted({t for t in near if t < T})


def check_large_head(ctx, w, q, s, x, tok, k, rows=None, what=""):
    T, V = x.shape[0], q.shape[0]
    assert unstored(T, V, k)
    got = head_score(ctx, w, x, tok, k)
    ctx.synchronize()
    check_rows(got, q, s, x, tok, k, rows or sample_rows(T), what)


def check_rows(got, q, s, x, tok, k, rows, what):
    logits = product(*quantize64(x[rows]), q, s, torch.float32)
    check_logprobs({n: v[rows] for n, v in got.items()}, logprobs64(logits, tok[rows], k), what)


@pytest.mark.parametrize("T,V,K,G,k,dtype", [(65, 600001, 16, 1, 1, "f32"), (200, 200001, 64, 2, 5, "bf16"),
                                             (203, 460001, 72, 1, 22, "f32"), (300, 330001, 33, 1, 23, "f16"),
                                             (257, 530003, 40, 3, 32, "f32"), (1100, 30011, 64, 1, 0, "f32"),
                                             (4000, 21001, 48, 0, 20, "bf16"), (513, 65537, 1000, 1, 8, "f32"),
                                             (130, 40000, 100, 1, 0, "f16")])
def test_large_head(ctx, T, V, K, G, k, dtype):
    x = torch.randn(T, K + 3, generator=torch.Generator().manual_seed(T + V)).to(DT[dtype]).cuda()[:, :K]
    w, q, s = head_of(ctx, V, V, K)
    tok = given(T, T, V, G)
    if G:
        tok[1] = -1
        tok[0, 0], tok[T - 1, 0] = 0, V - 1
    check_large_head(ctx, w, q, s, x, tok, k, what=(T, V, K))


@pytest.mark.parametrize("k", [5, 22, 32])
def test_large_head_ties(ctx, k):
    """Few distinct logits, each many times over: every list is full of equals,
    and the lower ids stand."""
    T, V, K = 200, 700001, 16
    g = torch.Generator().manual_seed(k)
    q = torch.randint(-1, 2, (V, K), generator=g, dtype=torch.int8).cuda()
    s = torch.full((V,), 0.25, device="cuda")
    w = ctx.wrap_i8(q, s)
    x = torch.randint(-1, 2, (T, K), generator=g).float().cuda()
    x[3] = 0.0                                  # all equal
    x[4] = 0.0
    x[4, 0] = 1.0                               # three values
    check_large_head(ctx, w, q, s, x, given(k, T, V, 1), k, rows=sample_rows(T)[:8] + [T - 1], what=k)


@pytest.mark.parametrize("k", [1, 20, 32])
def test_large_head_orders(ctx, k):
    """Logits that rise with the id insert themselves into every list."""
    T, V, K = 210, 640001, 16
    q = torch.ones(V, K, dtype=torch.int8, device="cuda")
    s = torch.linspace(1e-4, 0.02, V).cuda()
    w = ctx.wrap_i8(q, s)
    x = torch.ones(T, K, device="cuda")
    x[1::2] = -1.0                              # and falls
    check_large_head(ctx, w, q, s, x, given(k, T, V, 1), k, rows=[0, 1, 127, 128, T - 1], what=k)


def test_large_head_values_that_are_not_numbers(ctx):
    """NaN and infinity in x leave the other rows alone; a head scale that is NaN
    makes every row NaN; scales whose products overflow mask (-inf) what is
    negative and make a row with a positive one NaN."""
    T, V, K, k = 200, 680001, 32, 32
    g = torch.Generator().manual_seed(3)
    w, q, s = head_of(ctx, 9, V, K)
    x = torch.randn(T, K, generator=g).cuda()
    x[2, 5], x[3, 0], x[T - 1] = math.nan, math.inf, 0.0
    tok = given(4, T, V, 1)
    check_large_head(ctx, w, q, s, x, tok, k, what="x")
    s2 = s.clone()
    s2[V - 100:V - 7] = math.nan
    check_large_head(ctx, ctx.wrap_i8(q, s2), q, s2, x, tok, k, rows=[0, 2, 128, T - 1], what="nan")
    # all but ten channels masked in every row, then all of them
    x = x.nan_to_num(0.5, 0.5, 0.5).abs() + 0.1
    for live in (10, 0):
        q2, s2 = -q.abs().clamp(min=1), torch.full((V,), 3e38, device="cuda")
        if live:
            at = torch.arange(live, device="cuda") * 12345 + 7
            s2[at] = 0.01
        tok[:, 0] = 7
        tok[5, 0] = 8
        x2 = 1e3 * x
        check_large_head(ctx, ctx.wrap_i8(q2, s2), q2, s2, x2, tok, k, rows=[0, 5, 127, 128, T - 1], what=("masked", live))
    q2[99] = 1                                  # one positive product: +inf
    check_large_head(ctx, ctx.wrap_i8(q2, s2), q2, s2, x2, tok, k, rows=[0, 128], what="inf")


def test_large_head_tokens_outside_the_vocabulary(ctx):
    T, V, K = 200, 200001, 16
    assert unstored(T, V, 4)
    w, q, s = head_of(ctx, 10, V, K)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(11)).cuda()
    tok = torch.full((T, 2), -1, dtype=torch.int32, device="cuda")
    tok[0, 1], tok[T - 1, 0], tok[5] = V, -5, 2
    got = head_score(ctx, w, x, tok, 4)
    with pytest.raises(har_cuda.HarCudaError) as e:
        ctx.synchronize()
    assert e.value.status == har_cuda.ERR_DEVICE
    check_rows(got, q, s, x, tok, 4, sample_rows(T), "outside")


def test_large_head_captured_and_replayed(ctx):
    T, V, K, k = 200, 200001, 80, 7
    assert unstored(T, V, k)
    w, q, s = head_of(ctx, 12, V, K)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(13)).cuda()
    tok = given(14, T, V, 1)
    need = w.head_workspace(T, 1, k)
    work = torch.empty(need + 256, dtype=torch.uint8, device="cuda")
    work[need:] = 77
    o = outputs(T, 1, k)
    args = (w, x, tok, o["logprobs"], o["entropy"], o["ids"], o["top"])
    ctx.i8_head_logprobs(*args, workspace=work[:need])
    torch.cuda.synchronize()
    first = {n: v.clone() for n, v in o.items()}
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    try:
        with torch.cuda.stream(side):
            g.capture_begin()
            ctx.bind_torch_stream()
            ctx.i8_head_logprobs(*args, workspace=work[:need])
            g.capture_end()
    finally:
        ctx.bind_torch_stream()
    work[:need] = 255
    g.replay()
    torch.cuda.synchronize()
    for n, v in o.items():
        assert torch.equal(v, first[n]), n      # the same bits from any workspace
    x.mul_(-1.5)
    g.replay()
    torch.cuda.synchronize()
    check_rows(o, q, s, x, tok, k, sample_rows(T), "replayed")
    assert bool((work[need:] == 77).all())


def test_large_head_in_several_launches(ctx):
    """9,001 tokens in three launches, the last one shorter."""
    T, V, K, k = 9001, 4001, 64, 6
    w, q, s = head_of(ctx, 14, V, K)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(5)).cuda()
    tok = given(6, T, V, 1)
    rows = list(range(3)) + list(range(3000, 3200)) + list(range(6100, 6200)) + list(range(T - 100, T))
    check_large_head(ctx, w, q, s, x, tok, k, rows=rows, what="launches")


def test_stored_and_unstored_logits_agree(ctx):
    """The same rows on both paths: 64 of them alone, and among 300."""
    T, V, K, k = 300, 290001, 96, 20
    assert unstored(T, V, k)
    w, q, s = head_of(ctx, 16, V, K)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(17)).cuda()
    tok = given(18, T, V, 1)
    many, few = head_score(ctx, w, x, tok, k), head_score(ctx, w, x[100:164], tok[100:164], k)
    ctx.synchronize()
    assert torch.equal(many["ids"][100:164], few["ids"])
    # each sum is off by L 2^-22 at the most, L = V / 32 additions, and log by its half steps
    tol = 2 * (V / 32 * 2.0 ** -22 + 64 * 2.0 ** -24)
    for n in ("logprobs", "top"):
        assert float((many[n][100:164] - few[n]).abs().max()) <= tol, n


@pytest.mark.parametrize("T", [2, 70])
def test_many_given_tokens(ctx, T):
    """More given tokens a row than a block has threads, repeated ones and
    padding among them, from logits and from hidden states."""
    V, K, G = 900, 48, 1000
    w, q, s = head_of(ctx, 21, V, K)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(22)).cuda()
    tok = given(23, T, V, G)
    tok[:, ::7], tok[1, 500:600] = -1, 3
    logits = product(*quantize64(x), q, s, torch.float32)
    ref = logprobs64(logits, tok, 4)
    got = head_score(ctx, w, x, tok, 4)
    ctx.synchronize()
    check_logprobs(got, ref, "head")
    check_logprobs(score(ctx, logits.cuda(), tok, 4), ref, "logits")


def test_many_short_rows(ctx):
    """300,007 rows of 11 logits, and as many from hidden states."""
    T, V, K, k = 300_007, 11, 16, 3
    w, q, s = head_of(ctx, 24, V, K)
    x = torch.randn(T, K, device="cuda", generator=torch.Generator(device="cuda").manual_seed(25))
    tok = given(26, T, V, 1)
    got = head_score(ctx, w, x, tok, k)
    ctx.synchronize()
    check_rows(got, q, s, x, tok, k, sample_rows(T), "head")
    logits = torch.randn(T, V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(27))
    got = score(ctx, logits, tok, k)
    rows = sample_rows(T)
    check_logprobs({n: v[rows] for n, v in got.items()}, logprobs64(logits[rows], tok[rows], k), "logits")


def test_workspace_for_alternatives_serves_none(ctx):
    """A workspace of head_workspace(T, G, k) bytes holds a call without
    alternatives too, on either side of the sizes where the logits are stored."""
    for V in (3, 700, 40_000, 131_072):
        w, q, s = head_of(ctx, V, V, 32)
        for T in (1, 4, 5, 64, 65, 90, 257, 700, 4096, 4097, 9001):
            for k in (1, 8, 9, 32):
                assert 0 <= w.head_workspace(T, 1, 0) <= w.head_workspace(T, 1, k), (T, V, k)
    T, V = 130, 40_000
    w, q, s = head_of(ctx, 31, V, 32)
    x = torch.randn(T, 32, generator=torch.Generator().manual_seed(32)).cuda()
    tok = given(33, T, V, 1)
    work = torch.empty(w.head_workspace(T, 1, 5), dtype=torch.uint8, device="cuda")
    o = outputs(T, 1, 0)
    ctx.i8_head_logprobs(w, x, tok, o["logprobs"], o["entropy"], workspace=work)
    ctx.synchronize()
    check_rows(o, q, s, x, tok, 0, sample_rows(T), "none")


@pytest.mark.parametrize("T,k", [(257, 5), (129, 3), (225, 24), (290, 12)])
def test_large_head_with_few_tokens_in_the_last_warps(ctx, T, k):
    """A token tile with one to three live lanes in its last warp, over enough
    vocabulary tiles that its parts confer several times: lanes past T skip what
    the others do between two of the warp's reads of tensor memory."""
    V, K = 420_001, 16
    w, q, s = head_of(ctx, 41 + k, V, K)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(T)).cuda()
    tok = given(42, T, V, 1)
    rows = sorted({0, 127, 128, T // 2, 160, T - 3, T - 2, T - 1} & set(range(T)))
    check_large_head(ctx, w, q, s, x, tok, k, rows=rows, what=(T, k))


def test_head_of_one_context_on_two_streams_in_turn(ctx):
    """Head calls without a workspace, logits stored and not, on two streams that
    nobody orders, through one context: each has the workspace to itself."""
    V, K, k = 240_001, 64, 6
    w, q, s = head_of(ctx, 51, V, K)
    c = har_cuda.Context(0)
    sizes = (130, 20, 257, 64, 200, 300)
    xs = [torch.randn(T, K, generator=torch.Generator().manual_seed(T)).cuda() for T in sizes]
    toks = [given(T, T, V, 1) for T in sizes]
    assert {unstored(T, V, k) for T in sizes} == {True, False}
    outs = [outputs(T, 1, k) for T in sizes]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for turn in range(3):
        for i, o in enumerate(outs):
            with torch.cuda.stream(streams[(i + turn) % 2]):
                c.bind_torch_stream()
                c.i8_head_logprobs(w, xs[i], toks[i], o["logprobs"], o["entropy"], o["ids"], o["top"])
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        check_rows(o, q, s, xs[i], toks[i], k, [0, sizes[i] // 2, sizes[i] - 1], i)
    c.close()


def test_two_threads_with_few_and_many_alternatives():
    """A context and a stream a thread, one asking for 5 alternatives and one for
    24: how much shared memory the one's lists take is no matter to the other."""
    V, K, T, calls = 1_200_001, 16, 65, 1500
    errors = []

    def work(k):
        try:
            c = har_cuda.Context(0, use_torch_stream=False)
            w = c.wrap_i8(q, s)
            o = outputs(T, 1, k)
            space = torch.empty(w.head_workspace(T, 1, k), dtype=torch.uint8, device="cuda")
            torch.cuda.synchronize()
            start.wait(60)
            for _ in range(calls):
                c.i8_head_logprobs(w, x, tok, o["logprobs"], o["entropy"], o["ids"], o["top"], workspace=space)
            c.synchronize()
            results[k] = o
            c.close()
        except Exception as e:
            errors.append((k, e))

    assert unstored(T, V, 5) and unstored(T, V, 24)
    q = torch.randint(-127, 128, (V, K), dtype=torch.int8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(61))
    s = torch.full((V,), 0.01, device="cuda")
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(62)).cuda()
    tok = given(63, T, V, 1)
    results, start = {}, threading.Barrier(2)
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in (5, 24)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for k, o in results.items():
        check_rows(o, q, s, x, tok, k, [0, T - 1], k)
