"""8-bit integer products with scales per token and channel against their
definition in 64 bits, bit for bit: every rounding is part of the definition."""
import ctypes as C
import math

import pytest
import torch

import har_cuda
from score_util import product, quantize64

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ctx():
    c = har_cuda.Context(0)
    yield c
    c.synchronize()
    c.close()


def rows(seed, M, K, dtype="f32", pad=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K + pad, generator=g) * std
    return x.to(DT[dtype]).cuda()[:, :K]


def weights(ctx, seed, N, K, low=-127):
    """int8 rows at 16-byte strides; the bytes behind K are not zero."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(low, 128, (N, (K + 15) // 16 * 16), generator=g, dtype=torch.int8).cuda()[:, :K]
    s = (torch.rand(N, generator=g) * 0.01 + 1e-4).cuda()
    return ctx.wrap_i8(q, s), q, s


def quantized(ctx, x):
    M, K = x.shape
    q = har_cuda.i8_rows(M, K, x.device)
    s = torch.empty(M, device=x.device)
    ctx.i8_quantize(x, q, s)
    return q, s


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,K,pad", [(1, 1, 0), (3, 7, 2), (2, 8, 0), (9, 64, 8), (5, 1000, 0), (4, 1024, 0),
                                     (7, 1025, 0), (3, 2048, 3), (5, 2049, 0), (2, 4096, 0), (3, 4104, 8), (2, 8192, 0),
                                     (2, 8200, 0), (2, 16384, 0),
                                     (2, 16397, 0), (1, 40001, 0), (700, 130, 1)])
def test_quantize_rows(ctx, dtype, M, K, pad):
    x = rows(K * 7 + M, M, K, dtype, pad)
    q, s = quantized(ctx, x)
    rq, rs = quantize64(x)
    assert torch.equal(s.cpu(), rs)
    assert torch.equal(q.cpu().long(), rq)


def test_quantize_halves_zeros_and_extremes(ctx):
    K = 254
    x = torch.zeros(8, K)
    x[0] = torch.arange(K) - 126.5              # halves at scale 1 after the row's 127
    x[0, 0] = 127.0
    x[2, :3] = torch.tensor([1e-45, -1e-45, 0])  # scale rounds to zero
    x[3, :4] = torch.tensor([3e-43, -1e-43, 1e-44, 2e-43])  # a subnormal scale
    x[4, :3] = torch.tensor([3.4e38, -3.4e38, 1e38])
    x[5, 3] = math.nan
    x[6, 7] = -math.inf
    x[7, :2] = torch.tensor([-0.0, 5.0])
    q, s = quantized(ctx, x.cuda())
    rq, rs = quantize64(x)
    assert torch.equal(s.cpu().isnan(), rs.isnan()) and s.cpu().isnan().tolist() == [False] * 5 + [True] * 2 + [False]
    assert torch.equal(s.cpu().nan_to_num(7.0), rs.nan_to_num(7.0))
    assert torch.equal(q.cpu().long(), rq)
    assert s[1] == 0 and not q[1].any() and not q[5].any()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_quantize_next_to_halves(ctx, dtype):
    """Every quotient beside a half, for many divisors: x = (n + 1/2) s and its
    neighbours; the row's largest value fixes s."""
    g = torch.Generator().manual_seed(3)
    rows_ = 400
    top = (torch.rand(rows_, generator=g) + 0.5) * torch.exp2(torch.randint(-12, 12, (rows_,), generator=g).float())
    top = top.to(DT[dtype]).float()
    s = top / 127
    h = torch.arange(-127, 127).float() + 0.5
    mid = (h.unsqueeze(0) * s.unsqueeze(1)).to(DT[dtype])
    up = torch.nextafter(mid.float(), torch.full_like(mid.float(), math.inf)).to(DT[dtype])
    down = torch.nextafter(mid.float(), torch.full_like(mid.float(), -math.inf)).to(DT[dtype])
    x = torch.cat([mid, up, down], 1).clamp(-top.unsqueeze(1), top.unsqueeze(1)).to(DT[dtype])
    x = torch.cat([x, top.unsqueeze(1).to(DT[dtype]), -top.unsqueeze(1).to(DT[dtype])], 1)
    q, sc = quantized(ctx, x.cuda())
    rq, rs = quantize64(x)
    assert torch.equal(sc.cpu(), rs) and torch.equal(q.cpu().long(), rq)


def test_quantize_leaves_the_padding(ctx):
    buf = torch.full((5, 32), 77, dtype=torch.int8, device="cuda")
    s = torch.empty(5, device="cuda")
    for K in (17, 24, 31):
        buf.fill_(77)
        ctx.i8_quantize(rows(K, 5, K), buf[:, :K], s)
        assert (buf[:, K:] == 77).all()
    odd = torch.full((4, 13), 77, dtype=torch.int8, device="cuda")  # rows at odd addresses
    x = rows(3, 4, 9)
    ctx.i8_quantize(x, odd[:, 2:11], s[:4])
    assert torch.equal(odd[:, 2:11].cpu().long(), quantize64(x)[0])
    assert (odd[:, :2] == 77).all() and (odd[:, 11:] == 77).all()


SHAPES = [(1, 1, 1), (1, 3, 16), (1, 130, 2048), (2, 64, 15), (3, 127, 17), (4, 1000, 2051), (7, 129, 64),
          (8, 257, 128), (9, 33, 144), (15, 128, 256), (16, 300, 63), (17, 255, 129), (31, 1000, 512),
          (33, 513, 1040), (64, 128, 2048), (65, 140, 300), (128, 384, 1000), (129, 640, 96), (256, 129, 272),
          (257, 256, 4096), (300, 1031, 777), (513, 260, 1024), (700, 5, 33), (1025, 515, 160), (2050, 1300, 720), (513, 5003, 96), (4100, 300, 48), (16, 1000, 2048),
          (100, 700, 1153), (512, 1500, 1100), (40, 3000, 600),
          # 5 to 8 rows: of a small matrix, of one just too large, with the longest rows on either side
          (5, 1, 1), (6, 1000, 2051), (8, 4096, 2048), (8, 8200, 1100), (5, 3, 12285), (8, 70, 12300),
          # the longest rows that a block keeps, and longer ones
          (8, 40, 3060), (8, 40, 3080), (4, 70, 6140), (4, 70, 6150), (2, 33, 12280), (2, 33, 12300),
          (1, 9, 24570), (1, 9, 24580)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("ydtype", ["f32", "f16", "bf16"])
def test_linear_and_matmul(ctx, M, N, K, ydtype):
    x = rows(M + N + K, M, K, {"f32": "bf16", "f16": "f32", "bf16": "f16"}[ydtype], pad=K % 3)
    w, wq, ws = weights(ctx, M * N + K, N, K)
    rq, rs = quantize64(x)
    ref = product(rq, rs, wq, ws, DT[ydtype])
    buf = torch.full((M + 2, N + 5), 9.0, dtype=DT[ydtype], device="cuda")
    y = buf[1:M + 1, 2:N + 2]                     # rows of a wider buffer, odd offsets
    ctx.i8_linear(w, x, y)
    assert torch.equal(y.cpu(), ref)
    y.fill_(9)
    q, s = quantized(ctx, x)
    ctx.i8_matmul(w, q, s, y)
    assert torch.equal(y.cpu(), ref)
    whole = torch.full((M + 2, (N + 23) // 8 * 8), 9.0, dtype=DT[ydtype], device="cuda")
    z = whole[1:M + 1, 8:N + 8]                   # rows at multiples of 16 bytes
    ctx.i8_matmul(w, q, s, z)
    assert torch.equal(z.cpu(), ref)
    assert (whole[0] == 9).all() and (whole[M + 1] == 9).all()
    assert (whole[:, :8] == 9).all() and (whole[:, N + 8:] == 9).all()
    assert (buf[0] == 9).all() and (buf[M + 1] == 9).all()
    assert (buf[:, :2] == 9).all() and (buf[:, N + 2:] == 9).all()


@pytest.mark.parametrize("M", [1, 5, 40, 300])
def test_extreme_sums(ctx, M):
    """The longest row with every product at its largest, 128 * 128, and the
    quantiser's own 127 * 128: the 32-bit sum neither wraps nor saturates."""
    K, N = har_cuda.I8_MAX_K, 130
    wq = torch.full((N, K), -128, dtype=torch.int8, device="cuda")
    wq[1::2] = 127
    ws = torch.ones(N, device="cuda")
    w = ctx.wrap_i8(wq, ws)
    q = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
    s = torch.full((M,), 0.5, device="cuda")
    y = torch.empty(M, N, device="cuda")
    ctx.i8_matmul(w, q, s, y)
    assert torch.equal(y.cpu(), product(q.cpu(), s, wq, ws, torch.float32))
    x = torch.ones(M, K, device="cuda")
    ctx.i8_linear(w, x, y)
    rq, rs = quantize64(x)
    assert torch.equal(y.cpu(), product(rq, rs, wq, ws, torch.float32))


@pytest.mark.parametrize("M", [2, 6, 20, 200])
def test_rows_that_are_not_numbers(ctx, M):
    x = rows(5, M, 100)
    x[1, 3] = math.nan
    w, wq, ws = weights(ctx, 6, 70, 100)
    y = torch.empty(M, 70, device="cuda")
    ctx.i8_linear(w, x, y)
    rq, rs = quantize64(x)
    ref = product(rq, rs, wq, ws, torch.float32)
    assert y[1].isnan().all() and torch.equal(y.cpu().nan_to_num(3.0), ref.nan_to_num(3.0))


def test_weights_quantised_by_the_library(ctx):
    for dtype in DT:
        wf = rows(11, 300, 517, dtype, pad=3, std=0.02)
        w = ctx.i8_weights(wf)
        wq, ws = quantize64(wf)
        for M in (1, 3, 50):
            x = rows(12 + M, M, 517)
            y = torch.empty(M, 300, device="cuda")
            ctx.i8_linear(w, x, y)
            rq, rs = quantize64(x)
            assert torch.equal(y.cpu(), product(rq, rs, wq, ws, torch.float32)), (dtype, M)
        assert w.nbytes == 300 * 521
        w.free()


def test_repeated_row_and_single_row_strides(ctx):
    """A row repeated by stride 0, and single rows whose stride says nothing."""
    w, wq, ws = weights(ctx, 21, 40, 48)
    x = rows(22, 1, 48)
    y = torch.empty(6, 40, device="cuda")
    ctx.i8_linear(w, x.expand(6, 48), y)
    rq, rs = quantize64(x)
    assert torch.equal(y.cpu(), product(rq, rs, wq, ws, torch.float32).expand(6, 40))
    y1 = torch.empty(40, device="cuda").as_strided((1, 40), (1, 1))
    ctx.i8_linear(w, x.as_strided((1, 48), (3, 1)), y1)
    assert torch.equal(y1[0], y[0])
    w1 = ctx.wrap_i8(wq[:1].as_strided((1, 48), (5, 1)), ws[:1])
    y2 = torch.empty(6, 1, device="cuda")
    ctx.i8_linear(w1, x.expand(6, 48), y2)
    assert torch.equal(y2[:, 0], y[:, 0])


def test_no_rows(ctx):
    w, _, _ = weights(ctx, 31, 16, 16)
    ctx.i8_linear(w, torch.empty(0, 16, device="cuda"), torch.empty(0, 16, device="cuda"))
    ctx.i8_quantize(torch.empty(0, 16, device="cuda"), torch.empty(0, 16, dtype=torch.int8, device="cuda"),
                    torch.empty(0, device="cuda"))
    assert w.linear_workspace(0) == 0 and w.linear_workspace(-1) == -1


def test_refusals(ctx):
    w, wq, ws = weights(ctx, 41, 32, 48)
    x, y = rows(1, 4, 48), torch.empty(4, 32, device="cuda")
    q, s = quantized(ctx, x)
    E = har_cuda.HarCudaError

    def refused(status, f, *a, **k):
        with pytest.raises(E) as e:
            f(*a, **k)
        assert e.value.status == status, e.value

    refused(har_cuda.ERR_GEOMETRY, ctx.i8_linear, w, rows(1, 4, 47), y)
    refused(har_cuda.ERR_GEOMETRY, ctx.i8_linear, w, x, torch.empty(4, 31, device="cuda"))
    refused(har_cuda.ERR_GEOMETRY, ctx.i8_linear, w, x, torch.empty(3, 32, device="cuda"))
    refused(har_cuda.ERR_ARG, ctx.i8_linear, w, x.double(), y)
    refused(har_cuda.ERR_ARG, ctx.i8_linear, w, x.cpu(), y)
    refused(har_cuda.ERR_ARG, ctx.i8_linear, w, x.t().contiguous().t(), y)
    refused(har_cuda.ERR_GEOMETRY, ctx.i8_linear, w, x, torch.empty(1, 32, device="cuda").expand(4, 32))
    refused(har_cuda.ERR_GEOMETRY, ctx.i8_linear, w, x[0], y)
    refused(har_cuda.ERR_ARG, ctx.i8_matmul, w, q.float(), s, y)
    refused(har_cuda.ERR_GEOMETRY, ctx.i8_matmul, w, q, s[:3], y)
    # rows that do not start at multiples of 16 bytes
    refused(har_cuda.ERR_ARG, ctx.i8_matmul, w, torch.empty(4, 49, dtype=torch.int8, device="cuda")[:, :48], s, y)
    refused(har_cuda.ERR_ARG, ctx.wrap_i8, torch.empty(4, 64, dtype=torch.int8, device="cuda")[:, 1:49], s)
    refused(har_cuda.ERR_ARG, ctx.wrap_i8, wq, ws.double())
    refused(har_cuda.ERR_GEOMETRY, ctx.wrap_i8, torch.empty(1, 131072, dtype=torch.int8, device="cuda"), ws[:1])
    refused(har_cuda.ERR_GEOMETRY, ctx.i8_weights, torch.empty(2, 131072, device="cuda"))
    refused(har_cuda.ERR_GEOMETRY, ctx.i8_quantize, x, q[:3], s)
    refused(har_cuda.ERR_GEOMETRY, ctx.i8_quantize, x, torch.empty(1, 48, dtype=torch.int8, device="cuda").expand(4, 48), s)
    M = 64
    xs, ys = rows(2, M, 48), torch.empty(M, 32, device="cuda")
    assert w.linear_workspace(M) > 0
    refused(har_cuda.ERR_ARG, ctx.i8_linear, w, xs, ys, torch.empty(w.linear_workspace(M) - 1, dtype=torch.uint8, device="cuda"))
    refused(har_cuda.ERR_ARG, ctx.i8_linear, w, xs, ys,
            torch.empty(w.linear_workspace(M) + 16, dtype=torch.uint8, device="cuda")[1:])


@pytest.mark.parametrize("M", [1, 8, 48, 300])
def test_captured_and_replayed(ctx, M):
    """A captured call keeps only the caller's addresses: replays follow new
    inputs, also after calls that grow the context's arena; without a workspace
    a call that needs one is refused under capture."""
    w, wq, ws = weights(ctx, 51, 200, 320)
    x = rows(52, M, 320)
    y = torch.empty(M, 200, device="cuda")
    need = w.linear_workspace(M)
    work = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    ctx.i8_linear(w, x, y, workspace=work)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    refused = False
    try:
        with torch.cuda.stream(side):
            g.capture_begin()
            ctx.bind_torch_stream()
            if need:
                try:
                    ctx.i8_linear(w, x, y)
                except har_cuda.HarCudaError as e:
                    refused = e.status == har_cuda.ERR_ARG
            ctx.i8_linear(w, x, y, workspace=work)
            g.capture_end()
    finally:
        ctx.bind_torch_stream()
    assert refused == bool(need)
    big = torch.empty(4096, 200, device="cuda")
    ctx.i8_linear(w, rows(53, 4096, 320), big)      # the arena grows
    for seed in (54, 55):
        x.copy_(rows(seed, M, 320))
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        rq, rs = quantize64(x)
        assert torch.equal(y.cpu(), product(rq, rs, wq, ws, torch.float32))


def test_on_another_stream_and_device_order(ctx):
    """The calls run on the bound stream, behind work already queued on it."""
    w, wq, ws = weights(ctx, 61, 128, 256)
    x = rows(62, 33, 256)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    try:
        with torch.cuda.stream(side):
            ctx.bind_torch_stream()
            big = torch.randn(4096, 4096, device="cuda")
            for _ in range(8):
                big = big @ big * 1e-2
            late = x * 2
            y = torch.empty(33, 128, device="cuda")
            ctx.i8_linear(w, late, y)
            out = y.clone()
        side.synchronize()
    finally:
        ctx.bind_torch_stream()
    rq, rs = quantize64(x * 2)
    assert torch.equal(out.cpu(), product(rq, rs, wq, ws, torch.float32))


@pytest.mark.parametrize("M", [1, 40])
def test_weights_past_two_gigabytes(ctx, M):
    """Offsets past 2^31 in the weights and in y."""
    N, K = 1100003, 2048
    q = torch.randint(-127, 128, (N, K), dtype=torch.int8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    s = torch.rand(N, device="cuda") * 0.01
    w = ctx.wrap_i8(q, s)
    x = rows(71, M, K)
    pad = 60_000_000 if M > 1 else 0               # rows of y far apart: the last starts past 2^31
    y = torch.empty(M, N + pad, dtype=torch.float16, device="cuda")[:, :N]
    ctx.i8_linear(w, x, y)
    rq, rs = quantize64(x)
    for a, b in ((0, 300), (N // 2, N // 2 + 300), (N - 300, N)):
        assert torch.equal(y[:, a:b].cpu(), product(rq, rs, q[a:b], s[a:b], torch.float16)), (a, b)


def test_one_workspace_for_two_graphs_in_turn(ctx):
    """Two captured calls that share a workspace, replayed one after the other
    on one stream, keep to their own inputs and outputs."""
    w, wq, ws = weights(ctx, 81, 300, 256)
    xs = [rows(82 + i, 20 + 30 * i, 256) for i in range(2)]
    ys = [torch.empty(x.shape[0], 300, device="cuda") for x in xs]
    work = torch.empty(max(w.linear_workspace(x.shape[0]) for x in xs), dtype=torch.uint8, device="cuda")
    graphs, side = [], torch.cuda.Stream()
    try:
        for x, y in zip(xs, ys):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.stream(side):
                g.capture_begin()
                ctx.bind_torch_stream()
                ctx.i8_linear(w, x, y, workspace=work)
                g.capture_end()
            graphs.append(g)
    finally:
        ctx.bind_torch_stream()
    for i in (0, 1, 1, 0, 1):
        xs[i].mul_(-1.25)
        graphs[i].replay()
        torch.cuda.synchronize()
        rq, rs = quantize64(xs[i])
        assert torch.equal(ys[i].cpu(), product(rq, rs, wq, ws, torch.float32)), i


def test_weights_are_not_made_under_capture(ctx):
    """The handle's memory would be written by the graph; the capture goes on."""
    x = rows(71, 5, 64)
    w, wq, ws = weights(ctx, 72, 40, 64)
    y = torch.zeros(5, 40, device="cuda")
    work = torch.empty(max(16, w.linear_workspace(5)), dtype=torch.uint8, device="cuda")
    ctx.i8_linear(w, x, y, workspace=work)
    torch.cuda.synchronize()
    g, side, status = torch.cuda.CUDAGraph(), torch.cuda.Stream(), None
    try:
        with torch.cuda.stream(side):
            g.capture_begin()
            ctx.bind_torch_stream()
            try:
                ctx.i8_weights(x)
            except har_cuda.HarCudaError as e:
                status = e.status
            ctx.i8_linear(w, x, y, workspace=work)
            g.capture_end()
    finally:
        ctx.bind_torch_stream()
    assert status == har_cuda.ERR_ARG
    y.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y.cpu(), product(*quantize64(x), wq, ws, torch.float32))


def test_two_contexts_share_weights(ctx):
    """Two contexts on two streams use one handle at the same time, each with its
    own arena; with work of every kernel in flight on both."""
    K, N = 512, 1500
    w, wq, ws = weights(ctx, 81, N, K)
    other = har_cuda.Context(0)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    x = [rows(82, 300, K), rows(83, 300, K)]
    sizes = (1, 7, 40, 300)
    y = [[torch.empty(m, N, device="cuda") for m in sizes] for _ in x]
    torch.cuda.synchronize()
    try:
        for i, c in enumerate((ctx, other)):
            with torch.cuda.stream(streams[i]):
                c.bind_torch_stream()
        for _ in range(20):
            for j, m in enumerate(sizes):
                for i, c in enumerate((ctx, other)):
                    c.i8_linear(w, x[i][:m], y[i][j])
        torch.cuda.synchronize()
    finally:
        ctx.bind_torch_stream()
    for i in range(2):
        ref = product(*quantize64(x[i]), wq, ws, torch.float32)
        for j, m in enumerate(sizes):
            assert torch.equal(y[i][j].cpu(), ref[:m]), (i, m)
    other.close()


@pytest.mark.parametrize("M,N,K", [(1_500_007, 5, 16), (1_500_007, 129, 33), (70, 300_001, 40)])
def test_many_rows_or_channels(ctx, M, N, K):
    """Thousands of tiles along one side; rows from both ends and between."""
    x = torch.randn(M, K, device="cuda", generator=torch.Generator(device="cuda").manual_seed(M))
    w, wq, ws = weights(ctx, N, N, K)
    y = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    ctx.i8_linear(w, x, y)
    at = sorted({0, 1, 69, M // 3, M // 2, M - 2, M - 1} & set(range(M)))
    assert torch.equal(y[at].cpu(), product(*quantize64(x[at]), wq, ws, torch.bfloat16))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_new_weights_are_ready_for_any_stream(ctx, dtype):
    """Weights made behind long work on one stream, multiplied at once by another
    context on another: the handle is filled when the call returns."""
    N, K = 700, 512
    source, x = rows(91, N, K, dtype), rows(92, 40, K)
    other = har_cuda.Context(0)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    y = [torch.empty(m, N, device="cuda") for m in (1, 40)]
    big = torch.randn(8192, 8192, device="cuda")
    torch.cuda.synchronize()
    try:
        with torch.cuda.stream(streams[0]):
            ctx.bind_torch_stream()
            for _ in range(20):
                big = big @ big * 1e-2
            w = ctx.i8_weights(source)
        with torch.cuda.stream(streams[1]):
            other.bind_torch_stream()
            for out in y:
                other.i8_linear(w, x[:out.shape[0]], out)
        torch.cuda.synchronize()
    finally:
        ctx.bind_torch_stream()
    ref = product(*quantize64(x), *quantize64(source), torch.float32)
    for out in y:
        assert torch.equal(out.cpu(), ref[:out.shape[0]]), out.shape
    other.close()


def test_one_context_on_two_streams_in_turn(ctx):
    """Calls without a workspace on two streams that nobody orders, through one
    context: the second waits for the first's quantised rows to be done with,
    also where the workspace grows between two calls."""
    N, K = 3000, 1024
    w, wq, ws = weights(ctx, 94, N, K)
    c = har_cuda.Context(0)                          # its workspace starts empty
    sizes = (40, 900, 333, 2000, 1500, 64, 2600, 2600)
    xs = [rows(95 + i, m, K, ("f32", "bf16")[i % 2]) for i, m in enumerate(sizes)]
    ys = [torch.zeros(m, N, device="cuda") for m in sizes]
    streams = [torch.cuda.Stream(), torch.cuda.default_stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for turn in range(6):
        for i, (x, y) in enumerate(zip(xs, ys)):
            with torch.cuda.stream(streams[(i + turn) % 3]):
                c.bind_torch_stream()
                c.i8_linear(w, x, y)
    torch.cuda.synchronize()
    for i, (x, y) in enumerate(zip(xs, ys)):
        at = sorted({0, 1, sizes[i] // 2, sizes[i] - 1})
        assert torch.equal(y[at].cpu(), product(*quantize64(x[at]), wq, ws, torch.float32)), i
    c.close()


def test_stream_destroyed_before_the_next_is_bound(ctx):
    """A stream of the caller's that is gone when the context is bound to the
    next one: its handle is not used any more."""
    N, K, M = 500, 256, 70
    w, wq, ws = weights(ctx, 97, N, K)
    runtime = torch.cuda.cudart()
    y = [torch.zeros(M, N, device="cuda") for _ in range(4)]
    x = [rows(98 + i, M, K) for i in range(4)]
    torch.cuda.synchronize()
    try:
        for i in range(4):
            h = C.c_void_p()
            assert int(runtime.cudaStreamCreate(C.addressof(h))) == 0
            ctx.check(ctx.lib.har_cuda_ctx_set_stream(ctx.handle, h))
            ctx.i8_linear(w, x[i], y[i])
            ctx.synchronize()
            assert int(runtime.cudaStreamDestroy(h.value)) == 0
    finally:
        ctx.bind_torch_stream()
    ctx.i8_linear(w, x[0], y[0])
    torch.cuda.synchronize()
    for a, b in zip(x, y):
        assert torch.equal(b.cpu(), product(*quantize64(a), wq, ws, torch.float32))
