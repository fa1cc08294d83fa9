"""4-bit layers on the GPU: quantisation bit for bit, products within the bounds of their own arithmetic."""
import pytest
import torch

from cudnntest_amd import ops
from head_reference import assert_within, mx4_encode, mx4_pack, mx4_round, mx4_values, product_bound

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
INF, NAN = float("inf"), float("nan")


def features(rows, K, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, K, generator=g) * std * torch.exp(torch.randn(rows, 1, generator=g))
    return (x * (torch.rand(rows, K, generator=g) > 0.1)).to(dtype)


def check_quantize(x):
    q = ops.mx4_quantize(x.cuda())
    c, s = mx4_encode(x)
    pc, ps = mx4_pack(c, s)
    assert torch.equal(q.scales.cpu(), ps)
    assert torch.equal(q.codes.cpu(), pc)
    want = mx4_values(c, s, x.shape[1])
    for dt in DTYPES:
        got = ops.mx4_dequantize(q, dt).cpu()
        ref = want.to(dt)                                  # one rounding: exact in fp32 and bf16
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        assert torch.equal(got.nan_to_num(nan=0.0, posinf=INF, neginf=-INF), ref.nan_to_num(nan=0.0, posinf=INF, neginf=-INF))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 31), (3, 32), (5, 33), (8, 200), (7, 255), (2, 256), (9, 257), (333, 1001), (64, 4096)])
def test_quantize_and_back(rows, K, dtype):
    check_quantize(features(rows, K, dtype, rows * 1000 + K))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_borders(dtype):
    """Every midpoint of the grid and its neighbours, saturation between 6 and 8, signed zeros, at many scales."""
    v = [0.0, -0.0, .25, .26, .5, .74, .75, .76, 1.0, 1.25, 1.26, 1.74, 1.75, 2.0, 2.5, 2.51, 3.0, 3.49, 3.5, 4.0, 5.0, 5.01, 6.0, 6.5, 7.0, 7.9,
         -.25, -.75, -1.25, -2.5, -3.5, -5.0]
    rows = [torch.tensor(v).double() * 2.0 ** e for e in range(-12, 13)]
    check_quantize(torch.stack(rows).to(dtype))


def test_quantize_extremes():
    """Blocks of subnormals, of the type's largest values, of zeros; NaN and infinities mark their block, not the row."""
    x = torch.zeros(8, 96)
    x[0] = 1e-45 * torch.arange(96)
    x[1] = 3.4e38
    x[2] = torch.logspace(-44, 38, 96)
    x[3, 5], x[3, 40] = NAN, 1.0
    x[4, 64], x[4, 1] = INF, -2.0
    x[5, 33] = -INF
    x[6] = 2.0 ** -126 * torch.linspace(-1, 1, 96)
    check_quantize(x)
    check_quantize(x.to(torch.bfloat16))
    check_quantize((x.clamp(-60000, 60000)).to(torch.float16))


def test_quantize_views_at_any_address():
    base = features(1, 7 * 300 + 3, torch.bfloat16, 5).cuda().view(-1)
    for off in range(3):
        x = base[off:off + 7 * 300].view(7, 300)
        a, b = ops.mx4_quantize(x), ops.mx4_quantize(x.clone())
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


def run_product(M, N, K, dtype, bias, relu, seed=0, x=None, w=None):
    x = features(M, K, dtype, seed + 1) if x is None else x
    w = features(N, K, dtype, seed + 2, 0.05) if w is None else w
    b = torch.randn(N, generator=torch.Generator().manual_seed(seed)).to(dtype) if bias else None
    wq = ops.mx4_quantize(w.cuda())
    bd = b.cuda() if bias else None
    y = ops.mx4_linear(x.cuda(), wq, bias=bd, relu=relu)
    y2 = ops.mx4_gemm(ops.mx4_quantize(x.cuda()), wq, bias=bd, relu=relu, dtype=dtype)
    assert torch.equal(y.cpu().view(torch.uint8), y2.cpu().view(torch.uint8)), "linear and quantize + gemm differ"
    xv, wv = mx4_round(x), mx4_round(w)
    want = xv @ wv.t()
    if bias:
        want = want + b.double()
    if relu:
        want = torch.where(want < 0, torch.zeros_like(want), want)
    assert_within(y.cpu(), want, product_bound(xv, wv, b, want, dtype), "product")
    return y


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 10, 32), (1, 1000, 4096), (2, 33, 257), (5, 130, 800), (16, 1000, 1024), (17, 129, 96),
                                   (33, 257, 4100), (130, 259, 511), (301, 1001, 1031)])
def test_linear(M, N, K, dtype):
    run_product(M, N, K, dtype, bias=True, relu=(M + N) % 2 == 0, seed=M + N + K)


@pytest.mark.parametrize("M,N,K", [(1, 4096, 25088), (257, 4096, 520), (2100, 2050, 300)])
def test_linear_large(M, N, K):
    run_product(M, N, K, torch.bfloat16, bias=False, relu=False, seed=7)


def test_linear_exact_on_grid_values():
    """Operands on the 4-bit grid with one scale: every sum below 2^24 units is exact, so y is the rounded integer result."""
    g = torch.Generator().manual_seed(3)
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6])
    x = grid[torch.randint(0, 8, (70, 700), generator=g)] * torch.where(torch.rand(70, 700, generator=g) < .5, -1.0, 1.0)
    w = grid[torch.randint(0, 8, (150, 700), generator=g)]
    x[:, ::32], w[:, ::32] = 6.0, 6.0                      # every block's scale is 1
    x[:, -1], w[:, -1] = 6.0, 6.0
    y = ops.mx4_linear(x.cuda(), ops.mx4_quantize(w.cuda()))
    assert torch.equal(y.cpu().double(), x.double() @ w.double().t())


@pytest.mark.parametrize("M", [1, 20, 300])
def test_linear_nan_blocks_stay_visible(M):
    x, w = features(M, 300, torch.float32, 1), features(40, 300, torch.float32, 2)
    x[M // 2, 100] = NAN
    w[7, 3] = INF
    y = run_product(M, 40, 300, torch.float32, False, True, x=x, w=w).cpu()
    assert torch.isnan(y[M // 2]).all() and torch.isnan(y[:, 7]).all()
    assert int(torch.isnan(y).sum()) == 40 + M - 1


@pytest.mark.parametrize("M", [1, 16, 40, 300])
def test_out_rows_behind_the_last_are_left(M):
    x, wq = features(M, 512, torch.float16, 4).cuda(), ops.mx4_quantize(features(130, 512, torch.float16, 5).cuda())
    big = torch.full((M + 3, 130), 7.0, dtype=torch.float16, device="cuda")
    y = ops.mx4_linear(x, wq, out=big[:M])
    assert y.data_ptr() == big.data_ptr() and bool((big[M:] == 7.0).all())
    assert torch.equal(big[:M], ops.mx4_linear(x, wq))


def test_outputs_at_unaligned_addresses():
    x, wq = features(3, 256, torch.bfloat16, 4).cuda(), ops.mx4_quantize(features(33, 256, torch.bfloat16, 5).cuda())
    want = ops.mx4_linear(x, wq)
    buf = torch.zeros(3 * 33 + 8, dtype=torch.bfloat16, device="cuda")
    for off in range(1, 5):
        assert torch.equal(ops.mx4_linear(x, wq, out=buf[off:off + 99].view(3, 33)), want)


def test_rows_do_not_depend_on_their_batch_neighbours_values():
    """A row's result with garbage (NaN, huge values) in every other row is the row's result without them."""
    for M in (4, 40, 200):
        x = features(M, 1024, torch.float32, 9)
        wq = ops.mx4_quantize(features(300, 1024, torch.float32, 10).cuda())
        clean = ops.mx4_linear(x.cuda(), wq)
        dirty = x.clone()
        dirty[1::2] = NAN
        assert torch.equal(ops.mx4_linear(dirty.cuda(), wq)[0::2], clean[0::2])


@pytest.mark.parametrize("M,N,K", [(1, 512, 2048), (12, 700, 1000), (200, 512, 4096)])
def test_linear_in_a_graph_and_on_another_stream(M, N, K):
    x = features(M, K, torch.bfloat16, 1).cuda()
    w = ops.mx4_quantize(features(N, K, torch.bfloat16, 2).cuda())
    want = ops.mx4_linear(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.mx4_linear(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.mx4_linear(x, w)
    for k in range(4):
        x.copy_(features(M, K, torch.bfloat16, 20 + k))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.mx4_linear(x, w))


def test_codes_past_four_gigabytes():
    """Weights whose codes pass 2^32 bytes: the last rows' results are those of these rows on their own, bit for bit."""
    N, K = 270_000, 32768
    wq = ops.Mx4._empty(N, K, torch.device("cuda", 0))
    assert wq.codes.numel() > 1 << 32
    part = features(1000, K, torch.float16, 1).cuda()
    big = torch.empty(N, K, dtype=torch.float16, device="cuda")
    for r in range(0, N, 1000):
        torch.mul(part, 1.0 + (r % 7000) / 10000.0, out=big[r:r + 1000])
    ops.mx4_quantize(big, out=wq)
    tail = ops.mx4_quantize(big[-300:].clone())
    kb = K // 128
    assert torch.equal(wq.codes.view(kb, N, 64)[:, -300:], tail.codes.view(kb, 300, 64))
    del big
    for M in (1, 5, 20, 200):
        x = features(M, K, torch.float16, 2).cuda()
        y, want = ops.mx4_linear(x, wq), ops.mx4_linear(x, tail)
        if M <= 16:                                        # one kernel, one order of the sum
            assert torch.equal(y[:, -300:], want)
        else:
            assert (y[:, -300:].float() - want.float()).abs().max() <= 2 * 2.0 ** -11 * want.float().abs().max()
    back = ops.mx4_dequantize(wq, torch.float16)
    assert torch.equal(back[-300:], ops.mx4_dequantize(tail, torch.float16))


def test_two_streams_at_once():
    """Calls on two streams overlap: each has its own workspace and output."""
    jobs = [(features(M, 4096, torch.bfloat16, M).cuda(), ops.mx4_quantize(features(1000, 4096, torch.bfloat16, M + 1).cuda())) for M in (200, 203)]
    want = [ops.mx4_linear(x, w) for x, w in jobs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for k, (x, w) in enumerate(jobs):
            with torch.cuda.stream(streams[k]):
                got[k].append(ops.mx4_linear(x, w))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(y, want[k]) for y in got[k])
