"""Calls of the head that a program makes around the plain ones: several threads on one stream, an output over its input,
gradients whose terms cancel, long batches, graphs that share their memory."""
import threading

import pytest
import torch

from cudnntest_amd import ops
from head_reference import E32, Ce, assert_within

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def rand(shape, dtype, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def test_two_threads_on_one_stream():
    """4-bit layers that need a workspace, called by two threads that share the default stream: the allocator hands blocks
    of the same sizes to both, and a call's block must not come back before its launches are queued."""
    jobs = [(rand((M, 4096), torch.bfloat16, M), ops.mx4_quantize(rand((1000, 4096), torch.bfloat16, M + 1))) for M in (200, 203)]
    step = (lambda x, w: ops.mx4_linear(x, w), lambda x, w: ops.mx4_gemm(ops.mx4_quantize(x), w, dtype=torch.bfloat16))
    want = [[f(*j) for f in step] for j in jobs]
    torch.cuda.synchronize()
    got = [[], []]

    def work(k):
        for _ in range(40):
            got[k].append([f(*jobs[k]) for f in step])
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for k in range(2):
        assert len(got[k]) == 40
        assert all(torch.equal(y, ref) for ys in got[k] for y, ref in zip(ys, want[k]))


def gradients_and_reference(T, D, V, dtype, keep=None, common=0.0, std=1.5):
    """`common`: a component that all classes' weights share, in units of their own; `keep`: rows that are not ignored."""
    x = rand((T, D), dtype, T + D)
    w = ((rand((V, D), torch.float32, V + D) + common * rand((1, D), torch.float32, V)) * std / D ** 0.5).to(dtype)
    b = rand((V,), dtype, V, 0.5)
    target = torch.randint(0, V, (T,), generator=torch.Generator(device="cuda").manual_seed(T), device="cuda")
    if keep is not None:
        target[keep:] = -100
    grad = (torch.rand(T, generator=torch.Generator(device="cuda").manual_seed(V), device="cuda") + 0.5) / T
    loss, lse = ops.linear_cross_entropy(x, w, target, bias=b)
    got = ops.linear_cross_entropy_backward(grad, x, w, target, lse, bias=b)
    return got, Ce(x, w, target, b, -100, grad), (x, w, b, target, grad)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,D,V,keep,common,std", [
    (300, 64, 10, None, 0.0, 0.1),                         # few classes: dbias is a difference of sums that nearly cancel
    (1000, 64, 10, None, 0.0, 0.1),
    (2048, 40, 300, 4, 0.0, 1.5),                          # a padded batch with four rows that count
    (300, 64, 1000, 3, 0.0, 1.5),
    (1000, 64, 1000, None, 5.0, 1.5),                      # classes that share a component, which dx cancels
    (700, 64, 9000, None, 5.0, 1.5),
    (257, 72, 33, None, 0.0, 1.5),
    (2048, 64, 20000, None, 0.0, 1.5)])                    # several pieces of the vocabulary
def test_gradients_carry_no_rounding_of_dl(T, D, V, keep, common, std, dtype):
    """At any number of rows the gradients' error is that of their own rounding, also where the sums over dl cancel.

    dl as two values of the type is off by 2^-17 (bf16) or 2^-22 (f16) of itself; its probabilities carry the fp32 noise of
    their logits, D roundings of random sign of at most 2^-24 of the largest logit, and four more of the bias, the statistics
    and the exponent.  That error r relative to dl reaches a gradient as at most r times the sum of its terms' magnitudes."""
    got, ref, (x, w, b, target, grad) = gradients_and_reference(T, D, V, dtype, keep, common, std)
    X, W = x.double(), w.double()
    l = X @ W.t().contiguous() + b.double()
    g = torch.where(target != -100, grad.double(), torch.zeros_like(ref.lse))
    p = (l - ref.lse.unsqueeze(1)).exp()
    rows = torch.arange(T, device="cuda")[target != -100]
    p[rows, target[rows]] -= 1.0
    d = (p * g.unsqueeze(1)).abs()
    r = {torch.float16: 2.0 ** -22, torch.bfloat16: 2.0 ** -17}[dtype] + E32 * ((D ** 0.5 + 4) * l.abs().max() + 8)
    terms = (d @ W.abs(), d.t().contiguous() @ X.abs(), d.sum(0))
    for name, a, want, mag in zip(("dx", "dw", "dbias"), got, (ref.dx, ref.dw, ref.db), terms):
        best = (want.to(dtype).double() - want).norm()     # rounded once
        err = (a.double() - want).norm()
        assert err <= 1.05 * best + r * mag.norm(), f"{name}: {(err / best).item():.2f} of one rounding"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N", [(1, 4096), (3, 256), (8, 4096), (16, 1024), (20, 1024), (40, 512), (300, 1000)])
def test_layer_in_place(M, N, dtype):
    """`out` over x, exactly or in part: the bits of a separate output."""
    w, b = ops.mx4_quantize(rand((N, N), dtype, N, 0.05)), rand((N,), dtype, 5)
    x = rand((M, N), dtype, M)
    want = ops.mx4_linear(x, w, bias=b, relu=True)
    for off in (0, N, M * N // 2):
        buf = torch.zeros(2 * M * N, dtype=dtype, device="cuda")
        buf[:M * N] = x.view(-1)
        out = buf[off:off + M * N].view(M, N)
        y = ops.mx4_linear(buf[:M * N].view(M, N), w, bias=b, relu=True, out=out)
        assert y.data_ptr() == out.data_ptr() and torch.equal(y, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V", [(40, 300), (600, 9000), (1500, 300)])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_row_weight_that_is_not_finite_stays_in_its_row(T, V, bad, dtype):
    """The loss of one row overflowed: the other rows of dx are those of a finite weight, bit for bit (it was not the largest,
    so nothing else changes)."""
    D = 64
    x, w = rand((T, D), dtype, 1), rand((V, D), dtype, 2, 0.2)
    target = torch.randint(0, V, (T,), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    target[::9] = -100
    grad = (torch.rand(T, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda") + 0.5) / T
    grad[5] = 0.25 / T
    _, lse = ops.linear_cross_entropy(x, w, target)
    want = ops.linear_cross_entropy_backward(grad, x, w, target, lse)[0]
    grad[5] = bad
    dx, dw, _ = ops.linear_cross_entropy_backward(grad, x, w, target, lse)
    rest = torch.arange(T, device="cuda") != 5
    assert torch.equal(dx[rest], want[rest]) and bool(torch.isfinite(want.float()).all())
    assert not bool(torch.isfinite(dx[5].float()).any()) and not bool(torch.isfinite(dw.float()).any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,D,V", [(70001, 24, 40), (5000, 40, 1), (3001, 9000, 3), (20000, 130, 257), (257, 1, 128), (321, 4100, 129)])
def test_many_rows(T, D, V, dtype):
    """Long reductions of dw over two values a row, cut in parts or not, and the last stage of both passes ragged."""
    x, w, b = rand((T, D), dtype, T), rand((V, D), dtype, V, 1.5 / D ** 0.5), rand((V,), dtype, D, 0.5)
    target = torch.randint(0, V, (T,), generator=torch.Generator(device="cuda").manual_seed(T), device="cuda")
    target[::11] = -100
    grad = (torch.rand(T, generator=torch.Generator(device="cuda").manual_seed(V), device="cuda") + 0.5) / T
    ref = Ce(x, w, target, b, -100, grad)
    loss, lse = ops.linear_cross_entropy(x, w, target, bias=b)
    assert_within(lse, ref.lse, ref.lse_tol, "lse")
    assert_within(loss, ref.loss, ref.loss_tol, "loss")
    got = ops.linear_cross_entropy_backward(grad, x, w, target, lse, bias=b)
    for a, want, tol, name in zip(got, (ref.dx, ref.dw, ref.db), (ref.dx_tol, ref.dw_tol, ref.db_tol), ("dx", "dw", "dbias")):
        assert_within(a, want, tol, name)
    again = ops.linear_cross_entropy_backward(grad, x, w, target, lse, bias=b)
    assert all(torch.equal(a, c) for a, c in zip(got, again))


@pytest.mark.parametrize("T,V", [(300, 129), (600, 9000)])
def test_two_graphs_of_one_pool_and_a_side_stream(T, V):
    """Loss and gradients captured twice into graphs that share their memory, replayed in turn, and on a stream of its own."""
    def problem(seed):
        x, w = rand((T, 72), torch.bfloat16, seed), rand((V, 72), torch.bfloat16, seed + 1, 0.2)
        return x, w, torch.randint(0, V, (T,), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda"), rand((T,), torch.float32, seed + 2)

    def step(x, w, target, grad):
        loss, lse = ops.linear_cross_entropy(x, w, target)
        return (loss, lse) + ops.linear_cross_entropy_backward(grad, x, w, target, lse)[:2]
    jobs = [problem(10), problem(20)]
    want = [step(*j) for j in jobs]
    graphs, outs, pool = [], [], None
    for j in jobs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(step(*j))
        graphs.append(g)
        pool = g.pool()
    for _ in range(4):
        for k in (0, 1):
            graphs[k].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(outs[k], want[k]))
            assert all(torch.equal(a, c) for a, c in zip(step(*jobs[k]), want[k]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*jobs[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, want[0]))
