"""Softmax cross entropy and its gradient on the GPU against float64, within the bounds of their own arithmetic."""
import pytest
import torch

from cudnntest_amd import ops
from head_reference import Ce, assert_within

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
INF, NAN = float("inf"), float("nan")


def problem(T, D, V, dtype, seed=0, bias=True, ignore=True, std=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + T + D + V)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, w = r(T, D).to(dtype), (r(V, D) * std / D ** 0.5).to(dtype)
    b = (r(V) * 0.5).to(dtype) if bias else None
    target = torch.randint(0, V, (T,), generator=g, device="cuda")
    if ignore and T > 1:
        target[::7] = -100
    grad = (torch.rand(T, generator=g, device="cuda") + 0.5) / T
    return x, w, target, b, grad


def check(x, w, target, b, grad, ignore=-100):
    ref = Ce(x, w, target, b, ignore, grad)
    loss, lse = ops.linear_cross_entropy(x, w, target, bias=b, ignore_index=ignore)
    assert_within(lse, ref.lse, ref.lse_tol, "lse")
    assert_within(loss, ref.loss, ref.loss_tol, "loss")
    dx, dw, db = ops.linear_cross_entropy_backward(grad, x, w, target, lse, bias=b, ignore_index=ignore)
    assert_within(dx, ref.dx, ref.dx_tol, "dx")
    assert_within(dw, ref.dw, ref.dw_tol, "dw")
    if b is None:
        assert db is None
    else:
        assert_within(db, ref.db, ref.db_tol, "dbias")
    return loss, lse, dx, dw, db


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,D,V", [(1, 1, 1), (1, 3, 2), (1, 64, 1000), (2, 8, 129), (7, 33, 10), (32, 200, 1000), (63, 100, 130), (65, 129, 257),
                                   (128, 64, 128), (129, 72, 300), (250, 512, 1000), (300, 41, 333)])
def test_against_float64(T, D, V, dtype):
    check(*problem(T, D, V, dtype, bias=(T + V) % 2 == 0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,D,V,bias", [(1000, 96, 8200, True), (515, 136, 15013, False), (2049, 40, 2311, True)])
def test_many_tiles(T, D, V, dtype, bias):
    """Problems with more tiles than CUs: the statistics come from the tiles, ragged in every direction."""
    check(*problem(T, D, V, dtype, bias=bias))


@pytest.mark.parametrize("dtype,T,D,V", [(torch.bfloat16, 1030, 72, 70003), (torch.float32, 1100, 20, 33001), (torch.float16, 1030, 48, 66000)])
def test_several_pieces_of_the_vocabulary(dtype, T, D, V):
    check(*problem(T, D, V, dtype, bias=True))


@pytest.mark.parametrize("T,V", [(20, 300), (600, 9000)])
def test_masked_classes_and_rows(T, V):
    """-inf in the bias masks a class: probability and gradient 0; a masked target has an infinite loss."""
    x, w, target, b, grad = problem(T, 64, V, torch.float32, ignore=False)
    b[::2] = -INF
    target = target | 1                                    # odd: not masked
    target.clamp_(max=(V - 1) | 1)
    target[target >= V] = 1
    loss, lse, dx, dw, db = check(x, w, target, b, grad)
    assert bool((dw[::2] == 0).all()) and bool((db[::2] == 0).all())
    target[3] = 2
    loss, lse = ops.linear_cross_entropy(x, w, target, bias=b)
    assert loss[3].item() == INF and bool(torch.isfinite(torch.cat([loss[:3], loss[4:]])).all())


@pytest.mark.parametrize("T,V", [(5, 40), (600, 9000)])
def test_a_row_without_any_class(T, V):
    x, w, target, b, grad = problem(T, 32, V, torch.float32, ignore=False)
    b[:] = -INF
    loss, lse = ops.linear_cross_entropy(x, w, target, bias=b)
    assert bool((lse == -INF).all()) and bool(torch.isnan(loss).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V", [(40, 100), (600, 9000)])
def test_nan_rows_stay_in_their_rows(T, V, dtype):
    x, w, target, b, grad = problem(T, 64, V, dtype, ignore=False)
    loss0, lse0 = ops.linear_cross_entropy(x, w, target, bias=b)
    x[5, 3] = NAN
    x[9, 0] = INF
    target[11], target[12] = V, -5                          # no such class
    target[13] = -100
    loss, lse = ops.linear_cross_entropy(x, w, target, bias=b)
    bad = torch.tensor([5, 9], device="cuda")
    assert bool(torch.isnan(lse[bad]).all())
    ok = torch.ones(T, dtype=torch.bool, device="cuda")
    ok[bad] = False
    assert torch.equal(lse[ok], lse0[ok])
    ok[torch.tensor([11, 12, 13], device="cuda")] = False
    assert torch.equal(loss[ok], loss0[ok])
    assert bool(torch.isnan(loss[[5, 9, 11, 12]]).all()) and loss[13].item() == 0
    dx, dw, db = ops.linear_cross_entropy_backward(grad, x, w, target, lse, bias=b)
    assert bool(torch.isnan(dx[[5, 9, 11, 12]]).any(1).all()) and bool((dx[13] == 0).all())
    assert bool(torch.isfinite(dx[ok].float()).all())


@pytest.mark.parametrize("T,V", [(33, 100), (700, 9000)])
def test_all_rows_ignored(T, V):
    x, w, target, b, grad = problem(T, 40, V, torch.bfloat16)
    target.fill_(7)
    loss, lse = ops.linear_cross_entropy(x, w, target, bias=b, ignore_index=7)
    assert bool((loss == 0).all()) and bool(torch.isfinite(lse).all())
    x[0, 0] = NAN                                          # an ignored row's NaN goes nowhere but into its own lse
    _, lse = ops.linear_cross_entropy(x, w, target, bias=b, ignore_index=7)
    for g in ops.linear_cross_entropy_backward(grad, x, w, target, lse, bias=b, ignore_index=7):
        assert bool((g == 0).all())


def test_large_and_equal_logits():
    for T, V in ((10, 64), (600, 9000)):
        x, w, target, b, grad = problem(T, 16, V, torch.float32, std=4000.0, ignore=False)
        check(x, w, target, b, grad)
        x.zero_()
        loss, lse, *_ = check(x, w, target, None, grad)
        assert (lse - torch.log(torch.tensor(float(V)))).abs().max().item() < 1e-5


@pytest.mark.parametrize("T,D,V", [(50, 64, 500), (600, 64, 9000)])
def test_f16_gradients_of_tiny_weights(T, D, V):
    """Row weights of 1e-7: the probabilities' share would vanish in f16; dx is returned in f16, so w is scaled up."""
    x, w, target, b, grad = problem(T, D, V, torch.float16)
    w.mul_(16)
    x.div_(16)
    check(x, w, target, b, grad * 1e-3 * T)
    check(x, w, target, b, torch.zeros_like(grad))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,D,V", [(30, 64, 200), (600, 64, 9000)])
def test_views_at_any_address(T, D, V, dtype):
    x, w, target, b, grad = problem(T, D, V, dtype)
    want = check(x, w, target, b, grad)

    def moved(t, off):
        buf = torch.empty(t.numel() + 8, dtype=t.dtype, device="cuda")
        v = buf[off:off + t.numel()].view(t.shape)
        v.copy_(t)
        return v
    for off in (1, 3):
        args = [moved(t, off) for t in (x, w, target, b, grad)]
        loss, lse = ops.linear_cross_entropy(args[0], args[1], args[2], bias=args[3])
        assert torch.equal(loss, want[0]) and torch.equal(lse, want[1])
        got = ops.linear_cross_entropy_backward(args[4], args[0], args[1], args[2], lse, bias=args[3])
        for a, c in zip(got, want[2:]):
            assert torch.equal(a, c)


@pytest.mark.parametrize("T,V", [(40, 300), (700, 9000)])
def test_gradients_one_at_a_time_and_again(T, V):
    x, w, target, b, grad = problem(T, 64, V, torch.bfloat16)
    _, lse = ops.linear_cross_entropy(x, w, target, bias=b)
    every = ops.linear_cross_entropy_backward(grad, x, w, target, lse, bias=b)
    for k in range(3):
        got = ops.linear_cross_entropy_backward(grad, x, w, target, lse, bias=b, need=tuple(i == k for i in range(3)))
        assert [g is not None for g in got] == [i == k for i in range(3)]
        assert torch.equal(got[k], every[k])
    again = ops.linear_cross_entropy_backward(grad, x, w, target, lse, bias=b)
    assert all(torch.equal(a, c) for a, c in zip(every, again))


def test_gradient_against_differences():
    """d loss / d x, w, bias of the kernels against central differences of the kernels' own loss, fp32."""
    T, D, V = 9, 24, 37
    x, w, target, b, grad = problem(T, D, V, torch.float32, ignore=False)
    grad = torch.ones_like(grad)
    total = lambda: ops.linear_cross_entropy(x, w, target, bias=b)[0].double().sum().item()
    _, lse = ops.linear_cross_entropy(x, w, target, bias=b)
    grads = ops.linear_cross_entropy_backward(grad, x, w, target, lse, bias=b)
    # h = 2^-6: the loss (about 9 rows of 4) is off by 2 E32 (D + V + ..) in all, over 2 h: 2e-4; the third derivative of a
    # row's loss in one logit is below 0.1 and |w|, |x| below 4, so h^2/6 * 9 * 6.4 leaves 2.4e-3
    h = 2.0 ** -6
    for t, g in zip((x, w, b), grads):
        for i in range(0, t.numel(), max(1, t.numel() // 6)):
            at = t.view(-1)
            keep = at[i].item()
            at[i] = keep + h
            up, hi = total(), at[i].item()
            at[i] = keep - h
            down, lo = total(), at[i].item()
            at[i] = keep
            assert abs((up - down) / (hi - lo) - g.view(-1)[i].item()) < 3e-3


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,V", [(64, 1000), (600, 9000)])
def test_in_a_graph(T, V, dtype):
    x, w, target, b, grad = problem(T, 64, V, dtype)

    def step():
        loss, lse = ops.linear_cross_entropy(x, w, target, bias=b)
        return (loss, lse) + ops.linear_cross_entropy_backward(grad, x, w, target, lse, bias=b)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        nx = problem(T, 64, V, dtype, seed=k + 1)
        for a, c in zip((x, w, target, b, grad), nx):
            a.copy_(c)
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(out, step()):
            assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,D,V", [(256, 40, 700), (257, 40, 700), (255, 72, 33), (193, 64, 40000), (64, 200, 129), (200, 16, 140000)])
def test_dl_in_two_values(T, D, V, dtype):
    """Up to 256 rows dl is kept as two 16-bit values: the gradients' error is that of their own rounding, nothing of dl's."""
    x, w, target, b, grad = problem(T, D, V, dtype)
    loss, lse, dx, dw, db = check(x, w, target, b, grad)
    if T > 256:
        return
    ref = Ce(x, w, target, b, -100, grad)
    for got, want in ((dx, ref.dx), (dw, ref.dw), (db, ref.db)):
        best = (want.to(dtype).double() - want).norm()     # rounded once
        assert (got.double() - want).norm() <= 1.05 * best + 2e-5 * want.norm()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_equal_weights_share_no_rounding(dtype):
    """A mean over 1000 rows: 1/1000 is no 16-bit number, and its rounding must not scale the whole gradient."""
    x, w, target, b, grad = problem(1000, 64, 5000, dtype, std=0.1)
    grad.fill_(1.0 / 1000)
    ref = Ce(x, w, target, b, -100, grad)
    _, lse = ops.linear_cross_entropy(x, w, target, bias=b)
    dx, dw, db = ops.linear_cross_entropy_backward(grad, x, w, target, lse, bias=b)
    for got, want in ((dx, ref.dx), (dw, ref.dw)):
        # the projection on the exact gradient: a common factor would show as up to 2^-9 (bf16), 2^-12 (f16)
        factor = (got.double() * want).sum() / (want * want).sum()
        assert abs(factor.item() - 1.0) < 2.0 ** -11


def test_weights_past_four_gigabytes():
    """w of 4.6 GB: the rows' statistics and the gradients of the last classes."""
    T, D, V = 48, 16384, 140_000
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.empty(V, D, dtype=torch.bfloat16, device="cuda")
    for v in range(0, V, 10000):
        w[v:v + 10000] = torch.randn(10000, D, generator=g, device="cuda") / 128
    x = torch.randn(T, D, generator=g, device="cuda").to(torch.bfloat16)
    target = torch.randint(V - 2000, V, (T,), generator=g, device="cuda")
    grad = torch.full((T,), 1.0, device="cuda")
    loss, lse = ops.linear_cross_entropy(x, w, target)
    l = torch.cat([x.double() @ w[v:v + 10000].double().t().contiguous() for v in range(0, V, 10000)], 1)
    want = torch.logsumexp(l, 1)
    assert (lse - want).abs().max() < 1e-4
    assert (loss - (want - l[torch.arange(T), target])).abs().max() < 1e-4
    dx, dw, _ = ops.linear_cross_entropy_backward(grad, x, w, target, lse)
    d = (l - want[:, None]).exp()
    d[torch.arange(T, device="cuda"), target] -= 1.0
    ref = d[:, -2000:].t().contiguous() @ x.double()
    assert (dw[-2000:].double() - ref).norm() / ref.norm() < 2.5e-3
    ref = sum(d[:, v:v + 10000] @ w[v:v + 10000].double() for v in range(0, V, 10000))
    assert (dx.double() - ref).norm() / ref.norm() < 2.5e-3


def test_two_streams_and_threads_at_once():
    import threading
    jobs = [problem(70 + k, 256, 900, torch.bfloat16, seed=k) for k in range(2)]

    def step(p):
        x, w, target, b, grad = p
        loss, lse = ops.linear_cross_entropy(x, w, target, bias=b)
        return (loss,) + ops.linear_cross_entropy_backward(grad, x, w, target, lse, bias=b)
    want = [step(p) for p in jobs]
    torch.cuda.synchronize()
    got = [[], []]

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(8):
                got[k].append(step(jobs[k]))
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for k in range(2):
        assert len(got[k]) == 8
        for out in got[k]:
            assert all(torch.equal(a, c) for a, c in zip(out, want[k]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,D,V", [(40, 64, 100), (130, 33, 500), (300, 64, 400), (700, 64, 9000), (1, 64, 50)])
def test_what_ignored_rows_hold_reaches_nothing(T, D, V, dtype):
    """A padded batch: rows behind the last one hold NaN, infinities, garbage weights and are ignored."""
    x, w, target, b, grad = problem(T, D, V, dtype, ignore=False)
    off = torch.zeros(T, dtype=torch.bool, device="cuda")
    off[::3] = True
    off[-1] = True                                         # the last row, which also fills the reduction's last stage
    target[off] = -100
    want = ops.linear_cross_entropy(x, w, target, bias=b)
    want += ops.linear_cross_entropy_backward(grad, x, w, target, want[1], bias=b)
    x[off], grad[off] = NAN, INF
    x[-1, 0] = -INF
    loss, lse = ops.linear_cross_entropy(x, w, target, bias=b)
    assert torch.equal(loss, want[0]) and torch.equal(lse[~off], want[1][~off]) and bool(torch.isnan(lse[off]).all())
    for got, ref in zip(ops.linear_cross_entropy_backward(grad, x, w, target, lse, bias=b), want[2:]):
        assert torch.equal(got, ref)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,D,V", [(164, 211, 476), (66, 299, 664), (97, 64, 700), (33, 80, 1100), (129, 24, 3000), (200, 130, 2100), (65, 520, 66)])
def test_gradients_in_parts_of_two_values(T, D, V, dtype):
    """dl as two values, products in parts: sizes whose padded reductions have a stage more than twice the plain one's.
    The workspace comes in holding NaNs, so a part that is added without having been written shows."""
    x, w, target, b, grad = problem(T, D, V, dtype)
    torch.cuda.synchronize()
    trash = [torch.full((1 << k,), NAN, device="cuda") for k in range(16, 24)]
    del trash                                              # back to the allocator, for the calls below
    check(x, w, target, b, grad)
