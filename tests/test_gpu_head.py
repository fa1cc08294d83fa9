"""The head behind the convolution stack: features -> two 4-bit layers -> last layer's loss and gradients."""
import pytest
import torch

from cudnntest_amd import _lib, ops
from head_reference import Ce, assert_within, mx4_round, product_bound

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N", [1, 5, 33])
def test_network_with_its_head(N, dtype):
    g = torch.Generator(device="cuda").manual_seed(N)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g, device="cuda") * std).to(dtype)
    stack = ops.ConvStack(dtype, N, 3, 24, 24, [dict(K=32, relu=True, pool=True), dict(K=40, relu=True, pool=True)])
    stack.set_layer(0, r(32, 3, 3, 3, std=0.3), r(32, std=0.1))
    stack.set_layer(1, r(40, 32, 3, 3, std=0.1), r(40, std=0.1))
    x = stack.forward(r(N, 3, 24, 24)).flatten(1)                       # [N][40 * 6 * 6]
    assert x.shape == (N, 1440)
    fc = [(ops.mx4_quantize(r(300, 1440, std=0.04)), r(300, std=0.1)), (ops.mx4_quantize(r(200, 300, std=0.08)), r(200, std=0.1))]
    for w, b in fc:
        xv, wv = mx4_round(x), ops.mx4_dequantize(w).double().cpu()
        want = (xv @ wv.t() + b.double().cpu()).clamp(min=0)
        y = ops.mx4_linear(x, w, bias=b, relu=True)
        assert_within(y.cpu(), want, product_bound(xv, wv, b.cpu(), want, dtype), "layer")
        x = y
    w, b = r(50, 200, std=0.1), r(50, std=0.1)
    target = torch.randint(0, 50, (N,), generator=g, device="cuda")
    loss, lse = ops.linear_cross_entropy(x, w, target, bias=b)
    grad = torch.full((N,), 1.0 / N, device="cuda")
    dx, dw, db = ops.linear_cross_entropy_backward(grad, x, w, target, lse, bias=b)
    ref = Ce(x, w, target, b, grad=grad)
    for got, want, tol, what in ((loss, ref.loss, ref.loss_tol, "loss"), (dx, ref.dx, ref.dx_tol, "dx"), (dw, ref.dw, ref.dw_tol, "dw"),
                                 (db, ref.db, ref.db_tol, "dbias")):
        assert_within(got, want, tol, what)
    stack.close()


GUARD = 4096


def dirty_workspace(nbytes):
    """A workspace full of NaNs with a guard behind it."""
    return torch.full((nbytes + GUARD,), 0xFF, dtype=torch.uint8, device="cuda")


def guarded(shape, dtype):
    """An output full of NaNs with a guard behind it."""
    n = 1
    for s in shape:
        n *= s
    buf = torch.full((n + 64,), float("nan"), dtype=dtype, device="cuda")
    return buf, buf[:n].view(shape)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,D,V", [(1, 1, 1), (1, 700, 3000), (3, 33, 900), (40, 1000, 1000), (66, 299, 664), (164, 211, 476), (250, 1000, 1000), (257, 129, 333),
                                   (300, 2050, 70), (900, 64, 5000), (1500, 100, 9000), (1030, 24, 70000)])
def test_loss_reads_nothing_it_has_not_written(T, D, V, dtype):
    """The C calls with a workspace and outputs that hold NaNs: the bits of a clean call, and nothing behind their ends touched."""
    g = torch.Generator(device="cuda").manual_seed(T + D + V)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)
    x, w, b = r(T, D), r(V, D), r(V)
    target = torch.randint(0, V, (T,), generator=g, device="cuda")
    target[::5] = -100
    grad = torch.rand(T, generator=g, device="cuda")
    want = ops.linear_cross_entropy(x, w, target, bias=b)
    want += ops.linear_cross_entropy_backward(grad, x, w, target, want[1], bias=b)
    assert all(bool(torch.isfinite(t.float()).all()) for t in want)
    L, dt, s = _lib.load(), ops._DTYPES[dtype], torch.cuda.current_stream().cuda_stream
    outs = [guarded((T,), torch.float32), guarded((T,), torch.float32), guarded((T, D), dtype), guarded((V, D), dtype), guarded((V,), dtype)]
    for backward in (0, 1):
        n = L.wino_linear_cross_entropy_workspace_bytes(dt, T, D, V, x.data_ptr(), w.data_ptr(), backward)
        ws = dirty_workspace(n)
        head = (dt, T, D, V, x.data_ptr(), w.data_ptr(), b.data_ptr(), target.data_ptr(), -100)
        if backward:
            rc = L.wino_linear_cross_entropy_backward(*head, grad.data_ptr(), outs[1][1].data_ptr(), *(o[1].data_ptr() for o in outs[2:]), ws.data_ptr(), n, s)
        else:
            rc = L.wino_linear_cross_entropy(*head, outs[0][1].data_ptr(), outs[1][1].data_ptr(), ws.data_ptr(), n, s)
        assert rc == 0, L.wino_last_error()
        assert bool((ws[n:] == 0xFF).all()), "written behind the workspace"
    for (buf, got), ref in zip(outs, want):
        assert torch.equal(got, ref)
        assert bool(torch.isnan(buf[got.numel():]).all()), "written behind an output"


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 1000, 4096), (5, 77, 333), (17, 200, 9000), (33, 257, 129), (64, 4096, 1000), (200, 300, 8192), (301, 1000, 4097)])
def test_layers_read_nothing_they_have_not_written(M, N, K, dtype):
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)
    x, w, b = r(M, K), ops.mx4_quantize(r(N, K)), r(N)
    want = ops.mx4_linear(x, w, bias=b)
    assert bool(torch.isfinite(want.float()).all())
    L, dt, s = _lib.load(), ops._DTYPES[dtype], torch.cuda.current_stream().cuda_stream
    n = L.wino_mx4_workspace_bytes(M, N, K)
    ws, (buf, y) = dirty_workspace(n), guarded((M, N), dtype)
    assert L.wino_mx4_linear(dt, 0, M, N, K, x.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), b.data_ptr(), y.data_ptr(), ws.data_ptr(), n, s) == 0
    assert torch.equal(y, want) and bool(torch.isnan(buf[y.numel():]).all()) and bool((ws[n:] == 0xFF).all())
    geo = ops.mx4_geometry(M, K)
    codes, scales = dirty_workspace(geo["code_bytes"]), dirty_workspace(geo["scale_bytes"])
    assert L.wino_mx4_quantize(dt, M, K, x.data_ptr(), codes.data_ptr(), scales.data_ptr(), s) == 0
    q = ops.mx4_quantize(x)
    assert torch.equal(codes[:-GUARD], q.codes.view(-1)) and torch.equal(scales[:-GUARD], q.scales.view(-1))
    assert bool((codes[-GUARD:] == 0xFF).all()) and bool((scales[-GUARD:] == 0xFF).all())
    buf, back = guarded((M, K), dtype)
    assert L.wino_mx4_dequantize(dt, M, K, codes.data_ptr(), scales.data_ptr(), back.data_ptr(), s) == 0
    assert torch.equal(back, ops.mx4_dequantize(q, dtype)) and bool(torch.isnan(buf[back.numel():]).all())
