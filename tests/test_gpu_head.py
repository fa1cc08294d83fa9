"""The head behind the convolution stack: features -> two 4-bit layers -> last layer's loss and gradients."""
import pytest
import torch

from cudnntest_amd import ops
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
