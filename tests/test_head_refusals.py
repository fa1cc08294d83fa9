"""What the head's entry points refuse, on the CPU: arguments are checked before a GPU is touched."""
import ctypes

import pytest
import torch

from cudnntest_amd import _lib, ops

INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -4
P = ctypes.c_void_p(256)                                    # never dereferenced: validation fails first
ODD = ctypes.c_void_p(257)
OFF8 = ctypes.c_void_p(264)


def test_mx4_geometry():
    assert ops.mx4_geometry(3, 257) == dict(Kp=384, code_bytes=3 * 192, scale_bytes=4 * 12)
    assert ops.mx4_geometry(1, 1) == dict(Kp=128, code_bytes=64, scale_bytes=16)
    L = _lib.load()
    assert L.wino_mx4_geometry(0, 5, None, None, None) == INVALID
    assert L.wino_mx4_geometry(5, -1, None, None, None) == INVALID
    assert L.wino_mx4_geometry(5, (1 << 21) + 1, None, None, None) == UNSUPPORTED


def test_mx4_refusals():
    L = _lib.load()
    assert L.wino_mx4_quantize(9, 1, 32, P, P, P, None) == INVALID
    assert L.wino_mx4_quantize(0, 0, 32, P, P, P, None) == INVALID
    assert L.wino_mx4_quantize(0, 1, 32, None, P, P, None) == INVALID
    assert L.wino_mx4_quantize(0, 1, 32, ODD, P, P, None) == INVALID
    assert L.wino_mx4_quantize(0, 1, 32, P, OFF8, P, None) == INVALID
    assert b"16-byte" in L.wino_last_error()
    assert L.wino_mx4_dequantize(0, 1, 32, P, P, None, None) == INVALID
    assert L.wino_mx4_dequantize(0, 1, 32, P, OFF8, P, None) == INVALID
    assert L.wino_mx4_workspace_bytes(0, 1, 1) == 0
    assert L.wino_mx4_workspace_bytes(4, 8, 32) == 0        # few rows need none
    need = L.wino_mx4_workspace_bytes(40, 8, 32)
    assert need > 0
    gemm = lambda **k: L.wino_mx4_gemm(*[k.get(n, d) for n, d in (
        ("dtype", 0), ("flags", 0), ("M", 4), ("N", 8), ("K", 32), ("xc", P), ("xs", P), ("wc", P), ("ws", P), ("bias", P), ("y", P), ("work", P),
        ("bytes", need), ("stream", None))])
    assert gemm(dtype=3) == INVALID
    assert gemm(flags=2) == INVALID                         # pooling makes no sense here
    assert gemm(M=0) == INVALID
    assert gemm(N=-3) == INVALID
    assert gemm(K=0) == INVALID
    assert gemm(xc=None) == INVALID
    assert gemm(ws=None) == INVALID
    assert gemm(wc=OFF8) == INVALID
    assert gemm(y=None) == INVALID
    assert gemm(y=ODD) == INVALID
    assert gemm(bias=ODD) == INVALID
    assert gemm(work=OFF8) == INVALID
    lin = lambda x, work, nbytes: L.wino_mx4_linear(0, 0, 40, 8, 32, x, P, P, None, P, work, nbytes, None)
    assert lin(None, P, need) == INVALID
    assert lin(ODD, P, need) == INVALID
    assert lin(P, None, need) == WORKSPACE
    assert lin(P, P, need - 1) == WORKSPACE


def test_cross_entropy_refusals():
    L = _lib.load()
    size = lambda backward, T=4, D=32, V=10, dt=0: L.wino_linear_cross_entropy_workspace_bytes(dt, T, D, V, P, P, backward)
    assert size(0) > 0 and size(1) > size(0)
    assert size(0, T=0) == 0 and size(0, dt=7) == 0 and size(0, V=-1) == 0
    # rows that are not 16-byte aligned are copied: more workspace
    assert size(0, D=33) > size(0, D=36)
    assert L.wino_linear_cross_entropy_workspace_bytes(0, 4, 32, 10, ctypes.c_void_p(260), P, 0) > size(0)
    fwd = lambda **k: L.wino_linear_cross_entropy(*[k.get(n, d) for n, d in (
        ("dtype", 0), ("T", 4), ("D", 32), ("V", 10), ("x", P), ("w", P), ("bias", P), ("target", P), ("ignore", -100), ("loss", P), ("lse", P),
        ("work", P), ("bytes", size(0)), ("stream", None))])
    assert fwd(dtype=5) == INVALID
    for n in ("T", "D", "V"):
        assert fwd(**{n: 0}) == INVALID
    for n in ("x", "w", "target", "loss", "lse"):
        assert fwd(**{n: None}) == INVALID
        assert fwd(**{n: ODD}) == INVALID
    assert fwd(bias=ODD) == INVALID
    assert fwd(D=(1 << 21) + 1) == UNSUPPORTED
    assert fwd(V=(1 << 24) + 1) == UNSUPPORTED
    assert fwd(work=None) == WORKSPACE
    assert fwd(bytes=size(0) - 1) == WORKSPACE
    assert fwd(work=OFF8) == INVALID
    bwd = lambda **k: L.wino_linear_cross_entropy_backward(*[k.get(n, d) for n, d in (
        ("dtype", 0), ("T", 4), ("D", 32), ("V", 10), ("x", P), ("w", P), ("bias", P), ("target", P), ("ignore", -100), ("grad", P), ("lse", P),
        ("dx", P), ("dw", P), ("db", P), ("work", P), ("bytes", size(1)), ("stream", None))])
    for n in ("x", "w", "target", "grad", "lse"):
        assert bwd(**{n: None}) == INVALID
    for n in ("dx", "dw", "db"):
        assert bwd(**{n: ODD}) == INVALID
    assert bwd(dx=None, dw=None, db=None) == INVALID
    assert bwd(bytes=size(0) - 1) == WORKSPACE


def test_python_layer_refuses():
    x, t = torch.zeros(4, 32), torch.zeros(4, dtype=torch.int64)
    w = torch.zeros(10, 32)
    with pytest.raises(ValueError, match="GPU"):
        ops.mx4_quantize(x)
    with pytest.raises(ValueError, match="matrix"):
        ops.mx4_quantize(torch.zeros(4))
    with pytest.raises(TypeError):
        ops.mx4_quantize(x.double())
    q = ops.Mx4(torch.zeros(1, 4, 64, dtype=torch.uint8), torch.zeros(1, 4, 4, dtype=torch.uint8), 4, 32)
    with pytest.raises(ValueError):
        ops.Mx4(q.codes, q.scales, 4, 257)
    with pytest.raises(TypeError):
        ops.Mx4(q.codes.to(torch.int16), q.scales, 4, 32)
    with pytest.raises(ValueError, match="contiguous"):
        ops.Mx4(torch.zeros(1, 4, 128, dtype=torch.uint8)[..., ::2], q.scales, 4, 32)
    with pytest.raises(ValueError, match="GPU"):
        ops.mx4_dequantize(q)
    with pytest.raises(ValueError, match="GPU"):
        ops.mx4_gemm(q, q)
    with pytest.raises(ValueError, match="columns"):
        ops.mx4_linear(torch.zeros(4, 33), q)
    with pytest.raises(TypeError, match="bias"):
        ops.mx4_linear(x, q, bias=torch.zeros(5))
    with pytest.raises(TypeError, match="dtype"):
        ops.mx4_dequantize(q, torch.float64)
    with pytest.raises(ValueError):
        ops.mx4_linear(x, q, out=torch.zeros(4, 5))
    with pytest.raises(ValueError, match="GPU"):
        ops.linear_cross_entropy(x, w, t)
    with pytest.raises(TypeError, match="int64"):
        ops.linear_cross_entropy(x, w, t.int())
    with pytest.raises(TypeError, match="int64"):
        ops.linear_cross_entropy(x, w, t[:3])
    with pytest.raises(ValueError, match="columns"):
        ops.linear_cross_entropy(x, torch.zeros(10, 31), t)
    with pytest.raises(TypeError, match="dtype"):
        ops.linear_cross_entropy(x, w.half(), t)
    with pytest.raises(TypeError, match="grad"):
        ops.linear_cross_entropy_backward(t, x, w, t, torch.zeros(4))
