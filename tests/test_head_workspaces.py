"""How long the head's Python calls keep what they hand to the library, on the CPU: a workspace that is back with the
allocator before its launches are queued can be handed to another thread's call on the same stream."""
import ctypes
import weakref

import pytest
import torch

from cudnntest_amd import _lib, ops

BYTES = 12345


def calls():
    x, w, t = torch.zeros(40, 256), torch.zeros(10, 256), torch.zeros(40, dtype=torch.int64)
    g = ops.mx4_geometry(40, 256)
    q = ops.Mx4(torch.zeros(g["code_bytes"], dtype=torch.uint8), torch.zeros(g["scale_bytes"], dtype=torch.uint8), 40, 256)
    f = torch.zeros(40)
    return {"mx4_linear": lambda: ops.mx4_linear(x, q), "mx4_gemm": lambda: ops.mx4_gemm(q, q),
            "linear_cross_entropy": lambda: ops.linear_cross_entropy(x, w, t),
            "linear_cross_entropy_backward": lambda: ops.linear_cross_entropy_backward(f, x, w, t, f)}


@pytest.mark.parametrize("name", sorted(calls()))
def test_workspace_lives_until_the_call_has_returned(name, monkeypatch):
    made, seen = [], []
    real = torch.empty

    def empty(*size, **kw):
        t = real(*size, **kw)
        if size == (BYTES,):
            made.append((weakref.ref(t), t.data_ptr()))
        return t

    def call(device, fn, what, *args):
        # the launches are queued here
        assert made and all(at in args for _, at in made), "the workspace is not handed on"
        seen.extend(ref() is not None for ref, _ in made)
    monkeypatch.setattr(torch, "empty", empty)
    monkeypatch.setattr(ops, "_call", call)
    monkeypatch.setattr(ops, "_on_gpu", lambda q, device, what: None)
    monkeypatch.setattr(ops, "_ptr", lambda t: t.data_ptr())
    monkeypatch.setattr(ops, "_mx4_workspace_bytes", lambda *a: BYTES)
    monkeypatch.setattr(ops, "_ce_workspace_bytes", lambda *a: BYTES)
    calls()[name]()
    assert seen == [True]


def test_more_rows_than_a_reduction_counts_are_refused():
    """dw of 16-bit tensors reduces over two values a row: past 2^29 rows (256 GB of dl) the call is refused, not cut short."""
    L, P = _lib.load(), ctypes.c_void_p(256)
    size = lambda dt, T, backward: L.wino_linear_cross_entropy_workspace_bytes(dt, T, 1, 100, P, P, backward)
    for dt in (1, 2):
        assert size(dt, 1 << 29, 1) >= (1 << 29) * 128 * 2 * 2 and size(dt, (1 << 29) + 1, 1) == 0
        assert size(dt, (1 << 29) + 1, 0) > 0
        rc = L.wino_linear_cross_entropy_backward(dt, (1 << 29) + 1, 1, 100, P, P, None, P, -100, P, P, P, P, None, P, 1 << 60, None)
        assert rc == -2 and b"at most" in L.wino_last_error()
    assert size(0, (1 << 29) + 1, 1) > 0


@pytest.mark.parametrize("dt,e", [(0, 4), (1, 2), (2, 2)])
def test_output_over_the_input_of_few_rows_is_refused(dt, e):
    """One launch quantises x and writes y: every workgroup reads all of x, so y must not lie over it."""
    L, at = _lib.load(), 1 << 20
    linear = lambda M, N, K, y: L.wino_mx4_linear(dt, 0, M, N, K, ctypes.c_void_p(at), ctypes.c_void_p(1 << 30), ctypes.c_void_p(1 << 29), None,
                                                  ctypes.c_void_p(y), None, 0, None)
    M, N, K = 4, 512, 1024
    assert L.wino_mx4_workspace_bytes(M, N, K) == 0
    for y in (at, at + 64, at + M * K * e - e, at - M * N * e + e):
        assert linear(M, N, K, y) == -1 and b"overlap" in L.wino_last_error()


def test_sizes_past_32_bits_are_refused():
    """The C calls take int: a size past it must not arrive as its low 32 bits."""
    long = torch.empty((1 << 32) + 5, 1, device="meta")
    t, w = torch.zeros(5, dtype=torch.int64), torch.zeros(3, 1)
    q = ops.Mx4(torch.zeros(64, dtype=torch.uint8), torch.zeros(16, dtype=torch.uint8), 1, 1)
    f = torch.zeros(5)
    for call in (lambda: ops.mx4_quantize(long), lambda: ops.mx4_linear(long, q), lambda: ops.linear_cross_entropy(long, w, t),
                 lambda: ops.linear_cross_entropy(torch.zeros(5, 1), long, t), lambda: ops.linear_cross_entropy_backward(f, long, w, t, f),
                 lambda: ops.mx4_geometry((1 << 32) + 5, 1), lambda: ops.mx4_geometry(5, (1 << 32) + 1),
                 lambda: ops.Mx4(q.codes, q.scales, (1 << 32) + 1, 1)):
        with pytest.raises(ValueError, match="32 bits"):
            call()
