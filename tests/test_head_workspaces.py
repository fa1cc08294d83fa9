"""How long the head's Python calls keep what they hand to the library, on the CPU: a workspace that is back with the
allocator before its launches are queued can be handed to another thread's call on the same stream."""
import weakref

import pytest
import torch

from cudnntest_amd import ops

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
