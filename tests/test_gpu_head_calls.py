"""Calls of the head that a program makes around the plain ones: several threads on one stream."""
import threading

import pytest
import torch

from cudnntest_amd import ops

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
