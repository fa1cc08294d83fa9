"""What is measured of the classifier-head operators: the layers that follow the 3x3 convolution stack of the
image-classification network this library runs (a 512 x 7 x 7 feature map per image, two fully connected layers of
4096, one of 1000 classes), and the same operators at the sizes they have behind other feature extractors.

  mx4_values   a matrix quantised to microscaled 4-bit floating point (blocks of 32 along a row share one power-of-two
               scale, elements are e2m1) and read back as the values its codes stand for
  mx4_linear   y = relu?(x w^T + bias) with w kept in that format and x quantised to it on the way in
  loss         softmax cross entropy of the logits x w^T + bias per row, without the logits in memory
  loss_grad    the same, and the gradients of x, w and bias for given weights of the rows' losses

`own` selects what run() computes with: the plain forms below (elementary torch operations in 32 bits), or this
package's operators.
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_IGNORE = -100


# ---- cases -----------------------------------------------------------------------------------

def listed():
    return [
        # one image's features on their way into a 4-bit layer: the smallest call, latency counts
        dict(name="values_1x4096_bf16", op="mx4_values", rows=1, K=4096, dtype="bf16"),
        # a ragged batch of feature vectors whose length is no multiple of the block
        dict(name="values_333x1001_f16", op="mx4_values", rows=333, K=1001, dtype="f16"),
        # the first fully connected layer's weights, quantised once when a network is loaded
        dict(name="values_4096x25088_f32", op="mx4_values", rows=4096, K=25088, dtype="f32"),
        # the first fully connected layer for a single image: bound by reading the weights
        dict(name="linear_1x4096x25088_bf16", op="mx4_linear", M=1, N=4096, K=25088, bias=True, relu=True, dtype="bf16"),
        # the class scores of a batch of 32 images (the batch size of this library's benchmark)
        dict(name="linear_32x1000x4096_f16", op="mx4_linear", M=32, N=1000, K=4096, bias=True, relu=False, dtype="f16"),
        # an odd batch through the second fully connected layer, in the element type the convolutions default to
        dict(name="linear_301x4096x4096_f32", op="mx4_linear", M=301, N=4096, K=4096, bias=True, relu=True, dtype="f32"),
        # a large offline batch through a wide layer: bound by the multiplies
        dict(name="linear_4096x8192x8192_bf16", op="mx4_linear", M=4096, N=8192, K=8192, bias=False, relu=False, dtype="bf16"),
        # evaluating a batch of 32 images against 1000 classes
        dict(name="loss_32x1000x4096_f32", op="loss", T=32, V=1000, D=4096, bias=True, dtype="f32"),
        # evaluating a long run of rows against a large, odd vocabulary
        dict(name="loss_4096x50257x1024_bf16", op="loss", T=4096, V=50257, D=1024, bias=False, dtype="bf16"),
        # fine-tuning the last layer on a ragged batch of images
        dict(name="grad_250x1000x4096_f16", op="loss_grad", T=250, V=1000, D=4096, bias=True, dtype="f16"),
        # odd sizes in all three directions, fp32
        dict(name="grad_777x10007x1003_f32", op="loss_grad", T=777, V=10007, D=1003, bias=True, dtype="f32"),
        # a training step over a large vocabulary: the largest call
        dict(name="grad_2048x32000x2048_bf16", op="loss_grad", T=2048, V=32000, D=2048, bias=False, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["mx4_values", "mx4_linear", "loss", "loss_grad"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "mx4_values":
        rows, K = _log(rng, 1, 8192), _log(rng, 32, 25088)
        while rows * K > 4096 * 25088:
            rows = max(1, rows // 2)
        return dict(op=op, rows=rows, K=K, dtype=dtype)
    if op == "mx4_linear":
        M, N, K = _log(rng, 1, 4096), _log(rng, 10, 8192), _log(rng, 32, 25088)
        while M * N * K > 4096 * 8192 * 8192:
            M = max(1, M // 2)
        return dict(op=op, M=M, N=N, K=K, bias=rng.random() < 0.6, relu=rng.random() < 0.5, dtype=dtype)
    T, V, D = _log(rng, 1, 4096), _log(rng, 10, 50257), _log(rng, 64, 4096)
    cap = 2048 * 32000 * 2048 // (8 if dtype == "f32" else 1)
    if op == "loss":
        cap *= 1 if dtype == "f32" else 2
    while T * V * D > cap:
        T = max(1, T // 2)
        V = max(10, V * 3 // 4)
    return dict(op=op, T=T, V=V, D=D, bias=rng.random() < 0.5, dtype=dtype)


# ---- inputs ----------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def _features(g, rows, K, dtype):
    """Feature vectors: normal values, some rows larger, a tenth of the entries zero (what a ReLU leaves)."""
    x = _randn(g, rows, K)
    x *= torch.exp(_randn(g, rows, 1, std=0.5))
    x *= (torch.rand(rows, K, generator=g, device="cuda") >= 0.1)
    return x.to(dtype)


def prepare(case, seed):
    dt = _DT[case["dtype"]]
    g = _gen(seed)
    if case["op"] == "mx4_values":
        return dict(case=case, x=_features(g, case["rows"], case["K"], dt))
    if case["op"] == "mx4_linear":
        M, N, K = case["M"], case["N"], case["K"]
        st = dict(case=case, x=_features(g, M, K, dt))
        w = _randn(g, N, K, std=math.sqrt(2.0 / K)).to(dt)
        st["bias"] = _randn(g, N, std=0.1).to(dt) if case["bias"] else None
        if own:                                     # the weights' 4-bit form is made once, when a network is loaded
            from cudnntest_amd import ops
            st["w"] = ops.mx4_quantize(w)
        else:
            st["codes"], st["scales"] = _pack(*_encode(w))
        return st
    T, V, D = case["T"], case["V"], case["D"]
    st = dict(case=case, x=_features(g, T, D, dt), w=_randn(g, V, D, std=1.5 / math.sqrt(D)).to(dt))
    st["bias"] = _randn(g, V, std=0.5).to(dt) if case["bias"] else None
    target = torch.randint(0, V, (T,), generator=g, device="cuda")
    skip = torch.rand(T, generator=g, device="cuda") < 0.05          # rows without a label
    st["target"] = torch.where(skip, torch.full_like(target, _IGNORE), target)
    if case["op"] == "loss_grad":                   # the weight of each row's loss: a mean over the rows, weighted
        st["grad"] = (0.5 + torch.rand(T, generator=g, device="cuda")) / T
    return st


# ---- the plain forms -------------------------------------------------------------------------

def _pow2(e):
    """2^e in float64 from the exponent's bits: a library's power need not be exact."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _encode(x):
    """e2m1 codes (0..15) [rows, K rounded up to 32] and the biased exponents of the blocks' scales: the scale is
    2^(floor(log2(largest magnitude)) - 2), elements are rounded to nearest (ties to even) and saturate at 6."""
    rows, K = x.shape
    v = torch.zeros(rows, (K + 31) // 32 * 32, dtype=torch.float32, device=x.device)
    v[:, :K] = x
    b = v.view(rows, -1, 32)
    top = (b.abs().amax(-1).view(torch.int32) >> 23) & 255           # biased exponent of the largest magnitude
    scale = torch.where(top == 255, top, (top - 2).clamp(min=0))
    e = torch.where(top == 255, torch.zeros_like(scale), scale)
    r = b * _pow2(127 - e).float().unsqueeze(-1)
    m = r.abs()
    code = ((m > 0.25).int() + (m >= 0.75).int() + (m > 1.25).int() + (m >= 1.75).int() + (m > 2.5).int() +
            (m >= 3.5).int() + (m > 5.0).int())
    code = code + 8 * torch.signbit(r).int()
    code = torch.where((top == 255).unsqueeze(-1), torch.zeros_like(code), code)
    return code.view(rows, -1), scale


def _pack(code, scale):
    return (code[:, 0::2] | (code[:, 1::2] << 4)).to(torch.uint8), scale.to(torch.uint8)


_GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def _decode(code, scale, K):
    grid = torch.tensor(_GRID, device=code.device)
    s = _pow2(scale - 127)
    s = torch.where(scale == 255, torch.full_like(s, float("nan")), s)
    v = grid[code.long()].view(code.shape[0], -1, 32).double() * s.unsqueeze(-1)
    return v.float().view(code.shape[0], -1)[:, :K]


def _unpack(codes, scales, K):
    c = torch.stack((codes & 15, codes >> 4), dim=-1).view(codes.shape[0], -1)
    return _decode(c, scales.int(), K)


def _plain_logits(st):
    l = st["x"].float() @ st["w"].float().t()
    return l if st["bias"] is None else l + st["bias"].float()


def _plain_loss(st):
    l = _plain_logits(st)
    m = l.amax(-1, keepdim=True)
    lse = (l - m).exp().sum(-1).log() + m.squeeze(-1)
    tgt = st["target"]
    keep = tgt != _IGNORE
    picked = l.gather(1, torch.where(keep, tgt, torch.zeros_like(tgt)).unsqueeze(-1)).squeeze(-1)
    return torch.where(keep, lse - picked, torch.zeros_like(lse)), lse


def _plain_grad(st, lse):
    tgt = st["target"]
    keep = tgt != _IGNORE
    g = torch.where(keep, st["grad"], torch.zeros_like(st["grad"]))
    d = (_plain_logits(st) - lse.unsqueeze(-1)).exp()
    rows = torch.arange(d.shape[0], device=d.device)
    d[rows, torch.where(keep, tgt, torch.zeros_like(tgt))] -= 1.0
    d *= g.unsqueeze(-1)
    dt = st["x"].dtype
    dx = (d @ st["w"].float()).to(dt)
    dw = (d.t() @ st["x"].float()).to(dt)
    return dx, dw, None if st["bias"] is None else d.sum(0).to(dt)


# ---- one pass --------------------------------------------------------------------------------

def run(st):
    op = st["case"]["op"]
    if own:
        from cudnntest_amd import ops
        if op == "mx4_values":
            return ops.mx4_dequantize(ops.mx4_quantize(st["x"]), st["x"].dtype)
        if op == "mx4_linear":
            return ops.mx4_linear(st["x"], st["w"], bias=st["bias"], relu=st["case"]["relu"])
        loss, lse = ops.linear_cross_entropy(st["x"], st["w"], st["target"], bias=st["bias"], ignore_index=_IGNORE)
        if op == "loss":
            return loss, lse
        dx, dw, db = ops.linear_cross_entropy_backward(st["grad"], st["x"], st["w"], st["target"], lse,
                                                       bias=st["bias"], ignore_index=_IGNORE)
    else:
        if op == "mx4_values":
            x = st["x"]
            return _decode(*_encode(x), x.shape[1]).to(x.dtype)
        if op == "mx4_linear":
            x, K = st["x"], st["x"].shape[1]
            y = _decode(*_encode(x), K) @ _unpack(st["codes"], st["scales"], K).t()
            if st["bias"] is not None:
                y = y + st["bias"].float()
            return (y.clamp(min=0) if st["case"]["relu"] else y).to(x.dtype)
        loss, lse = _plain_loss(st)
        if op == "loss":
            return loss, lse
        dx, dw, db = _plain_grad(st, lse)
    return (loss, dx, dw) if db is None else (loss, dx, dw, db)


def work(case):
    s = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "mx4_values":
        n, blocks = case["rows"] * case["K"], case["rows"] * ((case["K"] + 31) // 32)
        # read, written as codes and scales, and those read back as values
        return dict(bytes=2 * n * s + 2 * (16 * blocks + blocks), flops=0)
    if case["op"] == "mx4_linear":
        M, N, K = case["M"], case["N"], case["K"]
        return dict(bytes=M * K * s + N * ((K + 31) // 32) * 17 + M * N * s + (N * s if case["bias"] else 0),
                    flops=2 * M * N * K)
    T, V, D = case["T"], case["V"], case["D"]
    b = T * D * s + V * D * s + (V * s if case["bias"] else 0) + T * 8 + T * 8
    if case["op"] == "loss":
        return dict(bytes=b, flops=2 * T * V * D)
    return dict(bytes=b + T * 4 + T * D * s + V * D * s + (V * s if case["bias"] else 0), flops=6 * T * V * D)


# ---- the definitions in 64 bits --------------------------------------------------------------

def _exact_values(x):
    rows, K = x.shape
    out = torch.empty(rows, K, dtype=torch.float64, device=x.device)
    step = max(1, (1 << 24) // max(K, 1))
    for r in range(0, rows, step):
        v = x[r:r + step].double()
        pad = (-K) % 32
        v = torch.nn.functional.pad(v, (0, pad)).reshape(v.shape[0], -1, 32)
        _, e = torch.frexp(v.abs().amax(-1, keepdim=True))           # |v| = f 2^e with f in [1/2, 1)
        scale = ((e.to(torch.int64) - 3).clamp(min=-127) + 1023).bitwise_left_shift(52).view(torch.float64)
        u = v / scale
        _, eu = torch.frexp(u)
        grid = ((eu.to(torch.int64) - 1).clamp(min=0) + 1022).bitwise_left_shift(52).view(torch.float64)   # e2m1's spacing around u
        q = (torch.round(u / grid) * grid).clamp(-6.0, 6.0)                # torch.round: ties to even
        out[r:r + step] = (q * scale).reshape(v.shape[0], -1)[:, :K]
    return out


def exact(case, seed):
    dt = _DT[case["dtype"]]
    g = _gen(seed)
    if case["op"] == "mx4_values":
        return _exact_values(_features(g, case["rows"], case["K"], dt))
    if case["op"] == "mx4_linear":
        M, N, K = case["M"], case["N"], case["K"]
        x = _features(g, M, K, dt)
        w = _randn(g, N, K, std=math.sqrt(2.0 / K)).to(dt)
        y = torch.matmul(_exact_values(x), _exact_values(w).t().contiguous())
        if case["bias"]:
            y += _randn(g, N, std=0.1).to(dt).double()
        return torch.relu(y) if case["relu"] else y
    T, V, D = case["T"], case["V"], case["D"]
    if T * V * D > 2e11 and case["op"] == "loss_grad":
        return None
    x = _features(g, T, D, dt).double()
    w = _randn(g, V, D, std=1.5 / math.sqrt(D)).to(dt).double()
    bias = _randn(g, V, std=0.5).to(dt).double() if case["bias"] else None
    target = torch.randint(0, V, (T,), generator=g, device="cuda")
    skip = torch.rand(T, generator=g, device="cuda") < 0.05
    grad = (0.5 + torch.rand(T, generator=g, device="cuda")) / T if case["op"] == "loss_grad" else None
    logits = torch.matmul(x, w.t().contiguous())
    if bias is not None:
        logits += bias
    lse = torch.logsumexp(logits, dim=1, keepdim=True)
    logp = logits - lse
    del logits
    loss = -torch.take_along_dim(logp, target[:, None], 1)[:, 0]
    loss[skip] = 0
    if case["op"] == "loss":
        return loss, lse[:, 0]
    d = torch.exp(logp)
    del logp
    d.scatter_add_(1, target[:, None], -torch.ones(T, 1, dtype=torch.float64, device="cuda"))
    d *= (grad.double() * ~skip)[:, None]
    out = (loss, torch.matmul(d, w), torch.matmul(d.t().contiguous(), x))
    return out if bias is None else out + (d.sum(0),)
