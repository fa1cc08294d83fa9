"""Plain 64-bit forms of the head's operators, and the bounds their tests use."""
import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # half a step, relative
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}   # half the smallest step
E32 = 2.0 ** -24
GRID = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def half_step(y, dtype):
    return y.abs() * U[dtype] + TINY[dtype]


def pow2(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def mx4_encode(x):
    """codes [rows][Kp], scale bytes [rows][Kp/32] of a matrix on the CPU, Kp a multiple of 128."""
    rows, K = x.shape
    Kp = (K + 127) // 128 * 128
    v = torch.zeros(rows, Kp, dtype=torch.float64)
    v[:, :K] = x.double()
    b = v.view(rows, Kp // 32, 32)
    top = b.abs().amax(-1)
    _, e = torch.frexp(top)
    byte = torch.where(top > 0, (e.long() - 1 - 2 + 127).clamp(0, 254), torch.zeros_like(e.long()))
    bad = ~torch.isfinite(b).all(-1)
    byte[bad] = 255
    u = b / pow2(torch.where(bad, torch.full_like(byte, 127), byte) - 127).unsqueeze(-1)
    # nearest of the grid; at equal distance the one with the even code
    d = (u.abs().clamp(max=6.0).unsqueeze(-1) - GRID).abs()
    near = d.amin(-1, keepdim=True)
    code = torch.arange(8)
    rank = torch.where(d == near, code % 2, torch.full_like(code, 9))
    c = rank.argmin(-1) + 8 * torch.signbit(u).long()
    c[bad] = 0
    return c.view(rows, Kp), byte


def mx4_pack(codes, scales):
    """The library's operand layout."""
    rows, Kp = codes.shape
    p = (codes[:, 0::2] | codes[:, 1::2] << 4).to(torch.uint8).view(rows, Kp // 128, 64).permute(1, 0, 2).contiguous()
    s = torch.zeros(Kp // 128, (rows + 3) // 4 * 4, 4, dtype=torch.uint8)
    s[:, :rows] = scales.to(torch.uint8).view(rows, Kp // 128, 4).permute(1, 0, 2)
    return p, s


def mx4_values(codes, scales, K):
    g = torch.cat([GRID, -GRID])[codes]
    s = pow2(scales - 127)
    s[scales == 255] = float("nan")
    return (g.view(codes.shape[0], -1, 32) * s.unsqueeze(-1)).view(codes.shape)[:, :K]


def mx4_round(x):
    c, s = mx4_encode(x.cpu())
    return mx4_values(c, s, x.shape[1])


def product_bound(xq, wq, bias, y, dtype):
    """|kernel - exact| for y = relu?(xq wq^T + bias): the products are exact, a sum of n of them in fp32 is off by at most
    n 2^-24 of the sum of magnitudes, in whatever order they are added; the bias adds one rounding, the store half a step."""
    n = xq.shape[1] + 1
    mag = xq.abs() @ wq.abs().t()
    if bias is not None:
        mag = mag + bias.double().abs()
    return n * E32 * mag + half_step(y, dtype)


class Ce:
    """Loss, lse and gradients in float64 from the tensors' own (rounded) values, with bounds for the kernels' results."""

    def __init__(self, x, w, target, bias=None, ignore=-100, grad=None):
        dt = x.dtype
        X, W = x.double(), w.double()
        T, D = X.shape
        V = W.shape[0]
        l = X @ W.t().contiguous()
        mag = X.abs() @ W.abs().t().contiguous()
        if bias is not None:
            l = l + bias.double()
            mag = mag + torch.where(torch.isfinite(bias), bias.double().abs(), torch.zeros(()).double().to(bias.device))
        keep = target != ignore
        safe = torch.where(keep, target, torch.zeros_like(target))
        self.lse = torch.logsumexp(l, 1)
        rows = torch.arange(T, device=x.device)
        self.loss = torch.where(keep, self.lse - l[rows, safe], torch.zeros_like(self.lse))
        # a logit: D products and a bias in fp32; lse moves by at most the largest change of a logit, plus the roundings of
        # exp, V additions (each relative to a sum of positive terms) and of the logarithm
        dl_logit = (D + 2) * E32 * mag
        fin = torch.where(torch.isfinite(l), dl_logit, torch.zeros_like(dl_logit))
        worst = fin.amax(1)
        spread = torch.where(torch.isfinite(l), (l - self.lse.unsqueeze(1)).abs(), torch.zeros_like(l))
        # terms of exp(l - max): off by (|l - max| + 4) 2^-24 relative, weighted by their share p
        p = (l - self.lse.unsqueeze(1)).exp()
        self.lse_tol = worst + ((p * (2 * spread + 8)).sum(1) + V + 8) * E32 + 4 * E32 * self.lse.abs()
        self.loss_tol = self.lse_tol + fin[rows, safe] + 2 * E32 * (self.lse.abs() + l[rows, safe].abs().nan_to_num(posinf=0))
        if grad is None:
            return
        g = torch.where(keep, grad.double(), torch.zeros_like(self.lse))
        hot = torch.zeros_like(p)
        hot[rows, safe] = 1.0
        d = (p - hot) * g.unsqueeze(1)
        # p: exponent off by the logit, lse (stored in fp32) and the arithmetic; then dl rounded to the type
        # (the exponential instruction returns 0 below the smallest normal number: off by less than 2^-126, absolute)
        dp = p * (fin + (self.lse_tol + E32 * self.lse.abs()).unsqueeze(1) + (4 * spread + 8) * E32) + 2.0 ** -126
        gmax = g.abs().max()
        floor = gmax * 2.0 ** -39 if dt == torch.float16 else TINY[dt]
        # (six more roundings: the subtraction, the row's weight made relative to the largest, its product, the way back)
        dd = (dp + 6 * E32 * (p + hot)) * g.abs().unsqueeze(1) + d.abs() * U[dt] + floor
        dd = torch.where(keep.unsqueeze(1), dd, torch.zeros_like(dd))
        ad = d.abs() + dd
        self.dx, self.dw, self.db = d @ W, d.t().contiguous() @ X, d.sum(0)
        self.dx_tol = dd @ W.abs() + (V + 2) * E32 * (ad @ W.abs()) + half_step(self.dx, dt) * (1 + U[dt])
        self.dw_tol = dd.t().contiguous() @ X.abs() + (T + 2) * E32 * (ad.t().contiguous() @ X.abs()) + half_step(self.dw, dt) * (1 + U[dt])
        self.db_tol = dd.sum(0) + (T + 2) * E32 * ad.sum(0) + half_step(self.db, dt) * (1 + U[dt])


def assert_within(got, want, tol, what):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaNs in other places"
    ok = torch.isnan(want) | (got == want) | ((got - want).abs() <= tol)
    if not bool(ok.all()):
        i = int((~ok).flatten().nonzero()[0])
        raise AssertionError(f"{what}: {int((~ok).sum())} of {ok.numel()} off, first at {i}: got {got.flatten()[i].item()!r}, "
                             f"want {want.flatten()[i].item()!r}, allowed {tol.expand_as(want).flatten()[i].item()!r}")
