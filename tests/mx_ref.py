"""Plain 64-bit forms of MXFP4 and of the fused norm, and the error bounds of the kernels.  TEST INFRASTRUCTURE ONLY."""

import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}     # largest relative error of one rounding
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}       # half of the smallest subnormal


def quantize(x):
    """x [R, K] -> (codes uint8 [R, K], scale codes uint8 [R, K/32]), by nearest grid point, ties to the even code."""
    rows, k = x.shape
    b = x.double().reshape(rows, k // 32, 32)
    bad = ~torch.isfinite(b).all(dim=-1)
    b = torch.where(bad.unsqueeze(-1), torch.zeros_like(b), b)
    top = b.abs().amax(dim=-1)
    _, e = torch.frexp(top)                                                # top = f * 2^e, f in [0.5, 1): floor(log2 top) = e - 1
    e = torch.where(top > 0, (e - 3).clamp(min=-127), torch.full_like(e, -127))
    size = torch.ldexp(b.abs(), -e.unsqueeze(-1))
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    border = (grid[1:] + grid[:-1]) / 2
    low, high = torch.bucketize(size, border), torch.bucketize(size, border, right=True)
    code = torch.where(low % 2 == 0, low, high)
    code = code + 8 * torch.signbit(b).long()
    scale = torch.where(bad, torch.full_like(e, 255), e + 127)
    return code.reshape(rows, k).to(torch.uint8), scale.to(torch.uint8)


def pack(codes):
    c = codes.view(codes.shape[0], -1, 2)
    return c[..., 0] | (c[..., 1] << 4)


def unpack(data):
    return torch.stack((data & 15, data >> 4), dim=-1).reshape(data.shape[0], -1)


def values(codes, scales):
    """fp64 values of codes [R, K] with scale codes [R, K/32]; 255 is NaN."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), dtype=torch.float64, device=codes.device)
    s = torch.exp2(scales.double() - 127.0)
    s = torch.where(scales == 255, torch.full_like(s, float("nan")), s)
    return grid[codes.long()] * s.repeat_interleave(32, dim=1)


def product_bound(a, b, exact, dtype, splits=8):
    """|kernel - exact| for fp32 accumulation: products of E2M1 values are exact; every 32 of them are added to the accumulator, which
    may drop its last bit (2^-23 of a partial sum, itself at most sum |a b|); the K split and the bias add a few more; one rounding."""
    size = a.abs() @ b.abs().t()
    adds = a.shape[1] // 32 + splits + 2
    return exact.abs() * HALF_STEP[dtype] * 1.001 + size * adds * 2.0 ** -23 + TINY[dtype]


def _norm(v, kind, eps):
    mean = v.mean(dim=-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    d = v - mean
    inv = 1.0 / torch.sqrt((d * d).mean(dim=-1, keepdim=True) + eps)
    return d * inv, inv, mean


def gated_norm(x, y=None, gate=None, residual_scale=1.0, post_norm=False, post_weight=None, weight=None, bias=None, scale=None, shift=None, kind="rms", eps=1e-6):
    """(r, h, bound of r, bound of h before their rounding), all fp64.

    u = 2^-24 is the error of one fp32 operation.  A sum of C values in the kernel is at most 32 sequential additions in a thread and
    11 levels of a tree, so a mean is off by at most 48 u times the mean of the absolute values; a mean of squares of values that
    are themselves off by d (rms) is off by that and by 2 d; a norm costs 4 operations more.  First order, with a factor 2 on top."""
    u = 2.0 ** -24
    f = lambda t: None if t is None else t.double()  # noqa: E731
    x, y, gate, post_weight, weight, bias, scale, shift = (f(t) for t in (x, y, gate, post_weight, weight, bias, scale, shift))

    def norm(v, off):
        n, inv, mean = _norm(v, kind, eps)
        off_mean = (48 * u * v.abs().mean(dim=-1, keepdim=True) + off.mean(dim=-1, keepdim=True)) if kind == "layer" else 0.0
        off_d = off + off_mean + u * (v - mean).abs()
        # relative error of 1 / sqrt(mean d^2 + eps)
        rel = 0.5 * (48 * u + 2 * (off_d * (v - mean).abs()).mean(dim=-1, keepdim=True) * inv * inv) + 4 * u
        return n, off_d * inv + n.abs() * rel

    if y is None:
        r, off = x, torch.zeros_like(x)
    else:
        z, off_z = y, torch.zeros_like(y)
        if post_norm:
            z, off_z = norm(y, off_z)
            if post_weight is not None:
                z, off_z = z * post_weight, (off_z + u * z.abs()) * post_weight.abs()
        if gate is not None:
            z, off_z = z * gate, (off_z + u * z.abs()) * gate.abs()
        # residual_scale reaches the kernel as fp32
        r = x + residual_scale * z
        off = abs(residual_scale) * (off_z + 2 * u * z.abs()) + u * r.abs()
    h, off_h = norm(r, off)
    if weight is not None:
        h, off_h = h * weight, (off_h + u * h.abs()) * weight.abs()
    if bias is not None:
        h = h + bias
        off_h = off_h + u * h.abs()
    if scale is not None:
        off_h = (off_h + 2 * u * h.abs()) * (1.0 + scale).abs() + u * h.abs()
        h = h * (1.0 + scale)
    if shift is not None:
        h = h + shift
        off_h = off_h + u * h.abs()
    return r, h, 2 * off, 2 * off_h


def within(got, exact, off, what):
    """got (16 or 32 bits) against exact, where the value before the rounding may be off by `off`."""
    dtype = got.dtype
    g = got.double()
    assert torch.equal(torch.isnan(g), torch.isnan(exact)), f"{what}: NaN in other places"
    fine = torch.isfinite(exact)
    err = (g - exact)[fine].abs()
    limit = (off + exact.abs() * HALF_STEP[dtype] * 1.001 + TINY[dtype])[fine]
    over = err > limit
    assert not over.any(), f"{what}: {int(over.sum())} of {over.numel()} out of bounds, worst {float((err / limit).max()):.3g} x the bound"
