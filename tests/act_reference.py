"""Plain 64-bit forms of the 8-bit activation checkpoints, from their definitions (include/camal_hip.h), on the CPU."""
import torch

BLOCK = 32
LARGEST = {"int8": 127.0, "e4m3": 448.0}
REACH = {"int8": 121, "e4m3": 119}  # the largest scale under which the largest code is still a float


def power(k):
    return ((k.long() + 1023) << 52).view(torch.float64)


def normalised(z, mean, invstd):
    """The float32 values that are quantised, in 64 bits."""
    return ((z.double() - mean.double()).float().double() * invstd.double()).float().double()


def side(x, gamma, beta):
    """Which side of the ReLU x is on: the sign of the float32 fma (which may underflow to zero)."""
    return (gamma.double() * x + beta.double()).float() > 0


def keep(x, fmt, gamma=None, beta=None):
    """-> (values [.., C] float64, scale bytes [.., C / 32]).  gamma given: behind a ReLU, the side is kept."""
    blocks = x.unflatten(-1, (-1, BLOCK))
    top = blocks.abs().amax(-1, keepdim=True)
    bad = ~(top <= LARGEST[fmt] * 2.0 ** REACH[fmt])
    mantissa, k = torch.frexp(torch.where(bad, 1.0, top) / LARGEST[fmt])
    k = torch.where(mantissa == 0.5, k - 1, k)
    k = torch.where(top == 0, -126, k).clamp(min=-126)
    s = power(k).expand_as(blocks)
    y = torch.where(bad, 0.0, blocks) / s
    step = torch.ones_like(y) if fmt == "int8" else power((torch.frexp(y)[1] - 1).clamp(min=-6) - 3)
    v = (y / step).round() * step
    v, y, step, s = (t.flatten(-2) for t in (v, y, step, s))
    if gamma is not None:
        other = torch.where(v < y, (y / step).ceil(), (y / step).floor()) * step
        wrong = side(v * s, gamma, beta) != side(x, gamma, beta)
        v = torch.where(wrong & ~bad.expand_as(blocks).flatten(-2), other, v)
    kept = torch.where(bad.expand_as(blocks).flatten(-2), torch.nan, v * s)
    return kept, torch.where(bad, 255, k + 127)[..., 0].to(torch.uint8)


def affine(x, gamma, beta):
    return gamma.double() * x + beta.double()


def activation(x, gamma, beta, relu=True, skip=None):
    u = affine(x, gamma, beta)
    a = torch.where(u <= 0, 0.0, u) if relu else u
    return a if skip is None else a + affine(*skip)


def operand(x, gamma, beta, relu=True, skip=None):
    """The activation as it enters the product: the float32 one, rounded to bf16."""
    u = affine(x, gamma, beta).float()
    a = torch.where(u <= 0, 0.0, u) if relu else u
    a = a if skip is None else a + affine(*skip).float()
    return a.bfloat16().double()


def norm_backward(da, x, invstd, gamma, beta, relu=True):
    """da [B, L, C] or [B, C].  -> dz, dgamma, dbeta, and the sums of magnitudes that error bounds need."""
    B, L, C = x.shape
    dy = (da.double() / L)[:, None, :].expand(B, L, C) if da.dim() == 2 else da.double()
    if relu:
        dy = torch.where(side(x, gamma, beta), dy, 0.0)
    n = B * L
    s1, s2 = dy.sum((0, 1)), (dy * x).sum((0, 1))
    gi = gamma.double() * invstd.double()
    dz = gi * (dy - s1 / n - x * (s2 / n))
    return dz, s2, s1, dict(dy=dy, abs1=dy.abs().sum((0, 1)), abs2=(dy * x).abs().sum((0, 1)), gi=gi.abs(), n=n)


def weight_grad(dz, a, ks, zero_pad=False):
    """-> dw [Cout, Cin, ks] and the sum of the products' magnitudes."""
    B, L, cin = a.shape
    at = torch.arange(L)
    d = dz.double().reshape(B * L, -1)
    dw = torch.empty(d.shape[1], cin, ks, dtype=torch.float64)
    mag = torch.empty_like(dw)
    for j in range(ks):
        p = at + j - ks // 2
        rows = a[:, p.clamp(0, L - 1)]
        if zero_pad:
            rows = rows * ((p >= 0) & (p < L)).double()[:, None]
        rows = rows.reshape(B * L, cin)
        dw[:, :, j] = d.t() @ rows
        mag[:, :, j] = d.abs().t() @ rows.abs()
    return dw, mag
