"""64-bit restatement of microscaled 4-bit floating point from its definition (test
infrastructure): e2m1 values in blocks of 16 with an e4m3 scale and one fp32 scale for
the tensor (nvfp4), or of 32 with a power of two (mxfp4, OCP MX v1.0)."""

from __future__ import annotations

import torch

from .block_ref import U32

BLOCK = {"nvfp4": 16, "mxfp4": 32}
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
# the values of e4m3 bytes 0 .. 126 (127 is NaN)
E4M3 = torch.tensor([(b & 7) * 2.0 ** -9 if b < 8 else (1 + (b & 7) / 8) * 2.0 ** ((b >> 3) - 7) for b in range(127)],
                    dtype=torch.float64)


def nearest(v, table):
    """Index of the entry of a rising table nearest to v >= 0; ties to the even index."""
    mid = (table[:-1] + table[1:]) / 2
    up = torch.searchsorted(mid, v.contiguous(), right=False)  # entries whose middle is below v
    tie = (up < mid.numel()) & (v == mid[up.clamp(max=mid.numel() - 1)])
    return torch.where(tie & (up % 2 == 1), up + 1, up)


def over_scale(x, scale):
    """x over the tensor's scale, as the format defines it: fp32 times fp32."""
    x = x.float()
    return x if scale is None else x * (torch.ones((), dtype=torch.float32) / scale.float().cpu())


def block_scales(most, fmt):
    """Bytes of the scales of blocks whose largest magnitudes are ``most`` (64 bits)."""
    fine = torch.isfinite(most)
    m = torch.where(fine, most, 1.0)
    if fmt == "nvfp4":
        return torch.where(fine, nearest((m / 6).clamp(max=448.0), E4M3), 127).to(torch.uint8)
    e = torch.frexp(m)[1] - 1 - 2 + 127
    return torch.where(fine, torch.where(m > 0, e.clamp(min=0), 0), 255).to(torch.uint8)


def scale_values(byte, fmt):
    b = byte.long()
    if fmt == "nvfp4":
        return torch.where(b < 127, E4M3[b.clamp(max=126)], float("nan"))
    return torch.where(b < 255, torch.exp2(b.double() - 127), float("nan"))


def quantize_ref(u, fmt):
    """u [.., K] already over the tensor's scale -> (values without that scale [.., K],
    scale bytes [.., K / block])."""
    b = u.double().cpu().unflatten(-1, (-1, BLOCK[fmt]))
    byte = block_scales(b.abs().amax(-1), fmt)  # (amax keeps a NaN)
    s = scale_values(byte, fmt)[..., None]
    q = torch.where(s > 0, b.abs() / s, 0.0)
    v = GRID[nearest(torch.nan_to_num(q, posinf=1e30), GRID)] * torch.where(torch.isnan(b), 1.0, torch.sign(b))
    return (v * s).flatten(-2), byte


def rows_scales(scales, K, fmt):
    """Granules [granules, rows, 16] -> [rows, K / block]."""
    return scales.cpu().transpose(0, 1).flatten(1)[:, : K // BLOCK[fmt]]


def values_ref(codes, scales, fmt):
    """codes [.., K / 2], scale bytes [.., K / block] -> values [.., K]."""
    c = codes.cpu().long()
    both = torch.stack([c & 15, c >> 4], dim=-1).flatten(-2)
    v = GRID[both & 7] * (1 - 2 * (both >> 3))
    return v * scale_values(scales.cpu(), fmt).repeat_interleave(BLOCK[fmt], dim=-1)


def pack(values, byte, fmt):
    """Values [.., K] of e2m1 times their blocks' scales -> codes [.., K / 2]."""
    s = scale_values(byte, fmt).repeat_interleave(BLOCK[fmt], dim=-1)
    v = torch.where(s > 0, values / s, 0.0)
    code = nearest(v.abs(), GRID) | (torch.signbit(v).long() << 3)
    pair = code.unflatten(-1, (-1, 2))
    return (pair[..., 0] | (pair[..., 1] << 4)).to(torch.uint8)


def product_ref(x, w, x_scale=None, w_scale=None, bias=None, silu_mul=False):
    """(y, bound): x [M, K] and w [N, K] in 64 bits. The bound is on fp32 sums of K terms,
    each off by at most U32 of the magnitudes so far, and a few roundings behind."""
    alpha = (1.0 if x_scale is None else float(x_scale)) * (1.0 if w_scale is None else float(w_scale))
    y, mag = alpha * (x @ w.T), alpha * (x.abs() @ w.abs().T) * ((x.shape[1] + 4) * U32)
    if bias is not None:
        y = y + bias.double()
        mag = mag + U32 * y.abs()
    if not silu_mul:
        return y, mag
    g, u, dg, du = y[:, 0::2], y[:, 1::2], mag[:, 0::2], mag[:, 1::2]
    act = g * g.sigmoid()
    # |silu'| <= 1.1; the exponential and the division, approximate: (6 + 1.173 |g|) 2^-23
    off = (8 + 1.2 * g.abs()) * U32 * (act * u).abs()
    return act * u, 1.1 * dg * (u.abs() + du) + act.abs() * du + off
