"""Float64 forms of the layer and head ops and their gradients, plain torch on
whatever device the inputs are, and the tolerances that their tests share.

Tolerances count roundings. A bf16 rounding is off by at most 2^-8 of the
value, an f32 one by 2^-24. A product of k terms on the matrix cores adds 16
products per instruction and k / 16 such sums one after another: with a factor
of 2 for sums that are cut off instead of rounded, it is within
(k / 16 + 20) 2^-23 of sum |x| |w| (`sum_tol`). A value near the middle of two
bf16 numbers may be rounded to the other one by the kernel; where a product
reads such values, the bound allows eight of them (`flips`) at the largest
factors.
"""
import math

import torch

F64 = torch.float64
BF16_STEP = 2.0 ** -8


def sum_tol(k):
    return (k / 16 + 20) * 2.0 ** -23


def flips(a, b):
    if a.numel() == 0 or b.numel() == 0:
        return 0.0
    return 8 * BF16_STEP * a.abs().max().item() * b.abs().max().item()


def out_tol(ref, dtype):
    return (BF16_STEP if dtype == torch.bfloat16 else 2.0 ** -24) * ref.abs()


def check(got, ref, tol, what):
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    got = got.double()
    assert torch.isfinite(got).all(), what
    over = ((got - ref).abs() - tol).max().item() if ref.numel() else 0.0
    assert over <= 0, (what, over, (got - ref).abs().max().item())


def act(name, z):
    """Value and slope."""
    if name is None:
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp_min(0), (z > 0).to(z.dtype)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu_erf":
        phi = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    u = math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    t = torch.tanh(u)
    du = math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * du


def r16(t):
    return t.to(torch.bfloat16).double()


def turn(v, rotary, sections, c, s, c2=None, s2=None, back=False):
    """The rotation of heads v [N, H, D] by tables c, s [N, columns], or its
    transpose."""
    if not rotary:
        return v
    if back:
        s, s2 = -s, None if s2 is None else -s2
    c, s = c[:, None, :], s[:, None, :]
    d = v.shape[-1]
    if sections == 3:
        a, b = v[..., 0:rotary:2], v[..., 1:rotary:2]
        out = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    elif sections == 1:
        h = rotary // 2
        a, b = v[..., :h], v[..., h:rotary]
        out = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        q, parts = d // 4, []
        for i, (cc, ss) in enumerate(((c, s), (c2[:, None, :], s2[:, None, :]))):
            a, b = v[..., 2 * i * q:(2 * i + 1) * q], v[..., (2 * i + 1) * q:(2 * i + 2) * q]
            parts += [a * cc - b * ss, b * cc + a * ss]
        return torch.cat(parts, -1)
    return torch.cat([out, v[..., rotary:]], -1)


def norm_rope(x, w, eps, rotary, sections, tables):
    """x [N, H, D] f64, w [H, D] or None (no norm)."""
    v = x if w is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    return turn(v, rotary, sections, *tables)


def norm_rope_bwd(dy, x, w, eps, rotary, sections, tables):
    """dx and dn * xhat per (token, head)."""
    dn = turn(dy, rotary, sections, *tables, back=True)
    if w is None:
        return dn, None
    inv = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    hat, wd = x * inv, dn * w
    return inv * (wd - hat * (wd * hat).mean(-1, keepdim=True)), dn * hat
