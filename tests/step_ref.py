"""Float64 forms of the residual norm and the pooling gradients, and the generator of the dropout,
in numpy's unsigned words. Tolerances count f32 roundings of 2^-24 (train_ref.py)."""
import numpy as np
import torch

import train_ref as R


def philox(c, key):
    """Philox 4x32-10: c [4, N] and key (two words), 32-bit words in uint64."""
    word = np.uint64(0xFFFFFFFF)
    k0, k1 = key
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = np.stack([(q >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), q & word,
                      (p >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p & word])
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def factor(m, n, dropout, seed, step, tag, device):
    """What dropout multiplies each element by [m, n], f64."""
    drop = round(dropout * 65536)
    if not drop:
        return torch.ones(m, n, dtype=R.F64, device=device)
    at = np.arange(m * n // 8, dtype=np.uint64)
    c = np.stack([at & np.uint64(0xFFFFFFFF), at >> np.uint64(32), np.full_like(at, tag & 0xFFFFFFFF),
                  np.full_like(at, step & 0xFFFFFFFF)])
    words = philox(c, (seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF)).T.astype("<u4")
    bits = np.ascontiguousarray(words).view("<u2").reshape(m, n)
    return torch.from_numpy(np.where(bits >= drop, 65536 / (65536 - drop), 0.0)).to(device)


def norm_err(n):
    """Relative error of 1 / rms: the squares' sum (8 values per lane and chunk one after another, at
    most 8 chunks, then a tree of 8 levels), and the mean, root and quotient."""
    return (8 * min(8, -(-n // 512)) + 24) * 2.0 ** -24


def add_norm(x, w, r, f, eps):
    h = x.double() * f + (0 if r is None else r.double())
    rms = torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    return h / rms * (1 if w is None else w.double()), h


def check_add_norm(y, h, x, w, r, f, eps, what):
    ry, rh = add_norm(x, w, r, f, eps)
    e_h = 2.0 ** -23 * ((x.double() * f).abs() + (0 if r is None else r.double().abs()))
    R.check(h, rh, e_h + R.out_tol(rh, h.dtype), what + " h")
    rms = torch.sqrt((rh * rh).mean(1, keepdim=True) + eps)
    wd = 1 if w is None else w.double().abs()
    e = norm_err(x.shape[1]) * ry.abs() + e_h / rms * wd + e_h.amax(1, keepdim=True) / rms * ry.abs()
    R.check(y, ry, e + R.out_tol(ry, y.dtype) + 1e-30, what + " y")


def check_add_norm_bwd(got, dy, h, w, dh, f, eps, what):
    dx, dres, dw = got
    m, n = h.shape
    hd, d = h.double(), dy.double()
    rms = torch.sqrt((hd * hd).mean(1, keepdim=True) + eps)
    hat, dn = hd / rms, d * (1 if w is None else w.double())
    mean, mean_abs = (dn * hat).mean(1, keepdim=True), (dn * hat).abs().mean(1, keepdim=True)
    past = 0 if dh is None else dh.double()
    g = (dn - hat * mean) / rms + past
    # 1 / rms enters up to three times, the mean's sum once
    e = 4 * norm_err(n) * (dn.abs() + hat.abs() * mean_abs) / rms + 2.0 ** -22 * (0 if dh is None else past.abs())
    if dres is not None:
        R.check(dres, g, e + R.out_tol(g, dres.dtype) + 1e-30, what + " dresidual")
    if dx is not None:
        R.check(dx, g * f, e * f * 1.01 + 2.0 ** -23 * (g * f).abs() + R.out_tol(g * f, dx.dtype) + 1e-30, what + " dx")
    if dw is not None:
        terms = d * hat
        R.check(dw, terms.sum(0), (norm_err(n) + (m + 64) * 2.0 ** -24) * terms.abs().sum(0) + 1e-30, what + " dweight")


def text_of(cu, rows):
    """Text of every row, -1 for none."""
    out = torch.full((rows,), -1, dtype=torch.long)
    for b in range(len(cu) - 1):
        out[cu[b]:cu[b + 1]] = b
    return out


def mean_bwd(dp, cu, rows, mean):
    """The gradient [rows, dim] in f64 and what its bound is relative to."""
    d = dp.double()
    size = d.abs()
    if mean is not None:
        s = torch.sqrt((mean.double() ** 2).sum(1, keepdim=True) + 1e-12)
        y = mean.double() / s
        d, size = (d - y * (d * y).sum(1, keepdim=True)) / s, (size + y.abs() * (d * y).abs().sum(1, keepdim=True)) / s
    lens = torch.tensor([max(1, b - a) for a, b in zip(cu[:-1], cu[1:])], device=dp.device)[:, None]
    pad = lambda t: torch.cat([t / lens, torch.zeros(1, t.shape[1], dtype=t.dtype, device=t.device)])
    at = text_of(cu, rows).to(dp.device)
    return pad(d)[at], pad(size)[at]


def last_bwd(dp, x, cu, w, eps):
    """dhidden and dweight in f64, and what their bounds are relative to."""
    dim = x.shape[1]
    out, size = (torch.zeros(x.shape, dtype=R.F64, device=x.device) for _ in range(2))
    dw, dw_size = (torch.zeros(dim, dtype=R.F64, device=x.device) for _ in range(2))
    wd = torch.ones(dim, dtype=R.F64, device=x.device) if w is None else w.double()
    for b in range(len(cu) - 1):
        if cu[b + 1] <= cu[b]:
            continue
        v, d = x[cu[b + 1] - 1].double(), dp[b].double()
        rms = torch.sqrt((v * v).mean() + eps)
        hat = v / rms
        z = hat * wd
        s = torch.sqrt((z * z).sum() + 1e-12)
        y = z / s
        dz = (d - y * (d @ y)) / s
        e = (d.abs() + y.abs() * (d * y).abs().sum()) / s
        dn = dz * wd
        out[cu[b + 1] - 1] = (dn - hat * (dn @ hat) / dim) / rms
        size[cu[b + 1] - 1] = (e * wd.abs()) / rms
        dw += dz * hat
        dw_size += e * hat.abs()
    return out, size, dw, dw_size
