"""Float64 gradients of packed attention, text by text, and how far a kernel may be
off that rounds P and dS to bf16 and sums in f32 (the steps and sums of train_ref.py).

With u = 2^-8 a bf16 rounding and t(k) = sum_tol(k) the bound of a sum of k products:
  s = scale q.k is off by e_s = scale t(d) |q|.|k| + 2^-21 |s|; the log-sum-exp of a row by the
  row's largest e_s and the rounding of n additions, 2^-24 n, and the exponent, a number of size
  |s| + |lse|, by 2^-22 of that; so P by P e_p with e_p the sum of these. dP and delta
  are off by t(d) |dO|.|v| and t(d) |dO|.|o|. Then
  dv: sum P (u + e_p) |dO|, its f32 sum t(n) sum P |dO|, and the last rounding;
  dS: e_ds = P |dP - delta| (u + e_p) + P (e_dP + e_delta), rounded to bf16 in the same u;
  dq: scale sum e_ds |k| + scale t(n) sum |dS| |k|, and the last rounding; dk likewise.
Products of two of these errors are below the slack of the bounds' sums (factor 1.01).
"""
import torch

import train_ref as R

U = R.BF16_STEP


def visible(t, causal, window, device):
    i = torch.arange(t, device=device)
    apart = i[None, :] - i[:, None]
    seen = torch.ones(t, t, dtype=torch.bool, device=device)
    if causal:
        seen &= apart <= 0
    if window >= 0:
        seen &= apart.abs() <= window
    return seen


def forward(q, k, v, starts, lengths, causal, window, scale):
    """out [N, Hq, D] in f64 (zeros outside every text)."""
    o = torch.zeros(q.shape, dtype=R.F64, device=q.device)
    g = q.shape[1] // k.shape[1]
    for a, t in zip(starts, lengths):
        qh, kh, vh = (x[a:a + t].double().transpose(0, 1) for x in (q, k, v))
        kh, vh = kh.repeat_interleave(g, 0), vh.repeat_interleave(g, 0)
        s = (qh @ kh.transpose(1, 2)) * scale
        s = s.masked_fill(~visible(t, causal, window, q.device), float("-inf"))
        o[a:a + t] = (torch.softmax(s, -1) @ vh).transpose(0, 1)
    return o


def backward(dout, q, k, v, out, starts, lengths, causal, window, scale):
    """((dq, its bound), (dk, ..), (dv, ..)) without the last rounding's share."""
    res = [[torch.zeros(x.shape, dtype=R.F64, device=q.device) for _ in range(2)] for x in (q, k, v)]
    g, hd = q.shape[1] // k.shape[1], q.shape[2]
    td = R.sum_tol(hd)
    for a, t in zip(starts, lengths):
        if t == 0:
            continue
        tn = R.sum_tol(t * g)
        qh, oh, gh = (x[a:a + t].double().transpose(0, 1) for x in (q, out, dout))
        kh, vh = (x[a:a + t].double().transpose(0, 1).repeat_interleave(g, 0) for x in (k, v))
        T = lambda x: x.transpose(1, 2)
        seen = visible(t, causal, window, q.device)
        s = (qh @ T(kh)) * scale
        e_s = (scale * td * (qh.abs() @ T(kh.abs())) + 2.0 ** -21 * s.abs()) * seen
        s = s.masked_fill(~seen, float("-inf"))
        lse = torch.logsumexp(s, -1, keepdim=True)
        p = torch.exp(s - lse)
        size = s.masked_fill(~seen, 0).abs() + lse.abs()
        e_p = e_s + e_s.max(-1, keepdim=True).values + 2.0 ** -24 * t + 2.0 ** -22 * size
        dp, delta = gh @ T(vh), (gh * oh).sum(-1, keepdim=True)
        e_dp = td * (gh.abs() @ T(vh.abs())) + td * (gh * oh).abs().sum(-1, keepdim=True)
        ds = p * (dp - delta)
        e_ds = (ds.abs() * (U + e_p) + p * e_dp) * 1.01
        pairs = ((scale * (ds @ kh), scale * (e_ds @ kh.abs() + tn * (ds.abs() @ kh.abs()))),
                 (scale * (T(ds) @ qh), scale * (T(e_ds) @ qh.abs() + tn * (T(ds.abs()) @ qh.abs()))),
                 (T(p) @ gh, 1.01 * (T(p * (U + e_p)) @ gh.abs()) + tn * (T(p) @ gh.abs())))
        for i, (x, e) in enumerate(pairs):
            for into, y in zip(res[i], (x, e)):
                if i:   # key heads: the sum over their query heads
                    y = y.view(-1, g, t, hd).sum(1)
                into[a:a + t] = y.transpose(0, 1)
    return res


def check(got, ref, what):
    for name, x, (y, e) in zip(("dq", "dk", "dv"), got, ref):
        if x is not None:
            R.check(x, y, e + R.out_tol(y, x.dtype) + 1e-30, f"{what} {name}")
