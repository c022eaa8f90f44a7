"""What a training step of an encoder needs beside ``perf/operators.py``, as
``inl_hip`` offers it, beside its plain forms.

Three operators: the gradients of packed attention, which recompute the
probabilities (``varlen_attention_bwd``); the residual stream's addition with
dropout from a counter and the root-mean-square norm behind it, forward and
backward (``add_rms_norm``, ``add_rms_norm_bwd``); and the gradients of the
pooled embedding (``pool_mean_bwd``, ``pool_last_bwd``). The plain forms are
elementary torch operations in float32, rounded once at the end, on padded
batches; ``exact`` computes the same outputs in float64, text by text.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

_BF16, _F32, _F64 = torch.bfloat16, torch.float32, torch.float64
EPS = 1e-6


def _inl():
    pkg = os.path.join(os.getcwd(), "im-not-llm_amd")
    if pkg not in sys.path:
        sys.path.insert(1, pkg)
    import inl_hip
    return inl_hip


def listed():
    return [
        # Gradients of one short query (0.6B embedder): nothing but latency.
        dict(name="attn_query_bwd", op="attn_bwd", texts=1, longest=23, mix="equal", q_heads=16, k_heads=8, dim=128,
             causal=True, window=-1),
        # A batch of passages of the 0.6B embedder: log-normal lengths.
        dict(name="attn_passages_bwd", op="attn_bwd", texts=64, longest=2048, mix="ragged", q_heads=16, k_heads=8,
             dim=128, causal=True, window=-1),
        # Long documents of the late-interaction tower: the most work here.
        dict(name="attn_long_bwd", op="attn_bwd", texts=4, longest=4096, mix="equal", q_heads=16, k_heads=2, dim=256,
             causal=True, window=-1),
        # EmbeddingGemma's sliding layers: one key head of 256, both directions.
        dict(name="attn_window_bwd", op="attn_bwd", texts=24, longest=2048, mix="spread", q_heads=3, k_heads=1,
             dim=256, causal=False, window=512),
        # The sparse encoder's local band over ragged texts.
        dict(name="attn_local_bwd", op="attn_bwd", texts=48, longest=1021, mix="spread", q_heads=12, k_heads=12,
             dim=64, causal=False, window=64),
        # The vision block: 64 images of 256 patches.
        dict(name="attn_patches_bwd", op="attn_bwd", texts=64, longest=256, mix="equal", q_heads=16, k_heads=16,
             dim=64, causal=False, window=-1),
        # One token's residual addition and norm: latency.
        dict(name="norm_token", op="norm", m=1, n=1024, x="bf16", stream="f32", out="bf16", dropout=0.0),
        # A batch of documents (EmbeddingGemma's width) in an f32 stream, with dropout.
        dict(name="norm_docs", op="norm", m=20011, n=768, x="bf16", stream="f32", out="bf16", dropout=0.1),
        # Its gradients.
        dict(name="norm_docs_bwd", op="norm_bwd", m=20011, n=768, x="bf16", stream="f32", out="bf16", dropout=0.1),
        # The 0.6B embedder's width in a bf16 stream, as large as a batch gets.
        dict(name="norm_stream_bwd", op="norm_bwd", m=65536, n=1024, x="bf16", stream="bf16", out="bf16",
             dropout=0.0),
        # Gradient of mean pooling with its unit length, back to every token.
        dict(name="pool_mean_bwd", op="mean_bwd", texts=96, longest=2048, mix="ragged", n=768, unit=True, x="bf16"),
        # Gradient of last-token pooling: final norm, unit length, zeros elsewhere.
        dict(name="pool_last_bwd", op="last_bwd", texts=64, longest=2048, mix="ragged", n=1024, x="bf16"),
    ]


def draw(rng):
    """One more case of the same ranges."""
    def log_int(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["attn_bwd"] * 5 + ["norm", "norm_bwd", "norm_bwd", "mean_bwd", "last_bwd"])
    mix = rng.choice(["ragged", "spread", "equal"])
    if op == "attn_bwd":
        q_heads, k_heads, dim = rng.choice([(16, 8, 128), (16, 2, 256), (3, 1, 256), (12, 12, 64), (16, 16, 64),
                                            (8, 1, 128), (5, 5, 128), (4, 2, 80), (6, 3, 40)])
        longest = log_int(2, 4096)   # (a text of one token alone has a gradient of nothing but rounding)
        most = max(1, min(256, int(5e8 / (q_heads * longest * longest))))
        return dict(op=op, texts=log_int(1, most), longest=longest, mix=mix, q_heads=q_heads, k_heads=k_heads,
                    dim=dim, causal=rng.random() < 0.5, window=rng.choice([-1, -1, 16, 64, 512]))
    if op in ("norm", "norm_bwd"):
        n = 8 * log_int(8, 512)
        return dict(op=op, m=log_int(1, 65536 * 1024 // max(n, 1024)), n=n, x=rng.choice(["bf16", "bf16", "f32"]),
                    stream=rng.choice(["f32", "bf16"]), out=rng.choice(["bf16", "bf16", "f32"]),
                    dropout=rng.choice([0.0, 0.1, 0.3]))
    n = 8 * log_int(8, 256)
    texts = log_int(1, 96)
    return dict(op=op, texts=texts, longest=log_int(1, 2048), mix=mix, n=n, x=rng.choice(["bf16", "f32"]),
                **(dict(unit=rng.random() < 0.7) if op == "mean_bwd" else {}))


def _lengths(case):
    """The batch's text lengths, the first the longest: part of the case, not of its seed."""
    texts, longest, mix = case["texts"], case["longest"], case["mix"]
    if mix == "equal":
        return [longest] * texts
    g = random.Random(7919 * texts + longest)
    if mix == "spread":
        return [longest] + [g.randint(max(1, longest // 8), longest) for _ in range(texts - 1)]
    # log-normal passages, as the attention benchmark draws them
    return [longest] + [max(1, min(longest, round(g.lognormvariate(math.log(max(1.0, longest / 11.4)), 1.0))))
                        for _ in range(texts - 1)]


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------

def _dt(name):
    return {"bf16": _BF16, "f32": _F32}[name]


def _pads(lengths):
    """Row of every (text, position) of the padded batch, and which are real."""
    lens = torch.tensor(lengths, device="cuda")
    first = torch.cumsum(lens, 0) - lens
    at = torch.arange(max(lengths), device="cuda")
    real = at[None, :] < lens[:, None]
    return torch.where(real, first[:, None] + at[None, :], torch.zeros_like(first)[:, None]), real


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * std

    s, op = dict(case), case["op"]
    if op == "attn_bwd":
        lengths = _lengths(case)
        n, hq, hk, d = sum(lengths), case["q_heads"], case["k_heads"], case["dim"]
        s["cu"] = [0] + list(np.cumsum(lengths).tolist())
        s["scale"] = d ** -0.5
        # q, k and v as slices of one projection's rows; scores of deviation 2
        rows = randn(n, hq + 2 * hk, d)
        rows[:, :hq] *= 2.0
        rows = rows.to(_BF16)
        s["q"], s["k"], s["v"] = rows[:, :hq], rows[:, hq:hq + hk], rows[:, hq + hk:]
        s["rows"], s["real"] = _pads(lengths)
        s["o"] = _attend(s).to(_BF16)          # what the forward left
        s["do"] = randn(n, hq, d, std=0.1).to(_BF16)
    elif op in ("norm", "norm_bwd"):
        m, n = case["m"], case["n"]
        s["w"] = (1 + 0.1 * randn(n)).to(_BF16)
        s["rng"] = torch.randint(0, 2 ** 31, (2,), generator=g, device="cuda", dtype=torch.int64)
        s["tag"] = 5
        if op == "norm":
            s["x"] = randn(m, n).to(_dt(case["x"]))
            s["r"] = randn(m, n, std=2.0).to(_dt(case["stream"]))
        else:
            s["h"] = randn(m, n, std=2.0).to(_dt(case["stream"]))
            s["dy"] = randn(m, n, std=0.1).to(_dt(case["out"]))
            s["dh"] = randn(m, n, std=0.1).to(_dt(case["stream"]))
    else:
        lengths = _lengths(case)
        rows, n = sum(lengths), case["n"]
        cu = torch.tensor([0] + list(np.cumsum(lengths).tolist()), dtype=torch.int32, device="cuda")
        s["cu"], s["total"] = cu, rows
        s["dp"] = randn(case["texts"], n, std=0.1)
        if op == "mean_bwd":
            # the means that the forward left (before their unit length)
            s["mean"] = randn(case["texts"], n, std=0.3) if case["unit"] else None
        else:
            s["x"] = randn(rows, n, std=2.0).to(_dt(case["x"]))
            s["w"] = (1 + 0.1 * randn(n)).to(_dt(case["x"]))
    return s


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------

def run(s):
    return _own(s) if own else _PLAIN[s["op"]](s)


def _own(s):
    inl, op = _inl(), s["op"]
    if op == "attn_bwd":
        return inl.varlen_attention_bwd(s["do"], s["q"], s["k"], s["v"], s["o"], s["cu"], causal=s["causal"],
                                        window=s["window"], scale=s["scale"])
    if op == "norm":
        return inl.add_rms_norm(s["x"], s["w"], residual=s["r"], eps=EPS, dropout=s["dropout"], rng=s["rng"],
                                tag=s["tag"], out_dtype=_dt(s["out"]))
    if op == "norm_bwd":
        return inl.add_rms_norm_bwd(s["dy"], s["h"], s["w"], dh=s["dh"], eps=EPS, dropout=s["dropout"], rng=s["rng"],
                                    tag=s["tag"], dx_dtype=_dt(s["x"]))
    if op == "mean_bwd":
        return inl.pool_mean_bwd(s["dp"], s["cu"], s["total"], mean=s["mean"], dtype=_dt(s["x"]))
    return inl.pool_last_bwd(s["dp"], s["x"], s["cu"], s["w"], eps=EPS)


# ---- plain forms: float32, rounded once at the end ----

def _padded(s, t):
    """[texts, heads, longest, dim] of packed rows, zeros where there is no token."""
    return (t[s["rows"]].float() * s["real"][:, :, None, None]).permute(0, 2, 1, 3)


def _packed(s, t):
    return t.permute(0, 2, 1, 3)[s["real"]]


def _probabilities(s):
    """Padded q and k, and the probabilities [texts, q_heads, longest, longest]."""
    group = s["q_heads"] // s["k_heads"]
    q, k = _padded(s, s["q"]), _padded(s, s["k"]).repeat_interleave(group, 1)
    z = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    at = torch.arange(s["longest"], device="cuda")
    apart = at[None, :] - at[:, None]
    seen = torch.ones_like(apart, dtype=torch.bool)
    if s["causal"]:
        seen = seen & (apart <= 0)
    if s["window"] >= 0:
        seen = seen & (apart.abs() <= s["window"])
    # (a row without a token sees itself)
    seen = (seen & s["real"][:, None, :]) | (apart == 0)
    z = torch.where(seen[:, None], z, torch.full_like(z[:1, :1, :1, :1], -math.inf))
    z = torch.exp(z - z.max(-1, keepdim=True).values)
    return q, k, z / z.sum(-1, keepdim=True)


def _attend(s):
    _, _, p = _probabilities(s)
    v = _padded(s, s["v"]).repeat_interleave(s["q_heads"] // s["k_heads"], 1)
    return _packed(s, torch.matmul(p, v))


def _attn_bwd(s):
    group = s["q_heads"] // s["k_heads"]
    q, k, p = _probabilities(s)
    do, o = _padded(s, s["do"]), _padded(s, s["o"])
    v = _padded(s, s["v"]).repeat_interleave(group, 1)
    dv = torch.matmul(p.transpose(-1, -2), do)
    ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    dq = torch.matmul(ds, k) * s["scale"]
    dk = torch.matmul(ds.transpose(-1, -2), q) * s["scale"]
    b, _, t, d = q.shape
    dk, dv = (x.view(b, s["k_heads"], group, t, d).sum(2) for x in (dk, dv))
    return _packed(s, dq).to(_BF16), _packed(s, dk).to(_BF16), _packed(s, dv).to(_BF16)


_LOW16, _LOW32 = 0xFFFF, 0xFFFFFFFF


def _mul_hi_lo(a, b):
    """High and low words of the product of a 32-bit number and 32-bit values in int64."""
    low, high = b * (a & _LOW16), b * (a >> 16)
    return (high + (low >> 16)) >> 16, ((high << 16) + low) & _LOW32


def _kept(s, m, n):
    """The dropout's mask, and what kept values are scaled by: 16 bits an element from the
    Philox 4x32-10 generator, a draw per 8 elements of the row-major matrix."""
    at = torch.arange(m * n // 8, device="cuda", dtype=torch.int64)
    seed, step = s["rng"][0], s["rng"][1]
    c0, c1 = at & _LOW32, at >> 32
    c2, c3 = torch.full_like(at, s["tag"]), (step & _LOW32).expand_as(at)
    k0, k1 = seed & _LOW32, (seed >> 32) & _LOW32
    for _ in range(10):
        h0, l0 = _mul_hi_lo(0xD2511F53, c0)
        h1, l1 = _mul_hi_lo(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & _LOW32, (k1 + 0xBB67AE85) & _LOW32
    words = torch.stack([c0, c1, c2, c3], 1)
    bits = torch.stack([words & _LOW16, words >> 16], 2).view(m, n)
    drop = round(s["dropout"] * 65536)
    return bits >= drop, 65536 / (65536 - drop)


def _dropped(s, x):
    if not s["dropout"]:
        return x
    keep, scale = _kept(s, *x.shape)
    return torch.where(keep, x * scale, torch.zeros_like(x))


def _norm(s):
    h = s["r"].float() + _dropped(s, s["x"].float())
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * s["w"].float()
    return y.to(_dt(s["out"])), h.to(s["r"].dtype)


def _norm_bwd(s):
    h, dy = s["h"].float(), s["dy"].float()
    inv = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
    hat, dn = h * inv, dy * s["w"].float()
    g = inv * (dn - hat * (dn * hat).mean(-1, keepdim=True)) + s["dh"].float()
    return _dropped(s, g).to(_dt(s["x"])), g.to(s["h"].dtype), (dy * hat).sum(0)


def _text_of(s):
    at = torch.arange(s["total"], device="cuda", dtype=torch.int32)
    return (at[:, None] >= s["cu"][None, 1:]).sum(1)


def _mean_bwd(s):
    d = s["dp"]
    if s["unit"]:
        size = torch.sqrt((s["mean"] * s["mean"]).sum(1, keepdim=True) + 1e-12)
        y = s["mean"] / size
        d = (d - y * (d * y).sum(1, keepdim=True)) / size
    d = d / (s["cu"][1:] - s["cu"][:-1])[:, None].float()
    return d[_text_of(s)].to(_dt(s["x"]))


def _last_bwd(s):
    last = s["cu"][1:].long() - 1
    x, w = s["x"][last].float(), s["w"].float()
    inv = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    hat = x * inv
    z = hat * w
    size = torch.sqrt((z * z).sum(1, keepdim=True) + 1e-12)
    y = z / size
    dz = (s["dp"] - y * (s["dp"] * y).sum(1, keepdim=True)) / size
    dn = dz * w
    dx = inv * (dn - hat * (dn * hat).mean(1, keepdim=True))
    out = torch.zeros_like(s["x"])
    out[last] = dx.to(out.dtype)
    return out, (dz * hat).sum(0)


_PLAIN = {"attn_bwd": _attn_bwd, "norm": _norm, "norm_bwd": _norm_bwd, "mean_bwd": _mean_bwd, "last_bwd": _last_bwd}


# --------------------------------------------------------------------------
# What a pass cannot do without
# --------------------------------------------------------------------------

def _pairs(t, causal, window):
    """Visible (query, key) pairs of a text of t tokens."""
    w = t if window < 0 else min(window, t - 1)
    back = t * w - w * (w + 1) // 2 if window >= 0 else t * (t - 1) // 2
    return t + back * (1 if causal else 2)


def work(case):
    op = case["op"]
    size = {"bf16": 2, "f32": 4}
    if op == "attn_bwd":
        lengths = _lengths(case)
        n, hq, hk, d = sum(lengths), case["q_heads"], case["k_heads"], case["dim"]
        pairs = sum(_pairs(t, case["causal"], case["window"]) for t in lengths)
        # q, out, dout; k, v; dq, dk, dv: five products over every visible pair
        return {"bytes": 2 * n * d * (4 * hq + 4 * hk), "flops": 10 * hq * d * pairs}
    if op == "norm":
        m, n = case["m"], case["n"]
        return {"bytes": m * n * (size[case["x"]] + 2 * size[case["stream"]] + size[case["out"]]) + 2 * n,
                "flops": 6 * m * n}
    if op == "norm_bwd":
        # h, dy, dh in; the stream's gradient out, and x's where it is another one
        m, n = case["m"], case["n"]
        same = not case["dropout"] and case["x"] == case["stream"]
        return {"bytes": m * n * (3 * size[case["stream"]] + size[case["out"]] + (0 if same else size[case["x"]]))
                + 6 * n, "flops": 12 * m * n}
    rows, n, texts = sum(_lengths(case)), case["n"], case["texts"]
    if op == "mean_bwd":
        return {"bytes": rows * n * size[case["x"]] + texts * n * (8 if case["unit"] else 4), "flops": rows * n}
    return {"bytes": rows * n * size[case["x"]] + texts * n * (4 + size[case["x"]]) + n * (4 + size[case["x"]]),
            "flops": 12 * texts * n}


# --------------------------------------------------------------------------
# The definitions in float64
# --------------------------------------------------------------------------

def _exact_attn(case, s):
    hq, hk, group = case["q_heads"], case["k_heads"], case["q_heads"] // case["k_heads"]
    dq, dk, dv = (torch.empty(x.shape, dtype=_F64, device="cuda") for x in (s["q"], s["k"], s["v"]))
    for a, b in zip(s["cu"][:-1], s["cu"][1:]):
        i = torch.arange(b - a, device="cuda")
        hidden = torch.zeros(b - a, b - a, dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden |= i[:, None] < i
        if case["window"] >= 0:
            hidden |= (i[:, None] - i).abs() > case["window"]
        for h in range(hk):
            heads = slice(h * group, (h + 1) * group)
            q, o, do = (s[x][a:b, heads].double().transpose(0, 1) for x in ("q", "o", "do"))
            k, v = s["k"][a:b, h].double(), s["v"][a:b, h].double()
            z = torch.matmul(q, k.t()).mul_(s["scale"]).masked_fill_(hidden, -math.inf)
            p = torch.softmax(z, dim=-1)
            g = p * (torch.matmul(do, v.t()) - (do * o).sum(dim=-1, keepdim=True))
            dq[a:b, heads] = torch.matmul(g, k).mul_(s["scale"]).transpose(0, 1)
            rows = group * (b - a)
            dk[a:b, h] = torch.matmul(g.reshape(rows, b - a).t(), q.reshape(rows, -1)) * s["scale"]
            dv[a:b, h] = torch.matmul(p.reshape(rows, b - a).t(), do.reshape(rows, -1))
    return dq, dk, dv


def _exact_factor(case, s):
    """What dropout multiplies each element by: the same draws, in numpy's unsigned words."""
    m, n = case["m"], case["n"]
    if not case["dropout"]:
        return torch.ones((), dtype=_F64, device="cuda")
    seed, step = (int(x) for x in s["rng"].tolist())
    word = np.uint64(0xFFFFFFFF)
    c = np.zeros((4, m * n // 8), dtype=np.uint64)
    at = np.arange(m * n // 8, dtype=np.uint64)
    c[0], c[1], c[2], c[3] = at & word, at >> np.uint64(32), s["tag"], step & 0xFFFFFFFF
    key = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = np.stack([(q >> np.uint64(32)) ^ c[1] ^ np.uint64(key[0]), q & word,
                      (p >> np.uint64(32)) ^ c[3] ^ np.uint64(key[1]), p & word])
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    bits = np.ascontiguousarray(c.T).astype("<u4").view("<u2").reshape(m, n)
    drop = round(case["dropout"] * 65536)
    return torch.from_numpy(np.where(bits >= drop, 65536 / (65536 - drop), 0.0)).to("cuda")


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "attn_bwd":
        return _exact_attn(case, s)
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if op == "norm":
        h = d["r"] + d["x"] * _exact_factor(case, s)
        return torch.nn.functional.normalize(h, dim=1, eps=0.0) * _rms_scale(h) * d["w"], h
    if op == "norm_bwd":
        rms = torch.sqrt(d["h"].square().mean(dim=1, keepdim=True) + EPS)
        e = d["dy"] * d["w"]
        g = e / rms - d["h"] * (e * d["h"]).mean(dim=1, keepdim=True) / rms ** 3 + d["dh"]
        return g * _exact_factor(case, s), g, (d["dy"] * d["h"] / rms).sum(dim=0)
    lens = (s["cu"][1:] - s["cu"][:-1]).long()
    if op == "mean_bwd":
        g = d["dp"]
        if case["unit"]:
            sq = d["mean"].square().sum(dim=1, keepdim=True) + 1e-12
            g = g * sq.rsqrt() - d["mean"] * (g * d["mean"]).sum(dim=1, keepdim=True) * sq ** -1.5
        return torch.repeat_interleave(g / lens.unsqueeze(1), lens, dim=0)
    end = s["cu"][1:].long() - 1
    x = d["x"][end].requires_grad_()
    w = d["w"].requires_grad_()
    z = x / torch.sqrt(x.square().mean(dim=1, keepdim=True) + EPS) * w
    y = z / torch.sqrt(z.square().sum(dim=1, keepdim=True) + 1e-12)
    dx, dw = torch.autograd.grad(y, (x, w), d["dp"])
    return torch.zeros(s["x"].shape, dtype=_F64, device="cuda").index_copy_(0, end, dx), dw


def _rms_scale(h):
    """|h| / rms(h): what a unit vector is multiplied by."""
    sq = h.square().sum(dim=1, keepdim=True)
    return torch.sqrt(sq / (sq / h.shape[1] + EPS))
