"""The trainable operators of an encoder layer and its head, as ``inl_hip``
offers them, beside their plain forms.

Four operators, each forward and backward: a linear layer with bias,
activation and residual in its epilogue (``dense``), the gated feed-forward
block (``gated_ffn``), softmax cross entropy over a vocabulary or over a
batch's documents without its logits (``softmax_xent``), and the per-head
norms of q and k with the position rotation (``norm_rope_qk``). The plain
forms are elementary torch operations in float32, rounded once at the end;
``exact`` computes the same outputs in float64.
"""
import math
import os
import sys

import torch

own = False

_BF16, _F32, _F64 = torch.bfloat16, torch.float32, torch.float64
IGNORE = -100


def _inl():
    pkg = os.path.join(os.getcwd(), "im-not-llm_amd")
    if pkg not in sys.path:
        sys.path.insert(1, pkg)
    import inl_hip
    return inl_hip


def listed():
    return [
        # One token through a projection with bias (4096 outputs: the fused
        # q/k/v rows of the 0.6B embedder): nothing but latency and weights.
        dict(name="dense_token", op="dense", m=1, n=4096, k=1024, act="none", bias=True, residual="none", out="bf16"),
        # The masked-language head of the sparse encoder over a ragged batch:
        # dense, bias and exact GELU.
        dict(name="dense_head", op="dense", m=20011, n=768, k=768, act="gelu_erf", bias=True, residual="none",
             out="bf16"),
        # Its gradients: input, weight and bias.
        dict(name="dense_head_bwd", op="dense_bwd", m=20011, n=768, k=768, act="gelu_erf", bias=True),
        # A projection back into an f32 residual stream.
        dict(name="dense_stream", op="dense", m=8192, n=1024, k=2048, act="none", bias=True, residual="f32",
             out="f32"),
        # One token through the feed-forward block (0.6B embedder).
        dict(name="ffn_token", op="ffn", m=1, hidden=1024, inner=2816, act="silu", residual=True, save=False),
        # EmbeddingGemma's block over a batch of documents, ragged row count.
        dict(name="ffn_docs", op="ffn", m=20011, hidden=768, inner=1152, act="gelu_tanh", residual=True, save=False),
        # A training step's block: all three weight gradients and dx.
        dict(name="ffn_train_bwd", op="ffn_bwd", m=16384, hidden=1024, inner=4096, act="silu"),
        # Contrastive loss: queries against every document of the batch.
        dict(name="xent_contrast", op="xent", m=1024, vocab=8192, hidden=1024, scale=50.0, bias=False, ignored=0.0),
        # Masked-language loss of the sparse encoder: its vocabulary, its
        # decoder bias, most positions ignored ones taken out, a few left in.
        dict(name="xent_vocab", op="xent", m=4099, vocab=50002, hidden=768, scale=1.0, bias=True, ignored=0.1),
        # Gradient over the largest vocabulary here (odd), the weights' too.
        dict(name="xent_vocab_bwd", op="xent_bwd", m=2048, vocab=151669, hidden=1024, scale=1.0, bias=False,
             ignored=0.1),
        # q and k of one query in f32, adjacent pairs rotated, half of the head.
        dict(name="rope_query", op="rope", m=23, q_heads=16, k_heads=8, dim=128, rotary=64, pairs="adjacent",
             dtype="f32", norm=True, longest=64),
        # The prologue's gradients over a batch of passages.
        dict(name="rope_passages_bwd", op="rope_bwd", m=32003, q_heads=16, k_heads=8, dim=128, rotary=128,
             pairs="half", dtype="bf16", norm=True, longest=2048),
    ]


def draw(rng):
    """One more case of the same ranges."""
    def log_int(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    def log8(lo, hi):
        return 8 * log_int(lo // 8, hi // 8)

    act = rng.choice(["none", "relu", "silu", "gelu_tanh", "gelu_erf"])
    gate = rng.choice(["silu", "gelu_tanh", "gelu_erf"])
    op = rng.choice(["dense", "dense", "dense_bwd", "ffn", "ffn", "ffn_bwd", "xent", "xent", "xent_bwd", "rope",
                     "rope_bwd"])
    if op == "dense":
        out = rng.choice(["bf16", "bf16", "f32"])
        return dict(op=op, m=log_int(1, 32768), n=log8(64, 4096), k=log8(64, 4096), act=act,
                    bias=rng.random() < 0.7, residual=rng.choice(["none", "bf16", "f32"]), out=out)
    if op == "dense_bwd":
        return dict(op=op, m=log_int(1, 32768), n=log8(64, 4096), k=log8(64, 4096), act=act,
                    bias=rng.random() < 0.7)
    if op == "ffn":
        return dict(op=op, m=log_int(1, 32768), hidden=log8(256, 2048), inner=log8(256, 4096), act=gate,
                    residual=rng.random() < 0.7, save=rng.random() < 0.5)
    if op == "ffn_bwd":
        return dict(op=op, m=log_int(1, 16384), hidden=log8(256, 1024), inner=log8(256, 4096), act=gate)
    if op in ("xent", "xent_bwd"):
        return dict(op=op, m=log_int(1, 4096 if op == "xent" else 2048), vocab=log_int(16, 151669),
                    hidden=log8(128, 1024), scale=rng.choice([1.0, 20.0, 50.0]), bias=rng.random() < 0.5,
                    ignored=rng.choice([0.0, 0.1, 0.5]))
    dim = rng.choice([64, 128, 256])
    return dict(op=op, m=log_int(1, 65536 * 128 // (2 * dim)), q_heads=rng.choice([3, 8, 12, 16]),
                k_heads=rng.choice([1, 2, 8]), dim=dim, rotary=rng.choice([dim, dim // 2]),
                pairs=rng.choice(["half", "adjacent"]), dtype=rng.choice(["bf16", "bf16", "f32"]),
                norm=rng.random() < 0.8, longest=rng.choice([512, 2048, 32768]))


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------

def _dt(name):
    return {"bf16": _BF16, "f32": _F32}[name]


def _tables(dim, longest):
    inv = 1e6 ** (-torch.arange(0, dim, 2, device="cuda", dtype=_F64) / dim)
    angle = torch.arange(longest, device="cuda", dtype=_F64)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * std

    op, m = case["op"], case["m"]
    s = dict(case)
    if op in ("dense", "dense_bwd"):
        n, k = case["n"], case["k"]
        s["x"] = randn(m, k).to(_BF16)
        s["w"] = randn(n, k, std=k ** -0.5).to(_BF16)
        s["b"] = randn(n, std=0.5) if case["bias"] else None
        if op == "dense":
            s["r"] = randn(m, n).to(_dt(case["residual"])) if case["residual"] != "none" else None
        else:
            z = s["x"].float() @ s["w"].float().T
            # what the forward left: the activation's input
            s["z"] = (z if s["b"] is None else z + s["b"]).to(_BF16) if case["act"] != "none" else None
            s["dy"] = randn(m, n, std=0.1).to(_BF16)
    elif op in ("ffn", "ffn_bwd"):
        hidden, inner = case["hidden"], case["inner"]
        s["x"] = randn(m, hidden).to(_BF16)
        s["wgu"] = randn(2 * inner, hidden, std=hidden ** -0.5).to(_BF16)
        s["wd"] = randn(hidden, inner, std=inner ** -0.5).to(_BF16)
        if op == "ffn":
            s["r"] = randn(m, hidden).to(_BF16) if case["residual"] else None
        else:
            gu = s["x"].float() @ s["wgu"].float().T
            s["h"] = (_act(case["act"], gu[:, :inner]) * gu[:, inner:]).to(_BF16)
            s["gu"] = gu.to(_BF16)
            s["dy"] = randn(m, hidden, std=0.1).to(_BF16)
    elif op in ("xent", "xent_bwd"):
        vocab, hidden = case["vocab"], case["hidden"]
        std = 1.0 if case["scale"] == 1.0 else hidden ** -0.5   # unit vectors under a temperature
        s["x"] = randn(m, hidden, std=std).to(_BF16)
        s["w"] = randn(vocab, hidden, std=hidden ** -0.5).to(_BF16)
        s["b"] = randn(vocab, std=0.5) if case["bias"] else None
        t = torch.randint(0, vocab, (m,), generator=g, device="cuda", dtype=torch.int32)
        drop = torch.rand(m, generator=g, device="cuda") < case["ignored"]
        s["t"] = torch.where(drop, torch.full_like(t, IGNORE), t)
        if op == "xent_bwd":
            s["lse"] = torch.logsumexp(_scores(s), 1)
            s["dl"] = torch.full((m,), 1.0 / m, device="cuda")
    else:
        heads, dim = case["q_heads"] + case["k_heads"], case["dim"]
        dt = _dt(case["dtype"])
        # the q and k heads of fused q/k/v rows, as a projection leaves them
        s["x"] = randn(m, heads + case["k_heads"], dim).to(dt)[:, :heads]
        s["wq"] = (1 + 0.1 * randn(dim)).to(dt)
        s["wk"] = (1 + 0.1 * randn(dim)).to(dt)
        s["cos"], s["sin"] = _tables(case["rotary"], case["longest"])
        s["pos"] = (torch.arange(m, device="cuda") % case["longest"]).to(torch.int32)
        if op == "rope_bwd":
            s["dy"] = randn(m, heads, dim).to(dt)
    return s


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------

def run(s):
    return _own(s) if own else _PLAIN[s["op"]](s)


def _own(s):
    inl, op = _inl(), s["op"]
    act = None if s.get("act") == "none" else s.get("act")
    if op == "dense":
        return inl.dense(s["x"], s["w"], s["b"], act=act, residual=s["r"], out_dtype=_dt(s["out"]))
    if op == "dense_bwd":
        return inl.dense_bwd(s["dy"], s["x"], s["w"], pre=s["z"], act=act, bias_grad=s["bias"])
    if op == "ffn":
        return inl.gated_ffn(s["x"], s["wgu"], s["wd"], act=act, residual=s["r"], save=s["save"])
    if op == "ffn_bwd":
        return inl.gated_ffn_bwd(s["dy"], s["x"], s["wgu"], s["wd"], s["gu"], s["h"], act=act)
    if op == "xent":
        return inl.softmax_xent(s["x"], s["w"], s["t"], bias=s["b"], scale=s["scale"], ignore_index=IGNORE)
    if op == "xent_bwd":
        return inl.softmax_xent_bwd(s["dl"], s["lse"], s["x"], s["w"], s["t"], bias=s["b"], scale=s["scale"],
                                    ignore_index=IGNORE)
    rope = dict(q_weight=s["wq"] if s["norm"] else None, k_weight=s["wk"] if s["norm"] else None, norm=s["norm"],
                eps=1e-6, rotary_dim=s["rotary"],
                sections=inl.ROPE_INTERLEAVED if s["pairs"] == "adjacent" else inl.ROPE_HALF)
    if op == "rope":
        return inl.norm_rope_qk(s["x"], s["q_heads"], s["pos"], s["cos"], s["sin"], **rope)
    return inl.norm_rope_qk_bwd(s["dy"], s["x"], s["q_heads"], s["pos"], s["cos"], s["sin"], **rope)


# ---- plain forms: float32, rounded once at the end ----

def _act(name, z):
    if name == "none":
        return z
    if name == "relu":
        return z.clamp_min(0)
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu_erf":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))


def _act_grad(name, z):
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        sg = 1 / (1 + torch.exp(-z))
        return sg * (1 + z * (1 - sg))
    if name == "gelu_erf":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def _dense(s):
    z = s["x"].float() @ s["w"].float().T
    if s["b"] is not None:
        z = z + s["b"]
    y = _act(s["act"], z)
    if s["r"] is not None:
        y = y + s["r"].float()
    return y.to(_dt(s["out"]))


def _dense_bwd(s):
    dz = s["dy"].float()
    if s["z"] is not None:
        dz = dz * _act_grad(s["act"], s["z"].float())
    return (dz @ s["w"].float()).to(_BF16), (dz.T @ s["x"].float()).to(_BF16), dz.sum(0) if s["bias"] else None


def _ffn(s):
    inner = s["inner"]
    gu = s["x"].float() @ s["wgu"].float().T
    h = _act(s["act"], gu[:, :inner]) * gu[:, inner:]
    y = h @ s["wd"].float().T
    if s["r"] is not None:
        y = y + s["r"].float()
    return (y.to(_BF16), gu.to(_BF16), h.to(_BF16)) if s["save"] else y.to(_BF16)


def _ffn_bwd(s):
    inner, dy, x = s["inner"], s["dy"].float(), s["x"].float()
    g, u = s["gu"][:, :inner].float(), s["gu"][:, inner:].float()
    dh = dy @ s["wd"].float()
    dgu = torch.cat([dh * u * _act_grad(s["act"], g), dh * _act(s["act"], g)], 1)
    return (dgu @ s["wgu"].float()).to(_BF16), (dgu.T @ x).to(_BF16), (dy.T @ s["h"].float()).to(_BF16)


def _scores(s):
    z = s["scale"] * (s["x"].float() @ s["w"].float().T)
    return z if s["b"] is None else z + s["b"]


def _xent(s):
    z, t = _scores(s), s["t"].long()
    top = z.max(1, keepdim=True).values
    lse = torch.log(torch.exp(z - top).sum(1)) + top[:, 0]
    at = z.gather(1, t.clamp_min(0)[:, None])[:, 0]
    return torch.where(t == IGNORE, torch.zeros_like(lse), lse - at), lse


def _xent_bwd(s):
    t = s["t"].long()
    dl = torch.where(t == IGNORE, torch.zeros_like(s["dl"]), s["dl"])
    p = torch.exp(_scores(s) - s["lse"][:, None])
    one = torch.arange(s["vocab"], device="cuda")[None, :] == t[:, None]
    p = (p - one.to(_F32)) * (dl * s["scale"])[:, None]
    return (p @ s["w"].float()).to(_BF16), (p.T @ s["x"].float()).to(_BF16), None


def _angles(s):
    return s["cos"][s["pos"].long()][:, None, :], s["sin"][s["pos"].long()][:, None, :]


def _halves(s, v):
    r = s["rotary"]
    return (v[..., 0:r:2], v[..., 1:r:2]) if s["pairs"] == "adjacent" else (v[..., :r // 2], v[..., r // 2:r])


def _joined(s, a, b, rest):
    ab = torch.stack([a, b], -1).flatten(-2) if s["pairs"] == "adjacent" else torch.cat([a, b], -1)
    return torch.cat([ab, rest], -1)


def _head_weights(s):
    return torch.cat([s["wq"].float().expand(s["q_heads"], -1), s["wk"].float().expand(s["k_heads"], -1)])


def _rope(s):
    v = s["x"].float()
    if s["norm"]:
        v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * _head_weights(s)
    c, sn = _angles(s)
    a, b = _halves(s, v)
    return _joined(s, a * c - b * sn, b * c + a * sn, v[..., s["rotary"]:]).to(s["x"].dtype)


def _rope_bwd(s):
    c, sn = _angles(s)
    a, b = _halves(s, s["dy"].float())
    dn = _joined(s, a * c + b * sn, b * c - a * sn, s["dy"][..., s["rotary"]:].float())
    if not s["norm"]:
        return dn.to(s["x"].dtype), None, None
    v = s["x"].float()
    inv = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6)
    hat, wdn = v * inv, dn * _head_weights(s)
    dw = dn * hat
    dx = inv * (wdn - hat * (wdn * hat).mean(-1, keepdim=True))
    return dx.to(s["x"].dtype), dw[:, :s["q_heads"]].sum((0, 1)), dw[:, s["q_heads"]:].sum((0, 1))


_PLAIN = {"dense": _dense, "dense_bwd": _dense_bwd, "ffn": _ffn, "ffn_bwd": _ffn_bwd, "xent": _xent,
          "xent_bwd": _xent_bwd, "rope": _rope, "rope_bwd": _rope_bwd}


# --------------------------------------------------------------------------
# What a pass cannot do without
# --------------------------------------------------------------------------

def work(case):
    op, m = case["op"], case["m"]
    size = {"bf16": 2, "f32": 4, "none": 0}
    if op in ("dense", "dense_bwd"):
        n, k = case["n"], case["k"]
        b = 4 * n if case["bias"] else 0
        if op == "dense":
            return {"bytes": 2 * (m * k + n * k) + b + m * n * (size[case["residual"]] + size[case["out"]]),
                    "flops": 2 * m * n * k}
        z = m * n * 2 if case["act"] != "none" else 0
        return {"bytes": 2 * (m * n + 2 * m * k + 2 * n * k) + z + b, "flops": 4 * m * n * k}
    if op in ("ffn", "ffn_bwd"):
        hidden, inner = case["hidden"], case["inner"]
        if op == "ffn":
            saved = 6 * m * inner if case["save"] else 0
            return {"bytes": 2 * (m * hidden * (3 if case["residual"] else 2) + 3 * hidden * inner) + saved,
                    "flops": 6 * m * hidden * inner}
        return {"bytes": 2 * (3 * m * hidden + 3 * m * inner + 6 * hidden * inner), "flops": 12 * m * hidden * inner}
    if op in ("xent", "xent_bwd"):
        v, hidden = case["vocab"], case["hidden"]
        b = 4 * v if case["bias"] else 0
        if op == "xent":
            return {"bytes": 2 * (m + v) * hidden + b + 12 * m, "flops": 2 * m * v * hidden}
        return {"bytes": 4 * (m + v) * hidden + b + 12 * m, "flops": 6 * m * v * hidden}
    row = (case["q_heads"] + case["k_heads"]) * case["dim"]
    e = size[case["dtype"]]
    tables = 4 * min(m, case["longest"]) * case["rotary"] + 4 * m
    return {"bytes": m * row * e * (2 if op == "rope" else 3) + tables,
            "flops": m * row * (10 if op == "rope" else 20)}


# --------------------------------------------------------------------------
# The definitions in float64
# --------------------------------------------------------------------------

def _phi(z):
    return 0.5 * torch.special.erfc(-z / math.sqrt(2.0))


def _f64_act(name, z):
    """The activation and its derivative."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), torch.where(z > 0, 1.0, 0.0).to(z)
    if name == "silu":
        sg = torch.sigmoid(z)
        return z * sg, sg + z * sg * torch.sigmoid(-z)
    if name == "gelu_erf":
        return z * _phi(z), _phi(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    # gelu_tanh(z) = z sigmoid(2u), u = sqrt(2 / pi) (z + 0.044715 z^3)
    two_u = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    sg = torch.sigmoid(two_u)
    slope = 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * z ** 2)
    return z * sg, sg + z * sg * torch.sigmoid(-two_u) * slope


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    op, act = case["op"], case.get("act")
    zero = torch.zeros((), dtype=_F64, device="cuda")
    if op == "dense":
        z = torch.matmul(d["x"], d["w"].t()) + d.get("b", zero)
        return _f64_act(act, z)[0] + d.get("r", zero)
    if op == "dense_bwd":
        dz = d["dy"] if act == "none" else d["dy"] * _f64_act(act, d["z"])[1]
        return (torch.matmul(dz, d["w"]), torch.matmul(dz.t().contiguous(), d["x"]),
                dz.sum(dim=0) if case["bias"] else None)
    if op == "ffn":
        gu = torch.matmul(d["x"], d["wgu"].t())
        gate, up = gu.split(case["inner"], dim=1)
        h = _f64_act(act, gate)[0] * up
        y = torch.matmul(h, d["wd"].t()) + d.get("r", zero)
        return (y, gu, h) if case["save"] else y
    if op == "ffn_bwd":
        gate, up = d["gu"].split(case["inner"], dim=1)
        value, slope = _f64_act(act, gate)
        dh = torch.matmul(d["dy"], d["wd"])
        dg, du = dh * up * slope, dh * value
        wg, wu = d["wgu"].split(case["inner"], dim=0)
        dx = torch.matmul(dg, wg) + torch.matmul(du, wu)
        dw = torch.cat([torch.matmul(dg.t().contiguous(), d["x"]), torch.matmul(du.t().contiguous(), d["x"])], dim=0)
        return dx, dw, torch.matmul(d["dy"].t().contiguous(), d["h"])
    if op in ("xent", "xent_bwd"):
        z = torch.matmul(d["x"] * case["scale"], d["w"].t()) + d.get("b", zero)
        keep = s["t"] != IGNORE
        rows = torch.nonzero(keep)[:, 0]
        cols = s["t"][rows].long()
        if op == "xent":
            lse = torch.logsumexp(z, dim=1)
            loss = torch.zeros_like(lse)
            loss[rows] = lse[rows] - z[rows, cols]
            return loss, lse
        grad = torch.exp(z.sub_(d["lse"].unsqueeze(1)))
        grad[rows, cols] -= 1.0
        grad *= (d["dl"] * keep * case["scale"]).unsqueeze(1)
        return torch.matmul(grad, d["w"]), torch.matmul(grad.t(), d["x"]), None
    # the rotation as a complex product, its gradient as the conjugate one
    turn = torch.complex(d["cos"], d["sin"])[s["pos"].long()].unsqueeze(1)
    r = case["rotary"]

    def rotate(v, by):
        if case["pairs"] == "adjacent":
            c = torch.view_as_complex(v[..., :r].contiguous().unflatten(-1, (r // 2, 2))) * by
            head = torch.view_as_real(c).flatten(-2)
        else:
            c = torch.complex(v[..., :r // 2].contiguous(), v[..., r // 2:r].contiguous()) * by
            head = torch.cat([c.real, c.imag], dim=-1)
        return torch.cat([head, v[..., r:]], dim=-1)

    q = case["q_heads"]
    w = torch.cat([d["wq"].repeat(q, 1), d["wk"].repeat(case["k_heads"], 1)], dim=0) if case["norm"] else zero + 1
    rms = torch.sqrt(d["x"].square().mean(dim=-1, keepdim=True) + 1e-6) if case["norm"] else zero + 1
    if op == "rope":
        return rotate(d["x"] / rms * w, turn)
    dn = rotate(d["dy"], turn.conj())
    if not case["norm"]:
        return dn, None, None
    e = dn * w
    dx = e / rms - d["x"] * (e * d["x"]).mean(dim=-1, keepdim=True) / rms ** 3
    dw = (dn * d["x"] / rms).sum(dim=0)
    return dx, dw[:q].sum(dim=0), dw[q:].sum(dim=0)
