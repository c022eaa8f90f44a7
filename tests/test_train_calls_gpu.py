"""How the layer and head ops are called: streams, layouts and forms of the
arguments beside those of tests/test_train_gpu.py."""
import pytest

import train_ref as R
from test_train_gpu import _rand

pytestmark = pytest.mark.gpu


def _ops(inl, torch, dev):
    """Every op as (call with stream=, bytes of its largest output)."""
    m, hidden, inner, vocab = 1024, 256, 512, 1024
    x, dy = _rand(torch, dev, (m, hidden), 1), _rand(torch, dev, (m, hidden), 2, 0.1)
    w = _rand(torch, dev, (hidden, hidden), 3, 1 / 16)
    gu, down = _rand(torch, dev, (2 * inner, hidden), 4, 1 / 16), _rand(torch, dev, (hidden, inner), 5, 1 / 16)
    wv = _rand(torch, dev, (vocab, hidden), 6, 1 / 16)
    t = torch.arange(m, device=dev, dtype=torch.int32)
    _, pre, h = inl.gated_ffn(x, gu, down, save=True)
    _, lse = inl.softmax_xent(x, wv, t)
    dl = torch.ones(m, device=dev)
    heads = x.view(m, 4, 64)
    return {
        "dense": (lambda s: inl.dense(x, w, act="silu", stream=s), 2 * m * hidden),
        "dense_bwd": (lambda s: inl.dense_bwd(dy, x, w, bias_grad=True, stream=s), 2 * m * hidden),
        "gated_ffn": (lambda s: inl.gated_ffn(x, gu, down, save=True, stream=s), 4 * m * inner),
        "gated_ffn_bwd": (lambda s: inl.gated_ffn_bwd(dy, x, gu, down, pre, h, stream=s), 2 * m * hidden),
        "softmax_xent": (lambda s: inl.softmax_xent(x, wv, t, stream=s), 4 * m),
        "softmax_xent_bwd": (lambda s: inl.softmax_xent_bwd(dl, lse, x, wv, t, stream=s), 2 * m * hidden),
        "norm_rope_qk_bwd": (lambda s: inl.norm_rope_qk_bwd(dy.view(m, 4, 64), heads, 2, stream=s), 2 * m * hidden),
    }


@pytest.mark.parametrize("op", ["dense", "dense_bwd", "gated_ffn", "gated_ffn_bwd", "softmax_xent", "softmax_xent_bwd",
                                "norm_rope_qk_bwd"])
def test_memory_of_a_call_on_another_stream(op, cuda, inl):
    """Blocks that were freed while work on the current stream still reads them are
    not taken by a call on another stream, which does not wait for that work."""
    import torch
    call, size = _ops(inl, torch, cuda)[op]
    flat = lambda out: [t for t in (out if isinstance(out, tuple) else (out,)) if t is not None]
    want = flat(call(None))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    a, b = (torch.randn(4096, 4096, device=cuda) for _ in range(2))
    blocks = [torch.full((n,), 7, dtype=torch.uint8, device=cuda) for n in (size, size, 1024, 4096, 1 << 20, 1 << 22, 1 << 24)]
    spans = [(t.data_ptr(), t.data_ptr() + t.numel()) for t in blocks]
    torch.cuda.synchronize()
    for _ in range(20):   # some milliseconds of work in front of the reads
        a = (a @ b).clamp_(-1, 1)
    seen = [t.clone() for t in blocks]
    del blocks
    got = flat(call(side))
    torch.cuda.synchronize()
    for t in got:
        assert not any(lo < t.data_ptr() + t.numel() * t.element_size() and t.data_ptr() < hi for lo, hi in spans)
    assert all((t == 7).all() for t in seen)
    assert all(torch.equal(u, v) for u, v in zip(got, want))


# row kernels, one per block of 16 columns, tiles of the three shapes, a split sum
@pytest.mark.parametrize("m,k", [(1, 8), (4, 40), (16, 72), (64, 72), (300, 2056), (5000, 72), (9000, 72)])
def test_gelu_erf_keeps_its_tail(m, k, cuda, inl):
    """v Phi(v) and its slope for v from -8 to 8 by their own size: the tail Phi(-|v|) is
    within 3e-4 of itself and 4e-7 of 1, and nothing cancels where it stands alone.
    An identity for weights makes v an input exactly."""
    import torch
    n = 1024 if m > 4000 else 264
    v = torch.linspace(-8, 8, n * 4, device=cuda).to(torch.bfloat16)
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=cuda)
    x[:, 5] = 1
    w = torch.zeros(4 * n, k, dtype=torch.bfloat16, device=cuda)
    w[:, 5] = v
    print(f"case=gelu tail {m} {k}", flush=True)
    d = v.double()
    tail = torch.special.erfc(d.abs() / 2 ** 0.5) / 2
    ref = torch.where(d < 0, d * tail, d * (1 - tail))
    # v Phi(v): the tail's error times v, two roundings
    tol = torch.where(d < 0, 3e-4 * ref.abs(), d.abs() * torch.minimum(3e-4 * tail, torch.full_like(tail, 4e-7))) + 2.0 ** -22 * ref.abs()
    for i in range(4):
        y = inl.dense(x, w[i * n:(i + 1) * n], act="gelu_erf", out_dtype=torch.float32)
        s = slice(i * n, (i + 1) * n)
        R.check(y, ref[s].expand(m, n), tol[s].expand(m, n), "y")
    # one row's bias gradient is its slope, Phi(v) + v phi(v)
    dens = d * torch.exp(-d * d / 2) / (2 * torch.pi) ** 0.5
    got = inl.dense_bwd(torch.ones(1, 4 * n, dtype=torch.bfloat16, device=cuda), x[:1], w, act="gelu_erf", pre=v[None, :],
                        bias_grad=True, dx_grad=False, dw_grad=False)[2]
    ref = torch.where(d < 0, tail, 1 - tail) + dens
    # (the exponent of the density, up to 47 in base 2, is off by 3 f32 steps of itself)
    R.check(got, ref, torch.minimum(3e-4 * tail, torch.full_like(tail, 4e-7)) + 2.0 ** -17 * dens.abs() + 2.0 ** -22 * ref.abs(), "slope")


def test_gelu_erf_far_values(cuda, inl):
    import torch
    v = torch.tensor([1e4, 3e38, float("inf"), -20, -1e4, -3e38, float("nan"), 0], device=cuda).to(torch.bfloat16)
    for m in (1, 16, 70):
        x = torch.ones(m, 8, dtype=torch.bfloat16, device=cuda)
        x[:, 1:] = 0
        w = torch.zeros(8, 8, dtype=torch.bfloat16, device=cuda)
        w[:, 0] = v
        y = inl.dense(x, w, act="gelu_erf", out_dtype=torch.float32)
        assert torch.equal(y[:, :3], v[:3].float().expand(m, 3)) and not y[:, 3:6].any() and not y[:, 7].any()
        assert torch.isnan(y[:, 6]).all()


@pytest.mark.parametrize("act", ["relu", "silu", "gelu_tanh", "gelu_erf"])
def test_slopes_of_far_values(act, cuda, inl):
    """Slopes of activations far out are 0 and 1, also where v^2 or v^3 leaves the range of
    f32, and NaN stays NaN; in the element-wise pass and in the products' epilogues."""
    import torch
    far = torch.tensor([20, 1e3, 1e12, 1e14, 1e18, 1e20, 1e30, 3e38], device=cuda)
    pre = torch.cat([far, -far, torch.full_like(far, float("nan"))]).to(torch.bfloat16)[None, :]
    ones = torch.ones(1, 24, dtype=torch.bfloat16, device=cuda)
    x, w = torch.zeros(1, 8, dtype=torch.bfloat16, device=cuda), torch.zeros(24, 8, dtype=torch.bfloat16, device=cuda)
    db = inl.dense_bwd(ones, x, w, act=act, pre=pre, bias_grad=True)[2]
    assert (db[:8] == 1).all() and (db[8:16].abs() <= 1e-7).all() and torch.isnan(db[16:]).all()
    # d_gate = dh up act'(gate) with dh = dy; dx of w_gate = identity is d_gate
    for m in (1, 300):
        gate = pre[:, :16].expand(m, 16)
        gu = torch.cat([gate, torch.ones_like(gate)], 1).contiguous()
        w_gu = torch.cat([torch.eye(16, device=cuda), torch.zeros(16, 16, device=cuda)]).to(torch.bfloat16)
        down = torch.zeros(16, 16, dtype=torch.bfloat16, device=cuda)
        down[0] = 1
        dy = torch.zeros(m, 16, dtype=torch.bfloat16, device=cuda)
        dy[:, 0] = 2.0 ** -20   # d_up = dh act(gate) stays in the range
        h = torch.zeros(m, 16, dtype=torch.bfloat16, device=cuda)
        dx, _, _ = inl.gated_ffn_bwd(dy, x.new_zeros(m, 16), w_gu, down, gu, h, act=act, dx_dtype=torch.float32)
        assert (dx[:, :8] == 2.0 ** -20).all() and (dx[:, 8:].abs() <= 1e-7 * 2.0 ** -20).all(), m


def test_prologue_forward_refusals(cuda, inl):
    """The forward refuses what its gradient refuses: nothing of it reaches a kernel."""
    import torch
    f = lambda *s, dtype=torch.float32: torch.ones(*s, dtype=dtype, device=cuda)
    x, rows, c = f(5, 3, 64), f(5, dtype=torch.int32), f(9, 32)
    for kw in (dict(rows=rows, cos=f(9, 64), sin=f(9, 64), rotary_dim=64, sections=3),
               dict(rows=rows.long(), cos=c, sin=c), dict(rows=rows[:4], cos=c, sin=c), dict(cos=c, sin=c),
               dict(rows=rows, cos=c), dict(rows=rows, cos=c.bfloat16(), sin=c.bfloat16()), dict(rows=rows.cpu(), cos=c, sin=c),
               dict(rows=rows, cos=c.cpu(), sin=c.cpu()), dict(out=f(5, 3, 32)), dict(out=f(4, 3, 64)), dict(out=f(1, 3, 64).expand(5, 3, 64)),
               dict(rotary_dim=8)):
        for call in (lambda: inl.norm_rope(x, **kw), lambda: inl.norm_rope_qk(x, 2, **kw)):
            with pytest.raises(inl.InlError):
                call()
    for w in (f(32), f(64, dtype=torch.bfloat16), f(64).cpu(), f(128)[::2]):
        for call in (lambda: inl.norm_rope(x, weight=w), lambda: inl.norm_rope_qk(x, 2, q_weight=w),
                     lambda: inl.norm_rope_qk(x, 2, k_weight=w)):
            with pytest.raises(inl.InlError):
                call()
    for t in (x[0], x.transpose(1, 2), f(5, 6, 64)[:, ::2], f(1, 3, 64).expand(5, 3, 64)):
        with pytest.raises(inl.InlError):
            inl.norm_rope_qk(t, 2)


@pytest.mark.parametrize("sections", [1, 3])
def test_prologue_forward_forms(sections, cuda, inl):
    """Longer rows and tables than are read, one token of any row stride, a weight that
    no norm uses, another stream: all as the plain call."""
    import torch
    x = _rand(torch, cuda, (5, 4, 64), 1)
    rows = torch.tensor([3, 0, 8, 1, 1, 7], dtype=torch.int32, device=cuda)
    c, s = _rand(torch, cuda, (9, 32), 2, 1, torch.float32), _rand(torch, cuda, (9, 32), 3, 1, torch.float32)
    w = _rand(torch, cuda, (64,), 4)
    kw = dict(rotary_dim=64, sections=sections)
    want = inl.norm_rope_qk(x, 3, rows[:5], c, s, q_weight=w, **kw)
    t64 = [v.double()[rows[:5].long()] for v in (c, s)]
    weights = torch.cat([w.double().expand(3, 64), torch.ones(1, 64, dtype=torch.float64, device=cuda)])
    ref = R.norm_rope(x.double(), weights, 1e-6, 64, sections, t64)
    R.check(want, ref, R.out_tol(ref, torch.bfloat16) + 2.0 ** -20 * ref.abs().amax(-1, keepdim=True), "y")
    assert torch.equal(inl.norm_rope_qk(x, 3, rows, c.view(9, 1, 32), torch.cat([s, s]), q_weight=w[None], **kw), want)
    one = torch.empty(1, 9, 64, dtype=torch.bfloat16, device=cuda).expand(1, 9, 64)[:, :4]
    one.copy_(x[2:3])
    assert torch.equal(inl.norm_rope_qk(one, 3, rows[2:], c, s, q_weight=w, **kw), want[2:3])
    plain = inl.norm_rope(x, rows, c, s, norm=False, **kw)
    assert torch.equal(inl.norm_rope(x, rows, c, s, norm=False, weight=w.float()[:1], **kw), plain)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = inl.norm_rope_qk(x, 3, rows, c, s, q_weight=w, stream=side, **kw)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_prologue_gradient_takes_the_forwards_arguments(cuda, inl):
    import torch
    x, dy = _rand(torch, cuda, (9, 3, 64), 1), _rand(torch, cuda, (9, 3, 64), 2)
    rows, c = torch.arange(9, dtype=torch.int32, device=cuda), _rand(torch, cuda, (9, 32), 3, 1, torch.float32)
    kw = dict(q_weight=x[0, 0], k_weight=x[1, 1], eps=1e-5, rotary_dim=64, sections=3, round_tables=True)
    inl.norm_rope_qk(x, 2, rows, c, c, round_norm=True, **kw)
    got = inl.norm_rope_qk_bwd(dy, x, 2, rows, c, c, round_norm=True, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, inl.norm_rope_qk_bwd(dy, x, 2, rows, c, c, **kw)))


# both sides of each border of the rules that choose a kernel for a few rows
@pytest.mark.parametrize("m,n,k", [(2, 16384, 1024), (2, 16392, 1016), (3, 8192, 2048), (4, 8200, 1016), (4, 4096, 4104),
                                   (5, 8192, 768), (16, 8192, 760), (16, 8200, 768), (16, 4104, 2048), (9, 40, 4096), (9, 40, 4104),
                                   (17, 4096, 2048), (32, 72, 2056), (32, 8192, 512), (32, 4104, 520)])
def test_dense_at_the_borders_of_few_rows(m, n, k, cuda, inl):
    from test_train_gpu import test_dense_few_rows
    test_dense_few_rows(m, n, k, "silu", cuda, inl)


@pytest.mark.parametrize("m,hidden,inner", [(4, 520, 6144), (3, 520, 6152), (4, 1024, 12288), (3, 1024, 12296), (16, 512, 4096),
                                            (5, 512, 4104), (16, 1024, 4104), (16, 1016, 4104), (32, 2048, 4096), (17, 2056, 264), (2, 264, 16400)])
def test_gated_ffn_at_the_borders_of_few_rows(m, hidden, inner, cuda, inl):
    from test_train_gpu import test_gated_ffn
    test_gated_ffn(m, hidden, inner, "gelu_erf", cuda, inl)
