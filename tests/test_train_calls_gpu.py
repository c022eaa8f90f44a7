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


# ---------------------------------------------------------------------------
# Padded rows in and out, with guards
# ---------------------------------------------------------------------------

def _padded(torch, dev, rows, cols, dtype, extra=24):
    """A [rows, cols] part of wider rows, a row behind them, everything 7."""
    whole = torch.full((rows + 2, cols + extra), 7.0, dtype=dtype, device=dev)
    return whole, whole[:rows, 8:8 + cols] if dtype == torch.bfloat16 else whole[:rows, 4:4 + cols]


def _only_inside_changed(torch, whole, part):
    part.fill_(7.0)
    return bool((whole == 7.0).all())


def _room(torch, dev, size_fn, desc):
    import ctypes
    n = ctypes.c_size_t()
    assert size_fn(desc, 1, ctypes.byref(n)) == 0
    return torch.empty(max(n.value, 16), dtype=torch.uint8, device=dev), n.value


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", [(3, 40, 24), (300, 136, 72), (2500, 264, 520)])
def test_gradients_into_padded_rows(m, n, k, dt, cuda, inl):
    """dx and dw of the linear layer, the block and cross entropy (several pieces of the
    vocabulary with the largest m) with row strides of their own: the bits of packed
    outputs, and nothing beside them is written. The binding packs its outputs, so
    these are calls of the C entries."""
    import torch
    from inl_hip import train as T
    dtype, code = (torch.bfloat16, 1) if dt == "bf16" else (torch.float32, 0)
    p, st = (lambda t: t.data_ptr()), torch.cuda.current_stream().cuda_stream
    x, dy, w = _rand(torch, cuda, (m, k), 1), _rand(torch, cuda, (m, n), 2, 0.1), _rand(torch, cuda, (n, k), 3, k ** -0.5)
    pre = _rand(torch, cuda, (m, n), 4)
    print(f"case=padded {m} {n} {k} {dt}", flush=True)
    want = inl.dense_bwd(dy, x, w, act="silu", pre=pre, dx_dtype=dtype, dw_dtype=dtype)
    (dxw, dx), (dww, dw) = _padded(torch, cuda, m, k, dtype), _padded(torch, cuda, n, k, dtype)
    d = T.DenseDesc(m, n, k, 0, 0, 0, 0, 0, dx.stride(0), dw.stride(0), 2, 0, 0, code, code)
    room, size = _room(torch, cuda, T._dense_ws, d)
    assert T._dense_bwd(d, p(dy), p(x), p(w), p(pre), p(dx), p(dw), None, p(room), size, st) == 0, inl.last_error()
    assert torch.equal(dx, want[0]) and torch.equal(dw, want[1])
    assert _only_inside_changed(torch, dxw, dx) and _only_inside_changed(torch, dww, dw)

    gu, down = _rand(torch, cuda, (2 * n, k), 5, k ** -0.5), _rand(torch, cuda, (k, n), 6, n ** -0.5)
    _, pre2, h = inl.gated_ffn(x, gu, down, save=True)
    want = inl.gated_ffn_bwd(x, x, gu, down, pre2, h, dx_dtype=dtype, dw_dtype=dtype)
    d = T.GatedFfnDesc(m, k, n, 0, 0, 0, dx.stride(0), 2, 0, 0, code, code)
    room, size = _room(torch, cuda, T._ffn_ws, d)
    dgu, dd = (torch.empty_like(t) for t in want[1:])
    assert T._ffn_bwd(d, p(x), p(x), p(gu), p(down), p(pre2), p(h), p(dx), p(dgu), p(dd), p(room), size, st) == 0
    assert all(torch.equal(a, b) for a, b in zip((dx, dgu, dd), want)) and _only_inside_changed(torch, dxw, dx)

    vocab = 2 ** 26 // m // 256 * 256 + 1031 if m > 2000 else n + 3
    wv, t = _rand(torch, cuda, (vocab, k), 7, k ** -0.5), torch.arange(m, device=cuda, dtype=torch.int32) % vocab
    _, lse = inl.softmax_xent(x, wv, t)
    dl = torch.full((m,), 1 / m, device=cuda)
    want = inl.softmax_xent_bwd(dl, lse, x, wv, t, dx_dtype=dtype, dw_dtype=dtype)
    dvw, dv = _padded(torch, cuda, vocab, k, dtype)
    d = T.SoftmaxXentDesc(m, vocab, k, 0, 0, dx.stride(0), dv.stride(0), 1.0, -100, code, code)
    room, size = _room(torch, cuda, T._xent_ws, d)
    assert T._xent_bwd(d, p(dl), p(lse), p(x), p(wv), None, p(t), p(dx), p(dv), None, p(room), size, st) == 0
    assert torch.equal(dx, want[0]) and torch.equal(dv, want[1])
    assert _only_inside_changed(torch, dxw, dx) and _only_inside_changed(torch, dvw, dv)


@pytest.mark.parametrize("m", [2, 20, 700])
def test_block_and_loss_on_strided_rows(m, cuda, inl):
    """Slices of wider rows in and out give what packed rows give."""
    import torch
    hidden, inner, vocab = 136, 200, 1001
    wide = lambda rows, cols, seed, std=1.0: _rand(torch, cuda, (rows, cols + 24), seed, std)[:, 8:8 + cols]
    x, dy, res, wv = wide(m, hidden, 1), wide(m, hidden, 2, 0.1), wide(m, hidden, 3), wide(vocab, hidden, 4, 0.08)
    gu, down = _rand(torch, cuda, (2 * inner, hidden), 5, 0.08), _rand(torch, cuda, (hidden, inner), 6, 0.07)
    c = lambda t: t.contiguous()
    print(f"case=strided {m}", flush=True)
    want = inl.gated_ffn(c(x), gu, down, residual=c(res), save=True)
    whole, out = _padded(torch, cuda, m, hidden, torch.bfloat16)
    got = inl.gated_ffn(x, gu, down, residual=res, save=True, out=out)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and _only_inside_changed(torch, whole, out)
    _, pre, h = want
    assert all(torch.equal(a, b) for a, b in zip(inl.gated_ffn_bwd(dy, x, gu, down, pre, h),
                                                 inl.gated_ffn_bwd(c(dy), c(x), gu, down, pre, h)))
    t = torch.arange(m, device=cuda, dtype=torch.int32)
    want = inl.softmax_xent(c(x), c(wv), t)
    assert all(torch.equal(a, b) for a, b in zip(inl.softmax_xent(x, wv, t), want))
    dl = torch.full((m,), 1 / m, device=cuda)
    want = inl.softmax_xent_bwd(dl, want[1], c(x), c(wv), t, bias_grad=True)
    assert all(torch.equal(a, b) for a, b in zip(inl.softmax_xent_bwd(dl, inl.softmax_xent(x, wv, t)[1], x, wv, t, bias_grad=True), want))


@pytest.mark.parametrize("m,vocab", [(9000, 9001), (17000, 9001)])
def test_softmax_xent_bwd_of_several_pieces(m, vocab, cuda, inl):
    """Two and three pieces of the vocabulary (2^26 / m columns each, 4,096 at least), the
    last one odd: dx adds up over them in f32."""
    from test_train_gpu import test_softmax_xent_bwd
    test_softmax_xent_bwd(m, vocab, 72, 1.0, True, cuda, inl)


# ---------------------------------------------------------------------------
# Forms of the prologue's gradient
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("types", [("bf16", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("weights,rounded", [(True, True), (False, False), (False, True)])
@pytest.mark.parametrize("n,hq,hk,d,rotary,sections", [(5, 2, 1, 64, 64, 1), (333, 16, 8, 128, 64, 3), (40, 6, 6, 64, 64, 2),
                                                       (2500, 8, 2, 32, 24, 3), (4000, 4, 4, 128, 128, 1)])
def test_prologue_gradient_forms(n, hq, hk, d, rotary, sections, weights, rounded, types, cuda, inl):
    """dy of the other type than x, norms without weights, tables rounded to bf16. The
    weight gradients' bound is of the sizes that are summed: a token's heads that
    went missing would show."""
    import torch
    from test_train_gpu import _tables
    tx, ty = ({"bf16": torch.bfloat16, "f32": torch.float32}[t] for t in types)
    heads = hq + hk
    x, dy = _rand(torch, cuda, (n, heads, d), 1, 1.0, tx), _rand(torch, cuda, (n, heads, d), 2, 1.0, ty)
    wq, wk = ((1 + _rand(torch, cuda, (d,), s, 0.2, torch.float32)).to(tx) for s in (3, 4))
    rows, tabs = _tables(torch, cuda, n, d, rotary, sections)
    kw = dict(q_weight=wq, k_weight=wk) if weights else {}
    print(f"case=rope_bwd forms {n} {hq} {hk} {d} {rotary} {sections} {types}", flush=True)
    dx, dq, dk = inl.norm_rope_qk_bwd(dy, x, hq, rows, tabs[0], tabs[1], rotary_dim=rotary, sections=sections, cos2=tabs[2],
                                      sin2=tabs[3], round_tables=rounded, **kw)
    t64 = [None if v is None else (R.r16(v) if rounded else v.double())[rows.long()] for v in tabs]
    w = torch.cat([wq.double().expand(hq, d), wk.double().expand(hk, d)]) if weights else torch.ones(heads, d, device=cuda, dtype=torch.float64)
    xd, dyd = x.double(), dy.double()
    ref, dw = R.norm_rope_bwd(dyd, xd, w, 1e-6, rotary, sections, t64)
    assert dx.dtype == tx
    inv = 1 / torch.sqrt((xd * xd).mean(-1, keepdim=True) + 1e-6)
    hat = xd * inv
    # sizes of what a rotation adds: |dy| turned by |cos| and -|sin|, backwards
    sizes = [None if v is None else v.abs() for v in t64]
    for i in (1, 3):
        sizes[i] = None if sizes[i] is None else -sizes[i]
    turned = R.turn(dyd.abs(), rotary, sections, *sizes)
    if rotary:   # (one of a pair takes the difference there: the sum bounds both)
        flip = R.turn(dyd.abs(), rotary, sections, *sizes, back=True)
        turned = torch.maximum(turned.abs(), flip.abs())
    # some 16 f32 roundings of each value's terms, and of the row's sum of d of them
    size = (w * turned).abs()
    mean = (size * hat.abs()).mean(-1, keepdim=True)
    R.check(dx, ref, R.out_tol(ref, tx) + (16 + d / 8) * 2.0 ** -24 * inv * (size + hat.abs() * mean), "dx")
    for got, q in ((dq, slice(0, hq)), (dk, slice(hq, heads))):
        part, each = dw[:, q], (turned * hat.abs())[:, q]
        terms = part.shape[0] * part.shape[1]
        # in order per lane, then over the lanes' groups and the workgroups: at most
        # 80 + terms / 64 additions on a value's way; 16 roundings of each term
        tol = (80 + terms / 64) * 2.0 ** -24 * part.abs().sum((0, 1)) + 16 * 2.0 ** -24 * each.sum((0, 1))
        R.check(got, part.sum((0, 1)), tol, "dweight")
        lost = part[n // 2].sum(0).abs()   # one token's heads
        assert (lost > 2 * tol).any(), "the bound would not see a lost token"


def test_prologue_gradient_weights_as_in_the_forward(cuda, inl):
    """The forms of a weight that the forward takes: any shape of head_dim values, and
    whatever it is where there is no norm."""
    import torch
    x, dy = _rand(torch, cuda, (9, 3, 64), 1), _rand(torch, cuda, (9, 3, 64), 2)
    w = _rand(torch, cuda, (64,), 3)
    for f in (inl.norm_rope_qk, inl.norm_rope_qk_bwd):
        a = (x,) if f is inl.norm_rope_qk else (dy, x)
        flat = lambda out: [t for t in (out if isinstance(out, tuple) else (out,)) if t is not None]
        for one, two in ((dict(q_weight=w[None], k_weight=w.view(8, 8)), dict(q_weight=w, k_weight=w)),
                         (dict(norm=False, q_weight=w.float()), dict(norm=False))):
            assert all(torch.equal(u, v) for u, v in zip(flat(f(*a, 2, **one)), flat(f(*a, 2, **two))))
        for bad in (w.float(), w[:32], w.cpu()):
            with pytest.raises(inl.InlError):
                f(*a, 2, q_weight=bad)


def test_softmax_xent_without_any_entry(cuda, inl):
    """A bias of -inf on the whole vocabulary leaves nothing: lse -inf, loss NaN but for
    ignored rows."""
    import torch
    for m, vocab in ((1, 3), (70, 1001), (300, 70)):
        x, w = _rand(torch, cuda, (m, 72), 1), _rand(torch, cuda, (vocab, 72), 2)
        t = torch.arange(m, device=cuda, dtype=torch.int32) % vocab
        t[m // 2] = -100
        loss, lse = inl.softmax_xent(x, w, t, bias=torch.full((vocab,), float("-inf"), device=cuda))
        assert (lse == float("-inf")).all() and loss[m // 2] == 0 and torch.isnan(loss[t >= 0]).all()


def test_columns_of_one_buffer_and_in_place(cuda, inl):
    """x, y, the residual and pre as columns of one buffer; the block in place on its
    residual stream; the linear layer there is refused."""
    import torch
    for m in (1, 9, 300):
        buf = _rand(torch, cuda, (m, 400), 1)
        x, y, res, pre = buf[:, :72], buf[:, 72:144], buf[:, 144:216], buf[:, 216:288]
        w = _rand(torch, cuda, (72, 72), 2, 0.1)
        want = inl.dense(x.clone(), w, act="silu", residual=res.clone())
        assert torch.equal(inl.dense(x, w, act="silu", residual=res, out=y, pre=pre), want)
        for kw in (dict(out=x), dict(out=x, residual=x), dict(pre=x), dict(out=y, pre=y), dict(residual=res, pre=res),
                   dict(out=buf[:, 64:136])):
            with pytest.raises(inl.InlError, match="overlap"):
                inl.dense(x, w, **kw)
        gu, down = _rand(torch, cuda, (400, 72), 3, 0.1), _rand(torch, cuda, (72, 200), 4, 0.1)
        want = inl.gated_ffn(x.clone(), gu, down, residual=x.clone())
        assert torch.equal(inl.gated_ffn(x, gu, down, residual=x, out=x), want) and torch.equal(x, want)


def test_captured_on_a_forked_stream(cuda, inl):
    """Calls with stream= inside a capture, on a stream that joined it: their memory is
    the graph's, and eager work between the replays leaves it alone."""
    import torch
    m, n, k = 500, 264, 136
    x, w, dy = _rand(torch, cuda, (m, k), 1), _rand(torch, cuda, (n, k), 2, 0.1), _rand(torch, cuda, (m, n), 3, 0.1)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        y = inl.dense(x, w, act="silu", stream=side)
        grads = inl.dense_bwd(dy, x, w, bias_grad=True, stream=side)
        also = inl.dense(x, w)
        here.wait_stream(side)
    for i in range(3):
        x.copy_(_rand(torch, cuda, (m, k), 10 + i))
        graph.replay()
        torch.cuda.synchronize()
        want = (inl.dense(x, w, act="silu"), *inl.dense_bwd(dy, x, w, bias_grad=True), inl.dense(x, w))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((y, *grads, also), want)), i
