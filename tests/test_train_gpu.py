"""The layer and head ops of include/inl_train.h and their gradients against
float64 (tests/train_ref.py, where the tolerances are derived)."""
import math

import pytest

import train_ref as R

pytestmark = pytest.mark.gpu
ACTS = [None, "relu", "silu", "gelu_tanh", "gelu_erf"]


def _rand(torch, dev, shape, seed, std=1.0, dtype=None):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * std).to(dtype or torch.bfloat16)


# ---------------------------------------------------------------------------
# Linear layer
# ---------------------------------------------------------------------------

def _dense_ref(x, w, b, act, res):
    z = x.double() @ w.double().T + (b.double() if b is not None else 0)
    size = x.double().abs() @ w.double().abs().T + (b.double().abs() if b is not None else 0)
    y = R.act(act, z)[0] + (res.double() if res is not None else 0)
    # slopes of the activations stay below 1.13; their own error is below 4 f32
    # steps and 2e-7 |z| (the normal distribution's polynomial); the bias and the
    # residual round once more each
    tol = 1.13 * R.sum_tol(x.shape[1]) * size + 3e-7 * z.abs() + 2.0 ** -22 * y.abs()
    return z, y, tol


# 1 to 4 and 5 to 32 rows have kernels of their own; sizes off every tile and off 32; k of many stages
SIZES = [(1, 8, 8), (2, 264, 72), (3, 72, 1032), (4, 1024, 512), (8, 40, 2048), (9, 8, 8), (64, 64, 64), (65, 136, 40),
         (129, 520, 264), (257, 72, 4104), (1000, 264, 96), (2051, 1032, 520)]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_dense(m, n, k, act, cuda, inl):
    import torch
    x, w = _rand(torch, cuda, (m, k), 1), _rand(torch, cuda, (n, k), 2, k ** -0.5)
    b = _rand(torch, cuda, (n,), 3, 0.5, torch.float32)
    i = SIZES.index((m, n, k)) + ACTS.index(act)
    bias = b if i % 3 else None
    res = [None, _rand(torch, cuda, (m, n), 4), _rand(torch, cuda, (m, n), 4, 1.0, torch.float32)][i % 3]
    out = [torch.bfloat16, torch.float32][(i // 2) % 2]
    pre = torch.empty(m, n, dtype=torch.bfloat16, device=cuda) if i % 2 else None
    print(f"case=dense {m} {n} {k} act={act}", flush=True)
    y = inl.dense(x, w, bias, act=act, residual=res, pre=pre, out_dtype=out)
    z, ref, tol = _dense_ref(x, w, bias, act, res)
    R.check(y, ref, tol + R.out_tol(ref, out), "y")
    if pre is not None:
        R.check(pre, z, tol + R.out_tol(z, torch.bfloat16), "pre")


def test_dense_strides_and_neighbours(cuda, inl):
    """Slices of wider rows in and out, the residual in place; memory around the
    written columns and rows stays as it was."""
    import torch
    for m, n, k in ((5, 72, 136), (300, 72, 136), (700, 520, 136)):
        xs, ws = _rand(torch, cuda, (m, k + 24), 5), _rand(torch, cuda, (n, k + 8), 6, k ** -0.5)
        ys = _rand(torch, cuda, (m + 2, n + 24), 7)
        before = ys.clone()
        x, w, y = xs[:, 8:8 + k], ws[:, :k], ys[:m, 16:16 + n]
        print(f"case=dense strides {m}", flush=True)
        inl.dense(x, w, None, act="silu", residual=y, out=y)
        _, ref, tol = _dense_ref(x, w, None, "silu", before[:m, 16:16 + n])
        R.check(y, ref, tol + R.out_tol(ref, torch.bfloat16), "y")
        ys[:m, 16:16 + n] = before[:m, 16:16 + n]
        assert torch.equal(ys, before)


def test_dense_garbage_stays_out(cuda, inl):
    """NaN behind every row and every tensor: none of it is read into a result."""
    import torch
    for m, n, k in ((3, 40, 24), (70, 136, 40), (333, 264, 72)):
        def holed(rows, cols, seed, std=1.0):
            t = torch.full((rows + 3, cols + 16), float("nan"), dtype=torch.bfloat16, device=cuda)
            t[:rows, :cols] = _rand(torch, cuda, (rows, cols), seed, std)
            return t[:rows, :cols]
        x, w, dy = holed(m, k, 8), holed(n, k, 9, k ** -0.5), holed(m, n, 10, 0.1)
        pre = holed(m, n, 11)
        print(f"case=dense garbage {m}", flush=True)
        y = inl.dense(x, w, act="gelu_tanh")
        _, ref, tol = _dense_ref(x, w, None, "gelu_tanh", None)
        R.check(y, ref, tol + R.out_tol(ref, torch.bfloat16), "y")
        got = inl.dense_bwd(dy, x, w, act="gelu_tanh", pre=pre, bias_grad=True)
        assert all(torch.isfinite(t).all() for t in got)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", [(1, 8, 8), (2, 72, 264), (31, 264, 72), (64, 64, 64), (257, 136, 1032), (1001, 520, 264),
                                   (5003, 264, 136), (2048, 1032, 2056)])
def test_dense_bwd(m, n, k, act, cuda, inl):
    import torch
    x, w = _rand(torch, cuda, (m, k), 11), _rand(torch, cuda, (n, k), 12, k ** -0.5)
    dy, pre = _rand(torch, cuda, (m, n), 13, 0.1), _rand(torch, cuda, (m, n), 14)
    f32 = (m + ACTS.index(act)) % 2 == 0
    dt = torch.float32 if f32 else torch.bfloat16
    print(f"case=dense_bwd {m} {n} {k} act={act}", flush=True)
    dx, dw, db = inl.dense_bwd(dy, x, w, act=act, pre=pre if act else None, bias_grad=True, dx_dtype=dt, dw_dtype=dt)
    dzf = dy.double() * R.act(act, pre.double())[1]
    dz = R.r16(dzf)
    fl = 0.0 if act is None else 1.0
    xd, wd = x.double(), w.double()
    ref = dz @ wd
    R.check(dx, ref, R.out_tol(ref, dt) + R.sum_tol(n) * (dz.abs() @ wd.abs()) + fl * R.flips(dz, wd), "dx")
    ref = dz.T.contiguous() @ xd
    R.check(dw, ref, R.out_tol(ref, dt) + R.sum_tol(m) * (dz.abs().T.contiguous() @ xd.abs()) + fl * R.flips(dz, xd), "dw")
    # f32 sums of 8 rows, 8 of those and m / 64 of those; the slope is within 2^-20 of 1.13
    R.check(db, dzf.sum(0), (m / 64 + 24) * 2.0 ** -24 * dzf.abs().sum(0) + 1.13 * 2.0 ** -20 * dy.double().abs().sum(0), "db")


def test_dense_bwd_differences(cuda, inl):
    """The gradients along random directions against central differences of the
    float64 forward."""
    import torch
    m, n, k = 130, 72, 136
    x, w = _rand(torch, cuda, (m, k), 15), _rand(torch, cuda, (n, k), 16, k ** -0.5)
    b, dy = _rand(torch, cuda, (n,), 17, 0.5, torch.float32), _rand(torch, cuda, (m, n), 18, 0.1)
    for act in ACTS[2:]:
        pre = torch.empty(m, n, dtype=torch.bfloat16, device=cuda)
        inl.dense(x, w, b, act=act, pre=pre)
        grads = inl.dense_bwd(dy, x, w, act=act, pre=pre, bias_grad=True, dx_dtype=torch.float32, dw_dtype=torch.float32)
        at = [x.double(), w.double(), b.double()]

        def f(p):
            return (dy.double() * R.act(act, p[0] @ p[1].T + p[2])[0]).sum().item()
        for i, g in enumerate(grads):
            v = _rand(torch, cuda, at[i].shape, 19 + i, 1.0, torch.float32).double()
            e = 1e-5
            up, down = [t.clone() for t in at], [t.clone() for t in at]
            up[i] += e * v
            down[i] -= e * v
            want = (f(up) - f(down)) / (2 * e)
            got = (g.double() * v).sum().item()
            # dz and pre are rounded: each moves a term dz t by at most 2^-8 of its own
            # size (pre through act'', below 1), independently: four deviations of the sum
            t = v @ at[1].T if i == 0 else at[0] @ v.T if i == 1 else v[None, :]
            z = pre.double()
            size = ((dy.double() * R.act(act, z)[1]).abs() + (dy.double() * z).abs()) * t.abs()
            assert abs(got - want) <= 4 * R.BF16_STEP * size.norm().item() + 1e-7 * abs(want), (act, i, got, want)


def test_dense_no_rows(cuda, inl):
    import torch
    x, w = _rand(torch, cuda, (0, 72), 1), _rand(torch, cuda, (40, 72), 2)
    assert inl.dense(x, w).shape == (0, 40)
    dx, dw, db = inl.dense_bwd(torch.empty(0, 40, dtype=torch.bfloat16, device=cuda), x, w, bias_grad=True)
    assert dx.shape == (0, 72) and not dw.any() and not db.any()


# ---------------------------------------------------------------------------
# Gated feed-forward block
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "gelu_erf", "relu"])
@pytest.mark.parametrize("m,hidden,inner", [(1, 8, 8), (2, 1032, 72), (7, 264, 520), (8, 64, 1024), (9, 72, 40),
                                            (65, 136, 200), (300, 264, 1032), (3001, 520, 264)])
def test_gated_ffn(m, hidden, inner, act, cuda, inl):
    import torch
    x = _rand(torch, cuda, (m, hidden), 21)
    wgu = _rand(torch, cuda, (2 * inner, hidden), 22, hidden ** -0.5)
    wd = _rand(torch, cuda, (hidden, inner), 23, inner ** -0.5)
    res = [None, _rand(torch, cuda, (m, hidden), 24), _rand(torch, cuda, (m, hidden), 24, 1.0, torch.float32)][m % 3]
    out = [torch.bfloat16, torch.float32][(m // 2) % 2]
    print(f"case=ffn {m} {hidden} {inner} {act}", flush=True)
    y, pre, h = inl.gated_ffn(x, wgu, wd, act=act, residual=res, save=True, out_dtype=out)
    assert torch.equal(y, inl.gated_ffn(x, wgu, wd, act=act, residual=res, out_dtype=out))
    gu = x.double() @ wgu.double().T
    gu_tol = R.sum_tol(hidden) * (x.double().abs() @ wgu.double().abs().T)
    R.check(pre, gu, gu_tol + R.out_tol(gu, torch.bfloat16), "pre")
    a, s = R.act(act, gu[:, :inner])
    ref = a * gu[:, inner:]
    h_tol = 1.13 * gu_tol[:, :inner] * gu[:, inner:].abs() + gu_tol[:, inner:] * a.abs() + \
        3e-7 * gu[:, :inner].abs() * gu[:, inner:].abs() + 2.0 ** -22 * ref.abs() + \
        1.13 * gu_tol[:, :inner] * gu_tol[:, inner:]
    R.check(h, ref, h_tol + R.out_tol(ref, torch.bfloat16), "h")
    hd, wdd = h.double(), wd.double()   # the h that the down projection read
    ref = hd @ wdd.T + (res.double() if res is not None else 0)
    R.check(y, ref, R.out_tol(ref, out) + R.sum_tol(inner) * (hd.abs() @ wdd.abs().T) + 2.0 ** -23 * ref.abs(), "y")


@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "gelu_erf", "relu"])
@pytest.mark.parametrize("m,hidden,inner", [(1, 8, 8), (3, 264, 72), (66, 136, 200), (777, 264, 520), (2050, 1032, 1032)])
def test_gated_ffn_bwd(m, hidden, inner, act, cuda, inl):
    import torch
    x, dy = _rand(torch, cuda, (m, hidden), 31), _rand(torch, cuda, (m, hidden), 32, 0.1)
    wgu = _rand(torch, cuda, (2 * inner, hidden), 33, hidden ** -0.5)
    wd = _rand(torch, cuda, (hidden, inner), 34, inner ** -0.5)
    pre, h = _rand(torch, cuda, (m, 2 * inner), 35), _rand(torch, cuda, (m, inner), 36)
    dt = torch.float32 if m % 2 else torch.bfloat16
    print(f"case=ffn_bwd {m} {hidden} {inner} {act}", flush=True)
    dx, dgu_w, dd_w = inl.gated_ffn_bwd(dy, x, wgu, wd, pre, h, act=act, dx_dtype=dt, dw_dtype=dt)
    dyd, wdd, xd, wgd = dy.double(), wd.double(), x.double(), wgu.double()
    dh = dyd @ wdd
    a, s = R.act(act, pre[:, :inner].double())
    dgu = R.r16(torch.cat([dh * pre[:, inner:].double() * s, dh * a], 1))
    # dh's own f32 error reaches dgu and from there the products: |u act'| and |act| times it
    dh_tol = R.sum_tol(hidden) * (dyd.abs() @ wdd.abs())
    e = torch.cat([1.13 * dh_tol * pre[:, inner:].double().abs(), dh_tol * a.abs()], 1) + 2.0 ** -20 * dgu.abs()
    ref = dgu @ wgd
    R.check(dx, ref, R.out_tol(ref, dt) + (R.sum_tol(2 * inner) * dgu.abs() + e) @ wgd.abs() + R.flips(dgu, wgd), "dx")
    ref = dgu.T.contiguous() @ xd
    R.check(dgu_w, ref, R.out_tol(ref, dt) + (R.sum_tol(m) * dgu.abs() + e).T.contiguous() @ xd.abs() + R.flips(dgu, xd), "dw_gate_up")
    ref = dyd.T.contiguous() @ h.double()
    R.check(dd_w, ref, R.out_tol(ref, dt) + R.sum_tol(m) * (dyd.abs().T.contiguous() @ h.double().abs()), "dw_down")


def test_gated_ffn_some_gradients(cuda, inl):
    """Gradients not asked for change nothing about the others."""
    import torch
    m, hidden, inner = 200, 72, 136
    x, dy = _rand(torch, cuda, (m, hidden), 31), _rand(torch, cuda, (m, hidden), 32, 0.1)
    wgu, wd = _rand(torch, cuda, (2 * inner, hidden), 33, 0.1), _rand(torch, cuda, (hidden, inner), 34, 0.1)
    _, pre, h = inl.gated_ffn(x, wgu, wd, save=True)
    whole = inl.gated_ffn_bwd(dy, x, wgu, wd, pre, h)
    a = inl.gated_ffn_bwd(dy, x, wgu, wd, pre, h, dw_grad=False)
    b = inl.gated_ffn_bwd(dy, x, wgu, wd, pre, h, dx_grad=False)
    assert torch.equal(a[0], whole[0]) and a[1] is None and a[2] is None
    assert b[0] is None and torch.equal(b[1], whole[1]) and torch.equal(b[2], whole[2])


# ---------------------------------------------------------------------------
# Softmax cross entropy
# ---------------------------------------------------------------------------

XENT = [(1, 1, 8, 1.0), (1, 50, 72, 1.0), (3, 129, 136, 1.0), (64, 64, 64, 20.0), (65, 1001, 264, 1.0),
        (130, 517, 40, 50.0), (700, 4099, 72, 1.0), (2100, 3001, 520, 0.5)]


def _xent_inputs(torch, dev, m, vocab, hidden, scale, ignored=True):
    x = _rand(torch, dev, (m, hidden), 41, 1.0 if scale <= 1 else hidden ** -0.5)
    w = _rand(torch, dev, (vocab, hidden), 42, hidden ** -0.5)
    b = _rand(torch, dev, (vocab,), 43, 0.5, torch.float32)
    g = torch.Generator(device=dev).manual_seed(44)
    t = torch.randint(0, vocab, (m,), generator=g, device=dev, dtype=torch.int32)
    if ignored and m > 2:
        t[::5] = -100
        t[1], t[2] = vocab - 1, 0
    return x, w, b, t


def _scores(x, w, b, scale):
    s = scale * (x.double() @ w.double().T) + (b.double() if b is not None else 0)
    tol = R.sum_tol(x.shape[1]) * abs(scale) * (x.double().abs() @ w.double().abs().T) + 2.0 ** -23 * s.abs()
    return s, tol


@pytest.mark.parametrize("m,vocab,hidden,scale", XENT)
@pytest.mark.parametrize("with_bias", [False, True])
def test_softmax_xent(m, vocab, hidden, scale, with_bias, cuda, inl):
    import torch
    x, w, b, t = _xent_inputs(torch, cuda, m, vocab, hidden, scale)
    b = b if with_bias else None
    print(f"case=xent {m} {vocab} {hidden}", flush=True)
    loss, lse = inl.softmax_xent(x, w, t, bias=b, scale=scale)
    s, tol = _scores(x, w, b, scale)
    want = torch.logsumexp(s, 1)
    # lse moves by at most the largest score's error; the sum of exponentials by
    # 3 f32 steps each and one per join of a block of at least 32 columns
    e = tol.max(1).values + (vocab / 32 + 40) * 2.0 ** -23 + 2.0 ** -22 * want.abs()
    R.check(lse, want, e, "lse")
    keep = t >= 0
    at = s.gather(1, t.clamp_min(0).long()[:, None])[:, 0]
    R.check(loss, torch.where(keep, want - at, 0.0), torch.where(keep, 2 * e, 0.0), "loss")


@pytest.mark.parametrize("m,vocab,hidden,scale", XENT + [(9000, 4700, 72, 1.0)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_softmax_xent_bwd(m, vocab, hidden, scale, with_bias, cuda, inl):
    """The last size takes two pieces of the vocabulary."""
    import torch
    x, w, b, t = _xent_inputs(torch, cuda, m, vocab, hidden, scale)
    b = b if with_bias else None
    dl = _rand(torch, cuda, (m,), 45, 1.0, torch.float32)
    s, tol = _scores(x, w, b, scale)
    lse = torch.logsumexp(s, 1).float()
    dt = torch.float32 if m % 2 else torch.bfloat16
    print(f"case=xent_bwd {m} {vocab} {hidden}", flush=True)
    dx, dw, db = inl.softmax_xent_bwd(dl, lse, x, w, t, bias=b, scale=scale, bias_grad=True, dx_dtype=dt, dw_dtype=dt)
    p = torch.exp(s - lse.double()[:, None])
    one = torch.arange(vocab, device=cuda)[None, :] == t.long()[:, None]
    d = torch.where(t >= 0, dl, 0.0).double()[:, None]
    g = R.r16(d * (p - one.double()))
    # the score's error moves p by that much of it; 2^-20 for exp and the product
    e = d.abs() * p * (tol + 2.0 ** -20) + 2.0 ** -22 * g.abs()
    xd, wd, a = x.double(), w.double(), abs(scale)
    ref = scale * (g @ wd)
    R.check(dx, ref, R.out_tol(ref, dt) + a * ((R.sum_tol(vocab) * g.abs() + e) @ wd.abs() + R.flips(g, wd)) +
            (vocab / 4096 + 1) * 2.0 ** -23 * ref.abs().max(), "dx")
    ref = scale * (g.T.contiguous() @ xd)
    R.check(dw, ref, R.out_tol(ref, dt) + a * ((R.sum_tol(m) * g.abs() + e).T.contiguous() @ xd.abs() + R.flips(g, xd)), "dw")
    R.check(db, g.sum(0), (m / 64 + 24) * 2.0 ** -24 * g.abs().sum(0) + e.sum(0) + 8 * R.BF16_STEP * g.abs().max(), "db")


def test_softmax_xent_targets_and_masks(cuda, inl):
    """Ignored rows have no loss and no gradient, whatever their scores are; a
    target outside the vocabulary is NaN; an entry masked by a bias of -inf or of
    the lowest float takes no part."""
    import torch
    m, vocab, hidden = 70, 300, 72
    x, w, b, t = _xent_inputs(torch, cuda, m, vocab, hidden, 1.0)
    b[100:250] = float("-inf")
    b[50] = torch.finfo(torch.float32).min
    t[(t >= 100) & (t < 250)] = 3
    t[t == 50] = 4
    loss, lse = inl.softmax_xent(x, w, t, bias=b)
    s, tol = _scores(x, w, b, 1.0)
    live = torch.ones(vocab, dtype=torch.bool, device=cuda)
    live[100:250] = False
    live[50] = False
    want = torch.logsumexp(s[:, live], 1)
    R.check(lse, want, tol[:, live].max() + 60 * 2.0 ** -23 + 2.0 ** -22 * want.abs(), "lse")
    assert (loss[t == -100] == 0).all()
    dl = torch.ones(m, device=cuda)
    dx, dw, db = inl.softmax_xent_bwd(dl, lse, x, w, t, bias=b, bias_grad=True)
    assert not dx[t == -100].any() and not dw[~live].any() and not db[~live].any()
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all()
    # every row ignored, and rows of NaN that are ignored
    xn = x.clone()
    xn[0] = float("nan")   # t[0] is ignored
    loss2, lse2 = inl.softmax_xent(xn, w, t, bias=b)
    assert torch.equal(loss2, loss) and torch.equal(lse2[1:], lse[1:])
    dx2, _, db2 = inl.softmax_xent_bwd(dl, lse2, xn, w, t, bias=b, bias_grad=True, dw_grad=False)
    assert torch.equal(dx2, dx) and torch.equal(db2, db)
    none = torch.full_like(t, -100)
    loss, lse = inl.softmax_xent(x, w, none)
    dx, dw, _ = inl.softmax_xent_bwd(dl, lse, x, w, none)
    assert not loss.any() and not dx.any() and not dw.any()
    for bad in (vocab, -1, 2 ** 31 - 1):
        tb = t.clone()
        tb[5] = bad
        lb, lse = inl.softmax_xent(x, w, tb)
        assert torch.isnan(lb[5]) and torch.isfinite(lb[torch.arange(m, device=cuda) != 5]).all()
        dx, _, _ = inl.softmax_xent_bwd(dl, lse, x, w, tb)
        assert torch.isnan(dx[5]).all() and torch.isfinite(dx[6:]).all()


def test_softmax_xent_wide_scores(cuda, inl):
    """Scores far apart: no overflow, and a row that knows its answer has a loss of
    0 within the scores' own error."""
    import torch
    m, vocab, hidden = 33, 200, 64
    w = torch.eye(vocab, hidden, device=cuda).to(torch.bfloat16) * 100
    x = torch.eye(m, hidden, device=cuda).to(torch.bfloat16) * 100
    t = torch.arange(m, device=cuda, dtype=torch.int32)
    loss, lse = inl.softmax_xent(x, w, t)
    assert torch.equal(loss, torch.zeros_like(loss)) and (lse == 10000).all()
    loss, lse = inl.softmax_xent(x, w, t, scale=-1.0)
    want = math.log(vocab - 1) + 10000
    assert ((loss.double() - want).abs() <= 2.0 ** -22 * want).all()


# ---------------------------------------------------------------------------
# q/k prologue
# ---------------------------------------------------------------------------

ROPE = [  # tokens, q heads, k heads, head_dim, rotary, sections
    (1, 1, 1, 8, 8, 1), (3, 2, 1, 16, 8, 3), (5, 3, 1, 64, 64, 1), (7, 4, 2, 64, 32, 3), (33, 16, 8, 128, 128, 1),
    (33, 16, 8, 128, 128, 3), (70, 3, 1, 256, 256, 1), (70, 3, 2, 256, 72, 3), (40, 5, 2, 128, 96, 1),
    (40, 6, 6, 64, 64, 2), (1030, 2, 1, 512, 512, 1), (600, 12, 12, 64, 0, 1), (2500, 8, 2, 32, 24, 3)]


def _tables(torch, dev, n, d, rotary, sections):
    cols = d // 4 if sections == 2 else rotary // 2
    g = torch.Generator(device=dev).manual_seed(54)
    a = torch.rand(2, 50, max(cols, 1), generator=g, device=dev) * 6.3
    rows = torch.randint(0, 50, (n,), generator=g, device=dev, dtype=torch.int32)
    t = [a[0].cos(), a[0].sin()] + ([a[1].cos(), a[1].sin()] if sections == 2 else [None, None])
    return rows, [v.contiguous() if v is not None else None for v in t]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("n,hq,hk,d,rotary,sections", ROPE)
def test_norm_rope_and_gradient(n, hq, hk, d, rotary, sections, norm, dtype, cuda, inl):
    import torch
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    heads = hq + hk
    x = _rand(torch, cuda, (n, heads + hk, d), 51, 1.0, dt)[:, :heads]   # q and k heads of q/k/v rows
    wq = (1 + _rand(torch, cuda, (d,), 52, 0.2, torch.float32)).to(dt)
    wk = (1 + _rand(torch, cuda, (d,), 53, 0.2, torch.float32)).to(dt)
    rows, tabs = _tables(torch, cuda, n, d, rotary, sections)
    if not rotary:
        rows, tabs = None, [None] * 4
    dy = _rand(torch, cuda, (n, heads, d), 55, 1.0, dt)
    kw = dict(q_weight=wq if norm else None, k_weight=wk if norm else None, norm=norm, rotary_dim=rotary,
              sections=sections, cos2=tabs[2], sin2=tabs[3])
    print(f"case=rope {n} {hq} {hk} {d} {rotary} {sections} {dtype}", flush=True)
    y = inl.norm_rope_qk(x, hq, rows, tabs[0], tabs[1], **kw)
    dx, dq, dk = inl.norm_rope_qk_bwd(dy, x, hq, rows, tabs[0], tabs[1], **kw)
    t64 = [v.double()[rows.long()] if v is not None else None for v in tabs]
    w = torch.cat([wq.double().expand(hq, d), wk.double().expand(hk, d)]) if norm else None
    xd, dyd = x.double(), dy.double()
    ref = R.norm_rope(xd, w, 1e-6, rotary, sections, t64)
    # some 8 f32 roundings per value and the two terms of a rotation, of the row's largest value
    big = lambda v: v.abs().amax(-1, keepdim=True)
    R.check(y, ref, R.out_tol(ref, dt) + 2.0 ** -20 * big(ref), "y")
    ref, dw = R.norm_rope_bwd(dyd, xd, w, 1e-6, rotary, sections, t64)
    # the two sums of a row (d / 8 terms a lane, then a tree) and 16 roundings, at
    # the row's largest dy weight / rms
    size = big(dyd) * (1.8 if norm else 1.0)
    if norm:
        size = size / torch.sqrt((xd * xd).mean(-1, keepdim=True) + 1e-6) * (1 + big(xd) / torch.sqrt((xd * xd).mean(-1, keepdim=True)))
    R.check(dx, ref, R.out_tol(ref, dt) + 32 * 2.0 ** -24 * 2 * size, "dx")
    if not norm:
        assert dq is None and dk is None
        return
    for got, part in ((dq, dw[:, :hq]), (dk, dw[:, hq:])):
        # in order per lane (tokens x heads / workgroups), then trees: bounded by
        # 64 + terms / 256 steps of the sum of sizes, and 16 roundings per term
        terms = part.shape[0] * part.shape[1]
        lim = (80 + terms / 64) * 2.0 ** -24 * (big(dyd)[:, :1] * 1.5 * (xd / torch.sqrt((xd * xd).mean(-1, keepdim=True) + 1e-6)).abs()).amax(0).amax(0) * terms
        R.check(got, part.sum((0, 1)), lim, "dweight")


def test_norm_rope_bwd_differences(cuda, inl):
    """Against central differences of the float64 forward, in f32."""
    import torch
    n, hq, hk, d = 9, 3, 2, 64
    x, dy = _rand(torch, cuda, (n, hq + hk, d), 61, 1.0, torch.float32), _rand(torch, cuda, (n, hq + hk, d), 62, 1.0, torch.float32)
    wq, wk = (1 + _rand(torch, cuda, (d,), s, 0.2, torch.float32) for s in (63, 64))
    for sections, rotary in ((1, 64), (3, 40), (2, 64)):
        rows, tabs = _tables(torch, cuda, n, d, rotary, sections)
        t64 = [v.double()[rows.long()] if v is not None else None for v in tabs]
        grads = inl.norm_rope_qk_bwd(dy, x, hq, rows, tabs[0], tabs[1], q_weight=wq, k_weight=wk, rotary_dim=rotary,
                                     sections=sections, cos2=tabs[2], sin2=tabs[3])
        at = [x.double(), wq.double(), wk.double()]

        def f(p):
            w = torch.cat([p[1].expand(hq, d), p[2].expand(hk, d)])
            return (dy.double() * R.norm_rope(p[0], w, 1e-6, rotary, sections, t64)).sum().item()
        for i, g in enumerate(grads):
            v = _rand(torch, cuda, at[i].shape, 65 + i, 1.0, torch.float32).double()
            e = 1e-5
            up, down = [t.clone() for t in at], [t.clone() for t in at]
            up[i] += e * v
            down[i] -= e * v
            want, got = (f(up) - f(down)) / (2 * e), (g.double() * v).sum().item()
            # f32 gradients: 2^-20 of the terms' sizes; the differences are good to 1e-8
            assert abs(got - want) <= 2.0 ** -20 * (g.double() * v).abs().sum().item() + 1e-7 * abs(want), (sections, i)


def test_norm_rope_bwd_in_place_and_bad_rows(cuda, inl):
    """dx over dy, dx as a slice of wider rows, and a token whose table row does
    not exist: NaN in its own gradient only (and in the weights')."""
    import torch
    n, hq, hk, d = 50, 4, 2, 128
    x, dy = _rand(torch, cuda, (n, hq + hk, d), 71), _rand(torch, cuda, (n, hq + hk, d), 72)
    wq, wk = _rand(torch, cuda, (d,), 73), _rand(torch, cuda, (d,), 74)
    rows, tabs = _tables(torch, cuda, n, d, d, 1)
    kw = dict(q_weight=wq, k_weight=wk)
    dx, dq, dk = inl.norm_rope_qk_bwd(dy, x, hq, rows, tabs[0], tabs[1], **kw)
    wide = torch.full((n, hq + 2 * hk, d), 7.0, dtype=torch.bfloat16, device=cuda)
    inl.norm_rope_qk_bwd(dy, x, hq, rows, tabs[0], tabs[1], out=wide[:, :hq + hk], **kw)
    assert torch.equal(wide[:, :hq + hk], dx) and (wide[:, hq + hk:] == 7).all()
    dy2 = dy.clone()
    got = inl.norm_rope_qk_bwd(dy2, x, hq, rows, tabs[0], tabs[1], out=dy2, **kw)
    assert torch.equal(dy2, dx) and torch.equal(got[1], dq) and torch.equal(got[2], dk)
    for bad in (50, -1, 2 ** 31 - 1):
        r = rows.clone()
        r[7] = bad
        b = inl.norm_rope_qk_bwd(dy, x, hq, r, tabs[0], tabs[1], **kw)
        keep = torch.arange(n, device=cuda) != 7
        assert torch.isnan(b[0][7]).all() and torch.equal(b[0][keep], dx[keep]) and torch.isnan(b[1]).all()
    # all heads q heads; no tokens
    only = inl.norm_rope_qk_bwd(dy, x, hq + hk, rows, tabs[0], tabs[1], q_weight=wq)
    assert only[2] is None and torch.equal(only[0][:, :hq], dx[:, :hq])
    none = inl.norm_rope_qk_bwd(dy[:0], x[:0], hq, rows[:0], tabs[0], tabs[1], **kw)
    assert none[0].shape == (0, hq + hk, d) and not none[1].any() and not none[2].any()


# ---------------------------------------------------------------------------
# Together, and how they are called
# ---------------------------------------------------------------------------

def _step(inl, torch, p):
    """A training step of what the ops cover of a layer and a head: projection,
    q/k prologue (its rows in place of attention's), block, loss and every
    gradient back to x."""
    n, heads, d = p["x"].shape[0], p["hq"] + p["hk"], p["d"]
    a = inl.dense(p["x"], p["w1"], p["b1"])
    q = inl.norm_rope_qk(a.view(n, heads, d), p["hq"], p["rows"], p["cos"], p["sin"], q_weight=p["wq"], k_weight=p["wk"])
    z = torch.empty(n, p["w2"].shape[0], dtype=torch.bfloat16, device=a.device)
    e = inl.dense(q.view(n, -1), p["w2"], p["b2"], act="gelu_erf", residual=p["x"], pre=z)
    f, gu, h = inl.gated_ffn(e, p["wgu"], p["wd"], residual=e, save=True)
    loss, lse = inl.softmax_xent(f, p["wv"], p["t"])
    dl = torch.full((n,), 1.0 / n, device=a.device)
    df, dwv, _ = inl.softmax_xent_bwd(dl, lse, f, p["wv"], p["t"])
    de, dwgu, dwd = inl.gated_ffn_bwd(df, e, p["wgu"], p["wd"], gu, h)
    de = de + df
    dq, dw2, db2 = inl.dense_bwd(de, q.view(n, -1), p["w2"], act="gelu_erf", pre=z, bias_grad=True)
    da, dwq, dwk = inl.norm_rope_qk_bwd(dq.view(n, heads, d), a.view(n, heads, d), p["hq"], p["rows"], p["cos"], p["sin"],
                                        q_weight=p["wq"], k_weight=p["wk"])
    dx, dw1, db1 = inl.dense_bwd(da.view(n, -1), p["x"], p["w1"], bias_grad=True)
    return dict(loss=loss, x=dx + de, w1=dw1, b1=db1, wq=dwq, wk=dwk, w2=dw2, b2=db2, wgu=dwgu, wd=dwd, wv=dwv)


def _step_inputs(torch, dev, n, seed=80):
    hidden, hq, hk, d, inner, vocab = 136, 3, 1, 64, 200, 1001
    r = lambda *s, std=1.0, dtype=None: _rand(torch, dev, s, seed + len(p), std, dtype)
    p = dict(hq=hq, hk=hk, d=d)
    p["x"] = r(n, hidden)
    p["w1"], p["b1"] = r(256, hidden, std=hidden ** -0.5), r(256, std=0.1, dtype=torch.float32)
    p["wq"], p["wk"] = (1 + r(d, std=0.1)), (1 + r(d, std=0.1))
    p["w2"], p["b2"] = r(hidden, 256, std=1 / 16), r(hidden, std=0.1, dtype=torch.float32)
    p["wgu"], p["wd"] = r(2 * inner, hidden, std=hidden ** -0.5), r(hidden, inner, std=inner ** -0.5)
    p["wv"] = r(vocab, hidden, std=hidden ** -0.5)
    g = torch.Generator(device=dev).manual_seed(seed)
    p["t"] = torch.randint(0, vocab, (n,), generator=g, device=dev, dtype=torch.int32)
    p["t"][::7] = -100
    p["rows"], tabs = _tables(torch, dev, n, d, d, 1)
    p["cos"], p["sin"] = tabs[0], tabs[1]
    return p


def _step_ref(torch, p):
    """The same step by autograd in float64."""
    v = {k: p[k].double().requires_grad_() for k in ("x", "w1", "b1", "wq", "wk", "w2", "b2", "wgu", "wd", "wv")}
    n, hq, hk, d, inner = p["x"].shape[0], p["hq"], p["hk"], p["d"], p["wd"].shape[1]
    a = v["x"] @ v["w1"].T + v["b1"]
    w = torch.cat([v["wq"].expand(hq, d), v["wk"].expand(hk, d)])
    c, s = p["cos"].double()[p["rows"].long()], p["sin"].double()[p["rows"].long()]
    q = R.norm_rope(a.view(n, hq + hk, d), w, 1e-6, d, 1, (c, s)).reshape(n, -1)
    e = R.act("gelu_erf", q @ v["w2"].T + v["b2"])[0] + v["x"]
    gu = e @ v["wgu"].T
    f = (R.act("silu", gu[:, :inner])[0] * gu[:, inner:]) @ v["wd"].T + e
    sc = f @ v["wv"].T
    t = p["t"].long()
    loss = torch.where(t >= 0, torch.logsumexp(sc, 1) - sc.gather(1, t.clamp_min(0)[:, None])[:, 0], 0.0)
    loss.sum().div(n).backward()
    return dict(loss=loss.detach(), **{k: t.grad for k, t in v.items()})


@pytest.mark.parametrize("n", [1, 40, 1300])
def test_training_step(n, cuda, inl):
    """Every gradient of the chain against float64 autograd. Each value passes some
    ten bf16 roundings on its way, independent ones: in norm within 10 x 2^-8."""
    import torch
    p = _step_inputs(torch, cuda, n)
    if n == 1:
        p["t"][0] = 5
    got, ref = _step(inl, torch, p), _step_ref(torch, p)
    for k in ref:
        err = (got[k].double() - ref[k]).norm().item()
        assert err <= 10 * 2.0 ** -8 * ref[k].norm().item(), (k, err / ref[k].norm().item())


def test_equal_calls_equal_bits(cuda, inl):
    import torch
    p = _step_inputs(torch, cuda, 900)
    a, b = _step(inl, torch, p), _step(inl, torch, p)
    assert all(torch.equal(a[k], b[k]) for k in a)


def test_captured_and_replayed(cuda, inl):
    """The step captured into a graph, replayed on new inputs with eager work
    between the replays."""
    import torch
    p, q = _step_inputs(torch, cuda, 500, 80), _step_inputs(torch, cuda, 500, 90)
    want = [_step(inl, torch, p), _step(inl, torch, q)]
    static = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in p.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(inl, torch, static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(inl, torch, static)
    for i in (0, 1, 0, 1):
        for k, v in (p, q)[i].items():
            if isinstance(v, torch.Tensor):
                static[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        eager = _step(inl, torch, (q, p)[i])
        assert all(torch.equal(out[k], want[i][k]) for k in out), i
        assert all(torch.equal(eager[k], want[1 - i][k]) for k in eager), i


def test_two_streams(cuda, inl):
    """Calls on two streams at a time, each with its own workspace."""
    import torch
    x, w = _rand(torch, cuda, (2000, 264), 1), _rand(torch, cuda, (520, 264), 2, 0.06)
    dy = _rand(torch, cuda, (2000, 520), 3, 0.1)
    want = inl.dense_bwd(dy, x, w, bias_grad=True)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [inl.dense_bwd(dy, x, w, bias_grad=True, stream=streams[i % 2]) for i in range(8)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_refusals(cuda, inl):
    import torch
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=cuda)
    x, w = z(4, 40), z(16, 40)
    bad = [
        lambda: inl.dense(z(4, 36), z(16, 36)), lambda: inl.dense(x, z(12, 40)), lambda: inl.dense(x, z(16, 48)),
        lambda: inl.dense(x, w, z(16)), lambda: inl.dense(x, w, z(8, dtype=torch.float32)),
        lambda: inl.dense(x, w, act="tanh"), lambda: inl.dense(x, w, residual=z(4, 8)),
        lambda: inl.dense(x.float(), w), lambda: inl.dense(x.cpu(), w), lambda: inl.dense(x, w.cpu()),
        lambda: inl.dense(z(4, 44)[:, :40], w), lambda: inl.dense(z(40, 4).T, w), lambda: inl.dense(z(4, 48)[:, 4:44], w),
        lambda: inl.dense(x, w, pre=z(4, 16, dtype=torch.float32)), lambda: inl.dense(x, w, out=z(4, 24)),
        lambda: inl.dense_bwd(z(4, 16), x, w, act="silu"), lambda: inl.dense_bwd(z(4, 8), x, w),
        lambda: inl.gated_ffn(x, z(32, 40), z(40, 8)), lambda: inl.gated_ffn(x, z(16, 40), z(40, 8), act=None),
        lambda: inl.gated_ffn(x, z(16, 48)[:, :40], z(40, 8)),
        lambda: inl.gated_ffn_bwd(x, x, z(16, 40), z(40, 8), z(4, 8), z(4, 8)),
        lambda: inl.softmax_xent(x, w, z(4, dtype=torch.int64)), lambda: inl.softmax_xent(x, w, z(3, dtype=torch.int32)),
        lambda: inl.softmax_xent(x, z(0, 40), z(4, dtype=torch.int32)),
        lambda: inl.softmax_xent(x, w, z(4, dtype=torch.int32), bias=z(16)),
        lambda: inl.softmax_xent_bwd(z(4), z(4, dtype=torch.float32), x, w, z(4, dtype=torch.int32)),
        lambda: inl.norm_rope_qk_bwd(z(4, 2, 64), z(4, 3, 64), 1), lambda: inl.norm_rope_qk_bwd(z(4, 3, 48), z(4, 3, 48), 1),
        lambda: inl.norm_rope_qk_bwd(z(4, 3, 64), z(4, 3, 64), 4),
        lambda: inl.norm_rope_qk(z(4, 3, 64), 1, z(4, dtype=torch.int32), z(9, 30, dtype=torch.float32),
                                 z(9, 30, dtype=torch.float32), rotary_dim=60, sections=3),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(inl.InlError):
            f()
            print("not refused:", i)


def test_softmax_xent_lowest_float_everywhere(cuda, inl):
    """A bias of the lowest float on every entry: all scores are that float, the
    softmax is uniform. -inf on all but one: that one has all of it."""
    import torch
    m, vocab, hidden = 20, 333, 72
    x, w, b, t = _xent_inputs(torch, cuda, m, vocab, hidden, 1.0, ignored=False)
    low = torch.full_like(b, torch.finfo(torch.float32).min)
    loss, lse = inl.softmax_xent(x, w, t, bias=low)
    assert (lse == low[0]).all()
    assert ((loss.double() - math.log(vocab)).abs() <= 2.0 ** -20).all()
    one = torch.full_like(b, float("-inf"))
    one[7] = 0
    t.fill_(7)
    loss, lse = inl.softmax_xent(x, w, t, bias=one)
    s, tol = _scores(x, w, None, 1.0)
    assert not loss.any() and ((lse.double() - s[:, 7]).abs() <= tol[:, 7]).all()
    dx, dw, db = inl.softmax_xent_bwd(torch.ones(m, device=cuda), lse, x, w, t, bias=one, bias_grad=True)
    # p of the one is 1 within the score's error, the others 0
    e = m * (tol[:, 7].max().item() * 2 + 2.0 ** -20)
    assert db.abs().max().item() <= e and dx.double().abs().max().item() <= e * w.double().abs().max().item() + 1e-30
    assert not dw[:7].any() and not dw[8:].any()


def test_dense_far_rows(cuda, inl):
    """Rows that start past 2^32 bytes, of x, y, the stored pre and the gradients."""
    import torch
    rows, wide, k, n = 280_000, 8192, 72, 40
    buf = torch.empty(rows, wide, dtype=torch.bfloat16, device=cuda)
    x, y, pre, dy = buf[:, 1024:1024 + k], buf[:, 2048:2048 + n], buf[:, 4096:4096 + n], buf[:, 6000:6000 + n]
    x.copy_(_rand(torch, cuda, (rows, k), 1))
    dy.copy_(_rand(torch, cuda, (rows, n), 2, 0.1))
    w = _rand(torch, cuda, (n, k), 3, k ** -0.5)
    print("case=dense far rows", flush=True)
    inl.dense(x, w, act="silu", pre=pre, out=y)
    z, ref, tol = _dense_ref(x, w, None, "silu", None)
    R.check(y, ref, tol + R.out_tol(ref, torch.bfloat16), "y")
    R.check(pre, z, tol + R.out_tol(z, torch.bfloat16), "pre")
    dx, dw, db = inl.dense_bwd(dy, x, w, act="silu", pre=pre, bias_grad=True)
    dz = R.r16(dy.double() * R.act("silu", pre.double())[1])
    ref = dz @ w.double()
    R.check(dx, ref, R.out_tol(ref, torch.bfloat16) + R.sum_tol(n) * (dz.abs() @ w.double().abs()) + R.flips(dz, w.double()), "dx")
    ref = dz.T.contiguous() @ x.double()
    # some 280,000 x 2^-14 values near the middle of two bf16 numbers, of either sign
    R.check(dw, ref, R.out_tol(ref, torch.bfloat16) + R.sum_tol(rows) * (dz.abs().T.contiguous() @ x.double().abs()) +
            2 * R.flips(dz, x.double()), "dw")


def test_first_call_in_a_capture(cuda, inl):
    """A shape that was never called before, captured at once."""
    import torch
    x, w = _rand(torch, cuda, (777, 200), 1), _rand(torch, cuda, (456, 200), 2, 0.07)
    dy = _rand(torch, cuda, (777, 456), 3, 0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = inl.dense(x, w)
        grads = inl.dense_bwd(dy, x, w, bias_grad=True)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        want = (inl.dense(x, w), *inl.dense_bwd(dy, x, w, bias_grad=True))
        assert all(torch.equal(a, b) for a, b in zip((y, *grads), want))


def test_results_do_not_depend_on_the_workspace(cuda, inl):
    """The C entries with a workspace of NaN and one of zeros, exactly as large as
    asked for, with guards behind it that stay as they were."""
    import ctypes

    import torch
    from inl_hip import train as T
    m, hidden, inner, vocab = 300, 136, 200, 1001
    x, dy = _rand(torch, cuda, (m, hidden), 1), _rand(torch, cuda, (m, hidden), 2, 0.1)
    wgu, wd = _rand(torch, cuda, (2 * inner, hidden), 3, 0.08), _rand(torch, cuda, (hidden, inner), 4, 0.07)
    wv = _rand(torch, cuda, (vocab, hidden), 5, 0.08)
    t = torch.arange(m, device=cuda, dtype=torch.int32)
    _, pre, h = inl.gated_ffn(x, wgu, wd, save=True)
    _, lse = inl.softmax_xent(x, wv, t)
    dl = torch.ones(m, device=cuda)
    st = torch.cuda.current_stream().cuda_stream
    p = lambda v: v.data_ptr()
    got = []
    for fill in (0, 255):
        def room(size_fn, desc, backward):
            n = ctypes.c_size_t()
            assert size_fn(desc, backward, ctypes.byref(n)) == 0
            buf = torch.full((n.value + 256,), fill, dtype=torch.uint8, device=cuda)
            return buf, n.value
        fd = T.GatedFfnDesc(m, hidden, inner, 0, 0, 0, 0, 2, 1, 0, 1, 1)
        xd = T.SoftmaxXentDesc(m, vocab, hidden, 0, 0, 0, 0, 1.0, -100, 1, 1)
        y, dx, dgu, dd = (torch.empty(s, dtype=torch.bfloat16, device=cuda)
                          for s in ((m, hidden), (m, hidden), (2 * inner, hidden), (hidden, inner)))
        loss, lse2 = torch.empty(m, device=cuda), torch.empty(m, device=cuda)
        dxx, dwv, db = torch.empty_like(x), torch.empty_like(wv), torch.empty(vocab, device=cuda)
        rooms = [room(T._ffn_ws, fd, 0), room(T._ffn_ws, fd, 1), room(T._xent_ws, xd, 0), room(T._xent_ws, xd, 1)]
        (a, na), (b, nb), (c, nc), (d, nd) = rooms
        assert T._ffn_fwd(fd, p(x), p(wgu), p(wd), None, p(y), None, None, p(a), na, st) == 0
        assert T._ffn_bwd(fd, p(dy), p(x), p(wgu), p(wd), p(pre), p(h), p(dx), p(dgu), p(dd), p(b), nb, st) == 0
        assert T._xent_fwd(xd, p(x), p(wv), None, p(t), p(loss), p(lse2), p(c), nc, st) == 0
        assert T._xent_bwd(xd, p(dl), p(lse), p(x), p(wv), None, p(t), p(dxx), p(dwv), p(db), p(d), nd, st) == 0
        torch.cuda.synchronize()
        assert all((buf[n:] == fill).all() for buf, n in rooms)
        got.append((y, dx, dgu, dd, loss, lse2, dxx, dwv, db))
    assert all(torch.equal(u, v) for u, v in zip(*got))


def test_overlapping_rows_and_wrong_ranks_are_refused(cuda, inl):
    """Expanded rows (the gradient of a sum) have a stride of 0, which the library
    reads as packed rows: they are refused, as are vectors for matrices."""
    import torch
    dev = cuda
    m, n, k = 24, 64, 32
    x, w, dy = (_rand(torch, dev, s, 7 + i) for i, s in enumerate([(m, k), (n, k), (m, n)]))
    wide = lambda cols: torch.ones((1, cols), dtype=torch.bfloat16, device=dev).expand(m, cols)
    gu, down = _rand(torch, dev, (2 * n, k), 20), _rand(torch, dev, (k, n), 21)
    targets = torch.zeros(m, dtype=torch.int32, device=dev)
    ones = torch.ones(m, device=dev)
    heads = _rand(torch, dev, (m, 3, 64), 22)
    flat = torch.ones((1, 3, 64), dtype=torch.bfloat16, device=dev).expand(m, 3, 64)
    slid = torch.zeros(m + k, dtype=torch.bfloat16, device=dev).as_strided((m, k), (1, 1))
    for call in (lambda: inl.dense(wide(k), w), lambda: inl.dense(slid, w), lambda: inl.dense(x[0], w),
                 lambda: inl.dense(x, w[0]), lambda: inl.dense(x, w, residual=wide(n)),
                 lambda: inl.dense(x, w, out=wide(n)), lambda: inl.dense_bwd(wide(n), x, w),
                 lambda: inl.dense_bwd(dy, x, w, act="silu", pre=wide(n)),
                 lambda: inl.gated_ffn(wide(k), gu, down), lambda: inl.gated_ffn(x, gu, down[0]),
                 lambda: inl.gated_ffn(x, gu, down, residual=wide(k)),
                 lambda: inl.softmax_xent(wide(k), w, targets), lambda: inl.softmax_xent(x[0], w, targets),
                 lambda: inl.softmax_xent(x, w, targets, ignore_index=2 ** 32),
                 lambda: inl.softmax_xent_bwd(ones[:1].expand(m), ones, x, w, targets),
                 lambda: inl.softmax_xent_bwd(ones, ones, x, wide(k), targets),
                 lambda: inl.norm_rope_qk_bwd(flat, heads, 2), lambda: inl.norm_rope_qk_bwd(heads, flat, 2),
                 lambda: inl.norm_rope_qk_bwd(heads, heads, 2, out=flat)):
        with pytest.raises(inl.InlError):
            call()
    one = torch.ones((1, k), dtype=torch.bfloat16, device=dev).expand(1, k)   # one row has no stride
    assert torch.equal(inl.dense(one, w), inl.dense(one.contiguous(), w))


@pytest.mark.parametrize("m", [1, 2])
def test_softmax_xent_very_wide(m, cuda, inl):
    """More vocabulary than a piece may be wide with a few rows."""
    test_softmax_xent(m, 2 ** 21 + 4099, 8, 1.0, True, cuda, inl)
    test_softmax_xent_bwd(m, 2 ** 21 + 4099, 8, 1.0, True, cuda, inl)


# both sides of the rules that choose a kernel for a few rows
FEW = [(5, 24, 40), (16, 1000, 1032), (16, 4096, 1024), (16, 4104, 2056), (17, 520, 264), (32, 4104, 72), (31, 264, 2040),
       (32, 8, 2056), (33, 264, 264), (4, 8200, 2040), (3, 8208, 2056)]


@pytest.mark.parametrize("act", [None, "gelu_erf"])
@pytest.mark.parametrize("m,n,k", FEW)
def test_dense_few_rows(m, n, k, act, cuda, inl):
    """With a neighbour on every side that stays as it was."""
    import torch
    x, w = _rand(torch, cuda, (m, k + 8), 1)[:, :k], _rand(torch, cuda, (n, k + 16), 2, k ** -0.5)[:, :k]
    b = _rand(torch, cuda, (n,), 3, 0.5, torch.float32)
    res = _rand(torch, cuda, (m, n), 4, 1.0, torch.float32 if m % 2 else torch.bfloat16)
    out = torch.full((m + 2, n + 16), 7.0, dtype=torch.bfloat16 if n % 16 else torch.float32, device=cuda)
    pre = torch.full((m + 2, n + 8), 7.0, dtype=torch.bfloat16, device=cuda)
    print(f"case=few {m} {n} {k} act={act}", flush=True)
    y = inl.dense(x, w, b, act=act, residual=res, pre=pre[1:-1, :n], out=out[1:-1, 8:-8])
    z, ref, tol = _dense_ref(x, w, b, act, res)
    R.check(y, ref, tol + R.out_tol(ref, out.dtype), "y")
    R.check(pre[1:-1, :n], z, tol + R.out_tol(z, torch.bfloat16), "pre")
    for t, inside in ((out, (slice(1, -1), slice(8, -8))), (pre, (slice(1, -1), slice(0, n)))):
        t[inside] = 7.0
        assert (t == 7.0).all()


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("m,hidden,inner", [(5, 40, 24), (16, 1024, 2816), (32, 1024, 4096), (24, 4104, 264), (33, 72, 136)])
def test_gated_ffn_few_rows(m, hidden, inner, act, cuda, inl):
    """Either product by either kernel."""
    test_gated_ffn(m, hidden, inner, act, cuda, inl)
