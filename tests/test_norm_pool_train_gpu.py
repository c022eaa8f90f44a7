"""The residual stream's addition, dropout and norm, and the pooling's gradients, against float64.
Bounds: step_ref.py."""
import pytest

import step_ref as S
import train_ref as R

pytestmark = pytest.mark.gpu


def _randn(torch, dev, shape, seed, std=1.0, dtype=None):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * std).to(dtype or torch.float32)


def _dt(torch, name):
    return torch.bfloat16 if name == "bf16" else torch.float32


NORM_CASES = [
    # one row, few rows, every width class (one wave per row to 2,048, a workgroup above), odd widths
    (1, 8, "bf16", "bf16", "bf16", 0.0), (1, 1024, "bf16", "f32", "bf16", 0.0), (3, 16, "f32", "f32", "f32", 0.5),
    (5, 504, "bf16", "f32", "bf16", 0.1), (7, 512, "f32", "bf16", "bf16", 0.0), (1025, 520, "bf16", "bf16", "f32", 0.3),
    (4099, 768, "bf16", "f32", "bf16", 0.1), (33, 1032, "f32", "f32", "bf16", 0.1), (130, 2048, "bf16", "bf16", "bf16", 0.2),
    (9, 2056, "bf16", "f32", "f32", 0.1), (70, 4096, "f32", "bf16", "bf16", 0.1), (1300, 4104, "bf16", "bf16", "bf16", 0.1),
    (6, 8192, "bf16", "f32", "bf16", 0.9), (5, 16384, "f32", "f32", "f32", 0.1), (3, 8200, "bf16", "bf16", "bf16", 0.0)]


@pytest.mark.parametrize("m,n,x,stream,out,dropout", NORM_CASES)
def test_add_rms_norm(m, n, x, stream, out, dropout, cuda, inl):
    import torch
    print(f"case=add_norm {m} {n} {x} {stream} {out} {dropout}", flush=True)
    xs = _randn(torch, cuda, (m, n), 1, 1.0, _dt(torch, x))
    r = _randn(torch, cuda, (m, n), 2, 2.0, _dt(torch, stream))
    seed, step, tag = 0x123456789ABCDEF, 77, 5
    rng = torch.tensor([seed, step], device=cuda)
    f = S.factor(m, n, dropout, seed, step, tag, cuda)
    for w in (_randn(torch, cuda, (n,), 3, 1.0, torch.bfloat16), _randn(torch, cuda, (n,), 4), None):
        for res in (r, None):
            y, h = inl.add_rms_norm(xs, w, residual=res, dropout=dropout, rng=rng, tag=tag, out_dtype=_dt(torch, out))
            torch.cuda.synchronize()
            S.check_add_norm(y, h, xs, w, res, f, 1e-6, "fwd")
    dy = _randn(torch, cuda, (m, n), 5, 0.1, _dt(torch, out))
    dh = _randn(torch, cuda, (m, n), 6, 0.1, _dt(torch, stream))
    for w in (_randn(torch, cuda, (n,), 3, 1.0, torch.bfloat16), None):
        for past in (dh, None):
            got = inl.add_rms_norm_bwd(dy, r, w, dh=past, dropout=dropout, rng=rng, tag=tag, dx_dtype=_dt(torch, x))
            torch.cuda.synchronize()
            assert (got[2] is None) == (w is None) and got[0].dtype == xs.dtype and got[1].dtype == r.dtype
            S.check_add_norm_bwd(got, dy, r, w, past, f, 1e-6, "bwd")


def test_many_rows(cuda, inl):
    """More rows than the gradient's workgroups take in one turn."""
    import torch
    m, n = 40001, 256
    h, dy = _randn(torch, cuda, (m, n), 1, 2.0, torch.bfloat16), _randn(torch, cuda, (m, n), 2, 0.1, torch.bfloat16)
    w = _randn(torch, cuda, (n,), 3)
    one = torch.ones((), dtype=torch.float64, device=cuda)
    S.check_add_norm_bwd(inl.add_rms_norm_bwd(dy, h, w), dy, h, w, None, one, 1e-6, "bwd")
    a, b = (inl.add_rms_norm_bwd(dy, h, w) for _ in range(2))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_far_values(cuda, inl):
    """Rows of zeros, tiny and large values, and NaN and infinities that stay in their row."""
    import torch
    m, n = 9, 264
    x = _randn(torch, cuda, (m, n), 1)
    x[0] = 0
    x[1] *= 1e-18
    x[2] *= 1e16
    one = torch.ones((), dtype=torch.float64, device=cuda)
    y, h = inl.add_rms_norm(x, eps=1e-12)
    S.check_add_norm(y, h, x, None, None, one, 1e-12, "far")
    assert not y[0].any() and h is x
    bad = x.clone()
    bad[4, 100], bad[7, 3] = float("nan"), float("inf")
    y2, _ = inl.add_rms_norm(bad, eps=1e-12)
    keep = [0, 1, 2, 3, 5, 6, 8]
    assert torch.equal(y2[keep], y[keep]) and torch.isnan(y2[4]).all()
    dy = _randn(torch, cuda, (m, n), 2, 0.1)
    good, got = inl.add_rms_norm_bwd(dy, x, eps=1e-12), inl.add_rms_norm_bwd(dy, bad, eps=1e-12)
    assert torch.equal(got[0][keep], good[0][keep])
    # what is dropped does not come back, whatever it was
    rng = torch.tensor([3, 4], device=cuda)
    f = S.factor(m, n, 0.5, 3, 4, 0, cuda)
    r = torch.zeros_like(x)
    _, h2 = inl.add_rms_norm(torch.full_like(x, float("nan")), residual=r, dropout=0.5, rng=rng)
    assert torch.equal(torch.isnan(h2), f != 0) and not h2[f == 0].any()


def test_strides_and_places(cuda, inl):
    """Rows of wider buffers; the sum in the residual's place, y in x's; the gradient in dy's and dh's."""
    import torch
    m, n = 37, 520
    wide = _randn(torch, cuda, (m, 3 * n), 1, 1.0, torch.bfloat16)
    x, r = wide[:, :n], wide[:, n:2 * n]
    w = _randn(torch, cuda, (n,), 2)
    y, h = inl.add_rms_norm(x.contiguous(), w, residual=r.contiguous())
    y2, h2 = inl.add_rms_norm(x, w, residual=r)
    assert torch.equal(y, y2) and torch.equal(h, h2)
    dy, dh = _randn(torch, cuda, (m, n), 3, 0.1, torch.bfloat16), _randn(torch, cuda, (m, n), 4, 0.1, torch.bfloat16)
    want = inl.add_rms_norm_bwd(dy, h, w, dh=dh)
    keep = wide[:, 2 * n:].clone()
    y3, h3 = inl.add_rms_norm(x, w, residual=r, out=x, sum_out=r)
    assert y3 is x and h3 is r and torch.equal(x, y) and torch.equal(r, h) and torch.equal(wide[:, 2 * n:], keep)
    got = inl.add_rms_norm_bwd(dy, r, w, dh=dh)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[0] is got[1]
    parts = inl.add_rms_norm_bwd(dy, r, w, dh=dh, residual_grad=False, weight_grad=False)
    assert torch.equal(parts[0], want[0]) and parts[1] is None and parts[2] is None
    parts = inl.add_rms_norm_bwd(dy, r, w, dh=dh, x_grad=False, dropout=0.5)
    assert parts[0] is None and torch.equal(parts[1], want[1])


def test_dropout_mask(cuda, inl):
    """The mask is the same in both directions, and another one for another seed, step or tag; how
    many are kept is binomial (six deviations)."""
    import torch
    m, n, p = 515, 1024, 0.25
    x = torch.ones(m, n, device=cuda)
    r = torch.zeros(m, n, device=cuda)
    masks = []
    for seed, step, tag in ((1, 1, 1), (2, 1, 1), (1, 2, 1), (1, 1, 2), (-5, 2 ** 31 + 7, 0xFFFFFFFF)):
        rng = torch.tensor([seed, step], device=cuda)
        _, h = inl.add_rms_norm(x, residual=r, dropout=p, rng=rng, tag=tag)
        f = S.factor(m, n, p, seed % 2 ** 64, step, tag, cuda)
        assert torch.equal(h.double() != 0, f != 0)
        kept = (h != 0).sum().item()
        assert abs(kept - m * n * (1 - p)) < 6 * (m * n * p * (1 - p)) ** 0.5
        dx, dres, _ = inl.add_rms_norm_bwd(x, x, dh=x, dropout=p, rng=rng, tag=tag)
        assert torch.equal(dx != 0, h != 0) and (dres != 0).all()
        masks.append(h != 0)
    for i in range(len(masks)):
        for j in range(i):
            same = (masks[i] == masks[j]).sum().item()
            assert abs(same - m * n * (p * p + (1 - p) ** 2)) < 6 * (m * n) ** 0.5 / 2


def test_captured_dropout_follows_the_step(cuda, inl):
    import torch
    m, n = 64, 768
    x, r = _randn(torch, cuda, (m, n), 1, 1.0, torch.bfloat16), _randn(torch, cuda, (m, n), 2)
    w = _randn(torch, cuda, (n,), 3)
    dy = _randn(torch, cuda, (m, n), 4, 0.1, torch.bfloat16)
    rng = torch.tensor([9, 0], device=cuda)

    def both():
        y, h = inl.add_rms_norm(x, w, residual=r, dropout=0.2, rng=rng, tag=3, out_dtype=torch.bfloat16)
        return (y, h) + inl.add_rms_norm_bwd(dy, h, w, dh=r, dropout=0.2, rng=rng, tag=3)
    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    seen = []
    for i in range(4):
        rng[1] += 1
        want = both()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
        seen.append(got[1].clone())
    assert not torch.equal(seen[0], seen[1])


CUS = [[0, 5], [0, 0, 1, 1, 40, 40], [0, 31, 32, 33, 97, 400], [0, 700], [0] + list(range(3, 603, 3))]


@pytest.mark.parametrize("extra", [0, 45])
@pytest.mark.parametrize("dim", [8, 64, 100, 768, 1024, 2048, 2056])
def test_pool_mean_bwd(dim, extra, cuda, inl):
    """Empty texts, texts that end inside a block of rows, rows behind the last text, odd widths."""
    import torch
    for cu in CUS:
        rows, texts = cu[-1] + extra, len(cu) - 1
        dp, mean = _randn(torch, cuda, (texts, dim), 1, 0.1), _randn(torch, cuda, (texts, dim), 2, 0.3)
        dev = torch.tensor(cu, dtype=torch.int32, device=cuda)
        for m in (None, mean):
            for dtype in (torch.bfloat16, torch.float32):
                print(f"case=pool_mean_bwd {dim} {texts} {rows} {m is not None} {dtype}", flush=True)
                if dtype == torch.bfloat16 and dim % 8:
                    wide = torch.full((rows, dim + 4), 7.0, dtype=dtype, device=cuda)
                    got = inl.pool_mean_bwd(dp, dev, rows, mean=m, out=wide[:, :dim])
                    assert (wide[:, dim:] == 7).all()
                else:
                    got = inl.pool_mean_bwd(dp, dev, rows, mean=m, dtype=dtype)
                torch.cuda.synchronize()
                ref, size = S.mean_bwd(dp, cu, rows, m)
                # two sums of dim terms, root, quotients
                R.check(got, ref, (dim / 256 + 24) * 2.0 ** -24 * 2 * size + R.out_tol(ref, dtype) + 1e-30, "dhidden")


def test_pool_mean_bwd_is_the_forwards(cuda, inl):
    """Against differences of pool_mean itself, through its unit length."""
    import torch
    cu = [0, 7, 40]
    dev = torch.tensor(cu, dtype=torch.int32, device=cuda)
    x, dp = _randn(torch, cuda, (40, 64), 1), _randn(torch, cuda, (2, 64), 2)
    way = _randn(torch, cuda, (40, 64), 3)
    mean = inl.pool_mean(x, dev)
    dx = inl.pool_mean_bwd(dp, dev, 40, mean=mean, dtype=torch.float32)

    def loss(v):
        m = torch.stack([v[a:b].mean(0) for a, b in zip(cu[:-1], cu[1:])])
        return ((m / torch.sqrt((m * m).sum(1, keepdim=True) + 1e-12)) * dp.double()).sum()
    h = 1e-5
    diff = (loss(x.double() + h * way) - loss(x.double() - h * way)) / (2 * h)
    _, size = S.mean_bwd(dp, cu, 40, mean)
    assert abs((dx.double() * way).sum() - diff) <= 2.0 ** -18 * (size * way.abs()).sum() + 1e-6


@pytest.mark.parametrize("extra", [0, 45])
@pytest.mark.parametrize("dim", [8, 100, 768, 1024, 2056])
def test_pool_last_bwd(dim, extra, cuda, inl):
    import torch
    for cu in CUS:
        rows, texts = cu[-1] + extra, len(cu) - 1
        dp = _randn(torch, cuda, (texts, dim), 1, 0.1)
        dev = torch.tensor(cu, dtype=torch.int32, device=cuda)
        for dtype, out in ((torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16), (torch.float32, torch.float32),
                           (torch.bfloat16, torch.float32)):
            if dim % 8 and torch.bfloat16 in (dtype, out):
                continue
            x = _randn(torch, cuda, (rows, dim), 3, 2.0, dtype)
            for w in (_randn(torch, cuda, (dim,), 4, 1.0, dtype), None):
                print(f"case=pool_last_bwd {dim} {texts} {rows} {dtype} {out} {w is not None}", flush=True)
                got, dw = inl.pool_last_bwd(dp, x, dev, w, dtype=out)
                torch.cuda.synchronize()
                ref, size, rdw, dw_size = S.last_bwd(dp, x, cu, w, 1e-6)
                e = (dim / 256 + 32) * 2.0 ** -24 * 4
                R.check(got, ref, e * size + R.out_tol(ref, out) + 1e-30, "dhidden")
                assert (dw is None) == (w is None)
                if dw is not None:
                    R.check(dw, rdw, (e + texts * 2.0 ** -24) * dw_size + 1e-30, "dweight")


def test_pool_gradients_in_a_graph(cuda, inl):
    """cu is read when the call runs: a replay follows it."""
    import torch
    dim, rows = 768, 300
    dp = _randn(torch, cuda, (3, dim), 1, 0.1)
    x, w = _randn(torch, cuda, (rows, dim), 2, 2.0, torch.bfloat16), _randn(torch, cuda, (dim,), 3, 1.0, torch.bfloat16)
    cu = torch.tensor([0, 10, 200, 300], dtype=torch.int32, device=cuda)
    both = lambda: (inl.pool_mean_bwd(dp, cu, rows),) + inl.pool_last_bwd(dp, x, cu, w)
    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for at in ([0, 10, 200, 300], [0, 0, 0, 1], [0, 99, 100, 250], [0, 10, 200, 300]):
        cu.copy_(torch.tensor(at, dtype=torch.int32))
        want = both()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), at
        ref, _ = S.mean_bwd(dp, at, rows, None)
        R.check(got[0], ref, R.out_tol(ref, torch.bfloat16) + 2.0 ** -22 * ref.abs(), at)


def test_streams(cuda, inl):
    import torch
    m, n = 700, 768
    x, r, w = _randn(torch, cuda, (m, n), 1, 1.0, torch.bfloat16), _randn(torch, cuda, (m, n), 2), _randn(torch, cuda, (n,), 3)
    dy = _randn(torch, cuda, (m, n), 4, 0.1, torch.bfloat16)
    cu = torch.tensor([0, 300, 700], dtype=torch.int32, device=cuda)
    dp = _randn(torch, cuda, (2, n), 5)
    calls = [lambda s: inl.add_rms_norm(x, w, residual=r, stream=s), lambda s: inl.add_rms_norm_bwd(dy, r, w, stream=s),
             lambda s: (inl.pool_mean_bwd(dp, cu, m, stream=s),),
             lambda s: inl.pool_last_bwd(dp, r, cu, w, stream=s)]
    want = [c(None) for c in calls]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = [[c(s) for c in calls] for s in sides]
        torch.cuda.synchronize()
        for one in got:
            for a, b in zip(one, want):
                assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_nothing_to_do(cuda, inl):
    import torch
    e = torch.empty(0, 64, dtype=torch.bfloat16, device=cuda)
    w = torch.ones(64, device=cuda)
    y, h = inl.add_rms_norm(e, w)
    assert y.shape == h.shape == (0, 64)
    dx, _, dw = inl.add_rms_norm_bwd(e, e, w)
    assert dx.shape == (0, 64) and not dw.any()
    cu = torch.zeros(3, dtype=torch.int32, device=cuda)
    dp = torch.ones(2, 64, device=cuda)
    assert not inl.pool_mean_bwd(dp, cu, 5).any() and inl.pool_mean_bwd(dp, cu, 0).shape == (0, 64)
    x = torch.ones(5, 64, device=cuda)
    dx, dw = inl.pool_last_bwd(dp, x, cu, w)
    assert not dx.any() and not dw.any()
    none = torch.empty(0, 64, device=cuda)
    assert not inl.pool_mean_bwd(none, cu[:1], 5).any()
    dx, dw = inl.pool_last_bwd(none, x, cu[:1], w)
    assert not dx.any() and not dw.any()
    dx, dw = inl.pool_last_bwd(dp, none, cu, w)
    assert dx.shape == (0, 64) and not dw.any()


def test_sum_in_x(cuda, inl):
    """The sum in x's place, with and without something to add; y in x's place where the sum is x."""
    import torch
    m, n = 21, 264
    r = _randn(torch, cuda, (m, n), 1, 1.0, torch.bfloat16)
    rng = torch.tensor([5, 6], device=cuda)
    for residual, dropout in ((r, 0.0), (None, 0.3), (r, 0.3), (None, 0.0)):
        x = _randn(torch, cuda, (m, n), 2, 1.0, torch.bfloat16)
        want = inl.add_rms_norm(x.clone(), residual=residual, dropout=dropout, rng=rng)
        y, h = inl.add_rms_norm(x, residual=residual, dropout=dropout, rng=rng, sum_out=x)
        assert h is x and torch.equal(y, want[0]) and torch.equal(x, want[1])
    x = _randn(torch, cuda, (m, n), 2, 1.0, torch.bfloat16)
    want = inl.add_rms_norm(x.clone())
    with pytest.raises(inl.InlError, match="overlaps"):
        inl.add_rms_norm(x, out=x, sum_out=x)
    y, h = inl.add_rms_norm(x, out=x)
    assert y is x and torch.equal(y, want[0]) and torch.equal(h, want[1])


def test_more_rows_than_one_grid_has_threads_for(cuda, inl):
    import torch
    m, n = 2 ** 26 + 5, 8
    x = torch.empty(m, n, dtype=torch.bfloat16, device=cuda)
    x[:] = _randn(torch, cuda, (1, n), 1, 1.0, torch.bfloat16)
    x[-3:] *= 2
    r = torch.zeros_like(x)
    y, h = inl.add_rms_norm(x, residual=r, eps=0.0)
    assert torch.equal(h, x)
    one = torch.ones((), dtype=torch.float64, device=cuda)
    for rows in (slice(0, 9), slice(2 ** 24 - 4, 2 ** 24 + 4), slice(m - 9, m)):
        S.check_add_norm(y[rows], h[rows], x[rows], None, None, one, 0.0, f"rows {rows}")
    assert torch.equal(y[1:-3], y[:1].expand(m - 4, n))
