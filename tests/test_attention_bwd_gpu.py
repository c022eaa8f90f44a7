"""Gradients of packed attention (inl_attn_varlen_bwd) against float64, at the lengths, masks,
head layouts and strides where they can go wrong. Bounds: attn_bwd_ref.py."""
import pytest

import attn_bwd_ref as A

pytestmark = pytest.mark.gpu


def _inputs(torch, dev, lengths, hq, hkv, hd, seed, std=1.5):
    g = torch.Generator(device=dev).manual_seed(seed)
    n = sum(lengths)
    rows = torch.randn(n, hq + 2 * hkv, hd, generator=g, device=dev)
    rows[:, :hq] *= std
    rows = rows.to(torch.bfloat16)
    dout = (0.1 * torch.randn(n, hq, hd, generator=g, device=dev)).to(torch.bfloat16)
    starts = [sum(lengths[:i]) for i in range(len(lengths))]
    return rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:], dout, starts, starts + [n]


def _case(inl, torch, dev, lengths, hq, hkv, hd, causal, window, seed=0, scale=None, **kw):
    print(f"case=attn_bwd {lengths} {hq}/{hkv} x {hd} causal={causal} window={window} {sorted(kw)}", flush=True)
    q, k, v, dout, starts, cu = _inputs(torch, dev, lengths, hq, hkv, hd, seed)
    scale = hd ** -0.5 if scale is None else scale
    out = A.forward(q, k, v, starts, lengths, causal, window, scale).to(torch.bfloat16)
    got = inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=causal, window=window, scale=scale, **kw)
    torch.cuda.synchronize()
    A.check(got, A.backward(dout, q, k, v, out, starts, lengths, causal, window, scale), lengths)
    return got


MASKS = [(False, -1), (True, -1), (False, 0), (False, 5), (True, 5), (False, 64), (True, 200)]


@pytest.mark.parametrize("causal,window", MASKS)
@pytest.mark.parametrize("hq,hkv,hd", [(2, 1, 64), (4, 2, 128), (3, 1, 256)])
def test_masks_and_lengths(hq, hkv, hd, causal, window, cuda, inl):
    """Lengths around the blocks of 32, 64 and 128 rows, texts of one token and of none."""
    import torch
    _case(inl, torch, cuda, [1, 0, 31, 32, 33, 0, 63, 65, 127, 129, 200, 2], hq, hkv, hd, causal, window)


@pytest.mark.parametrize("hd", [8, 16, 40, 72, 80, 120, 136, 192, 248])
def test_head_dims(hd, cuda, inl):
    import torch
    _case(inl, torch, cuda, [70, 3, 129], 4, 2, hd, True, -1, seed=hd)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (5, 5), (16, 2), (7, 1), (16, 8), (12, 12)])
def test_head_layouts(hq, hkv, cuda, inl):
    import torch
    _case(inl, torch, cuda, [100, 37], hq, hkv, 64, False, -1)
    _case(inl, torch, cuda, [100, 37], hq, hkv, 128, True, -1)


@pytest.mark.parametrize("lengths,hd,causal,window", [
    ([1537], 128, True, -1), ([1100, 5], 256, False, 512), ([2050], 64, False, 64), ([1], 128, True, -1),
    ([1100], 256, True, -1)])
def test_long_texts(lengths, hd, causal, window, cuda, inl):
    import torch
    _case(inl, torch, cuda, lengths, 2, 1, hd, causal, window)


def test_many_texts(cuda, inl):
    """More texts than a launch carries."""
    import torch
    g = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 9, (700,), generator=g).tolist()
    lengths[500] = 140
    _case(inl, torch, cuda, lengths, 2, 1, 64, False, -1)
    _case(inl, torch, cuda, [3] * 256, 2, 2, 64, True, -1)
    _case(inl, torch, cuda, [3] * 257, 2, 2, 64, True, -1)


def test_peaked_and_flat_scores(cuda, inl):
    """Scores in the hundreds, equal scores, and a scale near zero."""
    import torch
    for scale in (4.0, 1e-3, 1e-36):
        _case(inl, torch, cuda, [90, 130], 2, 1, 64, True, -1, scale=scale)


def test_f32_gradients_and_parts(cuda, inl):
    import torch
    got = _case(inl, torch, cuda, [90, 131], 4, 2, 128, True, -1, grad_dtype=torch.float32)
    assert all(x.dtype == torch.float32 for x in got)
    few = _case(inl, torch, cuda, [90, 131], 4, 2, 128, True, -1, grad_dtype=torch.float32, kv_grad=False)
    assert few[1] is None and few[2] is None and torch.equal(few[0], got[0])


def test_slices_of_one_row(cuda, inl):
    """dq, dk, dv into the heads of one fused row, and rows of no text left alone."""
    import torch
    lengths, hq, hkv, hd = [33, 64, 5], 4, 2, 80
    q, k, v, dout, starts, cu = _inputs(torch, cuda, lengths, hq, hkv, hd, 7)
    out = A.forward(q, k, v, starts, lengths, True, -1, hd ** -0.5).to(torch.bfloat16)
    want = inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=True)
    rows = torch.full((cu[-1] + 3, hq + 2 * hkv + 1, hd), 7.0, dtype=torch.bfloat16, device=cuda)
    parts = rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:hq + 2 * hkv]
    inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=True, grads=parts)
    torch.cuda.synchronize()
    for x, y in zip(parts, want):
        assert torch.equal(x[:cu[-1]], y)
    assert (rows[cu[-1]:] == 7).all() and (rows[:, -1] == 7).all()
    # only dk and dv
    again = torch.empty_like(rows)
    inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=True,
                             grads=(None, again[:, hq:hq + hkv], again[:, hq + hkv:hq + 2 * hkv]))
    assert torch.equal(again[:cu[-1], hq:hq + hkv], want[1]) and torch.equal(again[:cu[-1], hq + hkv:hq + 2 * hkv], want[2])


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_padded_batch(hd, cuda, inl):
    """Texts placed in a padded batch, whatever the padding holds; gradients made here are zero there."""
    import torch
    lengths, width, hq, hkv = [40, 1, 0, 130, 64], 140, 2, 1
    q, k, v, dout, starts, cu = _inputs(torch, cuda, lengths, hq, hkv, hd, 9)
    out = A.forward(q, k, v, starts, lengths, True, -1, hd ** -0.5).to(torch.bfloat16)
    want = inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=True)
    at = torch.cat([torch.arange(t) + width * b + (width - t if b % 2 else 0) for b, t in enumerate(lengths)]).to(cuda)
    seq = [width * b + (width - t if b % 2 else 0) for b, t in enumerate(lengths)]

    def pad(x):
        big = torch.full((width * len(lengths), *x.shape[1:]), float("nan"), dtype=x.dtype, device=cuda)
        big[at] = x
        return big
    got = inl.varlen_attention_bwd(pad(dout), pad(q), pad(k), pad(v), pad(out), cu, causal=True, seq_starts=seq)
    rest = torch.ones(width * len(lengths), dtype=torch.bool, device=cuda)
    rest[at] = False
    for x, y in zip(got, want):
        assert torch.equal(x[at], y) and not x[rest].any()


def test_not_finite_stays_in_its_text(cuda, inl):
    import torch
    for hd in (64, 128, 256):
        lengths = [70, 40, 70]
        q, k, v, dout, starts, cu = _inputs(torch, cuda, lengths, 2, 1, hd, 11)
        out = A.forward(q, k, v, starts, lengths, False, -1, hd ** -0.5).to(torch.bfloat16)
        want = inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=False)
        for t in (q, k, v, out, dout):
            for value in (float("inf"), float("nan")):
                one = t[75, 0, 3:4]
                keep = one.clone()
                one.fill_(value)
                got = inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=False)
                one.copy_(keep)
                for x, y in zip(got, want):
                    assert torch.equal(x[:70], y[:70]) and torch.equal(x[110:], y[110:])


def test_differences(cuda, inl):
    """Against differences of the forward's own loss sum(out dout) in float64."""
    import torch
    lengths, hq, hkv, hd = [19, 34], 2, 1, 64
    q, k, v, dout, starts, cu = _inputs(torch, cuda, lengths, hq, hkv, hd, 13)
    args = (starts, lengths, True, 16, hd ** -0.5)
    out = A.forward(q, k, v, *args).to(torch.bfloat16)
    got = inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=True, window=16, grad_dtype=torch.float32)
    _, bounds = zip(*A.backward(dout, q, k, v, out, *args))
    loss = lambda a, b, c: (A.forward(a, b, c, *args) * dout.double()).sum()
    base = [q.double(), k.double(), v.double()]
    g = torch.Generator(device=cuda).manual_seed(1)
    for i in range(3):
        way = torch.randn(base[i].shape, generator=g, device=cuda, dtype=torch.float64)
        h = 1e-4
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + h * way, base[i] - h * way
        diff = (loss(*up) - loss(*down)) / (2 * h)
        # `out` was rounded: delta is off by at most u |dO|.|o|, which meets P |k| or P |q| in dq and dk
        slack = 0.0
        if i < 2:
            full = A.forward(q, k, v, *args)
            e = A.U * (dout.double() * full).abs().sum(-1).max().item()
            slack = e * hd ** -0.5 * base[1 - i].abs().max().item() * way.abs().sum().item()
        tol = (bounds[i] * way.abs()).sum().item() + slack + 2.0 ** -23 * (got[i].double() * way).abs().sum().item() + 1e-6
        assert abs((got[i].double() * way).sum().item() - diff.item()) <= tol, i


def test_equal_calls_give_equal_bits(cuda, inl):
    import torch
    lengths = [300, 77, 513]
    for hq, hkv, hd in ((4, 2, 128), (3, 1, 256), (4, 4, 64)):
        q, k, v, dout, starts, cu = _inputs(torch, cuda, lengths, hq, hkv, hd, 15)
        out = A.forward(q, k, v, starts, lengths, False, 100, hd ** -0.5).to(torch.bfloat16)
        a, b = (inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=False, window=100) for _ in range(2))
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("texts", [3, 300])
def test_graph_replays(texts, cuda, inl):
    """Captured beside eager calls, two graphs with a workspace each, new values between replays."""
    import torch
    lengths = [40 + i % 7 for i in range(texts)]
    hq, hkv, hd = 4, 2, 128
    q, k, v, dout, starts, cu = _inputs(torch, cuda, lengths, hq, hkv, hd, 17)
    out = A.forward(q, k, v, starts, lengths, True, -1, hd ** -0.5).to(torch.bfloat16)
    call = lambda: inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=True)
    call()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, call()))
    for i in range(4):
        dout.mul_(-0.5)
        want = call()
        torch.cuda.synchronize()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, got in graphs:
            assert all(torch.equal(x, y) for x, y in zip(got, want)), i


def test_streams(cuda, inl):
    import torch
    lengths = [300, 77]
    q, k, v, dout, starts, cu = _inputs(torch, cuda, lengths, 4, 2, 128, 19)
    out = A.forward(q, k, v, starts, lengths, True, -1, 128 ** -0.5).to(torch.bfloat16)
    want = inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=True)
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = [inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=True, stream=s) for s in sides for _ in range(3)]
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(x, y) for x, y in zip(one, want))


def test_after_the_forward(cuda, inl):
    """With what varlen_attention itself leaves, in its three forms."""
    import torch
    for lengths, hq, hkv, hd, causal, window in (([300, 41], 16, 8, 128, True, -1), ([600, 90], 3, 1, 256, False, 512),
                                                 ([300, 33], 12, 12, 64, False, 64)):
        q, k, v, dout, starts, cu = _inputs(torch, cuda, lengths, hq, hkv, hd, 21)
        out = inl.varlen_attention(q, k, v, cu, causal=causal, window=window)
        got = inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=causal, window=window)
        torch.cuda.synchronize()
        A.check(got, A.backward(dout, q, k, v, out, starts, lengths, causal, window, hd ** -0.5), lengths)


def test_nothing_to_do(cuda, inl):
    import torch
    e = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=cuda)
    assert all(x.shape == (0, 2, 64) for x in inl.varlen_attention_bwd(e, e, e, e, e, [0], causal=True))
    assert all(x.shape == (0, 2, 64) for x in inl.varlen_attention_bwd(e, e, e, e, e, [0, 0, 0], causal=True))
    z = torch.randn(4, 2, 64, device=cuda).to(torch.bfloat16)
    assert not any(x.any() for x in inl.varlen_attention_bwd(z, z, z, z, z, [0, 0], causal=False))


@pytest.mark.parametrize("causal", [False, True])
def test_widest_window(causal, cuda, inl):
    """A window of any size up to 2^31 - 1 that covers the texts is no window."""
    import torch
    for hd in (64, 128, 256):
        lengths = [70, 1, 300]
        q, k, v, dout, starts, cu = _inputs(torch, cuda, lengths, 2, 1, hd, 13)
        out = A.forward(q, k, v, starts, lengths, causal, -1, hd ** -0.5).to(torch.bfloat16)
        A.check(inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=causal, window=2 ** 31 - 1),
                A.backward(dout, q, k, v, out, starts, lengths, causal, -1, hd ** -0.5), lengths)


def test_more_blocks_than_one_grid_has_threads_for(cuda, inl):
    """2^18 + 3 texts of one token and 64 heads: a key is all that its query sees, so dv is dout, and
    dq and dk are 0."""
    import torch
    n, h, hd = 2 ** 18 + 3, 64, 8
    g = torch.Generator(device=cuda).manual_seed(1)
    q, k, v, dout = (torch.randn(n, h, hd, generator=g, device=cuda).to(torch.bfloat16) for _ in range(4))
    dq, dk, dv = inl.varlen_attention_bwd(dout, q, k, v, v, list(range(n + 1)), causal=False)
    assert torch.equal(dv, dout)
    # dP - delta: delta has 8 roundings of 2^-24 at most of s = sum |dout v|; dP is added up from -delta on, 8
    # steps of 2^-23 (matrix instructions need not round to nearest) of 2 s
    few = (40 * 2.0 ** -24 * (dout.abs().float() * v.abs().float()).sum(-1, keepdim=True))
    assert (dq.float().abs() <= few * hd ** -0.5 * k.abs().float() * (1 + 2.0 ** -6)).all()
    assert (dk.float().abs() <= few * hd ** -0.5 * q.abs().float() * (1 + 2.0 ** -6)).all()
