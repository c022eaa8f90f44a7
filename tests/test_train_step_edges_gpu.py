"""Gradients of attention, residual norm and pooling where addresses are far apart, calls are captured over padded
batches, and outputs take the place of inputs."""
import pytest

import attn_bwd_ref as A
import step_ref as S

pytestmark = pytest.mark.gpu


def _randn(torch, dev, shape, seed, std=1.0, dtype=None):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * std).to(dtype or torch.float32)


def _apart(torch, x, rows, width, at):
    """Rows `at` of a buffer [rows, width] whose first columns hold x."""
    n, h, d = x.shape
    big = torch.empty(rows, width, dtype=x.dtype, device=x.device)
    view = big.as_strided((rows, h, d), (width, d, 1))
    view[at] = x
    return view


@pytest.mark.parametrize("hq,hkv,hd,causal,window", [(2, 1, 64, True, 16), (4, 2, 120, False, 40), (3, 1, 256, True, 20)])
def test_rows_far_apart(hq, hkv, hd, causal, window, cuda, inl):
    """A text whose rows of every tensor span more than 2^31 bytes, and one behind it that starts beyond 4 GiB: the same
    bits as from packed rows."""
    import torch
    lengths = [20_011, 3_001]
    n, width = sum(lengths), 1 << 16   # 128 KB a row in bf16
    q, dout = (_randn(torch, cuda, (n, hq, hd), i, 1.0, torch.bfloat16) for i in (1, 2))
    k, v = (_randn(torch, cuda, (n, hkv, hd), i, 1.0, torch.bfloat16) for i in (3, 4))
    cu = [0, lengths[0], n]
    out = inl.varlen_attention(q, k, v, cu, causal=causal, window=window)
    want = inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=causal, window=window)
    torch.cuda.synchronize()
    seq = [5, 40_000]
    rows = seq[1] + lengths[1]
    at = torch.cat([torch.arange(a, a + t) for a, t in zip(seq, lengths)]).to(cuda)
    far = [_apart(torch, x, rows, width, at) for x in (dout, q, k, v, out)]
    grads = [_apart(torch, torch.zeros_like(x), rows, width, at) for x in (q, k, v)]
    print(f"case=far rows={rows} stride={width} {hq}/{hkv} x {hd}", flush=True)
    got = inl.varlen_attention_bwd(*far, cu, causal=causal, window=window, seq_starts=seq, grads=grads)
    torch.cuda.synchronize()
    assert all(torch.equal(x[at], y) for x, y in zip(got, want))


def test_padded_batch_in_a_graph(cuda, inl):
    """The rows between the texts are 0 after every replay too."""
    import torch
    lengths, width, hq, hkv, hd = [60, 1, 0, 131, 64], 140, 4, 2, 64
    n = sum(lengths)
    cu = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    seq = [i * width for i in range(len(lengths))]
    rows = width * len(lengths)
    at = torch.cat([torch.arange(a, a + t) for a, t in zip(seq, lengths)]).to(cuda)
    rest = torch.ones(rows, dtype=torch.bool, device=cuda)
    rest[at] = False
    q, k, v, out, dout = (_randn(torch, cuda, (rows, h, hd), i, 1.0, torch.bfloat16)
                          for i, h in enumerate((hq, hkv, hkv, hq, hq)))
    call = lambda: inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=True, seq_starts=seq)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for i in range(4):
        for x in got:
            x.fill_(3.0)
        dout.mul_(-0.5)
        want = call()
        packed = inl.varlen_attention_bwd(*(x[at] for x in (dout, q, k, v, out)), cu, causal=True)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y, z in zip(got, want, packed):
            assert torch.equal(x, y) and torch.equal(x[at], z) and not x[rest].any(), i
    assert n == len(at)


@pytest.mark.parametrize("m,n", [(37, 520), (9, 2056), (1500, 264), (5, 16384)])
def test_norm_gradients_in_the_place_of_inputs(m, n, cuda, inl):
    """dx and dresidual in the places of dy, h and dh, by the library's own entry."""
    import ctypes

    import torch
    from inl_hip import train as T
    w = _randn(torch, cuda, (n,), 1)
    dy, h, dh = (_randn(torch, cuda, (m, n), i, 1.0, torch.bfloat16) for i in (2, 3, 4))
    rng = torch.tensor([7, 8], device=cuda)
    d = T.AddNormDesc(m=m, n=n, eps=1e-6, drop=13107, tag=2, x_dtype=1, stream_dtype=1, out_dtype=1, weight_dtype=0)
    need = ctypes.c_size_t()
    assert T._add_norm_ws(d, ctypes.byref(need)) == 0
    ws = torch.empty(max(16, need.value), dtype=torch.uint8, device=cuda)
    want = inl.add_rms_norm_bwd(dy, h, w, dh=dh, dropout=13107 / 65536, rng=rng, tag=2)
    for to in ((0, 1), (1, 0), (2, 0), (0, 2), (1, 2), (2, 1)):
        x = [t.clone() for t in (dy, h, dh)]
        dw = torch.empty(n, device=cuda)
        rc = T._add_norm_bwd(d, *(t.data_ptr() for t in x), w.data_ptr(), rng.data_ptr(), x[to[0]].data_ptr(),
                             x[to[1]].data_ptr(), dw.data_ptr(), ws.data_ptr(), need.value,
                             torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert rc == 0 and torch.equal(x[to[0]], want[0]) and torch.equal(x[to[1]], want[1]) and torch.equal(dw, want[2]), to
    x = dy.clone()
    assert T._add_norm_bwd(d, x.data_ptr(), h.data_ptr(), dh.data_ptr(), w.data_ptr(), rng.data_ptr(), x.data_ptr(),
                           x.data_ptr(), None, None, 0, None) == -1


def test_more_than_2_to_the_32_values(cuda, inl):
    """A matrix of more than 2^32 values: the first rows, those around 2^31 and 2^32 values, and the last."""
    import numpy as np
    import torch

    import train_ref as R
    m, n, drop = (1 << 20) + 5, 4104, 0.25
    x = torch.empty(m, n, dtype=torch.bfloat16, device=cuda)
    base = _randn(torch, cuda, (257, n), 1, 1.0, torch.bfloat16)
    for a in range(0, m, 257):
        x[a:a + 257] = base[:min(257, m - a)]
    r = torch.ones((), dtype=torch.bfloat16, device=cuda).expand(m, n).contiguous()
    w = _randn(torch, cuda, (n,), 3, 1.0, torch.bfloat16)
    seed, step, tag = 0xABCDEF987654321, 3, 9
    rng = torch.tensor([seed, step], device=cuda)
    y, h = inl.add_rms_norm(x, w, residual=r, dropout=drop, rng=rng, tag=tag)
    edge = [(1 << 31) // n - 2, (1 << 32) // n - 2]
    for a in (0, *edge, m - 5):
        rows = slice(a, a + 5)
        # the draws of these rows' groups
        at = np.arange(a * n // 8, (a + 5) * n // 8, dtype=np.uint64)
        c = np.stack([at & np.uint64(0xFFFFFFFF), at >> np.uint64(32), np.full_like(at, tag), np.full_like(at, step)])
        words = S.philox(c, (seed & 0xFFFFFFFF, seed >> 32)).T.astype("<u4")
        bits = np.ascontiguousarray(words).view("<u2").reshape(5, n)
        f = torch.from_numpy(np.where(bits >= 16384, 65536 / (65536 - 16384), 0.0)).to(cuda)
        S.check_add_norm(y[rows], h[rows], x[rows], w, r[rows], f, 1e-6, f"rows {a}")
    del y, r
    dx, dres, _ = inl.add_rms_norm_bwd(x, h, w, dropout=drop, rng=rng, tag=tag, weight_grad=False)
    for a in (0, *edge, m - 5):
        rows = slice(a, a + 5)
        at = np.arange(a * n // 8, (a + 5) * n // 8, dtype=np.uint64)
        c = np.stack([at & np.uint64(0xFFFFFFFF), at >> np.uint64(32), np.full_like(at, tag), np.full_like(at, step)])
        words = S.philox(c, (seed & 0xFFFFFFFF, seed >> 32)).T.astype("<u4")
        bits = np.ascontiguousarray(words).view("<u2").reshape(5, n)
        f = torch.from_numpy(np.where(bits >= 16384, 65536 / (65536 - 16384), 0.0)).to(cuda)
        S.check_add_norm_bwd((dx[rows], dres[rows], None), x[rows], h[rows], w, None, f, 1e-6, f"bwd rows {a}")
    # the pooling's gradient of as many
    del dx, dres, h
    cu = torch.tensor([3, 1 << 19, m - 4], dtype=torch.int32, device=cuda)
    dp = _randn(torch, cuda, (2, n), 5)
    inl.pool_mean_bwd(dp, cu, m, out=x)
    for a, text in ((0, None), (3, 0), (edge[0], None if edge[0] < 3 else 0), ((1 << 19) - 1, 0), (1 << 19, 1), (m - 5, 1), (m - 4, None)):
        want = torch.zeros(n, dtype=torch.float64, device=cuda)
        if text is not None:
            want = dp[text].double() / ((1 << 19) - 3 if text == 0 else m - 4 - (1 << 19))
        R.check(x[a], want, 2.0 ** -22 * want.abs() + R.out_tol(want, torch.bfloat16), f"mean row {a}")
    hid = torch.empty_like(x)
    ends = ((1 << 19) - 1, m - 5)
    for e in ends:
        hid[e] = base[e % 257]
    got, _ = inl.pool_last_bwd(dp, hid, cu, w, out=x)
    ref, size, _, _ = S.last_bwd(dp, torch.stack([hid[e] for e in ends]), [0, 1, 2], w, 1e-6)
    for i, e in enumerate(ends):
        R.check(got[e], ref[i], (n / 256 + 32) * 2.0 ** -22 * size[i] + R.out_tol(ref[i], torch.bfloat16) + 1e-30, f"last {e}")
        assert not got[e - 1].any() and not got[e + 1].any()
    assert not got[0].any() and not got[m - 1].any()
