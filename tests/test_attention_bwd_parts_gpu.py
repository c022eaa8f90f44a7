"""Gradients of packed attention by every kernel that the rule chooses among, over many stream tiles and more than one
block of own rows, against float64 (bounds: attn_bwd_ref.py). A kernel whose waves all have own rows of their own (one
part) is for batches that fill the GPU, so the batches here do."""
import pytest

import attn_bwd_ref as A

pytestmark = pytest.mark.gpu

# every length modulo 4, so most of a tile's and a block's; an empty text and texts of one and two tokens
RAGGED = [257 - 4 * i for i in range(64)] + [0, 1, 2]
WIDE = [300 - 7 * i for i in range(40)] + [0, 1, 2]


def _name(d, kv, parts):
    return "attn_bwd_pair_kernel<256>" if d == 256 and kv else f"attn_bwd_kernel<{d}, {str(kv).lower()}, {parts}>"


CASES = [
    # lengths, query / key heads, head_dim, causal, window, parts of dq, of dk and dv
    ([257] * 64, 16, 16, 64, False, -1, 1, 1), ([257] * 64, 16, 16, 64, False, 64, 1, 1),
    (RAGGED, 16, 16, 64, True, -1, 1, 1), (RAGGED, 16, 16, 40, False, 64, 1, 1), (RAGGED, 16, 16, 8, True, 33, 1, 1),
    (RAGGED, 24, 12, 64, False, -1, 1, 1), (RAGGED, 12, 12, 56, False, 0, 1, 1),
    ([257] * 64, 16, 8, 128, False, -1, 1, 1), (RAGGED, 16, 8, 128, False, 64, 1, 1),
    (RAGGED, 16, 8, 80, False, -1, 1, 1), (RAGGED, 16, 8, 120, False, 31, 1, 1), (RAGGED, 16, 8, 128, True, -1, 1, 2),
    (RAGGED, 16, 8, 72, True, 40, 1, 2), ([600] * 16, 16, 8, 128, False, -1, 1, 1), ([601] * 16, 10, 10, 128, False, 100, 1, 1),
    ([300] * 32, 3, 1, 256, True, -1, 1, 0), ([300] * 32, 3, 1, 256, False, 40, 1, 0), (WIDE, 6, 2, 256, True, -1, 1, 0),
    (WIDE, 6, 2, 192, False, -1, 1, 0), (WIDE, 6, 2, 136, True, 70, 1, 0), ([520] * 16, 16, 2, 256, False, -1, 1, 0),
    # few texts: two parts
    ([700, 1, 333], 2, 2, 64, False, -1, 2, 2), ([700, 1, 333], 2, 2, 48, True, 65, 2, 2),
    ([700, 1, 333], 4, 2, 128, False, -1, 2, 2), ([700, 1, 333], 4, 2, 104, True, -1, 2, 2),
    ([700, 1, 333], 3, 1, 256, True, -1, 2, 0), ([700, 1, 333], 3, 1, 200, False, 90, 2, 0)]


def _inputs(torch, dev, lengths, hq, hkv, hd, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    n = sum(lengths)
    rows = torch.randn(n, hq + 2 * hkv, hd, generator=g, device=dev)
    rows[:, :hq] *= 1.5
    rows = rows.to(torch.bfloat16)
    dout = (0.1 * torch.randn(n, hq, hd, generator=g, device=dev)).to(torch.bfloat16)
    starts = [sum(lengths[:i]) for i in range(len(lengths))]
    return rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:], dout, starts, starts + [n]


@pytest.mark.parametrize("lengths,hq,hkv,hd,causal,window,dq_parts,kv_parts", CASES)
def test_parts(lengths, hq, hkv, hd, causal, window, dq_parts, kv_parts, cuda, inl):
    import torch
    print(f"case=attn_bwd_parts {len(lengths)} to {max(lengths)} {hq}/{hkv} x {hd} causal={causal} window={window}", flush=True)
    q, k, v, dout, starts, cu = _inputs(torch, cuda, lengths, hq, hkv, hd, hd)
    wide = 64 if hd <= 64 else 128 if hd <= 128 else 256
    names = inl.attention_bwd_kernel_names(inl.make_attn_desc(cu, hq, hkv, hd, causal=causal, window=window))
    assert names == (_name(wide, False, dq_parts), _name(wide, True, kv_parts))
    scale = hd ** -0.5
    out = A.forward(q, k, v, starts, lengths, causal, window, scale).to(torch.bfloat16)
    got = inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=causal, window=window)
    torch.cuda.synchronize()
    ref = A.backward(dout, q, k, v, out, starts, lengths, causal, window, scale)
    A.check(got, ref, names)
    again = inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=causal, window=window)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    full = inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=causal, window=window, grad_dtype=torch.float32)
    torch.cuda.synchronize()
    A.check(full, ref, names)
    assert all(torch.equal(a.to(torch.bfloat16), b) for a, b in zip(full, got))


def test_every_kernel_is_among_the_cases():
    names = {_name(64 if c[3] <= 64 else 128 if c[3] <= 128 else 256, kv, parts)
             for c in CASES for kv, parts in ((False, c[6]), (True, c[7]))}
    assert names == {_name(d, kv, parts) for d in (64, 128, 256) for kv in (False, True) for parts in (1, 2)}


def test_a_padded_batch_in_one_part(cuda, inl):
    """Texts of a padded batch that fills the GPU, NaN in the padding, and the gradients in slices of one row whose
    padding and other heads stay as they were."""
    import torch
    for hq, hkv, hd, causal in ((16, 16, 64, False), (16, 8, 120, False), (6, 2, 256, True)):
        lengths = [200 - i for i in range(48)]
        q, k, v, dout, starts, cu = _inputs(torch, cuda, lengths, hq, hkv, hd, 5)
        names = inl.attention_bwd_kernel_names(inl.make_attn_desc(cu, hq, hkv, hd, causal=causal))
        assert names[0].endswith("false, 1>")
        out = A.forward(q, k, v, starts, lengths, causal, -1, hd ** -0.5).to(torch.bfloat16)
        want = inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=causal)
        width = max(lengths) + 3
        seq = [i * width for i in range(len(lengths))]
        at = torch.cat([torch.arange(a, a + t) for a, t in zip(seq, lengths)]).to(cuda)

        def pad(x):
            big = torch.full((width * len(lengths), *x.shape[1:]), float("nan"), dtype=x.dtype, device=cuda)
            big[at] = x
            return big
        rows = torch.full((width * len(lengths), hq + 2 * hkv + 1, hd), 7.0, dtype=torch.bfloat16, device=cuda)
        parts = rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:-1]
        inl.varlen_attention_bwd(pad(dout), pad(q), pad(k), pad(v), pad(out), cu, causal=causal, seq_starts=seq, grads=parts)
        torch.cuda.synchronize()
        rest = torch.ones(width * len(lengths), dtype=torch.bool, device=cuda)
        rest[at] = False
        assert all(torch.equal(x[at], y) for x, y in zip(parts, want)), names
        assert (rows[rest] == 7).all() and (rows[:, -1] == 7).all(), names


def test_not_finite_stays_in_its_text_in_one_part(cuda, inl):
    import torch
    for hq, hkv, hd, causal in ((16, 16, 64, True), (16, 8, 128, False), (6, 2, 256, False)):
        lengths = [130] * 48
        q, k, v, dout, starts, cu = _inputs(torch, cuda, lengths, hq, hkv, hd, 11)
        names = inl.attention_bwd_kernel_names(inl.make_attn_desc(cu, hq, hkv, hd, causal=causal))
        assert names[0].endswith("false, 1>")
        out = A.forward(q, k, v, starts, lengths, causal, -1, hd ** -0.5).to(torch.bfloat16)
        want = inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=causal)
        for t in (q, k, v, out, dout):
            one = t[5 * 130 + 60, 0, 3:4]
            keep = one.clone()
            one.fill_(float("nan"))
            got = inl.varlen_attention_bwd(dout, q, k, v, out, cu, causal=causal)
            one.copy_(keep)
            for x, y in zip(got, want):
                assert torch.equal(x[:650], y[:650]) and torch.equal(x[780:], y[780:]), names
