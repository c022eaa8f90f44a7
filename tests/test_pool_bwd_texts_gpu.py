"""The pooling's gradients over batches of 256 texts and more, where a row's text is found by a search in steps of 64, and
rows of odd widths, against float64 (bounds: step_ref.py)."""
import random

import pytest

import step_ref as S
import train_ref as R

pytestmark = pytest.mark.gpu


def _offsets(texts, first):
    """Runs of empty texts, texts of one to three rows (many ends in one block of rows) and some of several blocks."""
    g = random.Random(texts)
    cu, at = [first], first
    while len(cu) <= texts:
        kind = g.choice(["empty", "short", "short", "long"])
        for _ in range(1 if kind == "long" else g.randint(1, 70)):
            at += {"empty": 0, "short": g.randint(1, 3), "long": g.randint(30, 130)}[kind]
            cu.append(at)
    return cu[:texts + 1]


def _randn(torch, dev, shape, seed, std=1.0, dtype=None):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * std).to(dtype or torch.float32)


def _mean(torch, cuda, inl, cu, rows, dim, dtype):
    texts = len(cu) - 1
    dev = torch.tensor(cu, dtype=torch.int32, device=cuda)
    dp, mean = _randn(torch, cuda, (texts, dim), 1, 0.1), _randn(torch, cuda, (texts, dim), 2, 0.3)
    for m in (None, mean):
        got = inl.pool_mean_bwd(dp, dev, rows, mean=m, dtype=dtype)
        torch.cuda.synchronize()
        ref, size = S.mean_bwd(dp, cu, rows, m)
        R.check(got, ref, (dim / 256 + 24) * 2.0 ** -24 * 2 * size + R.out_tol(ref, dtype) + 1e-30, ("mean", texts, dim))


def _last(torch, cuda, inl, cu, rows, dim, dtype, out):
    texts = len(cu) - 1
    dev = torch.tensor(cu, dtype=torch.int32, device=cuda)
    dp, x = _randn(torch, cuda, (texts, dim), 1, 0.1), _randn(torch, cuda, (rows, dim), 3, 2.0, dtype)
    w = _randn(torch, cuda, (dim,), 4, 1.0, dtype)
    got, dw = inl.pool_last_bwd(dp, x, dev, w, dtype=out)
    torch.cuda.synchronize()
    ref, size, rdw, dw_size = S.last_bwd(dp, x, cu, w, 1e-6)
    e = (dim / 256 + 32) * 2.0 ** -24 * 4
    R.check(got, ref, e * size + R.out_tol(ref, out) + 1e-30, ("last", texts, dim))
    R.check(dw, rdw, (e + texts * 2.0 ** -24) * dw_size + 1e-30, ("dweight", texts, dim))


@pytest.mark.parametrize("first,extra", [(0, 0), (37, 45)])
@pytest.mark.parametrize("texts", [254, 255, 256, 257, 319, 4095, 4096, 5000])
def test_many_texts(texts, first, extra, cuda, inl):
    import torch
    cu = _offsets(texts, first)
    rows = cu[-1] + extra
    print(f"case=pool_bwd texts={texts} rows={rows} first={first}", flush=True)
    for dim in (8, 264, 5):
        _mean(torch, cuda, inl, cu, rows, dim, torch.bfloat16)
    _last(torch, cuda, inl, cu, rows, 264, torch.bfloat16, torch.bfloat16)


def test_only_empty_texts_and_one(cuda, inl):
    import torch
    for cu in ([0] * 300 + [33] * 700, [0] * 999 + [1], [40] * 1000, [0] + [70] * 999):
        _mean(torch, cuda, inl, cu, 100, 16, torch.float32)
        _last(torch, cuda, inl, cu, 100, 16, torch.float32, torch.float32)


@pytest.mark.parametrize("dim", [1, 7, 13, 100, 1025, 2057])
def test_odd_widths(dim, cuda, inl):
    """One column per lane: packed bf16 rows of odd widths, as input and as output."""
    import torch
    b, f = torch.bfloat16, torch.float32
    for cu in ([0, 0, 1, 1, 40, 40], [3, 31, 32, 33, 97, 200]):
        for dtype, out in ((b, b), (f, b), (b, f), (f, f)):
            print(f"case=pool_bwd odd {dim} {len(cu) - 1} {dtype} {out}", flush=True)
            _last(torch, cuda, inl, cu, cu[-1] + 7, dim, dtype, out)
            _mean(torch, cuda, inl, cu, cu[-1] + 7, dim, out)


def test_strided_odd_rows(cuda, inl):
    """Slices of wider bf16 buffers; what lies beside them stays."""
    import torch
    cu, dim, rows = [0, 5, 5, 64, 90], 99, 97
    dev = torch.tensor(cu, dtype=torch.int32, device=cuda)
    dp = _randn(torch, cuda, (4, dim), 1, 0.1)
    wide = _randn(torch, cuda, (rows, dim + 6), 2, 2.0, torch.bfloat16)
    x, w = wide[:, 3:3 + dim], _randn(torch, cuda, (dim,), 4, 1.0, torch.bfloat16)
    want, want_dw = inl.pool_last_bwd(dp, x.contiguous(), dev, w)
    into = torch.full((rows, dim + 4), 7.0, dtype=torch.bfloat16, device=cuda)
    got, dw = inl.pool_last_bwd(dp, x, dev, w, out=into[:, 1:1 + dim])
    assert torch.equal(got, want) and torch.equal(dw, want_dw)
    assert (into[:, 0] == 7).all() and (into[:, 1 + dim:] == 7).all()
    got = inl.pool_mean_bwd(dp, dev, rows, out=into[:, 1:1 + dim])
    assert torch.equal(got, inl.pool_mean_bwd(dp, dev, rows))
    assert (into[:, 0] == 7).all() and (into[:, 1 + dim:] == 7).all()
