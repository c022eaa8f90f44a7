"""The residual norm's and the pooling gradients' entries refuse bad arguments on the host, before
any GPU call: pointers here are made up and never read. And the dropout's generator by its
published values."""
import ctypes

import numpy as np
import pytest

import step_ref as S

MB = 1 << 20


@pytest.fixture(scope="module")
def T():
    from inl_hip import train
    return train


def _said(word):
    import inl_hip
    return word in inl_hip.last_error(), inl_hip.last_error()


def _desc(T, **kw):
    d = dict(m=4, n=64, eps=1e-6, drop=0, x_dtype=1, stream_dtype=0, out_dtype=1, weight_dtype=0)
    d.update(kw)
    return T.AddNormDesc(**d)


def test_generator():
    """The known answers published with the generator."""
    def draw(c, k):
        return [int(v) for v in S.philox(np.array(c, dtype=np.uint64)[:, None], k)[:, 0]]
    assert draw([0] * 4, (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert draw([0xFFFFFFFF] * 4, (0xFFFFFFFF, 0xFFFFFFFF)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


@pytest.mark.parametrize("fields,code,word", [
    (dict(m=-1), -1, "m must be"), (dict(n=0), -1, "n > 0"), (dict(n=60), -2, "multiple of 8"),
    (dict(n=16392), -2, "at most"), (dict(m=1 << 31), -2, "below"), (dict(x_dtype=2), -1, "dtypes"),
    (dict(stream_dtype=-1), -1, "dtypes"), (dict(weight_dtype=3), -1, "dtypes"), (dict(drop=65536), -1, "drop"),
    (dict(drop=-1), -1, "drop"), (dict(eps=-1.0), -1, "eps"), (dict(eps=float("nan")), -1, "eps"),
    (dict(x_stride=56), -1, "row stride"), (dict(h_stride=66), -1, "row stride"), (dict(y_stride=68), -1, "row stride")])
def test_norm_refusals(fields, code, word, T):
    d = _desc(T, **fields)
    assert T._add_norm(d, MB, 2 * MB, 3 * MB, 4 * MB, 5 * MB, 6 * MB, None) == code and all(_said(word))
    assert T._add_norm_bwd(d, MB, 2 * MB, 3 * MB, 4 * MB, 5 * MB, 6 * MB, 7 * MB, 8 * MB, 9 * MB, MB, None) == code


def test_norm_pointers(T):
    base = [MB, 2 * MB, 3 * MB, 4 * MB, 5 * MB, 6 * MB]   # x, residual, weight, rng, h, y
    call = lambda d, **kw: T._add_norm(d, *[kw.get(f"p{i}", p) for i, p in enumerate(base)], None)
    assert call(None) == -1
    for i in (0, 5):
        assert call(_desc(T), **{f"p{i}": None}) == -1 and all(_said("NULL"))
    for i in (0, 1, 2, 4, 5):
        assert call(_desc(T), **{f"p{i}": base[i] + 4}) == -1 and all(_said("aligned"))
    assert call(_desc(T, drop=5), p3=None) == -1 and all(_said("rng"))
    assert call(_desc(T, drop=5), p3=MB + 4) == -1 and all(_said("rng"))
    # outputs in another place of an input, in one another, in the weight
    assert call(_desc(T), p5=MB + 128) == -1 and all(_said("y overlaps x"))
    assert call(_desc(T), p5=2 * MB) == -1 and all(_said("y overlaps residual"))   # of another type
    assert call(_desc(T), p4=MB) == -1 and all(_said("h overlaps x"))
    assert call(_desc(T, stream_dtype=1), p4=6 * MB) == -1 and all(_said("y overlaps h"))
    assert call(_desc(T, stream_dtype=1), p4=2 * MB, h_stride=0, p5=2 * MB) == -1
    assert call(_desc(T, h_stride=128), p4=2 * MB) == -1 and all(_said("h overlaps residual"))
    assert call(_desc(T), p4=3 * MB) == -1 and all(_said("weight"))
    assert call(_desc(T, m=0), p0=None, p5=None) == 0


def test_norm_bwd_pointers(T):
    base = [MB * (i + 1) for i in range(9)]   # dy, h, dh, weight, rng, dx, dresidual, dweight, workspace
    call = lambda d, size=0, **kw: T._add_norm_bwd(d, *[kw.get(f"p{i}", p) for i, p in enumerate(base)], size, None)
    for i in (0, 1):
        assert call(_desc(T), **{f"p{i}": None}) == -1 and all(_said("NULL"))
    for i in (0, 1, 2, 3, 5, 6, 7):
        assert call(_desc(T), **{f"p{i}": base[i] + 4}) == -1 and all(_said("aligned"))
    assert call(_desc(T, drop=9), p4=None) == -1 and all(_said("rng"))
    assert call(_desc(T, dh_stride=32)) == -1 and call(_desc(T), p6=6 * MB) == -1 and all(_said("overlaps"))
    assert call(_desc(T), p7=2 * MB) == -1 and all(_said("dweight overlaps h"))
    assert call(_desc(T), p5=MB + 64) == -1 and all(_said("dx overlaps dy"))
    assert T._add_norm_ws(_desc(T), None) == -1
    n = ctypes.c_size_t()
    assert T._add_norm_ws(_desc(T, n=4), ctypes.byref(n)) == -2
    assert call(_desc(T), p5=None, p6=None, p7=None) == 0


def test_pool_refusals(T):
    mean = lambda n=3, cu=MB, dim=64, rows=9, stride=0, dt=1, dp=2 * MB, m=3 * MB, out=4 * MB: \
        T._pool_mean_bwd(n, cu, dim, rows, stride, dt, dp, m, out, None)
    for bad in (dict(n=-1), dict(dim=0), dict(rows=-1), dict(dt=2), dict(stride=32), dict(out=None), dict(cu=None),
                dict(dp=None), dict(dp=MB + 2), dict(out=MB + 1), dict(out=2 * MB + 64), dict(out=3 * MB), dict(out=MB),
                dict(m=3 * MB + 2)):
        assert mean(**bad) == -1, bad
    assert mean(rows=1 << 31) == -2
    assert mean(rows=0, out=None, cu=None, dp=None) == 0

    def last(n=3, cu=MB, dim=64, rows=9, stride=0, dt=1, dp=2 * MB, h=3 * MB, w=4 * MB, eps=1e-6, ds=0, ddt=1, out=5 * MB,
             dw=6 * MB, ws=7 * MB, size=0):
        return T._pool_last_bwd(n, cu, dim, rows, stride, dt, dp, h, w, eps, ds, ddt, out, dw, ws, size, None)
    for bad in (dict(n=-1), dict(dim=0), dict(rows=-1), dict(dt=2), dict(ddt=5), dict(stride=32), dict(ds=8), dict(out=None),
                dict(cu=None), dict(dp=None), dict(h=None), dict(eps=-1.0), dict(h=MB + 1), dict(w=MB + 1), dict(dw=MB + 2),
                dict(out=3 * MB), dict(dw=3 * MB), dict(dw=2 * MB), dict(out=4 * MB), dict(dw=5 * MB), dict(out=MB)):
        assert last(**bad) == -1, bad
    assert last() == -1 and all(_said("workspace"))
    assert last(ws=None, size=3 * 64 * 4) == -1 and all(_said("workspace"))
    n = ctypes.c_size_t()
    assert T._pool_last_ws(3, 64, ctypes.byref(n)) == 0 and n.value == 3 * 64 * 4
    assert T._pool_last_ws(-1, 64, ctypes.byref(n)) == -1 and T._pool_last_ws(3, 64, None) == -1
    assert last(rows=0, out=None, cu=None, dp=None, h=None, dw=None) == 0


def test_pool_grids(T):
    far = [(i + 1) << 44 for i in range(6)]
    for n, rows in ((3, 2 ** 29), (2 ** 24, 9), (2 ** 23, 2 ** 28), (2 ** 31 - 1, 9)):
        assert T._pool_mean_bwd(n, far[0], 8, rows, 0, 1, far[1], far[2], far[3], None) == -2 and all(_said("2^24"))
        assert T._pool_last_bwd(n, far[0], 8, rows, 0, 1, far[1], far[2], None, 1e-6, 0, 1, far[3], None, None, 0,
                                None) == -2 and all(_said("2^24"))


def test_bindings_check_tensors():
    import torch

    import inl_hip
    x = torch.zeros(4, 64)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    for call in (lambda: inl_hip.add_rms_norm(x), lambda: inl_hip.add_rms_norm_bwd(x, x),
                 lambda: inl_hip.pool_mean_bwd(x[:1], cu, 4), lambda: inl_hip.pool_last_bwd(x[:1], x, cu)):
        with pytest.raises(inl_hip.InlError, match="not a device tensor"):
            call()
    from inl_hip import train
    for bad in (-0.1, 1.0, 0.99999999, float("nan")):
        with pytest.raises(inl_hip.InlError, match="dropout"):
            train._drop(bad, None, 0)
    assert train._drop(0.0, None, 0) == (0, None) and train._drop(1e-6, None, 0) == (0, None)
    with pytest.raises(inl_hip.InlError, match="rng"):
        train._drop(0.1, None, 0)
    for bad in (-2 ** 31 - 1, 2 ** 32):
        with pytest.raises(inl_hip.InlError, match="tag"):
            train._tag(bad)
