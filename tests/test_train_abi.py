"""The C entries of include/inl_train.h refuse bad arguments on the host, before any
GPU call: pointers here are made up and never read."""
import ctypes

import pytest

P, ODD = 1 << 20, (1 << 20) + 8   # 16-byte aligned, and not


@pytest.fixture(scope="module")
def T():
    from inl_hip import train
    return train


def _dense(T, **kw):
    d = dict(m=4, n=16, k=40, out_dtype=1, residual_dtype=1, dx_dtype=1, dw_dtype=1)
    d.update(kw)
    return T.DenseDesc(**d)


def _ffn(T, **kw):
    d = dict(m=4, hidden=40, inner=16, act=2, out_dtype=1, residual_dtype=1, dx_dtype=1, dw_dtype=1)
    d.update(kw)
    return T.GatedFfnDesc(**d)


def _xent(T, **kw):
    d = dict(m=4, vocab=17, hidden=40, scale=1.0, ignore_index=-100, dx_dtype=1, dw_dtype=1)
    d.update(kw)
    return T.SoftmaxXentDesc(**d)


@pytest.mark.parametrize("fields,code,word", [
    (dict(m=-1), -1, "m must be"), (dict(n=0), -1, "n and k"), (dict(k=36), -2, "multiples of 8"),
    (dict(n=12), -2, "multiples of 8"), (dict(n=1 << 22), -2, "at most"), (dict(m=1 << 31), -2, "below"),
    (dict(act=5), -1, "unknown act"), (dict(act=-1), -1, "unknown act"), (dict(x_stride=32), -1, "x: the row stride"),
    (dict(w_stride=44), -2, "w: the row stride"), (dict(y_stride=1 << 22), -2, "2^21"),
    (dict(out_dtype=2), -1, "dtype"), (dict(residual_dtype=7), -1, "dtype"), (dict(pre_stride=8), -1, "pre")])
def test_dense_refusals(fields, code, word, T):
    import inl_hip
    assert T._dense_fwd(_dense(T, **fields), P, P, P, P, P, P, None, 0, None) == code
    assert word in inl_hip.last_error(), inl_hip.last_error()


def test_dense_pointers(T):
    import inl_hip
    for i in range(6):
        for bad in (ODD, None) if i not in (2, 3, 5) else (ODD,):
            args = [P] * 6
            args[i] = bad
            assert T._dense_fwd(_dense(T), *args, None, 0, None) == -1
    assert T._dense_fwd(None, P, P, P, P, P, P, None, 0, None) == -1
    for i in (0, 1, 2, 3):   # dy, x, w, pre
        args = [P] * 7
        args[i] = None
        assert T._dense_bwd(_dense(T, act=2), *args, None, 0, None) == -1
    assert T._dense_bwd(_dense(T, dw_dtype=3), *[P] * 7, None, 0, None) == -1
    assert T._dense_bwd(_dense(T, dx_stride=8), *[P] * 7, None, 0, None) == -1 and "dx" in inl_hip.last_error()
    n = ctypes.c_size_t()
    assert T._dense_ws(_dense(T, k=4), 0, ctypes.byref(n)) == -2
    assert T._dense_ws(_dense(T), 0, None) == -1
    # a few rows need none; nothing to do needs nothing
    assert T._dense_ws(_dense(T), 0, ctypes.byref(n)) == 0 and n.value == 0
    assert T._dense_fwd(_dense(T, m=0), None, None, None, None, None, None, None, 0, None) == 0


@pytest.mark.parametrize("fields,code,word", [
    (dict(m=-1), -1, "m must be"), (dict(hidden=36), -2, "multiples of 8"), (dict(inner=0), -1, "inner"),
    (dict(act=0), -1, "act"), (dict(act=9), -1, "act"), (dict(inner=1 << 21), -2, "at most"),
    (dict(x_stride=8), -1, "x: the row stride"), (dict(out_dtype=3), -1, "dtype")])
def test_gated_ffn_refusals(fields, code, word, T):
    import inl_hip
    assert T._ffn_fwd(_ffn(T, **fields), P, P, P, P, P, P, P, None, 0, None) == code
    assert word in inl_hip.last_error(), inl_hip.last_error()


def test_gated_ffn_pointers(T):
    import inl_hip
    assert T._ffn_fwd(_ffn(T), P, P, P, None, P, P, None, None, 0, None) == -1 and "together" in inl_hip.last_error()
    for i in (0, 1, 2, 4):
        args = [P] * 7
        args[i] = None
        assert T._ffn_fwd(_ffn(T), *args, None, 0, None) == -1
    for i in range(6):
        args = [P] * 9
        args[i] = ODD
        assert T._ffn_bwd(_ffn(T), *args, None, 0, None) == -1
    # the few-row forward keeps h in the workspace
    assert T._ffn_fwd(_ffn(T), *[P] * 7, None, 0, None) == -1 and "workspace" in inl_hip.last_error()
    assert T._ffn_fwd(_ffn(T), *[P] * 7, P, 8, None) == -1 and "need" in inl_hip.last_error()


@pytest.mark.parametrize("fields,code,word", [
    (dict(m=-1), -1, "m must be"), (dict(vocab=0), -1, "vocab"), (dict(hidden=36), -2, "multiple of 8"),
    (dict(vocab=1 << 29), -2, "at most"), (dict(w_stride=8), -1, "w: the row stride")])
def test_softmax_xent_refusals(fields, code, word, T):
    import inl_hip
    assert T._xent_fwd(_xent(T, **fields), *[P] * 6, None, 0, None) == code
    assert word in inl_hip.last_error(), inl_hip.last_error()
    assert T._xent_bwd(_xent(T, **fields), *[P] * 9, None, 0, None) == code


def test_softmax_xent_pointers(T):
    for i in (0, 1, 3, 4, 5):
        args = [P] * 6
        args[i] = None
        assert T._xent_fwd(_xent(T), *args, None, 0, None) == -1
    assert T._xent_fwd(_xent(T), P, P, ODD, P, P, P, None, 0, None) == -1
    for i in (0, 1, 2, 3, 5):
        args = [P] * 9
        args[i] = None
        assert T._xent_bwd(_xent(T), *args, None, 0, None) == -1
    assert T._xent_bwd(_xent(T, dx_dtype=5), *[P] * 9, None, 0, None) == -1


def test_norm_rope_bwd_refusals(T):
    import inl_hip
    def call(q=2, dq=P, dk=P, kw=P, dx_stride=0, x=P, dy=P, **kw_):
        d = inl_hip.NormRopeDesc()
        d.n_tokens, d.heads, d.head_dim, d.dtype, d.out_dtype, d.norm, d.eps = 4, 3, 64, 1, 1, 1, 1e-6
        d.rotary_dim, d.sections, d.table_rows = 64, 1, 9
        for k, v in kw_.items():
            setattr(d, k, v)
        return T._rope_bwd(d, q, dy, x, P, dx_stride, P, kw, P, P, P, None, None, dq, dk, None, 0, None)
    assert call(head_dim=48) == -2 and call(rotary_dim=60, sections=3) == -2 and call(sections=4) == -1
    assert call(q=0) == -1 and call(q=4) == -1 and call(q=3) == -1 and "k heads" in inl_hip.last_error()
    assert call(norm=0) == -1 and "no norm" in inl_hip.last_error()
    assert call(dx_stride=100) == -1 and call(x_row_stride=100) == -1 and call(x=ODD) == -1 and call(dy=None) == -1
    assert call(sections=2, rotary_dim=64) == -1   # axial without its second tables
    n = ctypes.c_size_t()
    assert T._rope_bwd_ws(None, ctypes.byref(n)) == -1


def test_adjacent_pairs_refusals():
    import inl_hip
    d = inl_hip.NormRopeDesc()
    d.n_tokens, d.heads, d.head_dim, d.dtype, d.out_dtype = 4, 3, 64, 1, 1
    d.sections, d.table_rows = 3, 9
    for rd in (4, 12, 72):
        d.rotary_dim = rd
        assert inl_hip._norm_rope(d, P, P, None, P, P, P, None, None, None) == -2


def test_package_imports_without_torch():
    """The layer ops need torch; the host-side entries of the package do not."""
    import subprocess
    import sys
    from pathlib import Path
    pkg = Path(__file__).resolve().parents[1] / "im-not-llm_amd"
    code = (f"import sys; sys.modules['torch'] = None; sys.path.insert(0, {str(pkg)!r}); import inl_hip; "
            "assert inl_hip.library_path().exists() and not hasattr(inl_hip, 'dense')")
    subprocess.run([sys.executable, "-c", code], check=True, timeout=120)


def test_stream_of_another_device(T):
    """Refused before anything is allocated or launched."""
    import types

    import inl_hip
    import torch
    x = types.SimpleNamespace(get_device=lambda: 0)
    s = types.SimpleNamespace(device=torch.device("cuda", 1), cuda_stream=P)
    for call in (lambda: T.dense(x, x, stream=s), lambda: T.dense_bwd(x, x, x, stream=s),
                 lambda: T.gated_ffn(x, x, x, stream=s), lambda: T.gated_ffn_bwd(x, x, x, x, x, x, stream=s),
                 lambda: T.softmax_xent(x, x, x, stream=s), lambda: T.softmax_xent_bwd(x, x, x, x, x, stream=s),
                 lambda: T.norm_rope_qk_bwd(x, x, 1, stream=s)):
        with pytest.raises(inl_hip.InlError, match="the stream is on cuda:1"):
            call()


def test_prologue_tables_and_rows():
    """What the prologue's kernels read by address is checked by the binding, forward
    and backward (host tensors here, whose device number is -1)."""
    import inl_hip
    import torch
    f = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype)
    rows = f(5, dtype=torch.int32)
    ok = lambda *a: inl_hip._rope_tables(*a, -1)
    assert ok(5, rows, 64, 128, 3, f(9, 32), f(9, 32), None, None) == 9
    assert ok(4, rows, 64, 128, 1, f(9, 1, 32), f(12, 32), None, None) == 9   # more than is read
    assert ok(5, rows, 128, 128, 2, f(5, 32), f(5, 32), f(5, 32), f(5, 32)) == 5
    for a in ((5, rows, 64, 128, 3, f(9, 64), f(9, 64), None, None),        # a column per feature
              (5, rows, 64, 128, 3, f(9, 32), f(9, 64), None, None),
              (5, rows, 64, 128, 1, f(9, 16), f(9, 16), None, None),
              (5, rows, 64, 128, 1, f(9, 32), f(8, 32), None, None),        # sin of fewer positions
              (5, rows, 64, 128, 1, f(9, 32), None, None, None),
              (5, rows, 64, 128, 1, None, f(9, 32), None, None),
              (5, rows, 64, 128, 1, f(288), f(288), None, None),
              (5, rows, 64, 128, 1, f(9, 32, dtype=torch.bfloat16), f(9, 32), None, None),
              (5, rows, 64, 128, 1, f(9, 64)[:, :32], f(9, 32), None, None),
              (5, rows, 64, 128, 1, f(32, 9).T, f(9, 32), None, None),
              (6, rows, 64, 128, 1, f(9, 32), f(9, 32), None, None),        # fewer rows than tokens
              (5, rows.long(), 64, 128, 1, f(9, 32), f(9, 32), None, None),
              (3, rows[::2], 64, 128, 1, f(9, 32), f(9, 32), None, None),
              (5, None, 64, 128, 1, f(9, 32), f(9, 32), None, None),
              (5, rows, 128, 128, 2, f(5, 32), f(5, 32), None, None),
              (5, rows, 128, 128, 2, f(5, 32), f(5, 32), f(5, 32), f(4, 32)),
              (5, rows, 128, 128, 2, f(5, 64), f(5, 64), f(5, 64), f(5, 64))):
        with pytest.raises(inl_hip.InlError):
            ok(*a)
    with pytest.raises(inl_hip.InlError, match="cuda:0"):   # another device than the tokens'
        inl_hip._rope_tables(5, rows, 64, 128, 1, f(9, 32), f(9, 32), None, None, 0)
    x = f(7, 5, 16)
    shape = x[:, :3].shape
    assert inl_hip._head_rows("x", x[:, :3], shape, -1) == 80
    assert inl_hip._head_rows("x", x[:1, :3].expand(1, 3, 16), (1, 3, 16), -1) == 48
    for t in (x, x[:, ::2], x[:, :3].float().transpose(1, 2), x[:1, :3].expand(7, 3, 16), x[:6, :3], f(7, 3, 32)[..., ::2]):
        with pytest.raises(inl_hip.InlError):
            inl_hip._head_rows("x", t, shape, -1)
    for call in (lambda: inl_hip.norm_rope(x), lambda: inl_hip.norm_rope_qk(x, 2)):
        with pytest.raises(inl_hip.InlError, match="not a device tensor"):
            call()


def test_prologue_of_no_tokens():
    """An empty tensor of rows has no address: no tokens is no error, forward or backward."""
    import inl_hip
    d = inl_hip.NormRopeDesc()
    d.n_tokens, d.heads, d.head_dim, d.dtype, d.out_dtype, d.norm, d.eps = 0, 3, 64, 1, 1, 1, 1e-6
    d.rotary_dim, d.table_rows = 64, 9
    for sections in (1, 3):
        d.sections = sections
        assert inl_hip._norm_rope(d, None, None, P, None, P, P, None, None, None) == 0, inl_hip.last_error()
        assert inl_hip._norm_rope_qk(d, 2, None, None, P, P, None, P, P, None, None, None) == 0
    d.n_tokens = 1
    assert inl_hip._norm_rope(d, P, P, P, None, P, P, None, None, None) == -1 and "rows" in inl_hip.last_error()


def test_dense_outputs_overlap_nothing(T):
    """y over x (a residual stream updated in place) would be written while it is read."""
    import inl_hip
    X, W, R, Y, PRE = (P + (i << 24) for i in range(5))
    kw = dict(m=300, n=40, k=40)

    def refused(x=X, w=W, res=None, y=Y, pre=None, **f):
        d = _dense(T, **{**kw, **f})
        rc = T._dense_fwd(d, x, w, None, res, y, pre, None, 0, None)
        return rc == -1 and "overlap" in inl_hip.last_error()
    assert refused(y=X) and refused(y=W) and refused(pre=X) and refused(pre=Y) and refused(res=R, pre=R)
    assert refused(res=X, y=X)                                  # residual in place, and x too
    assert refused(y=X + 16) and refused(y=X - 16)              # a shifted one
    assert refused(y=X + 300 * 80 - 16) and refused(y=X - 300 * 80 + 16)   # the ends
    assert refused(y=Y, res=Y, residual_dtype=0)                # another type at the same place
    assert refused(y=Y, res=Y, y_stride=48, residual_stride=56)
    assert refused(y=Y, res=Y + 16)
    assert refused(y=X + 80, x_stride=80, y_stride=88)          # strides that drift into each other


def test_rows_meet(T):
    """Against all pairs of rows, by way of the entry's refusal."""
    import random

    import inl_hip
    rng = random.Random(1)
    seen = set()
    for _ in range(4000):
        m, n, k = rng.choice([1, 2, 5]), 8 * rng.randint(1, 3), 8 * rng.randint(1, 3)
        xs = k + 8 * rng.randint(0, 6)
        ys = rng.choice([xs, n + 8 * rng.randint(0, 6)])
        if ys < n:
            continue
        at = P + 16 * rng.randint(-20, 20)
        want = any(P + 2 * i * xs < at + 2 * (j * ys + n) and at + 2 * j * ys < P + 2 * (i * xs + k)
                   for i in range(m) for j in range(m))
        # (a call that is not refused would go on to the card: where y misses x, w lies on y,
        # which is looked at next)
        d = _dense(T, m=m, n=n, k=k, x_stride=xs, y_stride=ys)
        assert T._dense_fwd(d, P, P + (1 << 24) if want else at, None, None, at, None, None, 0, None) == -1
        assert inl_hip.last_error().endswith("overlap of y and x" if want else "overlap of y and w")
        seen.add(want)
    assert seen == {True, False}


def test_norm_rope_bwd_overlaps(T):
    """dx over dy or x of another type or stride, or shifted. (A call that passes ends at
    the device or the workspace, which are looked at next.)"""
    import inl_hip

    def message(dx, dx_stride=0, dtype=1, out_dtype=1, ys=0):
        d = inl_hip.NormRopeDesc(5, 3, 64, 0, ys, dtype, out_dtype, 1, 1e-6, 0, 1, 0, 0, 0)
        assert T._rope_bwd(d, 2, P, P + (1 << 24), dx, dx_stride, None, None, None, None, None, None, None, P, P, None, 0, None) != 0
        return inl_hip.last_error()
    for dx, kw in ((P + 16, {}), (P, dict(dx_stride=200)), (P, dict(out_dtype=0)), (P, dict(dtype=0)), (P - 16, {}),
                   (P + (1 << 24), dict(dx_stride=256)), (P + (1 << 24) + 5 * 384 - 16, {}), (P + 128, dict(ys=384, dx_stride=384))):
        assert "overlaps" in message(dx, **kw), (dx, kw)
    for dx, kw in ((P, {}), (P + (1 << 24), {}), (P + 5 * 384, {}), (P + 384, dict(ys=384, dx_stride=384)), (1 << 24, {})):
        assert "overlaps" not in message(dx, **kw), (dx, kw)
