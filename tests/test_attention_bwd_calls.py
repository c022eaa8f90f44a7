"""What varlen_attention_bwd hands to the library, and what it refuses itself: its checks run here on tensors of the
host, with the library's call recorded instead of made."""
import pytest
import torch


@pytest.fixture
def call(monkeypatch):
    from inl_hip import train
    made = []
    monkeypatch.setattr(train, "_attn_bwd", lambda *a: made.append(a) or 0)
    monkeypatch.setattr(train, "_stream", lambda dev: None)
    monkeypatch.setattr(train, "_room", lambda n, dev: None)

    def run(grads=None, kv_grad=True, window=-1, grad_dtype=None):
        x = [torch.zeros(9, h, 64, dtype=torch.bfloat16) for h in (4, 2, 2, 4, 4)]
        q, k, v, out, dout = x
        del made[:]
        got = train._attn_grads.__wrapped__(-1, q, dout, k, v, out, [0, 4, 9], False, window, None, None, grad_dtype, grads,
                                            kv_grad)
        return got, made[0]
    return run


def _grads(dtype=torch.bfloat16):
    return tuple(torch.zeros(9, h, 64, dtype=dtype) for h in (4, 2, 2))


def test_kv_grad_leaves_given_tensors_alone(call):
    """Without kv_grad the dk and dv of `grads` are neither written nor returned."""
    g = _grads()
    got, args = call(grads=g, kv_grad=False)
    assert got[0] is g[0] and got[1] is None and got[2] is None
    assert args[7:10] == (g[0].data_ptr(), None, None)
    got, args = call(grads=g)
    assert all(a is b for a, b in zip(got, g)) and args[7:10] == tuple(t.data_ptr() for t in g)
    # nor does their type count
    got, args = call(grads=(g[0],) + _grads(torch.float32)[1:], kv_grad=False, grad_dtype=torch.bfloat16)
    assert got[1] is None and args[1].grad_dtype == 1
    got, args = call(kv_grad=False)
    assert got[0].shape == (9, 4, 64) and got[1] is None and args[8:10] == (None, None)


@pytest.mark.parametrize("window", [2 ** 31, 2 ** 32, 2 ** 32 + 3, -2, -2 ** 32 - 1])
def test_windows_beyond_32_bits_are_refused(window, call):
    """They would reach the library as their low 32 bits: 2^32 as a window of 0."""
    import inl_hip
    with pytest.raises(inl_hip.InlError, match="window"):
        call(window=window)


def test_windows(call):
    for window, want in ((None, -1), (-1, -1), (0, 0), (2 ** 31 - 1, 2 ** 31 - 1)):
        assert call(window=window)[1][0].window == want


def test_kernel_names():
    """By the batch's fill of a GPU of 256 compute units, each by the widest of its features."""
    import ctypes

    import inl_hip
    from inl_hip import train

    def names(lengths, hq, hkv, hd, causal=False, window=-1):
        cu = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
        return inl_hip.attention_bwd_kernel_names(inl_hip.make_attn_desc(cu, hq, hkv, hd, causal=causal, window=window))
    assert names([257] * 64, 16, 16, 40) == ("attn_bwd_kernel<64, false, 1>", "attn_bwd_kernel<64, true, 1>")
    assert names([900], 16, 16, 64) == ("attn_bwd_kernel<64, false, 2>", "attn_bwd_kernel<64, true, 2>")
    assert names([257] * 64, 16, 8, 72, True) == ("attn_bwd_kernel<128, false, 1>", "attn_bwd_kernel<128, true, 2>")
    assert names([300] * 32, 3, 1, 256, True) == ("attn_bwd_kernel<256, false, 1>", "attn_bwd_pair_kernel<256>")
    assert names([23], 16, 8, 128, True) == ("attn_bwd_kernel<128, false, 1>", "attn_bwd_kernel<128, true, 1>")
    assert names([0, 0], 2, 2, 64) == ("none", "none")
    d = inl_hip.make_attn_desc([0, 5], 2, 2, 64, causal=False)
    name = ctypes.c_char_p()
    assert train._attn_bwd_name(d, 2, ctypes.byref(name)) == -1 and train._attn_bwd_name(d, 0, None) == -1
    assert train._attn_bwd_name(None, 0, ctypes.byref(name)) == -1 and name.value is None
    with pytest.raises(inl_hip.InlError, match="bf16"):
        inl_hip.attention_bwd_kernel_names(inl_hip.make_attn_desc([0, 5], 2, 2, 64, causal=False, dtype="f32"))


_EMPTY = """
import sys
sys.path[:0] = {path!r}
import inl_hip
from inl_hip import train as T
MB = 1 << 20
# no texts: dpooled and mean are empty, wherever they point; cu lies in dhidden and is what is refused
a = T._pool_mean_bwd(0, MB + 64, 8, 100, 8, 1, MB + 32, MB + 48, MB, None)
assert a == -1 and "overlaps" in inl_hip.last_error(), (a, inl_hip.last_error())
b = T._pool_last_bwd(0, MB + 64, 8, 100, 8, 1, MB + 32, 2 * MB, None, 1e-6, 8, 1, MB, None, None, 0, None)
assert b == -1 and "overlaps" in inl_hip.last_error(), (b, inl_hip.last_error())
"""


def test_empty_tensors_inside_an_output():
    """An empty dpooled whose address lies in dhidden shares no byte with it (in a process of its own: the check of the
    overlap divided by its length)."""
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", _EMPTY.format(path=sys.path)], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stderr[-800:])


@pytest.mark.parametrize("stride", [1 << 24, 1 << 31, 1 << 40, 1 << 60, 1 << 61, 1 << 62])
def test_rows_that_lie_far_apart_are_refused(stride):
    """A text's rows are addressed with 32 bits: no stride passes as its low bits."""
    import inl_hip
    from inl_hip import train as T
    far = [(i + 1) << 44 for i in range(8)]
    for name in ("q", "k", "v", "o"):
        d = inl_hip.make_attn_desc([0, 1], 2, 2, 64, causal=True, **{f"{name}_row_stride": stride})
        assert T._attn_bwd(d, T.AttnGrads(grad_dtype=1), *far, None, 0, None) == -2, name
        assert "4 GiB" in inl_hip.last_error()
    d = inl_hip.make_attn_desc([0, 1], 2, 2, 64, causal=True)
    for name in ("do", "dq", "dk", "dv"):
        g = T.AttnGrads(**{f"{name}_row_stride": stride, "grad_dtype": 0})
        assert T._attn_bwd(d, g, *far, None, 0, None) == -2 and "4 GiB" in inl_hip.last_error(), name
