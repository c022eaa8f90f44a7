"""inl_attn_varlen_bwd refuses bad arguments on the host, before any GPU call: pointers here are
made up and never read."""
import ctypes

import pytest

MB = 1 << 20


@pytest.fixture(scope="module")
def T():
    from inl_hip import train
    return train


def _call(T, lengths=(5, 0, 9), ptrs=None, ws=None, ws_bytes=0, starts=None, grads=None, cu=None, dtype="bf16",
          out_dtype="bf16", hq=4, hkv=2, hd=64, no_grads=False, **kw):
    import inl_hip
    cu = cu or [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    d = inl_hip.make_attn_desc(cu, hq, hkv, hd, causal=True, dtype=dtype, out_dtype=out_dtype, seq_starts=starts)
    for k, v in kw.items():
        setattr(d, k, v)
    p = [MB * (i + 1) for i in range(8)]   # q, k, v, out, dout, dq, dk, dv: far apart
    for i, v in (ptrs or {}).items():
        p[i] = v
    g = T.AttnGrads(**{"grad_dtype": 1, **(grads or {})})
    return T._attn_bwd(d, None if no_grads else g, *p, ws, ws_bytes, None)


def _said(word):
    import inl_hip
    return word in inl_hip.last_error()


def test_types_and_shapes(T):
    assert _call(T, dtype="f32", out_dtype="f32") == -2 and _said("bf16")
    assert _call(T, out_dtype="f32") == -2
    assert _call(T, hd=60) == -2 and _call(T, hd=264) == -2 and _call(T, hq=3) == -1
    assert _call(T, cu=[0, 5, 3]) == -1 and _call(T, cu=[1, 5, 9]) == -1
    assert _call(T, window=-2) == -1 and _call(T, scale=0.0) == -1 and _call(T, scale=float("nan")) == -1
    assert _call(T, grads=dict(grad_dtype=2)) == -1 and _said("grad_dtype")
    assert _call(T, no_grads=True) == -1
    assert T._attn_bwd(None, None, *[None] * 8, None, 0, None) == -1


@pytest.mark.parametrize("i", range(8))
def test_pointers(i, T):
    assert _call(T, ptrs={i: MB * (i + 1) + 8}) == -1 and _said("aligned")
    if i < 5:
        assert _call(T, ptrs={i: None}) == -1 and _said("non-null")


def test_strides(T):
    for name in ("q", "k", "v", "o"):
        assert _call(T, **{f"{name}_row_stride": 64}) == -1
        assert _call(T, **{f"{name}_row_stride": 260}) == -1
    for name in ("do", "dq", "dk", "dv"):
        assert _call(T, grads={f"{name}_row_stride": 64}) == -1 and _said("stride")
        assert _call(T, grads={f"{name}_row_stride": 261}) == -1
    # 4 GiB of one text's rows
    assert _call(T, lengths=(4096,), q_row_stride=1 << 19, ptrs={i: (i + 1) << 40 for i in range(8)}) == -2 and _said("span")


def test_overlaps(T):
    assert _call(T, ptrs={5: MB}) == -1 and _said("dq overlaps q")
    assert _call(T, ptrs={6: 7 * MB + 16, 7: 7 * MB}) == -1 and _said("dv overlaps dk")
    assert _call(T, ptrs={7: 5 * MB + 64}) == -1 and _said("dv overlaps dout")
    assert _call(T, ptrs={6: None}) == -1 and _said("together")
    # slices of one row do not
    row = (4 + 2 + 2) * 64
    slices = {5: 9 * MB, 6: 9 * MB + 4 * 128, 7: 9 * MB + 6 * 128}
    assert _call(T, ptrs=slices, grads=dict(dq_row_stride=row, dk_row_stride=row, dv_row_stride=row)) == -1
    assert _said("workspace")
    assert _call(T, ptrs={**slices, 7: 9 * MB + 5 * 128},
                 grads=dict(dq_row_stride=row, dk_row_stride=row, dv_row_stride=row)) == -1 and _said("dv overlaps dk")


def test_texts_of_a_padded_batch(T):
    assert _call(T, starts=[0, 0, 20]) == -1 and _said("workspace")
    assert _call(T, starts=[0, 0, 4]) == -1 and _said("texts overlap")
    assert _call(T, lengths=(5, 3, 9), starts=[10, 12, 20]) == -1 and _said("texts overlap")
    assert _call(T, starts=[-1, 0, 20]) == -1


def test_workspace(T):
    import inl_hip
    n = ctypes.c_size_t()
    d = inl_hip.make_attn_desc([0, 5, 14], 4, 2, 64, causal=True)
    assert T._attn_bwd_ws(d, ctypes.byref(n)) == 0 and n.value >= 2 * 4 * 14 * 4
    assert _call(T, ws=None) == -1 and _said("workspace")
    assert _call(T, ws=9 * MB + 8, ws_bytes=MB) == -1 and _call(T, ws=9 * MB, ws_bytes=n.value - 1) == -1
    assert T._attn_bwd_ws(d, None) == -1 and T._attn_bwd_ws(None, ctypes.byref(n)) == -1
    # nothing to do needs nothing
    d = inl_hip.make_attn_desc([0, 0], 4, 2, 64, causal=True)
    assert T._attn_bwd_ws(d, ctypes.byref(n)) == 0 and n.value == 0
    assert _call(T, lengths=(0, 0), ptrs={i: None for i in range(8)}) == 0
    assert _call(T, ptrs={5: None, 6: None, 7: None}) == 0


def test_binding_checks_tensors():
    import torch

    import inl_hip
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(inl_hip.InlError, match="not a device tensor"):
        inl_hip.varlen_attention_bwd(x, x, x, x, x, [0, 4], causal=True)


def test_listing_check_finds_missing_waits():
    """A descriptor word that v_readfirstlane wrote is read five wait states later at the earliest."""
    import importlib.util
    from pathlib import Path
    path = Path(__file__).resolve().parent.parent / "im-not-llm_amd" / "asmcheck.py"
    spec = importlib.util.spec_from_file_location("asmcheck_waits", path)
    check = importlib.util.module_from_spec(spec)
    import sys
    sys.modules[spec.name] = check
    spec.loader.exec_module(check)
    head = "_kernel:\n\tv_readfirstlane_b32 s61, v3\n\ts_mov_b32 m0, s4\n"
    load = "\tbuffer_load_dwordx4 v3, s[60:63], 0 offen lds\n"
    assert len(check.check_sgpr_waits(head + "\ts_nop 0\n" + load)) == 1
    assert len(check.check_sgpr_waits(head + "\ts_nop 2\n" + load)) == 1
    assert not check.check_sgpr_waits(head + "\ts_nop 3\n" + load)
    assert not check.check_sgpr_waits(head + "\ts_mov_b32 s61, s7\n" + load)
    assert not check.check_sgpr_waits("_kernel:\n\tv_readfirstlane_b32 s40, v3\n" + load)
    assert not check.check_sgpr_waits(head + "_other:\n" + load)


def test_too_many_blocks(T):
    """The span of a text allows it, the number of blocks does not."""
    far = {i: (i + 1) << 44 for i in range(8)}
    assert _call(T, lengths=[1] * 300, hq=1 << 20, hkv=1, hd=8, ptrs=far) == -2 and _said("blocks")
