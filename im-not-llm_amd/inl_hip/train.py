"""Layer and head ops with their gradients (``include/inl_train.h``): a linear
layer with bias, activation and residual, the gated feed-forward block, softmax
cross entropy without its scores, and the gradients of the q/k prologue.

Gradients are plain functions of what the forward left (no autograd graph is
kept): a ``torch.autograd.Function`` or a training loop calls them in its own
backward. Outputs and workspaces come from torch's allocator, so calls can be
captured into a graph.
"""
from __future__ import annotations

import contextlib
import ctypes

from . import (INL_BF16, INL_F32, InlError, NormRopeDesc, _check, _dtype_code, _lib, _sig, _stream_ptr, c_i32, c_i64,
               c_void_p)

ACTS = {None: 0, "none": 0, "relu": 1, "silu": 2, "gelu_tanh": 3, "gelu_erf": 4}
ROPE_HALF, ROPE_AXIAL, ROPE_INTERLEAVED = 1, 2, 3

_size_p = ctypes.POINTER(ctypes.c_size_t)


class DenseDesc(ctypes.Structure):
    _fields_ = [(n, c_i64) for n in ("m", "n", "k", "x_stride", "w_stride", "y_stride", "residual_stride",
                                     "pre_stride", "dx_stride", "dw_stride")] + \
               [(n, c_i32) for n in ("act", "out_dtype", "residual_dtype", "dx_dtype", "dw_dtype")]


class GatedFfnDesc(ctypes.Structure):
    _fields_ = [(n, c_i64) for n in ("m", "hidden", "inner", "x_stride", "y_stride", "residual_stride",
                                     "dx_stride")] + \
               [(n, c_i32) for n in ("act", "out_dtype", "residual_dtype", "dx_dtype", "dw_dtype")]


class SoftmaxXentDesc(ctypes.Structure):
    _fields_ = [(n, c_i64) for n in ("m", "vocab", "hidden", "x_stride", "w_stride", "dx_stride", "dw_stride")] + \
               [("scale", ctypes.c_float)] + [(n, c_i32) for n in ("ignore_index", "dx_dtype", "dw_dtype")]


def _ptrs(n):
    return [c_void_p] * n


_dense_ws = _sig("inl_dense_workspace_size", ctypes.c_int, ctypes.POINTER(DenseDesc), c_i32, _size_p)
_dense_fwd = _sig("inl_dense_fwd", ctypes.c_int, ctypes.POINTER(DenseDesc), *_ptrs(7), ctypes.c_size_t, c_void_p)
_dense_bwd = _sig("inl_dense_bwd", ctypes.c_int, ctypes.POINTER(DenseDesc), *_ptrs(8), ctypes.c_size_t, c_void_p)
_ffn_ws = _sig("inl_gated_ffn_workspace_size", ctypes.c_int, ctypes.POINTER(GatedFfnDesc), c_i32, _size_p)
_ffn_fwd = _sig("inl_gated_ffn_fwd", ctypes.c_int, ctypes.POINTER(GatedFfnDesc), *_ptrs(8), ctypes.c_size_t, c_void_p)
_ffn_bwd = _sig("inl_gated_ffn_bwd", ctypes.c_int, ctypes.POINTER(GatedFfnDesc), *_ptrs(10), ctypes.c_size_t,
                c_void_p)
_xent_ws = _sig("inl_softmax_xent_workspace_size", ctypes.c_int, ctypes.POINTER(SoftmaxXentDesc), c_i32, _size_p)
_xent_fwd = _sig("inl_softmax_xent_fwd", ctypes.c_int, ctypes.POINTER(SoftmaxXentDesc), *_ptrs(7), ctypes.c_size_t,
                 c_void_p)
_xent_bwd = _sig("inl_softmax_xent_bwd", ctypes.c_int, ctypes.POINTER(SoftmaxXentDesc), *_ptrs(10), ctypes.c_size_t,
                 c_void_p)
_rope_bwd_ws = _sig("inl_norm_rope_bwd_workspace_size", ctypes.c_int, ctypes.POINTER(NormRopeDesc), _size_p)
_rope_bwd = _sig("inl_norm_rope_qk_bwd", ctypes.c_int, ctypes.POINTER(NormRopeDesc), c_i32, *_ptrs(3), c_i64,
                 *_ptrs(10), ctypes.c_size_t, c_void_p)


def _on(t):
    """The device of ``t`` as the current one: the library launches there."""
    import torch
    if not t.is_cuda:
        raise InlError(-1, f"not a device tensor ({t.device})")
    if t.device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(t.device)


def _mat(name, t, shape, dtypes, like):
    """``t`` as rows of a matrix for the library, which sees only a pointer: its
    shape, type and device, and contiguous rows. Returns the row stride."""
    if tuple(t.shape) != tuple(shape):
        raise InlError(-1, f"{name}: shape {tuple(t.shape)}, need {tuple(shape)}")
    if t.dtype not in dtypes:
        raise InlError(-1, f"{name}: dtype {t.dtype}, need {' or '.join(str(d) for d in dtypes)}")
    if t.device != like.device:
        raise InlError(-1, f"{name}: on {t.device}, x is on {like.device}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise InlError(-1, f"{name}: rows must be contiguous")
    return t.stride(0) if t.dim() > 1 and t.shape[0] > 1 else t.shape[-1]


def _vec(name, t, n, dtype, like):
    if t is None:
        return None
    if tuple(t.shape) != (n,) or t.dtype != dtype or t.device != like.device or (n > 1 and t.stride(0) != 1):
        raise InlError(-1, f"{name}: need contiguous {dtype} [{n}] on {like.device}, got {t.dtype} {tuple(t.shape)} "
                           f"on {t.device}")
    return t.data_ptr()


def _types():
    import torch
    return (torch.bfloat16,), (torch.bfloat16, torch.float32)


def _act(act, gated=False):
    if act not in ACTS or (gated and not ACTS[act]):
        raise InlError(-1, f"unknown act {act!r}")
    return ACTS[act]


def _workspace(size_fn, desc, like, *args):
    import torch
    n = ctypes.c_size_t()
    _check(size_fn(ctypes.byref(desc), *args, ctypes.byref(n)))
    return torch.empty(n.value, dtype=torch.uint8, device=like.device) if n.value else None


def _done(stream, *tensors):
    """Tensors allocated here that work on another stream than the current one
    uses: the allocator must not hand their memory out before it is done."""
    import torch
    if stream is None or stream == torch.cuda.current_stream():
        return
    for t in tensors:
        if t is not None:
            t.record_stream(stream)


def _ptr(t):
    return None if t is None else t.data_ptr()


# ---------------------------------------------------------------------------
# Linear layer
# ---------------------------------------------------------------------------

def dense(x, w, bias=None, *, act=None, residual=None, pre=None, out=None, out_dtype=None, stream=None):
    """``act(x @ w.T + bias) + residual`` (``inl_dense_fwd``): bf16 ``x [m, k]``
    and ``w [n, k]``, f32 ``bias [n]``, ``act`` one of None, "relu", "silu",
    "gelu_tanh", "gelu_erf", ``residual [m, n]`` bf16 or f32 (it may be
    ``out``). ``pre``: a bf16 ``[m, n]`` tensor that receives ``x @ w.T + bias`` for
    ``dense_bwd``. n and k are multiples of 8; rows may be strided."""
    import torch
    b16, any_ = _types()
    m, k = x.shape
    n = w.shape[0]
    with _on(x):
        d = DenseDesc(m=m, n=n, k=k, act=_act(act))
        d.x_stride, d.w_stride = _mat("x", x, (m, k), b16, x), _mat("w", w, (n, k), b16, x)
        made = out is None
        if made:
            out = torch.empty((m, n), dtype=out_dtype or torch.bfloat16, device=x.device)
        d.y_stride, d.out_dtype = _mat("out", out, (m, n), any_, x), _dtype_code(out.dtype)
        if residual is not None:
            d.residual_stride = _mat("residual", residual, (m, n), any_, x)
            d.residual_dtype = _dtype_code(residual.dtype)
        if pre is not None:
            d.pre_stride = _mat("pre", pre, (m, n), b16, x)
        ws = _workspace(_dense_ws, d, x, 0)
        _check(_dense_fwd(ctypes.byref(d), x.data_ptr(), w.data_ptr(), _vec("bias", bias, n, torch.float32, x),
                          _ptr(residual), out.data_ptr(), _ptr(pre), _ptr(ws), ws.numel() if ws is not None else 0,
                          _stream_ptr(stream)))
        _done(stream, ws, out if made else None)
    return out


def dense_bwd(dy, x, w, *, act=None, pre=None, bias_grad=False, dx_grad=True, dw_grad=True, dx_dtype=None,
              dw_dtype=None, stream=None):
    """``(dx, dw, dbias)`` of ``dense`` from bf16 ``dy [m, n]`` (``inl_dense_bwd``);
    ``pre`` is what the forward stored (not needed without an activation). dx and dw are
    bf16 unless ``dx_dtype``/``dw_dtype`` say float32, dbias f32; what is not asked
    for is None. The residual's gradient is ``dy``."""
    import torch
    b16, _ = _types()
    m, n = dy.shape
    k = x.shape[1]
    with _on(x):
        d = DenseDesc(m=m, n=n, k=k, act=_act(act))
        d.x_stride, d.w_stride = _mat("x", x, (m, k), b16, x), _mat("w", w, (n, k), b16, x)
        d.y_stride = _mat("dy", dy, (m, n), b16, x)
        if d.act:
            if pre is None:
                raise InlError(-1, "dense_bwd: an activation needs pre")
            d.pre_stride = _mat("pre", pre, (m, n), b16, x)
        else:
            pre = None
        dx = torch.empty((m, k), dtype=dx_dtype or torch.bfloat16, device=x.device) if dx_grad else None
        dw = torch.empty((n, k), dtype=dw_dtype or torch.bfloat16, device=x.device) if dw_grad else None
        db = torch.empty(n, dtype=torch.float32, device=x.device) if bias_grad else None
        d.dx_dtype = _dtype_code(dx.dtype) if dx_grad else INL_BF16
        d.dw_dtype = _dtype_code(dw.dtype) if dw_grad else INL_BF16
        ws = _workspace(_dense_ws, d, x, 1)
        _check(_dense_bwd(ctypes.byref(d), dy.data_ptr(), x.data_ptr(), w.data_ptr(), _ptr(pre), _ptr(dx), _ptr(dw),
                          _ptr(db), _ptr(ws), ws.numel() if ws is not None else 0, _stream_ptr(stream)))
        _done(stream, ws, dx, dw, db)
    return dx, dw, db


# ---------------------------------------------------------------------------
# Gated feed-forward block
# ---------------------------------------------------------------------------

def gated_ffn(x, w_gate_up, w_down, *, act="silu", residual=None, save=False, out=None, out_dtype=None, stream=None):
    """``(act(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T + residual``
    (``inl_gated_ffn_fwd``): bf16 ``x [m, hidden]``, ``w_gate_up [2 inner, hidden]``
    (gate rows, then up rows) and ``w_down [hidden, inner]``, both packed; ``act``
    "silu", "gelu_tanh", "gelu_erf" or "relu". ``save=True`` returns ``(out, pre,
    h)`` with what ``gated_ffn_bwd`` reads: the gate and up products ``[m, 2
    inner]`` and ``h [m, inner]``, bf16."""
    import torch
    b16, any_ = _types()
    m, hidden = x.shape
    inner = w_down.shape[1]
    with _on(x):
        d = GatedFfnDesc(m=m, hidden=hidden, inner=inner, act=_act(act, True))
        d.x_stride = _mat("x", x, (m, hidden), b16, x)
        _packed("w_gate_up", w_gate_up, (2 * inner, hidden), x)
        _packed("w_down", w_down, (hidden, inner), x)
        made = out is None
        if made:
            out = torch.empty((m, hidden), dtype=out_dtype or torch.bfloat16, device=x.device)
        d.y_stride, d.out_dtype = _mat("out", out, (m, hidden), any_, x), _dtype_code(out.dtype)
        if residual is not None:
            d.residual_stride = _mat("residual", residual, (m, hidden), any_, x)
            d.residual_dtype = _dtype_code(residual.dtype)
        pre = torch.empty((m, 2 * inner), dtype=torch.bfloat16, device=x.device) if save else None
        h = torch.empty((m, inner), dtype=torch.bfloat16, device=x.device) if save else None
        ws = _workspace(_ffn_ws, d, x, 0)
        _check(_ffn_fwd(ctypes.byref(d), x.data_ptr(), w_gate_up.data_ptr(), w_down.data_ptr(), _ptr(residual),
                        out.data_ptr(), _ptr(pre), _ptr(h), _ptr(ws), ws.numel() if ws is not None else 0,
                        _stream_ptr(stream)))
        _done(stream, ws, pre, h, out if made else None)
    return (out, pre, h) if save else out


def _packed(name, t, shape, like):
    if _mat(name, t, shape, _types()[0], like) != shape[1]:
        raise InlError(-1, f"{name}: must be packed")


def gated_ffn_bwd(dy, x, w_gate_up, w_down, pre, h, *, act="silu", dx_grad=True, dw_grad=True, dx_dtype=None,
                  dw_dtype=None, stream=None):
    """``(dx, dw_gate_up, dw_down)`` of ``gated_ffn`` from bf16 ``dy [m, hidden]`` and
    the ``pre`` and ``h`` that the forward saved (``inl_gated_ffn_bwd``); bf16 unless
    ``dx_dtype``/``dw_dtype`` say float32."""
    import torch
    b16, _ = _types()
    m, hidden = x.shape
    inner = w_down.shape[1]
    with _on(x):
        d = GatedFfnDesc(m=m, hidden=hidden, inner=inner, act=_act(act, True))
        d.x_stride, d.y_stride = _mat("x", x, (m, hidden), b16, x), _mat("dy", dy, (m, hidden), b16, x)
        for name, t, shape in (("w_gate_up", w_gate_up, (2 * inner, hidden)), ("w_down", w_down, (hidden, inner)),
                               ("pre", pre, (m, 2 * inner)), ("h", h, (m, inner))):
            _packed(name, t, shape, x)
        wd = dw_dtype or torch.bfloat16
        dx = torch.empty((m, hidden), dtype=dx_dtype or torch.bfloat16, device=x.device) if dx_grad else None
        dgu = torch.empty((2 * inner, hidden), dtype=wd, device=x.device) if dw_grad else None
        ddown = torch.empty((hidden, inner), dtype=wd, device=x.device) if dw_grad else None
        d.dx_dtype = _dtype_code(dx.dtype) if dx_grad else INL_BF16
        d.dw_dtype = _dtype_code(wd)
        ws = _workspace(_ffn_ws, d, x, 1)
        _check(_ffn_bwd(ctypes.byref(d), dy.data_ptr(), x.data_ptr(), w_gate_up.data_ptr(), w_down.data_ptr(),
                        pre.data_ptr(), h.data_ptr(), _ptr(dx), _ptr(dgu), _ptr(ddown), _ptr(ws),
                        ws.numel() if ws is not None else 0, _stream_ptr(stream)))
        _done(stream, ws, dx, dgu, ddown)
    return dx, dgu, ddown


# ---------------------------------------------------------------------------
# Softmax cross entropy
# ---------------------------------------------------------------------------

def _xent_desc(x, w, scale, ignore_index):
    b16, _ = _types()
    m, hidden = x.shape
    d = SoftmaxXentDesc(m=m, vocab=w.shape[0], hidden=hidden, scale=float(scale), ignore_index=int(ignore_index))
    d.x_stride, d.w_stride = _mat("x", x, (m, hidden), b16, x), _mat("w", w, (w.shape[0], hidden), b16, x)
    return d


def softmax_xent(x, w, targets, *, bias=None, scale=1.0, ignore_index=-100, stream=None):
    """``(loss, lse)``, f32 ``[m]``, of the scores ``scale * x @ w.T + bias``, which are
    not stored (``inl_softmax_xent_fwd``): bf16 ``x [m, hidden]`` and ``w [vocab,
    hidden]`` (a decoder, or the documents of a batch with ``scale`` = 1 /
    temperature), f32 ``bias [vocab]``, int32 ``targets [m]``. Rows whose target is
    ``ignore_index`` have loss 0; a target outside the vocabulary gives NaN."""
    import torch
    m = x.shape[0]
    with _on(x):
        d = _xent_desc(x, w, scale, ignore_index)
        loss, lse = torch.empty((2, m), dtype=torch.float32, device=x.device).unbind(0)
        ws = _workspace(_xent_ws, d, x, 0)
        _check(_xent_fwd(ctypes.byref(d), x.data_ptr(), w.data_ptr(), _vec("bias", bias, d.vocab, torch.float32, x),
                         _vec("targets", targets, m, torch.int32, x), loss.data_ptr(), lse.data_ptr(), _ptr(ws),
                         ws.numel() if ws is not None else 0, _stream_ptr(stream)))
        _done(stream, ws, loss, lse)
    return loss, lse


def softmax_xent_bwd(dloss, lse, x, w, targets, *, bias=None, scale=1.0, ignore_index=-100, dx_grad=True,
                     dw_grad=True, bias_grad=False, dx_dtype=None, dw_dtype=None, stream=None):
    """``(dx, dw, dbias)`` of ``softmax_xent`` from f32 ``dloss [m]`` and the forward's
    ``lse`` (``inl_softmax_xent_bwd``); dx and dw bf16 unless ``dx_dtype``/``dw_dtype``
    say float32, dbias f32; what is not asked for is None."""
    import torch
    m, f32 = x.shape[0], torch.float32
    with _on(x):
        d = _xent_desc(x, w, scale, ignore_index)
        dx = torch.empty(x.shape, dtype=dx_dtype or torch.bfloat16, device=x.device) if dx_grad else None
        dw = torch.empty(w.shape, dtype=dw_dtype or torch.bfloat16, device=x.device) if dw_grad else None
        db = torch.empty(d.vocab, dtype=f32, device=x.device) if bias_grad else None
        d.dx_dtype = _dtype_code(dx.dtype) if dx_grad else INL_BF16
        d.dw_dtype = _dtype_code(dw.dtype) if dw_grad else INL_BF16
        ws = _workspace(_xent_ws, d, x, 1)
        _check(_xent_bwd(ctypes.byref(d), _vec("dloss", dloss, m, f32, x), _vec("lse", lse, m, f32, x), x.data_ptr(),
                         w.data_ptr(), _vec("bias", bias, d.vocab, f32, x), _vec("targets", targets, m, torch.int32, x),
                         _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), ws.numel() if ws is not None else 0,
                         _stream_ptr(stream)))
        _done(stream, ws, dx, dw, db)
    return dx, dw, db


# ---------------------------------------------------------------------------
# q/k prologue
# ---------------------------------------------------------------------------

def _heads(name, t, shape, like):
    if tuple(t.shape) != tuple(shape) or t.device != like.device:
        raise InlError(-1, f"{name}: shape {tuple(t.shape)} on {t.device}, need {tuple(shape)} on {like.device}")
    if t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != t.shape[2]):
        raise InlError(-1, f"{name}: heads must be contiguous inside a token row")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1] * t.shape[2]


def norm_rope_qk_bwd(dy, x, q_heads, rows=None, cos=None, sin=None, *, q_weight=None, k_weight=None, eps=1e-6,
                     norm=True, rotary_dim=None, sections=1, cos2=None, sin2=None, round_tables=False, out=None,
                     weight_grad=True, stream=None):
    """``(dx, dq_weight, dk_weight)`` of ``norm_rope_qk`` from ``dy [N, heads,
    head_dim]`` and the forward's ``x`` (``inl_norm_rope_qk_bwd``); the other
    arguments as in the forward. dx has x's dtype (``out`` may be a slice of wider rows), the
    weight gradients are f32 ``[head_dim]`` and None without a norm, with
    ``weight_grad=False`` or, dk_weight, where all heads are q heads."""
    import torch
    n, heads, hd = x.shape
    with _on(x):
        d = NormRopeDesc()
        d.n_tokens, d.heads, d.head_dim = n, heads, hd
        d.x_row_stride, d.y_row_stride = _heads("x", x, (n, heads, hd), x), _heads("dy", dy, (n, heads, hd), x)
        d.dtype, d.out_dtype = _dtype_code(x.dtype), _dtype_code(dy.dtype)
        d.norm, d.eps = int(bool(norm)), float(eps)
        d.rotary_dim = int((hd if cos is not None else 0) if rotary_dim is None else rotary_dim)
        d.sections, d.round_tables = int(sections), int(bool(round_tables))
        d.table_rows = int(cos.shape[0]) if cos is not None else 0
        if d.rotary_dim:
            width = hd // 4 if sections == ROPE_AXIAL else d.rotary_dim // 2
            for name, t in (("cos", cos), ("sin", sin), ("cos2", cos2), ("sin2", sin2)):
                if t is None and name in ("cos2", "sin2") and sections != ROPE_AXIAL:
                    continue
                if t is None or tuple(t.shape) != (d.table_rows, width) or t.dtype != torch.float32 \
                        or not t.is_contiguous() or t.device != x.device:
                    raise InlError(-1, f"{name}: need contiguous f32 [{d.table_rows}, {width}] on {x.device}")
            _vec("rows", rows, n, torch.int32, x)
        made = out is None
        if made:
            out = torch.empty((n, heads, hd), dtype=x.dtype, device=x.device)
        elif out.dtype != x.dtype:
            raise InlError(-1, f"out: dtype {out.dtype}, need {x.dtype}")
        ds = _heads("out", out, (n, heads, hd), x)
        grads = bool(norm and weight_grad)
        dq = torch.empty(hd, dtype=torch.float32, device=x.device) if grads else None
        dk = torch.empty(hd, dtype=torch.float32, device=x.device) if grads and q_heads < heads else None
        ws = _workspace(_rope_bwd_ws, d, x) if grads else None
        _check(_rope_bwd(ctypes.byref(d), int(q_heads), dy.data_ptr(), x.data_ptr(), out.data_ptr(), ds,
                         _vec("q_weight", q_weight, hd, x.dtype, x), _vec("k_weight", k_weight, hd, x.dtype, x),
                         _ptr(rows), _ptr(cos), _ptr(sin), _ptr(cos2), _ptr(sin2), _ptr(dq), _ptr(dk), _ptr(ws),
                         ws.numel() if ws is not None else 0, _stream_ptr(stream)))
        _done(stream, ws, dq, dk, out if made else None)
    return out, dq, dk
