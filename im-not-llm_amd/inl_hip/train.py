"""Layer and head ops with their gradients (``include/inl_train.h``): a linear
layer with bias, activation and residual, the gated feed-forward block, softmax
cross entropy without its scores, the residual stream's addition with dropout and
norm, and the gradients of the q/k prologue, of attention and of the pooled embedding.

Gradients are plain functions of what the forward left (outputs carry no autograd
graph, whatever ``requires_grad`` says of the inputs): a ``torch.autograd.Function`` or
a training loop calls them in its own backward. Outputs and workspaces come from torch's allocator, so calls can be
captured into a graph. With ``stream=`` a call works there and takes its memory there;
that its inputs are ready on that stream, and that their memory is not handed on
before it is done (``record_stream``), is up to the caller, as it is that the current
stream waits before it uses the outputs.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import (INL_BF16, INL_F32, AttnDesc, InlError, NormRopeDesc, _check, _cu_array, _dtype_code, _head_rows,
               _head_weight, _rope_tables, _sig, c_i32, c_i64, c_void_p, desc_rows, make_attn_desc)

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


class AttnGrads(ctypes.Structure):
    _fields_ = [(n, c_i64) for n in ("do_row_stride", "dq_row_stride", "dk_row_stride", "dv_row_stride")] + \
               [("grad_dtype", c_i32)]


class AddNormDesc(ctypes.Structure):
    _fields_ = [(n, c_i64) for n in ("m", "n", "x_stride", "residual_stride", "h_stride", "y_stride", "dh_stride")] + \
               [("eps", ctypes.c_float)] + \
               [(n, c_i32) for n in ("drop", "tag", "x_dtype", "stream_dtype", "out_dtype", "weight_dtype")]


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


_attn_bwd_ws = _sig("inl_attn_bwd_workspace_size", ctypes.c_int, ctypes.POINTER(AttnDesc), _size_p)
_attn_bwd_name = _sig("inl_attn_bwd_kernel_name", ctypes.c_int, ctypes.POINTER(AttnDesc), c_i32,
                      ctypes.POINTER(ctypes.c_char_p))
_attn_bwd = _sig("inl_attn_varlen_bwd", ctypes.c_int, ctypes.POINTER(AttnDesc), ctypes.POINTER(AttnGrads), *_ptrs(9),
                 ctypes.c_size_t, c_void_p)
_add_norm = _sig("inl_add_rms_norm_fwd", ctypes.c_int, ctypes.POINTER(AddNormDesc), *_ptrs(7))
_add_norm_ws = _sig("inl_add_rms_norm_bwd_workspace_size", ctypes.c_int, ctypes.POINTER(AddNormDesc), _size_p)
_add_norm_bwd = _sig("inl_add_rms_norm_bwd", ctypes.c_int, ctypes.POINTER(AddNormDesc), *_ptrs(9), ctypes.c_size_t,
                     c_void_p)
_pool_mean_bwd = _sig("inl_pool_mean_bwd", ctypes.c_int, c_i32, c_void_p, c_i32, c_i64, c_i64, c_i32, *_ptrs(4))
_pool_last_ws = _sig("inl_pool_last_bwd_workspace_size", ctypes.c_int, c_i32, c_i32, _size_p)
_pool_last_bwd = _sig("inl_pool_last_bwd", ctypes.c_int, c_i32, c_void_p, c_i32, c_i64, c_i64, c_i32, *_ptrs(3),
                      ctypes.c_float, c_i64, c_i32, *_ptrs(3), ctypes.c_size_t, c_void_p)

_BF16, _F32 = torch.bfloat16, torch.float32
_B16, _ANY = (_BF16,), (_BF16, _F32)
_CODE = {_BF16: INL_BF16, _F32: INL_F32}


def _at_home(call):
    """Runs ``call(device, first, *args)`` with the device of its first tensor as the
    current one and ``stream`` (the last argument; None: the current one) as the
    current stream: the library launches there, and workspaces and outputs come from
    that stream's memory. A block of another stream's could still be in use by work
    queued there, which ``stream`` does not wait for."""
    @functools.wraps(call)
    def wrapped(first, *args):
        *args, stream = args
        dev = first.get_device()
        if dev < 0:
            raise InlError(-1, f"not a device tensor ({first.device})")
        if stream is not None:
            if stream.device.index != dev:   # a launch there would use this device's addresses
                raise InlError(-1, f"the stream is on {stream.device}, the tensors on cuda:{dev}")
            callers = torch.cuda.current_stream(dev)
            if stream != callers:
                with torch.cuda.stream(stream):
                    made = call(dev, first, *args)
                # the caller goes on with them on its own stream, once that has waited
                for t in made if isinstance(made, tuple) else (made,):
                    if t is not None:
                        t.record_stream(callers)
                return made
        if dev == torch._C._cuda_getDevice():
            return call(dev, first, *args)
        with torch.cuda.device(dev):
            return call(dev, first, *args)
    return wrapped


def _mat(name, t, rows, cols, dtypes, dev):
    """``t`` as rows of a matrix for the library, which sees only a pointer: its
    shape, type and device, and contiguous rows. Returns the row stride."""
    if t.shape != (rows, cols):
        raise InlError(-1, f"{name}: shape {tuple(t.shape)}, need {(rows, cols)}")
    if t.dtype not in dtypes:
        raise InlError(-1, f"{name}: dtype {t.dtype}, need {' or '.join(str(d) for d in dtypes)}")
    if t.get_device() != dev:
        raise InlError(-1, f"{name}: on {t.device}, need cuda:{dev}")
    row, col = t.stride()
    if col != 1 and cols > 1:
        raise InlError(-1, f"{name}: rows must be contiguous")
    if rows <= 1:
        return cols
    if row < cols:   # expanded rows, too: the library reads a stride of 0 as packed
        raise InlError(-1, f"{name}: rows overlap (strides {(row, col)})")
    return row


def _matrix(name, t):
    shape = t.shape
    if len(shape) != 2:
        raise InlError(-1, f"{name}: shape {tuple(shape)}, need two dimensions")
    return shape


def _packed(name, t, rows, cols, dev):
    if _mat(name, t, rows, cols, _B16, dev) != cols:
        raise InlError(-1, f"{name}: must be packed")


def _vec(name, t, n, dtype, dev):
    if t is None:
        return None
    if t.dtype != dtype or t.shape != (n,) or t.get_device() != dev or (n > 1 and t.stride(0) != 1):
        raise InlError(-1, f"{name}: need contiguous {dtype} [{n}] on cuda:{dev}, got {t.dtype} {tuple(t.shape)} on "
                           f"{t.device}")
    return t.data_ptr()


def _act(act, gated=False):
    code = ACTS.get(act)
    if code is None or (gated and not code):
        raise InlError(-1, f"unknown act {act!r}")
    return code


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(op, dev, backward, *sizes):
    """By the sizes alone (``dev``: the plan behind them counts compute units)."""
    desc, size_fn, fields = {"dense": (DenseDesc, _dense_ws, ("m", "n", "k", "act")),
                             "gated_ffn": (GatedFfnDesc, _ffn_ws, ("m", "hidden", "inner", "act")),
                             "softmax_xent": (SoftmaxXentDesc, _xent_ws, ("m", "vocab", "hidden"))}[op]
    n = ctypes.c_size_t()
    _check(size_fn(desc(**dict(zip(fields, sizes))), backward, ctypes.byref(n)))
    return n.value


def _room(n, dev):
    return torch.empty(n, dtype=torch.uint8, device=dev) if n else None


def _stream(dev):
    return torch._C._cuda_getCurrentRawStream(dev)


def _ptr(t):
    return None if t is None else t.data_ptr()


# ---------------------------------------------------------------------------
# Linear layer
# ---------------------------------------------------------------------------

@_at_home
def _dense(dev, x, w, bias, act, residual, pre, out, out_dtype):
    m, k = _matrix("x", x)
    n = _matrix("w", w)[0]
    code = _act(act)
    xs, ws = _mat("x", x, m, k, _B16, dev), _mat("w", w, n, k, _B16, dev)
    if out is None:
        out = x.new_empty((m, n), dtype=out_dtype)
    ys = _mat("out", out, m, n, _ANY, dev)
    rs = rd = ps = 0
    if residual is not None:
        rs, rd = _mat("residual", residual, m, n, _ANY, dev), _CODE[residual.dtype]
    if pre is not None:
        ps = _mat("pre", pre, m, n, _B16, dev)
    bp = _vec("bias", bias, n, _F32, dev)
    d = DenseDesc(m, n, k, xs, ws, ys, rs, ps, 0, 0, code, _CODE[out.dtype], rd, 0, 0)
    size = _workspace_bytes("dense", dev, 0, m, n, k, code)
    room = _room(size, dev)
    _check(_dense_fwd(d, x.data_ptr(), w.data_ptr(), bp, _ptr(residual), out.data_ptr(), _ptr(pre), _ptr(room), size,
                      _stream(dev)))
    return out


def dense(x, w, bias=None, *, act=None, residual=None, pre=None, out=None, out_dtype=None, stream=None):
    """``act(x @ w.T + bias) + residual`` (``inl_dense_fwd``): bf16 ``x [m, k]``
    and ``w [n, k]``, f32 ``bias [n]``, ``act`` one of None, "relu", "silu",
    "gelu_tanh", "gelu_erf", ``residual [m, n]`` bf16 or f32 (it may be
    ``out``; ``x`` may not). ``pre``: a bf16 ``[m, n]`` tensor that receives ``x @ w.T + bias`` for
    ``dense_bwd``. n and k are multiples of 8; rows may be strided."""
    return _dense(x, w, bias, act, residual, pre, out, out_dtype, stream)


@_at_home
def _dense_grads(dev, x, dy, w, act, pre, bias_grad, dx_grad, dw_grad, dx_dtype, dw_dtype):
    m, k = _matrix("x", x)
    n = _matrix("w", w)[0]
    code = _act(act)
    if not code:
        pre = None
    elif pre is None:
        raise InlError(-1, "dense_bwd: an activation needs pre")
    xs, ws, ys = _mat("x", x, m, k, _B16, dev), _mat("w", w, n, k, _B16, dev), _mat("dy", dy, m, n, _B16, dev)
    ps = _mat("pre", pre, m, n, _B16, dev) if pre is not None else 0
    dx = x.new_empty((m, k), dtype=dx_dtype) if dx_grad else None
    dw = x.new_empty((n, k), dtype=dw_dtype) if dw_grad else None
    db = x.new_empty(n, dtype=_F32) if bias_grad else None
    d = DenseDesc(m, n, k, xs, ws, ys, 0, ps, 0, 0, code, 0, 0, _dtype_code(dx_dtype or _BF16),
                  _dtype_code(dw_dtype or _BF16))
    size = _workspace_bytes("dense", dev, 1, m, n, k, code)
    room = _room(size, dev)
    _check(_dense_bwd(d, dy.data_ptr(), x.data_ptr(), w.data_ptr(), _ptr(pre), _ptr(dx), _ptr(dw), _ptr(db),
                      _ptr(room), size, _stream(dev)))
    return dx, dw, db


def dense_bwd(dy, x, w, *, act=None, pre=None, bias_grad=False, dx_grad=True, dw_grad=True, dx_dtype=None,
              dw_dtype=None, stream=None):
    """``(dx, dw, dbias)`` of ``dense`` from bf16 ``dy [m, n]`` (``inl_dense_bwd``);
    ``pre`` is what the forward stored (not needed without an activation). dx and dw are
    bf16 unless ``dx_dtype``/``dw_dtype`` say float32, dbias f32; what is not asked
    for is None. The residual's gradient is ``dy``."""
    return _dense_grads(x, dy, w, act, pre, bias_grad, dx_grad, dw_grad, dx_dtype, dw_dtype, stream)


# ---------------------------------------------------------------------------
# Gated feed-forward block
# ---------------------------------------------------------------------------

@_at_home
def _ffn(dev, x, w_gate_up, w_down, act, residual, save, out, out_dtype):
    m, hidden = _matrix("x", x)
    inner = _matrix("w_down", w_down)[1]
    code = _act(act, True)
    xs = _mat("x", x, m, hidden, _B16, dev)
    _packed("w_gate_up", w_gate_up, 2 * inner, hidden, dev)
    _packed("w_down", w_down, hidden, inner, dev)
    if out is None:
        out = x.new_empty((m, hidden), dtype=out_dtype)
    ys = _mat("out", out, m, hidden, _ANY, dev)
    rs = rd = 0
    if residual is not None:
        rs, rd = _mat("residual", residual, m, hidden, _ANY, dev), _CODE[residual.dtype]
    pre = x.new_empty((m, 2 * inner)) if save else None
    h = x.new_empty((m, inner)) if save else None
    d = GatedFfnDesc(m, hidden, inner, xs, ys, rs, 0, code, _CODE[out.dtype], rd, 0, 0)
    size = _workspace_bytes("gated_ffn", dev, 0, m, hidden, inner, code)
    room = _room(size, dev)
    _check(_ffn_fwd(d, x.data_ptr(), w_gate_up.data_ptr(), w_down.data_ptr(), _ptr(residual), out.data_ptr(),
                    _ptr(pre), _ptr(h), _ptr(room), size, _stream(dev)))
    return (out, pre, h) if save else out


def gated_ffn(x, w_gate_up, w_down, *, act="silu", residual=None, save=False, out=None, out_dtype=None, stream=None):
    """``(act(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T + residual``
    (``inl_gated_ffn_fwd``): bf16 ``x [m, hidden]``, ``w_gate_up [2 inner, hidden]``
    (gate rows, then up rows) and ``w_down [hidden, inner]``, both packed; ``act``
    "silu", "gelu_tanh", "gelu_erf" or "relu". ``save=True`` returns ``(out, pre,
    h)`` with what ``gated_ffn_bwd`` reads: the gate and up products ``[m, 2
    inner]`` and ``h [m, inner]``, bf16."""
    return _ffn(x, w_gate_up, w_down, act, residual, save, out, out_dtype, stream)


@_at_home
def _ffn_grads(dev, x, dy, w_gate_up, w_down, pre, h, act, dx_grad, dw_grad, dx_dtype, dw_dtype):
    m, hidden = _matrix("x", x)
    inner = _matrix("w_down", w_down)[1]
    code = _act(act, True)
    xs, ys = _mat("x", x, m, hidden, _B16, dev), _mat("dy", dy, m, hidden, _B16, dev)
    for name, t, rows, cols in (("w_gate_up", w_gate_up, 2 * inner, hidden), ("w_down", w_down, hidden, inner),
                                ("pre", pre, m, 2 * inner), ("h", h, m, inner)):
        _packed(name, t, rows, cols, dev)
    wd = dw_dtype or _BF16
    dx = x.new_empty((m, hidden), dtype=dx_dtype) if dx_grad else None
    dgu = x.new_empty((2 * inner, hidden), dtype=wd) if dw_grad else None
    ddown = x.new_empty((hidden, inner), dtype=wd) if dw_grad else None
    d = GatedFfnDesc(m, hidden, inner, xs, ys, 0, 0, code, 0, 0, _dtype_code(dx_dtype or _BF16), _dtype_code(wd))
    size = _workspace_bytes("gated_ffn", dev, 1, m, hidden, inner, code)
    room = _room(size, dev)
    _check(_ffn_bwd(d, dy.data_ptr(), x.data_ptr(), w_gate_up.data_ptr(), w_down.data_ptr(), pre.data_ptr(),
                    h.data_ptr(), _ptr(dx), _ptr(dgu), _ptr(ddown), _ptr(room), size, _stream(dev)))
    return dx, dgu, ddown


def gated_ffn_bwd(dy, x, w_gate_up, w_down, pre, h, *, act="silu", dx_grad=True, dw_grad=True, dx_dtype=None,
                  dw_dtype=None, stream=None):
    """``(dx, dw_gate_up, dw_down)`` of ``gated_ffn`` from bf16 ``dy [m, hidden]`` and
    the ``pre`` and ``h`` that the forward saved (``inl_gated_ffn_bwd``); bf16 unless
    ``dx_dtype``/``dw_dtype`` say float32."""
    return _ffn_grads(x, dy, w_gate_up, w_down, pre, h, act, dx_grad, dw_grad, dx_dtype, dw_dtype, stream)


# ---------------------------------------------------------------------------
# Softmax cross entropy
# ---------------------------------------------------------------------------

def _xent_desc(dev, x, w, scale, ignore_index, dx_dtype=None, dw_dtype=None):
    m, hidden = _matrix("x", x)
    vocab = _matrix("w", w)[0]
    if not -2 ** 31 <= ignore_index < 2 ** 31:
        raise InlError(-1, f"ignore_index {ignore_index} is no int32")
    return SoftmaxXentDesc(m, vocab, hidden, _mat("x", x, m, hidden, _B16, dev), _mat("w", w, vocab, hidden, _B16, dev),
                           0, 0, scale, ignore_index, _dtype_code(dx_dtype or _BF16), _dtype_code(dw_dtype or _BF16))


def _xent_room(d, dev, backward):
    size = _workspace_bytes("softmax_xent", dev, backward, d.m, d.vocab, d.hidden)
    return _room(size, dev), size


@_at_home
def _xent(dev, x, w, targets, bias, scale, ignore_index):
    d = _xent_desc(dev, x, w, scale, ignore_index)
    loss, lse = x.new_empty(d.m, dtype=_F32), x.new_empty(d.m, dtype=_F32)
    room, size = _xent_room(d, dev, 0)
    _check(_xent_fwd(d, x.data_ptr(), w.data_ptr(), _vec("bias", bias, d.vocab, _F32, dev),
                     _vec("targets", targets, d.m, torch.int32, dev), loss.data_ptr(), lse.data_ptr(), _ptr(room), size,
                     _stream(dev)))
    return loss, lse


def softmax_xent(x, w, targets, *, bias=None, scale=1.0, ignore_index=-100, stream=None):
    """``(loss, lse)``, f32 ``[m]``, of the scores ``scale * x @ w.T + bias``, which are
    not stored (``inl_softmax_xent_fwd``): bf16 ``x [m, hidden]`` and ``w [vocab,
    hidden]`` (a decoder, or the documents of a batch with ``scale`` = 1 /
    temperature), f32 ``bias [vocab]``, int32 ``targets [m]``. Rows whose target is
    ``ignore_index`` have loss 0; a target outside the vocabulary gives NaN."""
    return _xent(x, w, targets, bias, scale, ignore_index, stream)


@_at_home
def _xent_grads(dev, x, dloss, lse, w, targets, bias, scale, ignore_index, dx_grad, dw_grad, bias_grad, dx_dtype,
                dw_dtype):
    d = _xent_desc(dev, x, w, scale, ignore_index, dx_dtype, dw_dtype)
    dx = x.new_empty(x.shape, dtype=dx_dtype) if dx_grad else None
    dw = x.new_empty(w.shape, dtype=dw_dtype) if dw_grad else None
    db = x.new_empty(d.vocab, dtype=_F32) if bias_grad else None
    room, size = _xent_room(d, dev, 1)
    _check(_xent_bwd(d, _vec("dloss", dloss, d.m, _F32, dev), _vec("lse", lse, d.m, _F32, dev), x.data_ptr(),
                     w.data_ptr(), _vec("bias", bias, d.vocab, _F32, dev),
                     _vec("targets", targets, d.m, torch.int32, dev), _ptr(dx), _ptr(dw), _ptr(db), _ptr(room), size,
                     _stream(dev)))
    return dx, dw, db


def softmax_xent_bwd(dloss, lse, x, w, targets, *, bias=None, scale=1.0, ignore_index=-100, dx_grad=True,
                     dw_grad=True, bias_grad=False, dx_dtype=None, dw_dtype=None, stream=None):
    """``(dx, dw, dbias)`` of ``softmax_xent`` from f32 ``dloss [m]`` and the forward's
    ``lse`` (``inl_softmax_xent_bwd``); dx and dw bf16 unless ``dx_dtype``/``dw_dtype``
    say float32, dbias f32; what is not asked for is None."""
    return _xent_grads(x, dloss, lse, w, targets, bias, scale, ignore_index, dx_grad, dw_grad, bias_grad, dx_dtype,
                       dw_dtype, stream)


# ---------------------------------------------------------------------------
# q/k prologue
# ---------------------------------------------------------------------------

@_at_home
def _rope_grads(dev, x, dy, q_heads, rows, cos, sin, q_weight, k_weight, eps, norm, rotary_dim, sections, cos2, sin2,
                round_tables, out, weight_grad):
    shape = x.shape
    if len(shape) != 3:
        raise InlError(-1, f"x: shape {tuple(shape)}, need [tokens, heads, head_dim]")
    n, heads, hd = shape
    d = NormRopeDesc()
    d.n_tokens, d.heads, d.head_dim = shape
    d.x_row_stride, d.y_row_stride = _head_rows("x", x, shape, dev), _head_rows("dy", dy, shape, dev)
    d.dtype, d.out_dtype = _dtype_code(x.dtype), _dtype_code(dy.dtype)
    d.norm, d.eps = int(bool(norm)), eps
    d.rotary_dim = int((hd if cos is not None else 0) if rotary_dim is None else rotary_dim)
    d.sections, d.round_tables = int(sections), int(bool(round_tables))
    if d.rotary_dim > 0:
        d.table_rows = _rope_tables(n, rows, d.rotary_dim, hd, d.sections, cos, sin, cos2, sin2, dev)
    if out is None:
        out = torch.empty(shape, dtype=x.dtype, device=dev)
    elif out.dtype != x.dtype:
        raise InlError(-1, f"out: dtype {out.dtype}, need {x.dtype}")
    ds = _head_rows("out", out, shape, dev)
    grads = bool(norm and weight_grad)
    dq = torch.empty(hd, dtype=_F32, device=dev) if grads else None
    dk = torch.empty(hd, dtype=_F32, device=dev) if grads and q_heads < heads else None
    size = ctypes.c_size_t()
    if grads:
        _check(_rope_bwd_ws(d, ctypes.byref(size)))
    room = _room(size.value, dev)
    wp = wp2 = None   # (as in the forward: not looked at without a norm)
    if norm:
        wp, wp2 = _head_weight("q_weight", q_weight, x.dtype, hd, dev), _head_weight("k_weight", k_weight, x.dtype, hd, dev)
    _check(_rope_bwd(d, int(q_heads), dy.data_ptr(), x.data_ptr(), out.data_ptr(), ds, wp, wp2, _ptr(rows), _ptr(cos),
                     _ptr(sin), _ptr(cos2), _ptr(sin2), _ptr(dq), _ptr(dk), _ptr(room), size.value, _stream(dev)))
    return out, dq, dk


def norm_rope_qk_bwd(dy, x, q_heads, rows=None, cos=None, sin=None, *, q_weight=None, k_weight=None, eps=1e-6,
                     norm=True, rotary_dim=None, sections=1, cos2=None, sin2=None, round_tables=False, round_norm=False,
                     out=None, weight_grad=True, stream=None):
    """``(dx, dq_weight, dk_weight)`` of ``norm_rope_qk`` from ``dy [N, heads,
    head_dim]`` and the forward's ``x`` (``inl_norm_rope_qk_bwd``); the other
    arguments as in the forward (``round_norm`` changes nothing, gradients pass the
    rounding unchanged; dy has the forward's output dtype). dx has x's dtype (``out`` may be a slice of wider rows), the
    weight gradients are f32 ``[head_dim]`` and None without a norm, with
    ``weight_grad=False`` or, dk_weight, where all heads are q heads."""
    del round_norm
    return _rope_grads(x, dy, q_heads, rows, cos, sin, q_weight, k_weight, eps, norm, rotary_dim, sections, cos2, sin2,
                       round_tables, out, weight_grad, stream)


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------

def _head_tensor(name, t, rows, heads, hd, dtype, dev):
    """The stride between the token rows of ``t [rows or more, heads, hd]``."""
    shape = t.shape
    if len(shape) == 3:   # (the usual form first: a short batch waits for these checks)
        row, head, one = t.stride()
        n, h, d = shape
        if n >= rows and n > 1 and h == heads and d == hd and t.dtype is dtype and one == 1 \
                and (head == hd or heads == 1) and row >= heads * hd and t.get_device() == dev:
            return row
    if len(shape) != 3 or shape[1:] != (heads, hd):
        raise InlError(-1, f"{name}: shape {tuple(shape)}, need [rows, {heads}, {hd}]")
    if t.dtype is not dtype:
        raise InlError(-1, f"{name}: dtype {t.dtype}, need {dtype}")
    if shape[0] < rows:
        raise InlError(-1, f"{name}: {shape[0]} rows, the texts cover {rows}")
    return _head_rows(name, t, shape, dev)


@_at_home
def _attn_grads(dev, q, dout, k, v, out, cu_seqlens, causal, window, scale, seq_starts, grad_dtype, grads, kv_grad):
    if len(q.shape) != 3 or len(k.shape) != 3:
        raise InlError(-1, f"q, k: shapes {tuple(q.shape)}, {tuple(k.shape)}, need [rows, heads, head_dim]")
    n, hq, hd = q.shape
    nk, hkv, _ = k.shape
    texts = len(cu_seqlens) - 1
    window = -1 if window is None else int(window)
    if not -1 <= window < 2 ** 31:   # (its low 32 bits would be another window)
        raise InlError(-1, f"window {window} must be -1 or in [0, 2^31)")
    if seq_starts is None:
        cu, starts = _cu_array(cu_seqlens), None
        rows = cu[texts] if texts > 0 else 0
    else:
        d = make_attn_desc(cu_seqlens, hq, hkv, hd, causal=causal, seq_starts=seq_starts)   # checks the lengths
        cu, starts, rows = d._cu_keepalive, d._starts_keepalive, desc_rows(d)
    d = AttnDesc(texts, cu, hq, hkv, hd, bool(causal), window,
                 hd ** -0.5 if scale is None else scale, INL_BF16, INL_BF16,
                 _head_tensor("q", q, rows, hq, hd, _BF16, dev), _head_tensor("k", k, rows, hkv, hd, _BF16, dev),
                 _head_tensor("v", v, rows, hkv, hd, _BF16, dev), _head_tensor("out", out, rows, hq, hd, _BF16, dev), 0,
                 starts)
    dos = _head_tensor("dout", dout, rows, hq, hd, _BF16, dev)
    if grads is None:
        # rows of no text have no gradient: they are zero in tensors made here
        made = torch.zeros if starts is not None or n != rows or nk != rows else torch.empty
        dt = grad_dtype or _BF16
        dq = made((n, hq, hd), dtype=dt, device=q.device)
        dk = dv = None
        if kv_grad:
            dk, dv = made((nk, hkv, hd), dtype=dt, device=q.device), made((nk, hkv, hd), dtype=dt, device=q.device)
        g = AttnGrads(dos, 0, 0, 0, _dtype_code(dt))
    else:
        dq, dk, dv = grads if kv_grad else (grads[0], None, None)
        dt = next((t.dtype for t in (dq, dk, dv) if t is not None), _BF16)
        if grad_dtype is not None and grad_dtype is not dt:
            raise InlError(-1, f"grads: dtype {dt}, grad_dtype {grad_dtype}")
        strides = [0 if t is None else _head_tensor(name, t, rows, heads, hd, dt, dev)
                   for name, t, heads in (("dq", dq, hq), ("dk", dk, hkv), ("dv", dv, hkv))]
        g = AttnGrads(dos, *strides, _dtype_code(dt))
    # inl_attn_bwd_workspace_size, or as much as a table of all the texts more
    size = (8 * hq * max(rows, 0) + 255 & ~255) + (12 * texts if texts > 256 else 0)
    room = _room(size, dev)
    _check(_attn_bwd(d, g, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr(), _ptr(dq),
                     _ptr(dk), _ptr(dv), _ptr(room), size, _stream(dev)))
    return dq, dk, dv


def varlen_attention_bwd(dout, q, k, v, out, cu_seqlens, *, causal, window=-1, scale=None, seq_starts=None,
                         grad_dtype=None, grads=None, kv_grad=True, stream=None):
    """``(dq, dk, dv)`` of ``varlen_attention`` from bf16 ``dout [N, Hq, D]`` and the
    forward's bf16 ``out`` (``inl_attn_varlen_bwd``); the other arguments as in the
    forward. The probabilities are recomputed. dq, dk and dv are bf16 unless
    ``grad_dtype`` says float32 (P and dS are rounded to bf16 in between all the same);
    ``kv_grad=False`` leaves dk and dv out (None), those of ``grads`` as they were.
    ``grads=(dq, dk, dv)`` are tensors to write, slices of one ``[N, Hq + 2 Hkv, D]`` row
    among them, None where not wanted; their rows outside every text are left as they
    were, and zero in tensors made here."""
    return _attn_grads(q, dout, k, v, out, cu_seqlens, causal, window, scale, seq_starts, grad_dtype, grads, kv_grad,
                       stream)


def attention_bwd_kernel_names(desc):
    """The kernels that ``varlen_attention_bwd`` launches for ``desc`` (``make_attn_desc``): the one that
    makes dq, and the one that makes dk and dv (``inl_attn_bwd_kernel_name``)."""
    names = []
    for kv in (0, 1):
        name = ctypes.c_char_p()
        _check(_attn_bwd_name(desc, kv, ctypes.byref(name)))
        names.append(name.value.decode())
    return tuple(names)


# ---------------------------------------------------------------------------
# The residual stream: addition, dropout, norm
# ---------------------------------------------------------------------------

def _drop(dropout, rng, dev, draws=True):
    """The dropped share in 1 / 65536 and the address of the generator's state."""
    if not 0.0 <= dropout < 1.0 or round(dropout * 65536) > 65535:
        raise InlError(-1, f"dropout {dropout} must be in [0, 1)")
    drop = round(dropout * 65536)
    if not drop or not draws:
        return drop, None
    if rng is None or rng.dtype is not torch.int64 or rng.shape != (2,) or rng.get_device() != dev \
            or rng.stride(0) != 1:
        raise InlError(-1, f"rng: dropout needs contiguous torch.int64 [2] on cuda:{dev}"
                           + ("" if rng is None else f", got {rng.dtype} {tuple(rng.shape)} on {rng.device}"))
    return drop, rng.data_ptr()


def _tag(tag):
    if not -2 ** 31 <= tag < 2 ** 32:
        raise InlError(-1, f"tag {tag} is no 32-bit number")
    return tag - 2 ** 32 if tag >= 2 ** 31 else tag


def _norm_weight(weight, n, dev):
    if weight is None:
        return INL_F32, None
    if weight.dtype not in _ANY:
        raise InlError(-1, f"weight: dtype {weight.dtype}, need torch.bfloat16 or torch.float32")
    return _CODE[weight.dtype], _vec("weight", weight, n, weight.dtype, dev)


@_at_home
def _norm_fwd(dev, x, weight, residual, eps, dropout, rng, tag, out, sum_out, out_dtype, sum_dtype):
    m, n = _matrix("x", x)
    drop, rp = _drop(dropout, rng, dev)
    xs = _mat("x", x, m, n, _ANY, dev)
    rs = 0
    if residual is not None:
        rs = _mat("residual", residual, m, n, _ANY, dev)
        sum_dtype = sum_dtype or residual.dtype
        if sum_dtype is not residual.dtype:
            raise InlError(-1, f"sum_dtype {sum_dtype}: the residual is {residual.dtype}")
    wd, wp = _norm_weight(weight, n, dev)
    if out is None:
        out = x.new_empty((m, n), dtype=out_dtype)
    ys = _mat("out", out, m, n, _ANY, dev)
    h, plain = sum_out, residual is None and not drop   # the sum of nothing is x itself
    if h is None:
        sd = sum_dtype or x.dtype
        # (and y may not take its place)
        kept = plain and sd is x.dtype and out.untyped_storage().data_ptr() != x.untyped_storage().data_ptr()
        h = x if kept else x.new_empty((m, n), dtype=sd)
    else:
        kept = False
        if sum_dtype is not None and sum_dtype is not h.dtype:
            raise InlError(-1, f"sum_out: dtype {h.dtype}, need {sum_dtype}")
    hs = _mat("sum_out", h, m, n, _ANY, dev)
    d = AddNormDesc(m, n, xs, rs, hs, ys, 0, eps, drop, _tag(tag), _CODE[x.dtype], _CODE[h.dtype], _CODE[out.dtype], wd)
    _check(_add_norm(d, x.data_ptr(), _ptr(residual), wp, rp, None if kept else h.data_ptr(), out.data_ptr(),
                     _stream(dev)))
    return out, h


def add_rms_norm(x, weight=None, *, residual=None, eps=1e-6, dropout=0.0, rng=None, tag=0, out=None, sum_out=None,
                 out_dtype=None, sum_dtype=None, stream=None):
    """``(y, h)`` with ``h = residual + drop(x)`` and ``y = h / sqrt(mean(h^2) + eps) * weight``
    (``inl_add_rms_norm_fwd``): bf16 or f32 ``x [m, n]`` and ``weight [n]``, ``residual [m, n]`` or
    None; n a multiple of 8, at most 16384; rows may be strided. h has the residual's dtype (without
    one ``sum_dtype``, x's by default; without dropout too it is x itself, where ``out`` is not) and may
    go into ``sum_out``, which may be x or the residual itself; y has x's dtype unless ``out_dtype`` says
    otherwise. ``dropout``: the probability (in steps of 1 / 65536); its draws come from ``rng``, int64
    ``[2]`` on the device (seed, step), and ``tag``, a number of this place in the model; no mask is
    kept."""
    return _norm_fwd(x, weight, residual, eps, dropout, rng, tag, out, sum_out, out_dtype, sum_dtype, stream)


@_at_home
def _norm_grads(dev, h, dy, weight, dh, eps, dropout, rng, tag, x_grad, residual_grad, weight_grad, dx_dtype):
    m, n = _matrix("h", h)
    drop, rp = _drop(dropout, rng, dev, x_grad)
    hs, ys = _mat("h", h, m, n, _ANY, dev), _mat("dy", dy, m, n, _ANY, dev)
    ds = 0
    if dh is not None:
        ds = _mat("dh", dh, m, n, (h.dtype,), dev)
    wd, wp = _norm_weight(weight, n, dev)
    if dx_dtype is None:
        dx_dtype = dy.dtype
    # without dropout x's gradient is the residual's, in its own dtype
    same = x_grad and not drop and dx_dtype is h.dtype
    dres = h.new_empty((m, n)) if residual_grad or same else None
    dx = h.new_empty((m, n), dtype=dx_dtype) if x_grad and not same else None
    dw = h.new_empty(n, dtype=_F32) if weight_grad and weight is not None else None
    d = AddNormDesc(m, n, 0, 0, hs, ys, ds, eps, drop, _tag(tag), _dtype_code(dx_dtype), _CODE[h.dtype],
                    _CODE[dy.dtype], wd)
    size = ctypes.c_size_t()
    if dw is not None:
        _check(_add_norm_ws(d, ctypes.byref(size)))
    room = _room(size.value, dev)
    _check(_add_norm_bwd(d, dy.data_ptr(), h.data_ptr(), _ptr(dh), wp, rp, _ptr(dx), _ptr(dres), _ptr(dw), _ptr(room),
                         size.value, _stream(dev)))
    return dres if same else dx, dres if residual_grad else None, dw


def add_rms_norm_bwd(dy, h, weight=None, *, dh=None, eps=1e-6, dropout=0.0, rng=None, tag=0, x_grad=True,
                     residual_grad=True, weight_grad=True, dx_dtype=None, stream=None):
    """``(dx, dresidual, dweight)`` of ``add_rms_norm`` from ``dy [m, n]`` (y's dtype) and the ``h`` that
    it returned (``inl_add_rms_norm_bwd``); ``dh`` (h's dtype) is the gradient that reaches h past the
    norm. ``dropout``, ``rng`` and ``tag`` as in the forward, with the step it had. dresidual has h's
    dtype, dx dy's unless ``dx_dtype`` says otherwise (without dropout, and of one dtype, they are one
    tensor), dweight f32 ``[n]`` (None without a weight); what is not asked for is None."""
    return _norm_grads(h, dy, weight, dh, eps, dropout, rng, tag, x_grad, residual_grad, weight_grad, dx_dtype, stream)


# ---------------------------------------------------------------------------
# Pooled embedding
# ---------------------------------------------------------------------------

def _pooled(name, t, texts, dim, dev):
    if t.shape != (texts, dim) or t.dtype is not _F32 or t.get_device() != dev or not t.is_contiguous():
        raise InlError(-1, f"{name}: need contiguous torch.float32 {(texts, dim)} on cuda:{dev}, got {t.dtype} "
                           f"{tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _offsets(cu, dev):
    if len(cu.shape) != 1 or cu.shape[0] < 1 or cu.dtype is not torch.int32 or cu.get_device() != dev \
            or not cu.is_contiguous():
        raise InlError(-1, f"cu: need contiguous torch.int32 [texts + 1] on cuda:{dev}, got {cu.dtype} "
                           f"{tuple(cu.shape)} on {cu.device}")
    return cu.shape[0] - 1


def _grad_rows(out, shape, dtype, like, dev):
    if out is None:
        out = like.new_empty(shape, dtype=dtype)
    elif dtype is not None and out.dtype is not dtype:
        raise InlError(-1, f"out: dtype {out.dtype}, need {dtype}")
    return out, _mat("out", out, *shape, _ANY, dev)


@_at_home
def _mean_grads(dev, dpooled, cu, rows, mean, dtype, out):
    texts, dim = _matrix("dpooled", dpooled)
    if _offsets(cu, dev) != texts:
        raise InlError(-1, f"cu: {cu.shape[0] - 1} texts, dpooled has {texts}")
    dp = _pooled("dpooled", dpooled, texts, dim, dev)
    mp = None if mean is None else _pooled("mean", mean, texts, dim, dev)
    out, stride = _grad_rows(out, (int(rows), dim), dtype if out is not None else dtype or _BF16, dpooled, dev)
    _check(_pool_mean_bwd(texts, cu.data_ptr(), dim, int(rows), stride, _CODE[out.dtype], dp, mp, out.data_ptr(),
                          _stream(dev)))
    return out


def pool_mean_bwd(dpooled, cu, rows, *, mean=None, dtype=None, out=None, stream=None):
    """The gradient ``[rows, dim]`` of ``pool_mean``'s hidden rows from f32 ``dpooled [texts, dim]``
    (``inl_pool_mean_bwd``): bf16 unless ``dtype`` says float32, 0 in rows of no text. ``mean``: with
    ``normalize=True`` in the forward, what it gives with ``normalize=False``, f32 ``[texts, dim]``."""
    return _mean_grads(dpooled, cu, rows, mean, dtype, out, stream)


@_at_home
def _last_grads(dev, dpooled, hidden, cu, weight, eps, dtype, out, weight_grad):
    rows, dim = _matrix("hidden", hidden)
    texts = _offsets(cu, dev)
    dp = _pooled("dpooled", dpooled, texts, dim, dev)
    hs = _mat("hidden", hidden, rows, dim, _ANY, dev)
    wp = _vec("weight", weight, dim, hidden.dtype, dev)
    out, stride = _grad_rows(out, (rows, dim), dtype if out is not None else dtype or hidden.dtype, hidden, dev)
    dw = hidden.new_empty(dim, dtype=_F32) if weight_grad and weight is not None else None
    size = 4 * texts * dim if dw is not None and texts > 1 else 0
    room = _room(size, dev)
    _check(_pool_last_bwd(texts, cu.data_ptr(), dim, rows, hs, _CODE[hidden.dtype], dp, hidden.data_ptr(), wp, eps,
                          stride, _CODE[out.dtype], out.data_ptr(), _ptr(dw), _ptr(room), size, _stream(dev)))
    return out, dw


def pool_last_bwd(dpooled, hidden, cu, weight=None, *, eps=1e-6, round_norm=False, dtype=None, out=None,
                  weight_grad=True, stream=None):
    """``(dhidden, dweight)`` of ``pool_last`` from f32 ``dpooled [texts, dim]`` and the forward's
    arguments (``inl_pool_last_bwd``; ``round_norm`` changes nothing, gradients pass the rounding
    unchanged). dhidden has hidden's dtype unless ``dtype`` says otherwise and is 0 but in the
    texts' last rows; dweight is f32 ``[dim]``, None without a weight."""
    del round_norm
    return _last_grads(dpooled, hidden, cu, weight, eps, dtype, out, weight_grad, stream)
