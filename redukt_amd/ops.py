"""Operators of libredukt_gpu.so on the caller's own device tensors (include/redukt_ops.h).

The gated delta rule for one token (`delta_step`) and for whole sequences (`delta_chunk`), int8
codes of activation rows (`quantize_rows`) and the product of codes with a scale per token and
channel (`int8_matmul`).  Arguments are torch tensors on one GPU; work is queued on torch's
current stream of that GPU, or on `stream`, a hipStream_t's value.  Outputs and workspaces that a
call allocates belong to torch's current stream, so for another one they are passed in, and the
caller keeps all tensors until that stream is done with them.  Outputs overlap no input (but a state
pool its own next states).  No model needs to be open.  The operators have no gradients: tensors
that ask for one, states and outputs among them, are refused while torch records them, and tensors
with a tangent always.  Wrong arguments raise `ffi.BackendError` (INVALID_ARGUMENT) and launch
nothing; there is no CPU fallback.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import ffi

NORMALIZE = 1      # REDUKT_DELTA_NORMALIZE
DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class DeltaRows(ctypes.Structure):
    """redukt_delta_rows."""
    _fields_ = [("dtype", ctypes.c_uint32), ("rows", ctypes.c_uint32), ("hk", ctypes.c_uint32), ("hv", ctypes.c_uint32),
                ("dk", ctypes.c_uint32), ("dv", ctypes.c_uint32), ("flags", ctypes.c_uint32), ("scale", ctypes.c_float),
                ("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("out", ctypes.c_void_p),
                ("q_stride", ctypes.c_int64), ("k_stride", ctypes.c_int64), ("v_stride", ctypes.c_int64),
                ("out_stride", ctypes.c_int64), ("g", ctypes.c_void_p), ("beta", ctypes.c_void_p),
                ("g_stride", ctypes.c_int64), ("beta_stride", ctypes.c_int64)]


class QuantizeRows(ctypes.Structure):
    """redukt_quantize_rows."""
    _fields_ = [("dtype", ctypes.c_uint32), ("rows", ctypes.c_uint32), ("cols", ctypes.c_uint32), ("x", ctypes.c_void_p),
                ("x_stride", ctypes.c_int64), ("codes", ctypes.c_void_p), ("codes_stride", ctypes.c_int64),
                ("scales", ctypes.c_void_p)]


class Int8Matmul(ctypes.Structure):
    """redukt_int8_matmul."""
    _fields_ = [("dtype", ctypes.c_uint32), ("m", ctypes.c_uint32), ("n", ctypes.c_uint32), ("k", ctypes.c_uint32),
                ("x", ctypes.c_void_p), ("x_stride", ctypes.c_int64), ("x_scales", ctypes.c_void_p),
                ("w", ctypes.c_void_p), ("w_stride", ctypes.c_int64), ("w_scales", ctypes.c_void_p),
                ("bias", ctypes.c_void_p), ("out", ctypes.c_void_p), ("out_stride", ctypes.c_int64)]


_lib = None


def _load() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        L = ffi.PluginLibrary().lib
        p, u32, u64 = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_uint64
        L.redukt_op_delta_step.argtypes = [ctypes.POINTER(DeltaRows), p, u32, p, p]
        L.redukt_op_delta_chunk.argtypes = [ctypes.POINTER(DeltaRows), p, u32, p, p, u32, p, p, u64, p]
        L.redukt_op_delta_chunk_workspace.argtypes = [ctypes.POINTER(DeltaRows), u32]
        L.redukt_op_delta_chunk_workspace.restype = u64
        L.redukt_op_quantize_rows.argtypes = [ctypes.POINTER(QuantizeRows), p]
        L.redukt_op_int8_matmul.argtypes = [ctypes.POINTER(Int8Matmul), p]
        for f in ("delta_step", "delta_chunk", "quantize_rows", "int8_matmul"):
            getattr(L, "redukt_op_" + f).restype = ctypes.c_int32
        _lib = L
    return _lib


def _refuse(what: str) -> None:
    raise ffi.BackendError(ffi.BackendResult.INVALID_ARGUMENT, what)


def _done(code: int, what: str) -> None:
    if code:
        raise ffi.BackendError(ffi.BackendResult.from_code(code), what)


def _sizes(op: str, *sizes: int) -> None:
    """The library's fields for sizes have 32 bits, and ctypes would drop what is above."""
    bits = 0
    for s in sizes:
        bits |= s
    if bits >> 31:
        _refuse(f"{op}: sizes {sizes} are not within 0 and 2^31 - 1")


def _check(op: str, device: int, name: str, t, dtype, shape) -> None:
    """t is a tensor on GPU `device` of this type and shape (None: any size)."""
    if not isinstance(t, torch.Tensor):
        _refuse(f"{op}: {name} is not a tensor")
    if t.get_device() != device:
        _refuse(f"{op}: {name} is on {t.device}, not on GPU {device}")
    if t.dtype is not dtype:
        _refuse(f"{op}: {name} is {t.dtype}, not {dtype}")
    got = t.shape
    if got != shape and (len(got) != len(shape) or any(w is not None and w != s for w, s in zip(shape, got))):
        _refuse(f"{op}: {name} has shape {tuple(t.shape)}, not {tuple('*' if w is None else w for w in shape)}")


def _device(op: str, t) -> int:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _refuse(f"{op}: tensors on a GPU are needed")
    return t.get_device()


def _stream(op: str, stream: Optional[int], device: int, allocates: bool) -> int:
    current = torch._C._cuda_getCurrentRawStream(device)
    if stream is None or stream == current:
        return current
    if allocates:
        _refuse(f"{op}: on a stream that is not torch's current one, outputs and workspace are passed in")
    return stream


def _no_gradients(op: str, *tensors) -> None:
    """Refuses tensors (None: left out) that ask for a gradient while torch records them, or have a tangent.  Called where one
    requires a gradient or somebody computes tangents (_tangents)."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        _refuse(f"{op}: a tensor asks for a gradient, which this operator has not (detach it, or use torch.no_grad())")
    if _tangents() and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        _refuse(f"{op}: a tensor has a tangent, which this operator would drop")


def _tangents() -> bool:
    return forward_ad._current_level >= 0


def _row_stride(op: str, name: str, t, width: int) -> int:
    """Elements from a row of t [rows, ...] to the next, whose rows are contiguous and of `width` elements."""
    if t.is_contiguous():
        return width
    shape, strides = t.shape, t.stride()
    want = 1
    for i in range(len(shape) - 1, 0, -1):
        if shape[i] != 1 and strides[i] != want:
            _refuse(f"{op}: the rows of {name} are not contiguous")
        want *= shape[i]
    return strides[0] if shape[0] > 1 else want


def _rows(op: str, q, k, v, g, beta, out, scale, normalize) -> Tuple[DeltaRows, torch.Tensor, int]:
    device = _device(op, q)
    if q.dtype not in DTYPES or q.dim() != 3:
        _refuse(f"{op}: q [rows, key heads, dk] is bfloat16, float16 or float32")
    dtype, shape = q.dtype, q.shape
    T, hk, dk = shape
    try:       # (all at once; what is wrong is looked for only if something is)
        wide, gates = v.shape, g.shape
        fine = (k.shape == shape and wide[0] == T and gates == wide[:2] and beta.shape == gates and len(wide) == 3
                and k.dtype is dtype and v.dtype is dtype and g.dtype is torch.float32 and beta.dtype is torch.float32
                and k.get_device() == v.get_device() == g.get_device() == beta.get_device() == device)
    except (AttributeError, IndexError, TypeError):
        fine = False
    if not fine:
        _check(op, device, "k", k, dtype, shape)
        _check(op, device, "v", v, dtype, (T, None, None))
        _check(op, device, "g", g, torch.float32, tuple(v.shape[:2]))
        _check(op, device, "beta", beta, torch.float32, tuple(v.shape[:2]))
        _refuse(f"{op}: tensors do not belong together")
    if q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad or beta.requires_grad or _tangents():
        _no_gradients(op, q, k, v, g, beta)
    _, hv, dv = wide
    if (T | hk | dk | hv | dv) >> 31:
        _sizes(op, T, hk, dk, hv, dv)
    if out is None:
        out = torch.empty_like(v) if v.is_contiguous() else torch.empty(wide, dtype=dtype, device=q.device)
    else:
        _check(op, device, "out", out, dtype, wide)
        _no_gradients(op, out)
    wk, wv = hk * dk, hv * dv
    if scale is None:
        scale = dk ** -0.5 if dk else 0.0
    a = DeltaRows(DTYPES[dtype], T, hk, hv, dk, dv, NORMALIZE if normalize else 0, scale, q.data_ptr(), k.data_ptr(),
                  v.data_ptr(), out.data_ptr(), _row_stride(op, "q", q, wk), _row_stride(op, "k", k, wk),
                  _row_stride(op, "v", v, wv), _row_stride(op, "out", out, wv), g.data_ptr(), beta.data_ptr(),
                  _row_stride(op, "g", g, hv), _row_stride(op, "beta", beta, hv))
    return a, out, device


def _pool(op: str, device: int, name: str, t, a: DeltaRows) -> None:
    try:
        if (t.dtype is torch.float32 and t.shape[1:] == (a.hv, a.dk, a.dv) and t.is_contiguous() and t.get_device() == device):
            if t.requires_grad or _tangents():
                _no_gradients(op, t)
            return
    except AttributeError:
        pass
    _check(op, device, name, t, torch.float32, (None, a.hv, a.dk, a.dv))
    _refuse(f"{op}: {name} is not contiguous")


def _slots(op: str, device: int, slots, n: int) -> Optional[int]:
    if slots is None:
        return None
    _check(op, device, "slots", slots, torch.int32, (n,))
    if not slots.is_contiguous():
        _refuse(f"{op}: slots is not contiguous")
    return slots.data_ptr()


def delta_step(q, k, v, g, beta, states, slots=None, out=None, scale: Optional[float] = None, normalize: bool = False,
               stream: Optional[int] = None):
    """The gated delta rule for one token of each of n entries (at most 65,536); states are stepped in place.

    q, k [n, key heads, dk] and v [n, value heads, dv] in bfloat16, float16 or float32; g (log
    decay) and beta (write strength) [n, value heads] float32; states [slots, value heads, dk,
    dv] float32.  Entry i steps slot slots[i] (int32; None: slot i); -1 leaves entry i's output
    and state as they are; a slot out of range, or named by an earlier entry, gives NaN outputs
    and touches no state.  scale: of the outputs (None: dk ** -0.5).  normalize: k and q are
    divided by sqrt(sum of squares + 1e-6) first.  Returns out [n, value heads, dv] (allocated
    if None).  dk is 64 or 128, dv a multiple of 32 up to 256; rows may be strided (slices of
    one projection's output), by whole 16 bytes.
    """
    op = "delta_step"
    allocates = out is None
    a, out, device = _rows(op, q, k, v, g, beta, out, scale, normalize)
    on = _stream(op, stream, device, allocates)
    _pool(op, device, "states", states, a)
    code = _load().redukt_op_delta_step(ctypes.byref(a), states.data_ptr(), states.shape[0],
                                        _slots(op, device, slots, a.rows), on)
    _done(code, op)
    # (these were written unseen by torch, which counts writes for what autograd has saved)
    increment_version(states if allocates else (states, out))
    return out


def delta_chunk_workspace(tokens: int, sequences: int, hk: int, hv: int, dk: int, dv: int, dtype) -> int:
    """Bytes of workspace that `delta_chunk` needs for these sizes."""
    if dtype not in DTYPES:
        _refuse("delta_chunk_workspace: bfloat16, float16 or float32")
    _sizes("delta_chunk_workspace", tokens, sequences, hk, hv, dk, dv)
    return _load().redukt_op_delta_chunk_workspace(ctypes.byref(DeltaRows(DTYPES[dtype], tokens, hk, hv, dk, dv)), sequences)


def delta_chunk(q, k, v, g, beta, cu_seqlens, state_in=None, state_out=None, slots=None, out=None,
                scale: Optional[float] = None, normalize: bool = False, workspace=None, stream: Optional[int] = None):
    """The gated delta rule over packed sequences: rows cu_seqlens[i] to cu_seqlens[i + 1] of
    q, k, v, g and beta (as in `delta_step`) are sequence i, from the state in slot slots[i]
    (None: i) of state_in (None: zeros); its final state goes to that slot of state_out (None:
    not wanted; state_in itself: in place).  cu_seqlens int32, none decreasing, within the rows.
    A slot of -1 leaves the sequence out; slots out of range, or named before while state_out
    is given, give NaN rows.  Returns out [rows, value heads, dv]; rows of no sequence are not
    written.  At most 65,536 sequences.  States and float32 outputs are as exact as float32 sums,
    16-bit outputs are summed from factors of 16 bits.  workspace: a uint8 tensor of
    `delta_chunk_workspace` bytes that nothing else uses meanwhile (allocated if None).
    """
    op = "delta_chunk"
    allocates = out is None or workspace is None
    given = () if out is None and workspace is None else [t for t in (out, workspace) if t is not None]
    a, out, device = _rows(op, q, k, v, g, beta, out, scale, normalize)
    on = _stream(op, stream, device, allocates)
    _check(op, device, "cu_seqlens", cu_seqlens, torch.int32, (None,))
    n = cu_seqlens.shape[0] - 1
    if n < 0 or not cu_seqlens.is_contiguous():
        _refuse(f"{op}: cu_seqlens holds one value more than there are sequences")
    if n > 65536:
        _refuse(f"{op}: more than 65,536 sequences")
    n_slots = 0
    for name, pool in (("state_in", state_in), ("state_out", state_out)):
        if pool is not None:
            _pool(op, device, name, pool, a)
            n_slots = pool.shape[0]
    if state_in is not None and state_out is not None and state_in.shape[0] != state_out.shape[0]:
        _refuse(f"{op}: state_in and state_out differ in slots")
    L = _load()
    need = L.redukt_op_delta_chunk_workspace(ctypes.byref(a), n)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    else:
        _check(op, device, "workspace", workspace, torch.uint8, (None,))
        if not workspace.is_contiguous():      # (its bytes are counted by its elements)
            _refuse(f"{op}: workspace is not contiguous")
    code = L.redukt_op_delta_chunk(ctypes.byref(a), cu_seqlens.data_ptr(), n,
                                   None if state_in is None else state_in.data_ptr(),
                                   None if state_out is None else state_out.data_ptr(), n_slots,
                                   _slots(op, device, slots, n), workspace.data_ptr(), workspace.numel(), on)
    _done(code, op)
    if state_out is not None:
        increment_version(state_out)
    if given:
        increment_version(given)
    return out


def quantize_rows(x, codes=None, scales=None, stream: Optional[int] = None):
    """int8 codes of each row of x [rows, cols] (bfloat16, float16 or float32) with the library's
    recipe: scale = max|x| / 127 (1 where that is 0), code = x / scale rounded with halves away
    from zero, each step in float32; NaN counts for nothing and becomes 0.  Returns (codes int8
    [rows, cols], scales float32 [rows]), allocated if None.  Rows may be strided.
    """
    op = "quantize_rows"
    device = _device(op, x)
    if x.dtype not in DTYPES or x.dim() != 2:
        _refuse(f"{op}: x [rows, cols] is bfloat16, float16 or float32")
    if x.requires_grad or _tangents():
        _no_gradients(op, x)
    on = _stream(op, stream, device, codes is None or scales is None)
    given = [t for t in (codes, scales) if t is not None]
    rows, cols = x.shape
    _sizes(op, rows, cols)
    if codes is None:
        codes = torch.empty_like(x, dtype=torch.int8, memory_format=torch.contiguous_format)
    else:
        _check(op, device, "codes", codes, torch.int8, (rows, cols))
    if scales is None:
        scales = torch.empty((rows,), dtype=torch.float32, device=x.device)
    else:
        _check(op, device, "scales", scales, torch.float32, (rows,))
        _no_gradients(op, scales)
        if not scales.is_contiguous():
            _refuse(f"{op}: scales is not contiguous")
    a = QuantizeRows(DTYPES[x.dtype], rows, cols, x.data_ptr(), _row_stride(op, "x", x, cols), codes.data_ptr(),
                     _row_stride(op, "codes", codes, cols), scales.data_ptr())
    _done(_load().redukt_op_quantize_rows(ctypes.byref(a), on), op)
    if given:
        increment_version(given)
    return codes, scales


def int8_matmul(x, x_scales, w, w_scales, bias=None, out=None, dtype=torch.bfloat16, stream: Optional[int] = None):
    """out[i, j] = (x[i] . w[j]) x_scales[i] w_scales[j] + bias[j]: int8 codes x [tokens, k] and w
    [channels, k] with float32 scales per token and channel; exact integer sums, rounded once
    to `dtype` (bfloat16, float16 or float32; out's type where out is given).  Any sizes, k up to
    131,000; fastest where k and the strides of x and w are multiples of 16.
    """
    op = "int8_matmul"
    device = _device(op, x)
    f32 = torch.float32
    try:       # (all at once; what is wrong is looked for only if something is)
        (m, k), (n, wk) = x.shape, w.shape
        fine = (x.dtype is torch.int8 and w.dtype is torch.int8 and wk == k and x_scales.dtype is f32 and w_scales.dtype is f32
                and x_scales.shape == (m,) and w_scales.shape == (n,) and x_scales.is_contiguous() and w_scales.is_contiguous()
                and w.get_device() == x_scales.get_device() == w_scales.get_device() == device
                and (bias is None or (bias.dtype is f32 and bias.shape == (n,) and bias.is_contiguous()
                                      and bias.get_device() == device)))
    except (AttributeError, TypeError, ValueError):
        fine = False
    if not fine:
        _check(op, device, "x", x, torch.int8, (None, None))
        _check(op, device, "w", w, torch.int8, (None, x.shape[1]))
        _check(op, device, "x_scales", x_scales, f32, (x.shape[0],))
        _check(op, device, "w_scales", w_scales, f32, (w.shape[0],))
        if bias is not None:
            _check(op, device, "bias", bias, f32, (w.shape[0],))
        _refuse(f"{op}: scales and bias are contiguous")
    if x_scales.requires_grad or w_scales.requires_grad or (bias is not None and bias.requires_grad) or _tangents():
        _no_gradients(op, x_scales, w_scales, bias)
    _sizes(op, m, n, k)
    allocates = out is None
    on = _stream(op, stream, device, allocates)
    if allocates:
        if dtype not in DTYPES:
            _refuse(f"{op}: dtype is bfloat16, float16 or float32")
        out = torch.empty((m, n), dtype=dtype, device=x.device)
    else:
        if not isinstance(out, torch.Tensor) or out.dtype not in DTYPES:
            _refuse(f"{op}: out is bfloat16, float16 or float32")
        _check(op, device, "out", out, out.dtype, (m, n))
        _no_gradients(op, out)
    a = Int8Matmul(DTYPES[out.dtype], m, n, k, x.data_ptr(), _row_stride(op, "x", x, k), x_scales.data_ptr(), w.data_ptr(),
                   _row_stride(op, "w", w, k), w_scales.data_ptr(), None if bias is None else bias.data_ptr(),
                   out.data_ptr(), _row_stride(op, "out", out, n))
    _done(_load().redukt_op_int8_matmul(ctypes.byref(a), on), op)
    if not allocates:
        increment_version(out)
    return out
