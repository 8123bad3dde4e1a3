"""Operators of libredukt_gpu.so on the caller's own device tensors (include/redukt_ops.h).

The gated delta rule for one token (`delta_step`) and for whole sequences (`delta_chunk`), the
selective scan likewise (`scan_step`, `scan_chunk`) and its gradients (`scan_grad`, `scan`), int8
codes of activation rows (`quantize_rows`) and the product of codes with a scale per token and
channel (`int8_matmul`), e4m3 codes with a scale for blocks of 128 (`quantize_blocks`) and their
product (`fp8_matmul`), and tokens drawn from logits (`sample`).  Arguments are torch tensors on one GPU; work is queued on torch's
current stream of that GPU, or on `stream`, a hipStream_t's value.  Outputs and workspaces that a
call allocates belong to torch's current stream, so for another one they are passed in, and the
caller keeps all tensors until that stream is done with them.  Outputs overlap no input (but a state
pool its own next states).  No model needs to be open.  The operators but `scan` have no gradients: tensors
that ask for one, states and outputs among them, are refused while torch records them, and tensors
with a tangent always.  Wrong arguments raise `ffi.BackendError` (INVALID_ARGUMENT) and launch
nothing; there is no CPU fallback.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Tuple

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


class ScanRows(ctypes.Structure):
    """redukt_scan_rows."""
    _fields_ = [("dtype", ctypes.c_uint32), ("rows", ctypes.c_uint32), ("channels", ctypes.c_uint32), ("groups", ctypes.c_uint32),
                ("n", ctypes.c_uint32), ("x", ctypes.c_void_p), ("dt", ctypes.c_void_p), ("z", ctypes.c_void_p),
                ("b", ctypes.c_void_p), ("c", ctypes.c_void_p), ("out", ctypes.c_void_p), ("x_stride", ctypes.c_int64),
                ("dt_stride", ctypes.c_int64), ("z_stride", ctypes.c_int64), ("b_stride", ctypes.c_int64),
                ("c_stride", ctypes.c_int64), ("out_stride", ctypes.c_int64), ("a", ctypes.c_void_p), ("d", ctypes.c_void_p),
                ("dt_bias", ctypes.c_void_p)]


class ScanGradients(ctypes.Structure):
    """redukt_scan_grads."""
    _fields_ = [("dout", ctypes.c_void_p), ("dx", ctypes.c_void_p), ("ddt", ctypes.c_void_p), ("dz", ctypes.c_void_p),
                ("db", ctypes.c_void_p), ("dc", ctypes.c_void_p), ("dout_stride", ctypes.c_int64), ("dx_stride", ctypes.c_int64),
                ("ddt_stride", ctypes.c_int64), ("dz_stride", ctypes.c_int64), ("db_stride", ctypes.c_int64),
                ("dc_stride", ctypes.c_int64), ("da", ctypes.c_void_p), ("dd", ctypes.c_void_p), ("ddt_bias", ctypes.c_void_p)]


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


class QuantizeBlocks(ctypes.Structure):
    """redukt_quantize_blocks."""
    _fields_ = [("dtype", ctypes.c_uint32), ("rows", ctypes.c_uint32), ("cols", ctypes.c_uint32), ("block_rows", ctypes.c_uint32),
                ("x", ctypes.c_void_p), ("x_stride", ctypes.c_int64), ("codes", ctypes.c_void_p), ("codes_stride", ctypes.c_int64),
                ("scales", ctypes.c_void_p)]


class Fp8Matmul(ctypes.Structure):
    """redukt_fp8_matmul."""
    _fields_ = Int8Matmul._fields_


class Sample(ctypes.Structure):
    """redukt_sample."""
    _fields_ = [("dtype", ctypes.c_uint32), ("rows", ctypes.c_uint32), ("vocab", ctypes.c_uint32), ("logits", ctypes.c_void_p),
                ("logits_stride", ctypes.c_int64), ("u", ctypes.c_void_p), ("temperature", ctypes.c_float), ("top_p", ctypes.c_float),
                ("min_p", ctypes.c_float), ("top_k", ctypes.c_int32), ("temperatures", ctypes.c_void_p), ("top_ps", ctypes.c_void_p),
                ("min_ps", ctypes.c_void_p), ("top_ks", ctypes.c_void_p), ("tokens", ctypes.c_void_p)]


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
        L.redukt_op_scan_step.argtypes = [ctypes.POINTER(ScanRows), p, u32, p, p]
        L.redukt_op_scan_chunk.argtypes = [ctypes.POINTER(ScanRows), p, u32, p, p, u32, p, p, u64, p]
        L.redukt_op_scan_chunk_workspace.argtypes = [ctypes.POINTER(ScanRows), u32]
        L.redukt_op_scan_chunk_workspace.restype = u64
        L.redukt_op_scan_grad.argtypes = [ctypes.POINTER(ScanRows), ctypes.POINTER(ScanGradients), p, u32, p, p, p, p, u64, p]
        L.redukt_op_scan_grad_workspace.argtypes = [ctypes.POINTER(ScanRows), u32]
        L.redukt_op_scan_grad_workspace.restype = u64
        L.redukt_op_quantize_blocks.argtypes = [ctypes.POINTER(QuantizeBlocks), p]
        L.redukt_op_fp8_matmul.argtypes = [ctypes.POINTER(Fp8Matmul), p]
        L.redukt_op_sample.argtypes = [ctypes.POINTER(Sample), p]
        for f in ("delta_step", "delta_chunk", "scan_step", "scan_chunk", "scan_grad", "quantize_rows", "int8_matmul", "quantize_blocks",
                  "fp8_matmul", "sample"):
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
    if not isinstance(slots, torch.Tensor) or slots.dtype is not torch.int32 or slots.shape != (n,) or slots.get_device() != device:
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


def _scan_rows(op: str, x, dt, a, b, c, d, z, dt_bias, out) -> Tuple[ScanRows, int]:
    """The rows, with every tensor checked (out None: none is written)."""
    device = _device(op, x)
    f32, dtype = torch.float32, x.dtype
    if dtype not in DTYPES or x.dim() != 2:
        _refuse(f"{op}: x [rows, channels] is bfloat16, float16 or float32")
    shape = x.shape
    T, channels = shape
    try:       # (all at once; what is wrong is looked for only if something is)
        bc, n = b.shape, a.shape[1]
        fine = (dt.shape == shape and bc == c.shape and len(bc) == 3 and bc[0] == T and bc[2] == n and a.shape == (channels, n)
                and dt.dtype is dtype and b.dtype is dtype and c.dtype is dtype and a.dtype is f32 and a.is_contiguous()
                and dt.get_device() == a.get_device() == b.get_device() == c.get_device() == device
                and (z is None or (z.shape == shape and z.dtype is dtype and z.get_device() == device))
                and (d is None or (d.shape == shape[1:] and d.dtype is f32 and d.get_device() == device and d.is_contiguous()))
                and (dt_bias is None or (dt_bias.shape == shape[1:] and dt_bias.dtype is f32 and dt_bias.get_device() == device
                                         and dt_bias.is_contiguous())))
    except (AttributeError, IndexError, TypeError):
        fine = False
    if not fine:
        _check(op, device, "dt", dt, dtype, (T, channels))
        _check(op, device, "a", a, f32, (channels, None))
        _check(op, device, "b", b, dtype, (T, None, a.shape[1]))
        _check(op, device, "c", c, dtype, tuple(b.shape))
        for name, t, of, want in (("z", z, dtype, (T, channels)), ("d", d, f32, (channels,)), ("dt_bias", dt_bias, f32, (channels,))):
            if t is not None:
                _check(op, device, name, t, of, want)
        _refuse(f"{op}: a, d and dt_bias are contiguous")
    groups = bc[1]
    if (T | channels | groups | n) >> 31:
        _sizes(op, T, channels, groups, n)
    if out is not None and (not isinstance(out, torch.Tensor) or out.shape != shape or out.dtype is not dtype or out.get_device() != device):
        _check(op, device, "out", out, dtype, shape)
    wide, null = groups * n, None
    # (rows that are not contiguous have their steps looked up)
    return ScanRows(DTYPES[dtype], T, channels, groups, n, x.data_ptr(), dt.data_ptr(), z.data_ptr() if z is not null else null, b.data_ptr(),
                    c.data_ptr(), out.data_ptr() if out is not null else null,
                    channels if x.is_contiguous() else _row_stride(op, "x", x, channels),
                    channels if dt.is_contiguous() else _row_stride(op, "dt", dt, channels),
                    channels if z is null or z.is_contiguous() else _row_stride(op, "z", z, channels),
                    wide if b.is_contiguous() else _row_stride(op, "b", b, wide), wide if c.is_contiguous() else _row_stride(op, "c", c, wide),
                    channels if out is null or out.is_contiguous() else _row_stride(op, "out", out, channels), a.data_ptr(),
                    d.data_ptr() if d is not null else null, dt_bias.data_ptr() if dt_bias is not null else null), device


def _scan_pool(op: str, device: int, name: str, t, a: ScanRows, slots: Optional[int] = None) -> None:
    try:
        got = t.shape
        if (t.dtype is torch.float32 and got[1:] == (a.channels, a.n) and (slots is None or got[0] == slots) and t.is_contiguous()
                and t.get_device() == device):
            return
    except (AttributeError, IndexError):
        pass
    _check(op, device, name, t, torch.float32, (slots, a.channels, a.n))
    _refuse(f"{op}: {name} is not contiguous")


def _sequences(op: str, device: int, cu_seqlens) -> int:
    _check(op, device, "cu_seqlens", cu_seqlens, torch.int32, (None,))
    n = cu_seqlens.shape[0] - 1
    if n < 0 or not cu_seqlens.is_contiguous():
        _refuse(f"{op}: cu_seqlens holds one value more than there are sequences")
    if n > 65536:
        _refuse(f"{op}: more than 65,536 sequences")
    return n


def _workspace(op: str, device: int, workspace, need: int):
    if workspace is None:
        return torch.empty(need, dtype=torch.uint8, device=torch.device("cuda", device) if device >= 0 else "cpu")
    _check(op, device, "workspace", workspace, torch.uint8, (None,))
    if not workspace.is_contiguous():      # (its bytes are counted by its elements)
        _refuse(f"{op}: workspace is not contiguous")
    return workspace


def _asks(*tensors) -> bool:
    """Whether one (None: left out) requires a gradient, or somebody computes tangents."""
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return forward_ad._current_level >= 0


def scan_step(x, dt, a, b, c, states, d=None, z=None, dt_bias=None, slots=None, out=None, stream: Optional[int] = None):
    """The selective scan for one token of each of n entries (at most 65,536); states are stepped in place.

    With s = softplus(dt + dt_bias), a channel's state h takes a token as h <- e^(s a) h + s x B and
    gives out = (C . h + d x) silu(z).  x, dt, z [n, channels] and b, c [n, groups, size] in bfloat16,
    float16 or float32 (one type); a [channels, size], d and dt_bias [channels] and states [slots,
    channels, size] float32.  z, d and dt_bias may be left out.  size is 8, 16, 32 or 64; with several
    groups each has a multiple of 64 channels.  Entry i steps slot slots[i] (int32; None: slot i); -1 leaves
    entry i's output and state as they are; a slot out of range, or named by an earlier entry, gives NaN
    outputs and touches no state.  Returns out [n, channels] (allocated if None); rows may be strided, a and states
    begin on 16 bytes.
    """
    op = "scan_step"
    allocates = out is None
    if allocates:
        _device(op, x)
        out = torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    r, device = _scan_rows(op, x, dt, a, b, c, d, z, dt_bias, out)
    on = _stream(op, stream, device, allocates)
    _scan_pool(op, device, "states", states, r)
    if _asks(x, dt, a, b, c, states, d, z, dt_bias, out):
        _no_gradients(op, x, dt, a, b, c, d, z, dt_bias, states, out)
    code = _load().redukt_op_scan_step(ctypes.byref(r), states.data_ptr(), states.shape[0], _slots(op, device, slots, r.rows), on)
    _done(code, op)
    increment_version(states if allocates else (states, out))
    return out


def _scan_sizes(op: str, tokens: int, sequences: int, channels: int, groups: int, size: int) -> ScanRows:
    _sizes(op, tokens, sequences, channels, groups, size)
    return ScanRows(0, tokens, channels, groups, size)


def scan_chunk_workspace(tokens: int, sequences: int, channels: int, groups: int, size: int) -> int:
    """Bytes of workspace that `scan_chunk` needs for these sizes."""
    a = _scan_sizes("scan_chunk_workspace", tokens, sequences, channels, groups, size)
    return _load().redukt_op_scan_chunk_workspace(ctypes.byref(a), sequences)


def scan_chunk(x, dt, a, b, c, cu_seqlens, d=None, z=None, dt_bias=None, state_in=None, state_out=None, slots=None, out=None,
               workspace=None, stream: Optional[int] = None):
    """The selective scan over packed sequences: rows cu_seqlens[i] to cu_seqlens[i + 1] of x, dt, z, b
    and c (as in `scan_step`) are sequence i, from the state in slot slots[i] (None: i) of state_in (None:
    zeros); its final state goes to that slot of state_out (None: not wanted; state_in itself: in
    place).  cu_seqlens int32, none decreasing, within the rows.  A slot of -1 leaves the sequence out;
    slots out of range, or named before while state_out is given, give NaN rows.  Returns out [rows,
    channels]; rows of no sequence are not written.  At most 65,536 sequences, whose results depend on
    nothing else in the call.  workspace: a uint8 tensor of `scan_chunk_workspace` bytes that nothing else
    uses meanwhile (allocated if None).  For training, `scan` is the same with gradients.
    """
    op = "scan_chunk"
    allocates = out is None or workspace is None
    given = [t for t in (state_out, out, workspace) if t is not None]
    if out is None:
        _device(op, x)
        out = torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    r, device = _scan_rows(op, x, dt, a, b, c, d, z, dt_bias, out)
    on = _stream(op, stream, device, allocates)
    n = _sequences(op, device, cu_seqlens)
    n_slots = 0
    for name, pool in (("state_in", state_in), ("state_out", state_out)):
        if pool is not None:
            _scan_pool(op, device, name, pool, r)
            n_slots = pool.shape[0]
    if state_in is not None and state_out is not None and state_in.shape[0] != state_out.shape[0]:
        _refuse(f"{op}: state_in and state_out differ in slots")
    if _asks(x, dt, a, b, c, d, z, dt_bias, state_in, state_out, out):
        _no_gradients(op, x, dt, a, b, c, d, z, dt_bias, state_in, state_out, out)
    L = _load()
    workspace = _workspace(op, device, workspace, L.redukt_op_scan_chunk_workspace(ctypes.byref(r), n))
    code = L.redukt_op_scan_chunk(ctypes.byref(r), cu_seqlens.data_ptr(), n, None if state_in is None else state_in.data_ptr(),
                                  None if state_out is None else state_out.data_ptr(), n_slots, _slots(op, device, slots, n),
                                  workspace.data_ptr(), workspace.numel(), on)
    _done(code, op)
    if given:
        increment_version(given)
    return out


class ScanGrads(NamedTuple):
    """Gradients of `scan_grad`'s inputs, by their names; None for what was not given."""
    x: torch.Tensor
    dt: torch.Tensor
    a: torch.Tensor
    b: torch.Tensor
    c: torch.Tensor
    d: Optional[torch.Tensor]
    z: Optional[torch.Tensor]
    dt_bias: Optional[torch.Tensor]
    state_in: Optional[torch.Tensor]


def scan_grad_workspace(tokens: int, sequences: int, channels: int, groups: int, size: int) -> int:
    """Bytes of workspace that `scan_grad` needs for these sizes."""
    a = _scan_sizes("scan_grad_workspace", tokens, sequences, channels, groups, size)
    return _load().redukt_op_scan_grad_workspace(ctypes.byref(a), sequences)


def scan_grad(dout, x, dt, a, b, c, cu_seqlens, d=None, z=None, dt_bias=None, state_in=None, dstate_out=None, grads=None,
              workspace=None, stream: Optional[int] = None) -> ScanGrads:
    """The backward pass of the selective scan over packed sequences: the gradients of sum(dout * out) +
    sum(dstate_out * final states) by everything that goes in.  Inputs as in `scan_chunk`; state_in and
    dstate_out [sequences, channels, size] or None for zeros (without state_in, its gradient is None).
    Gradients have their inputs' types; rows of no sequence have gradients of zero.  Everything is formed anew from
    the inputs: nothing of the forward pass is needed.  grads: a ScanGrads of tensors to write (allocated if
    None).  workspace: a uint8 tensor of `scan_grad_workspace` bytes that nothing else uses meanwhile (allocated
    if None).
    """
    op = "scan_grad"
    allocates = grads is None or workspace is None
    r, device = _scan_rows(op, x, dt, a, b, c, d, z, dt_bias, None)
    on = _stream(op, stream, device, allocates)
    n = _sequences(op, device, cu_seqlens)
    _check(op, device, "dout", dout, x.dtype, (r.rows, r.channels))
    for name, pool in (("state_in", state_in), ("dstate_out", dstate_out)):
        if pool is not None:
            _scan_pool(op, device, name, pool, r, n)
    inputs = (x, dt, a, b, c, d, z, dt_bias, state_in)
    if grads is None:
        made = ScanGrads(*(None if t is None else torch.empty_like(t, memory_format=torch.contiguous_format) for t in inputs))
    else:
        if not isinstance(grads, tuple) or len(grads) != len(inputs):
            _refuse(f"{op}: grads is a ScanGrads")
        made = ScanGrads(*grads)
        for name, t, g in zip(ScanGrads._fields, inputs, made):
            if t is None and g is None:
                continue
            if t is None or g is None:
                _refuse(f"{op}: grads.{name} is given where {name} is, and only there")
            _check(op, device, "grads." + name, g, t.dtype, t.shape)
            if name in ("a", "d", "dt_bias", "state_in") and not g.is_contiguous():
                _refuse(f"{op}: grads.{name} is not contiguous")
    if _asks(dout, dstate_out, *inputs, *made):
        _no_gradients(op, dout, dstate_out, *inputs, *made)

    def at(t):
        return None if t is None else t.data_ptr()

    wide = r.groups * r.n
    g = ScanGradients(dout.data_ptr(), made.x.data_ptr(), made.dt.data_ptr(), at(made.z), made.b.data_ptr(), made.c.data_ptr(),
                      _row_stride(op, "dout", dout, r.channels), _row_stride(op, "grads.x", made.x, r.channels),
                      _row_stride(op, "grads.dt", made.dt, r.channels),
                      0 if made.z is None else _row_stride(op, "grads.z", made.z, r.channels),
                      _row_stride(op, "grads.b", made.b, wide), _row_stride(op, "grads.c", made.c, wide), made.a.data_ptr(),
                      at(made.d), at(made.dt_bias))
    L = _load()
    own = workspace is not None
    workspace = _workspace(op, device, workspace, L.redukt_op_scan_grad_workspace(ctypes.byref(r), n))
    code = L.redukt_op_scan_grad(ctypes.byref(r), ctypes.byref(g), cu_seqlens.data_ptr(), n, at(state_in), at(dstate_out),
                                 at(made.state_in), workspace.data_ptr(), workspace.numel(), on)
    _done(code, op)
    written = ([t for t in made if t is not None] if grads is not None else []) + ([workspace] if own else [])
    if written:
        increment_version(written)
    return made


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, a, b, c, cu_seqlens, d, z, dt_bias, state_in):
        final = torch.empty((max(cu_seqlens.shape[0] - 1, 0),) + tuple(a.shape), dtype=torch.float32, device=x.device)
        # (a row of no sequence is a zero: what is left out of a loss by a factor of 0 may not be NaN)
        out = torch.zeros_like(x, memory_format=torch.contiguous_format)
        scan_chunk(x, dt, a, b, c, cu_seqlens, d, z, dt_bias, state_in, final, out=out)
        ctx.save_for_backward(x, dt, a, b, c, cu_seqlens, d, z, dt_bias, state_in)
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dfinal):
        x, dt, a, b, c, cu_seqlens, d, z, dt_bias, state_in = ctx.saved_tensors
        if dout is None:
            dout = torch.zeros_like(x)
        g = scan_grad(dout.contiguous(), x, dt, a, b, c, cu_seqlens, d, z, dt_bias, state_in,
                      None if dfinal is None else dfinal.contiguous())
        return g.x, g.dt, g.a, g.b, g.c, None, g.d, g.z, g.dt_bias, g.state_in


def scan(x, dt, a, b, c, cu_seqlens, d=None, z=None, dt_bias=None, state_in=None):
    """`scan_chunk` for training: (out, final states), from the states state_in [sequences, channels, size]
    (None: zeros), with gradients for every floating-point input (once; tangents are refused).  Rows of no
    sequence have outputs and gradients of zero.  On torch's current stream; the backward pass runs `scan_grad`
    on the stream of the forward pass.  To capture it, let no graph of an eager pass over the same leaves live.
    """
    op = "scan"
    _device(op, x)
    n = _sequences(op, x.get_device(), cu_seqlens)
    _check(op, x.get_device(), "a", a, torch.float32, (None, None))      # (the final states take their size from it)
    if _tangents():
        with torch.no_grad():
            _no_gradients(op, x, dt, a, b, c, d, z, dt_bias, state_in)
    if state_in is not None:
        _check(op, x.get_device(), "state_in", state_in, torch.float32, (n, None, None))
    return _Scan.apply(x, dt, a, b, c, cu_seqlens, d, z, dt_bias, state_in)


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


E4M3 = torch.float8_e4m3fn


def quantize_blocks(x, block_rows: int = 1, codes=None, scales=None, stream: Optional[int] = None):
    """e4m3 codes of x [rows, cols] (bfloat16, float16 or float32) with one scale for each 128 columns of a row
    (block_rows 1: activations) or of 128 rows (block_rows 128: weights): scale = max|x| / 448, at least 2^-126,
    code = x / scale to the nearest, each step in float32; NaN does not count and stays NaN.  Returns (codes
    float8_e4m3fn [rows, cols], scales float32 [ceil(rows / block_rows), ceil(cols / 128)]), allocated if None.  Rows
    may be strided.
    """
    op = "quantize_blocks"
    device = _device(op, x)
    if x.dtype not in DTYPES or x.dim() != 2:
        _refuse(f"{op}: x [rows, cols] is bfloat16, float16 or float32")
    if block_rows != 1 and block_rows != 128:
        _refuse(f"{op}: block_rows is 1 or 128")
    if x.requires_grad or _tangents():
        _no_gradients(op, x)
    on = _stream(op, stream, device, codes is None or scales is None)
    given = [t for t in (codes, scales) if t is not None]
    rows, cols = x.shape
    _sizes(op, rows, cols)
    blocks = (-(-rows // block_rows), -(-cols // 128))
    if codes is None:
        codes = torch.empty_like(x, dtype=E4M3, memory_format=torch.contiguous_format)
    else:
        _check(op, device, "codes", codes, E4M3, (rows, cols))
        _no_gradients(op, codes)
    if scales is None:
        scales = torch.empty(blocks, dtype=torch.float32, device=x.device)
    else:
        _check(op, device, "scales", scales, torch.float32, blocks)
        _no_gradients(op, scales)
        if not scales.is_contiguous():
            _refuse(f"{op}: scales is not contiguous")
    a = QuantizeBlocks(DTYPES[x.dtype], rows, cols, block_rows, x.data_ptr(), _row_stride(op, "x", x, cols), codes.data_ptr(),
                       _row_stride(op, "codes", codes, cols), scales.data_ptr())
    _done(_load().redukt_op_quantize_blocks(ctypes.byref(a), on), op)
    if given:
        increment_version(given)
    return codes, scales


def fp8_matmul(x, x_scales, w, w_scales, bias=None, out=None, dtype=torch.bfloat16, stream: Optional[int] = None):
    """The product of e4m3 codes x [tokens, k] and w [channels, k] with float32 scales for blocks of 128 columns,
    x_scales [tokens, ceil(k / 128)] and w_scales [ceil(channels / 128), ceil(k / 128)] (`quantize_blocks` with block_rows
    1 and 128): out[i, j] = the sum over blocks b of (x[i] . w[j] over b) x_scales[i, b] w_scales[j // 128, b], + bias[j], rounded
    once to `dtype` (bfloat16, float16 or float32; out's type where out is given).  float32 outputs are as exact as float32
    sums of exact products.  For 16-bit outputs the products of eight neighbouring columns are added with 13 bits below the largest one's
    exponent, and all else in float32: beside the rounding they are off by at most 7 * 2^-13 of the largest product of each
    eight, times its scales (about 1.5e-5 of a result with random codes; more of one that large products cancel out in, for
    which float32 outputs are the way).  Any sizes, k up to
    1,048,576; fastest where k and the strides of x and w are multiples of 16.
    """
    op = "fp8_matmul"
    device = _device(op, x)
    f32 = torch.float32
    try:       # (all at once; what is wrong is looked for only if something is)
        (m, k), (n, wk) = x.shape, w.shape
        blocks = -(-k // 128)
        fine = (x.dtype is E4M3 and w.dtype is E4M3 and wk == k and x_scales.dtype is f32 and w_scales.dtype is f32
                and x_scales.shape == (m, blocks) and w_scales.shape == (-(-n // 128), blocks) and x_scales.is_contiguous()
                and w_scales.is_contiguous() and w.get_device() == x_scales.get_device() == w_scales.get_device() == device
                and (bias is None or (bias.dtype is f32 and bias.shape == (n,) and bias.is_contiguous()
                                      and bias.get_device() == device)))
    except (AttributeError, TypeError, ValueError):
        fine = False
    if not fine:
        _check(op, device, "x", x, E4M3, (None, None))
        _check(op, device, "w", w, E4M3, (None, x.shape[1]))
        _check(op, device, "x_scales", x_scales, f32, (x.shape[0], -(-x.shape[1] // 128)))
        _check(op, device, "w_scales", w_scales, f32, (-(-w.shape[0] // 128), -(-x.shape[1] // 128)))
        if bias is not None:
            _check(op, device, "bias", bias, f32, (w.shape[0],))
        _refuse(f"{op}: scales and bias are contiguous")
    if x.requires_grad or w.requires_grad or x_scales.requires_grad or w_scales.requires_grad or (bias is not None and bias.requires_grad) or _tangents():
        _no_gradients(op, x, w, x_scales, w_scales, bias)
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
    a = Fp8Matmul(DTYPES[out.dtype], m, n, k, x.data_ptr(), _row_stride(op, "x", x, k), x_scales.data_ptr(), w.data_ptr(),
                  _row_stride(op, "w", w, k), w_scales.data_ptr(), None if bias is None else bias.data_ptr(),
                  out.data_ptr(), _row_stride(op, "out", out, n))
    _done(_load().redukt_op_fp8_matmul(ctypes.byref(a), on), op)
    if not allocates:
        increment_version(out)
    return out


def sample(logits, u, temperature=1.0, top_k=None, top_p=None, min_p=None, out=None, stream: Optional[int] = None):
    """Draws a token from each row of logits [rows, vocab] (bfloat16, float16 or float32; vocab at most 1,048,576) by the
    random numbers u [rows] float32 in [0, 1).

    Token i weighs e^((l_i - max) / temperature) in whole steps of 2^-42; -inf and NaN weigh nothing.  Kept are, by
    falling logits and equal ones by index, the top_k first; of these, those before which less than top_p of their sum has
    come; of these, those that weigh min_p of the largest or more.  The token is the first by index up to which the kept
    weights' sum is over u times the whole one: sums are exact, so it depends on nothing but the row.  temperature, top_p and
    min_p are numbers or float32 tensors [rows], top_k a number or an int32 tensor; None (and top_k <= 0, top_p >= 1, min_p <=
    0) keeps all.  A temperature of 0 takes the first of the largest.  Rows may be strided.  Returns out int32 [rows]
    (allocated if None); -1 for a row with no logit over -inf.
    """
    op = "sample"
    device = _device(op, logits)
    if logits.dtype not in DTYPES or logits.dim() != 2:
        _refuse(f"{op}: logits [rows, vocab] is bfloat16, float16 or float32")
    rows, vocab = logits.shape
    _sizes(op, rows, vocab)

    asks = logits.requires_grad or _tangents()

    def per_row(name, t, dtype):
        nonlocal asks
        if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.shape != (rows,) or t.get_device() != device:
            _check(op, device, name, t, dtype, (rows,))
        if not t.is_contiguous():
            _refuse(f"{op}: {name} is not contiguous")
        asks = asks or t.requires_grad
        return t.data_ptr()

    def setting(name, v, dtype, none):
        """(the number for all rows, the address of one for each)"""
        if v is None:
            return none, None
        if isinstance(v, torch.Tensor):
            return none, per_row(name, v, dtype)
        try:
            return (min(max(int(v), -1), 2 ** 31 - 1) if dtype is torch.int32 else float(v)), None
        except (OverflowError, TypeError, ValueError):
            _refuse(f"{op}: {name} is a number or a tensor [rows]")

    f32 = torch.float32
    at_u = per_row("u", u, f32)
    (t, ts), (p, ps), (m, ms) = setting("temperature", temperature, f32, 1.0), setting("top_p", top_p, f32, 1.0), setting("min_p", min_p, f32, 0.0)
    k, ks = setting("top_k", top_k, torch.int32, 0)
    if asks:
        _no_gradients(op, logits, u, *(v if isinstance(v, torch.Tensor) else None for v in (temperature, top_p, min_p)))
    allocates = out is None
    on = _stream(op, stream, device, allocates)
    if allocates:
        out = torch.empty((rows,), dtype=torch.int32, device=logits.device)
    a = Sample(DTYPES[logits.dtype], rows, vocab, logits.data_ptr(), _row_stride(op, "logits", logits, vocab), at_u, t, p, m, k, ts, ps, ms, ks,
               per_row("out", out, torch.int32))
    _done(_load().redukt_op_sample(ctypes.byref(a), on), op)
    if not allocates:
        increment_version(out)
    return out
