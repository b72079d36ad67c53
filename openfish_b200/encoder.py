"""Operators of the transformer encoder in front of the CRF head (include/openfish_b200.h): attention over packed
sequences, the product of 8-bit integers, and the residual norm that feeds it.

Tensors are torch CUDA tensors of one device; the calls queue their kernels on ``stream`` (a torch.cuda.Stream of that
device; its current stream by default) and return.  On another stream than the current one, it is the caller who lets ``stream`` wait for what makes
the inputs, and the current stream for the results; the memory of both is kept until the streams are done with it, so that no tensor has to be
held on to.  Arguments that cannot be served raise before anything is queued:
TypeError and ValueError for what is no such tensor, OpenfishError for what the library refuses.  The operators serve: no
gradient passes through them.
"""
import contextlib
import ctypes as C
import math
import struct

NORM_KINDS = {"none": 0, "layer": 1, "rms": 2}


class AttentionArgs(C.Structure):
    """openfish_b200_attention_t."""
    _fields_ = ([(n, C.c_int) for n in ("dtype", "head_dim", "q_heads", "kv_heads", "sequences", "max_q", "max_k", "window_left",
                                        "window_right")]
                + [("scale", C.c_float), ("q_rows", C.c_longlong), ("k_rows", C.c_longlong)]
                + [(n, C.c_void_p) for n in ("q_start", "k_start", "q_used", "k_used", "q", "k", "v", "out")]
                + [(n, C.c_longlong) for n in ("q_stride_row", "q_stride_head", "k_stride_row", "k_stride_head", "v_stride_row",
                                               "v_stride_head", "out_stride_row", "out_stride_head")]
                + [("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)])


class MatmulI8Args(C.Structure):
    """openfish_b200_matmul_i8_t."""
    _fields_ = ([("dtype", C.c_int), ("cols", C.c_int), ("depth", C.c_int), ("rows", C.c_longlong)]
                + [(n, C.c_void_p) for n in ("x", "w", "x_scale", "w_scale", "bias", "out")]
                + [(n, C.c_longlong) for n in ("x_stride", "w_stride", "out_stride")])


class NormArgs(C.Structure):
    """openfish_b200_norm_t."""
    _fields_ = ([("dtype", C.c_int), ("kind", C.c_int), ("width", C.c_int), ("eps", C.c_float), ("residual_scale", C.c_float),
                 ("rows", C.c_longlong)]
                + [(n, C.c_void_p) for n in ("x", "residual", "weight", "bias", "out", "q", "q_scale")]
                + [(n, C.c_longlong) for n in ("x_stride", "residual_stride", "out_stride", "q_stride")])


def _packer(args):
    """The struct's fields from a tuple of numbers (an address of 0 for NULL): a fifth of the time that a ctypes.Structure takes,
    which a call on a single token would notice."""
    code = {C.c_int: "i", C.c_float: "f", C.c_longlong: "q", C.c_void_p: "P", C.c_size_t: "N"}
    packer = struct.Struct("@" + "".join(code[t] for _, t in args._fields_))
    assert packer.size == C.sizeof(args)

    def pack(*fields):
        try:
            return packer.pack(*fields)
        except (struct.error, OverflowError) as e:
            raise ValueError("a size or number that the library does not take: %s" % e) from None
    return pack


_pack_attention, _pack_matmul_i8, _pack_norm = _packer(AttentionArgs), _packer(MatmulI8Args), _packer(NormArgs)
_pack_room = struct.Struct("@PN").pack  # the last fields of AttentionArgs: the workspace


def declare(L):
    """The argument types of the encoder's entry points in the loaded library (a struct's address: ctypes.byref of it, or its
    bytes)."""
    for name in ("attention", "matmul_i8", "norm"):
        f = getattr(L, "openfish_b200_" + name)
        f.restype, f.argtypes = None, [C.c_void_p, C.c_void_p]
    L.openfish_b200_attention_workspace.restype, L.openfish_b200_attention_workspace.argtypes = C.c_size_t, [C.c_void_p]
    L.openfish_b200_encoder_wait.restype, L.openfish_b200_encoder_wait.argtypes = None, [C.c_void_p]


_of = _torch = None


def _ready():
    """The package, its library loaded, and torch."""
    global _of, _torch
    if _of is None:
        import torch

        import openfish_b200
        openfish_b200.lib()
        _of, _torch = openfish_b200, torch
    return _of._lib or _of.lib()


def _code(dtype):
    if dtype is _torch.float16:
        return 0
    if dtype is _torch.bfloat16:
        return 1
    raise TypeError("float16 or bfloat16, not %s" % dtype)


def _tensor(name, x, dims):
    if not isinstance(x, _torch.Tensor) or not x.is_cuda or x.dim() != dims:
        raise TypeError("%s must be a CUDA tensor of %d dimensions" % (name, dims))


def _want(name, x, shape, dtype, device):
    """The address of a CUDA tensor of this shape, type and device (its index) whose rows are contiguous."""
    if (isinstance(x, _torch.Tensor) and x.dtype is dtype and x.get_device() == device and x.shape == shape
            and (not shape or shape[-1] < 2 or x.stride()[-1] == 1)):
        return x.data_ptr()
    if not isinstance(x, _torch.Tensor) or not x.is_cuda or x.dtype is not dtype:
        raise TypeError("%s must be a CUDA %s tensor" % (name, dtype))
    if x.shape != shape:
        raise ValueError("%s has shape %s, not %s" % (name, tuple(x.shape), tuple(shape)))
    if x.get_device() != device:
        raise ValueError("%s is on cuda:%d, not on cuda:%d" % (name, x.get_device(), device))
    raise ValueError("%s: the elements of a row must lie next to each other" % name)


def _elsewhere(device):
    """What a call needs around it where it does not go to the current device: None, or a context."""
    return None if device == _torch.cuda.current_device() else _torch.cuda.device(device)


def _of_device(stream, device):
    if stream.device.index != device:
        raise ValueError("the stream is on %s, the tensors on cuda:%d" % (stream.device, device))
    return stream


def _on_stream(stream, call, *tensors):
    """call() on that stream, in whose allocations it makes its results.  The inputs' memory is not given to others before the stream is done with
    it, nor the results' before the caller's current stream is."""
    device = stream.device
    current = _torch.cuda.current_stream(device)
    with _torch.cuda.stream(stream):
        results = call()
    if stream != current:
        for t in tensors:
            if isinstance(t, _torch.Tensor):
                t.record_stream(stream)
        for t in results if isinstance(results, tuple) else (results,):
            if t is not None:
                t.record_stream(current)
    return results


def _check(L):
    if L.openfish_b200_last_status():
        _of._check()


def _attention_fields(q, k, v, q_start, k_start, max_q, max_k, out, q_used, k_used, causal, window, scale):
    """The struct's fields but the workspace's, checked."""
    _tensor("q", q, 3)
    _tensor("k", k, 3)
    dtype, device, int32 = q.dtype, q.get_device(), _torch.int32
    code, shape, kv_shape = _code(dtype), q.shape, k.shape
    if kv_shape[2] != shape[2]:
        raise ValueError("k has heads of %d, q of %d" % (kv_shape[2], shape[2]))
    if not isinstance(q_start, _torch.Tensor) or q_start.dim() != 1 or q_start.shape[0] < 1:
        raise TypeError("q_start must be a CUDA int32 tensor of at least one element")
    starts = q_start.shape
    sequences = starts[0] - 1
    at = (_want("q_start", q_start, starts, int32, device), _want("k_start", k_start, starts, int32, device),
          0 if q_used is None else _want("q_used", q_used, (sequences,), int32, device),
          0 if k_used is None else _want("k_used", k_used, (sequences,), int32, device),
          _want("q", q, shape, dtype, device), _want("k", k, kv_shape, dtype, device), _want("v", v, kv_shape, dtype, device),
          _want("out", out, shape, dtype, device))
    left, right = (-1, -1) if window is None else window
    if causal and right != 0:
        right = 0
    return ((code, shape[2], shape[1], kv_shape[1], sequences, max_q, max_k, left, right,
             1.0 / math.sqrt(shape[2] or 1) if scale is None else scale, shape[0], kv_shape[0]) + at
            + q.stride()[:2] + k.stride()[:2] + v.stride()[:2] + out.stride()[:2])


def attention(q, k, v, q_start, k_start, max_q, max_k, q_used=None, k_used=None, causal=False, window=None, scale=None, out=None,
              workspace=None, stream=None):
    """openfish_b200_attention: q [q_rows][q_heads][head_dim], k and v [k_rows][kv_heads][head_dim]; sequence s has the rows
    q_start[s]:q_start[s+1] and k_start[s]:k_start[s+1] (int32 on the device), or the first q_used[s] / k_used[s] of them.
    max_q, max_k: at least the longest sequence's.  window (left, right): how many keys before and behind its own place a
    query sees, -1 for all; causal: none behind.  scale: 1/sqrt(head_dim) by default.  Returns out (rows behind a sequence's
    used queries are not written).  workspace: a uint8 tensor of attention_workspace_bytes; made where it is not given."""
    L = _ready()
    _tensor("q", q, 3)
    device = q.get_device()
    if stream is not None:
        return _on_stream(_of_device(stream, device), lambda: attention(q, k, v, q_start, k_start, max_q, max_k, q_used, k_used, causal, window, scale,
                                                                        out, workspace),
                          q, k, v, q_start, k_start, q_used, k_used, out, workspace)
    around = _elsewhere(device)
    if around is not None:
        with around:
            return attention(q, k, v, q_start, k_start, max_q, max_k, q_used, k_used, causal, window, scale, out, workspace)
    if out is None:
        out = q.new_empty(q.shape)
    fields = _attention_fields(q, k, v, q_start, k_start, max_q, max_k, out, q_used, k_used, causal, window, scale)
    args = _pack_attention(*fields, 0, 0)
    if workspace is None:
        need = L.openfish_b200_attention_workspace(args)
        if need:  # the stream's allocator takes it back in order
            workspace = q.new_empty(need, dtype=_torch.uint8)
    if workspace is not None:
        room = _pack_room(_want("workspace", workspace, workspace.shape, _torch.uint8, device), workspace.numel())
        args = args[: -len(room)] + room
    L.openfish_b200_attention(_torch._C._cuda_getCurrentRawStream(device), args)
    _check(L)
    return out


def attention_workspace_bytes(q, k, v, q_start, k_start, max_q, max_k, q_used=None, k_used=None, causal=False, window=None, scale=None,
                              out=None):
    """openfish_b200_attention_workspace of that call."""
    L = _ready()
    fields = _attention_fields(q, k, v, q_start, k_start, max_q, max_k, q if out is None else out, q_used, k_used, causal, window, scale)
    with _elsewhere(q.get_device()) or contextlib.nullcontext():
        need = L.openfish_b200_attention_workspace(_pack_attention(*fields, 0, 0))
    _check(L)
    return need


def matmul_i8(x, x_scale, w, w_scale, bias=None, dtype=None, out=None, stream=None):
    """openfish_b200_matmul_i8: x [rows][depth] and w [cols][depth] int8 (as quantize_i8 gives them), x_scale [rows] and
    w_scale [cols] float32, bias [cols] of the result's type.  Returns out [rows][cols] (dtype: float16 by default)."""
    L = _ready()
    _tensor("x", x, 2)
    _tensor("w", w, 2)
    device = x.get_device()
    if stream is not None:
        return _on_stream(_of_device(stream, device), lambda: matmul_i8(x, x_scale, w, w_scale, bias, dtype, out), x, x_scale, w, w_scale, bias, out)
    around = _elsewhere(device)
    if around is not None:
        with around:
            return matmul_i8(x, x_scale, w, w_scale, bias, dtype, out)
    (rows, depth), cols = x.shape, w.shape[0]
    if out is None:
        dtype = dtype or _torch.float16
        out = x.new_empty((rows, cols), dtype=dtype)
    elif dtype is None:
        dtype = out.dtype
    int8, float32 = _torch.int8, _torch.float32
    L.openfish_b200_matmul_i8(_torch._C._cuda_getCurrentRawStream(device), _pack_matmul_i8(
        _code(dtype), cols, depth, rows, _want("x", x, x.shape, int8, device), _want("w", w, (cols, depth), int8, device),
        _want("x_scale", x_scale, (rows,), float32, device), _want("w_scale", w_scale, (cols,), float32, device),
        0 if bias is None else _want("bias", bias, (cols,), dtype, device), _want("out", out, (rows, cols), dtype, device),
        x.stride(0), w.stride(0), out.stride(0)))
    _check(L)
    return out


def norm(x, kind, weight=None, bias=None, eps=1e-5, residual=None, residual_scale=1.0, out=None, quantize=False, stream=None):
    """openfish_b200_norm of the rows of x [rows][width] + residual_scale * residual; kind "layer", "rms" or "none".  Returns
    out, or (out, q, q_scale) with quantize=True: the rows in 8 bits (int8 [rows][width], each row on a 16-byte boundary as
    matmul_i8 wants it) and their scales.  out=False: no result in 16 bits (None in its place).  out may be x or residual."""
    L = _ready()
    if kind not in NORM_KINDS:
        raise ValueError("kind must be one of %s" % ", ".join(NORM_KINDS))
    _tensor("x", x, 2)
    device = x.get_device()
    if stream is not None:
        return _on_stream(_of_device(stream, device), lambda: norm(x, kind, weight, bias, eps, residual, residual_scale, out, quantize),
                          x, weight, bias, residual, out)
    around = _elsewhere(device)
    if around is not None:
        with around:
            return norm(x, kind, weight, bias, eps, residual, residual_scale, out, quantize)
    dtype, shape = x.dtype, x.shape
    rows, width = shape
    if out is None:
        out = x.new_empty(shape)
    q = q_scale = None
    if quantize:
        stride = (width + 15) // 16 * 16
        q = x.new_empty((rows, stride), dtype=_torch.int8)
        if stride != width:
            q = q[:, :width]
        q_scale = x.new_empty(rows, dtype=_torch.float32)
    L.openfish_b200_norm(_torch._C._cuda_getCurrentRawStream(device), _pack_norm(
        _code(dtype), NORM_KINDS[kind], width, eps, residual_scale, rows, _want("x", x, shape, dtype, device),
        0 if residual is None else _want("residual", residual, shape, dtype, device),
        0 if weight is None else _want("weight", weight, (width,), dtype, device),
        0 if bias is None else _want("bias", bias, (width,), dtype, device),
        0 if out is False else _want("out", out, shape, dtype, device), q.data_ptr() if quantize else 0,
        q_scale.data_ptr() if quantize else 0, x.stride(0), 0 if residual is None else residual.stride(0),
        0 if out is False else out.stride(0), stride if quantize else 0))
    _check(L)
    out = None if out is False else out
    return (out, q, q_scale) if quantize else out


def quantize_i8(x, stream=None):
    """The rows of x [rows][width] in 8 bits: (q, scale), x ~ q * scale[:, None] (norm of kind "none").  For tokens, and once
    for the weights of a product."""
    return norm(x, "none", out=False, quantize=True, stream=stream)[1:]


def encoder_wait(stream=None):
    """openfish_b200_encoder_wait: waits for the stream (default: the current one) and raises if a kernel of these operators has
    given up waiting on its device since the calling thread's last such call (or its first call of the operator)."""
    L = _ready()
    stream = stream or _torch.cuda.current_stream()
    with _elsewhere(stream.device.index) or contextlib.nullcontext():
        L.openfish_b200_encoder_wait(stream.cuda_stream)
    _check(L)


def selfcheck_encoder_wait(kernels=3, limit_us=1000, stream=None):
    """openfish_b200_selfcheck_encoder_wait on the stream (default: the current one), for attention (1), matmul_i8 (2) or both: the status
    code.  The next encoder_wait has to raise, the one after it not."""
    L = _ready()
    stream = stream or _torch.cuda.current_stream()
    with _elsewhere(stream.device.index) or contextlib.nullcontext():
        return int(L.openfish_b200_selfcheck_encoder_wait(stream.cuda_stream, kernels, limit_us))
