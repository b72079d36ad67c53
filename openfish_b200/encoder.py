"""Operators of the transformer encoder in front of the CRF head (include/openfish_b200.h): attention over packed
sequences, the product of 8-bit integers, and the residual norm that feeds it.

Tensors are torch CUDA tensors of one device; the calls queue their kernels on ``stream`` (a torch.cuda.Stream of that
device; its current stream by default) and return.  Arguments that cannot be served raise before anything is queued:
TypeError and ValueError for what is no such tensor, OpenfishError for what the library refuses.
"""
import contextlib
import ctypes as C
import math

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
                + [(n, C.c_longlong) for n in ("x_stride", "w_stride", "out_stride")]
                + [("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)])


class NormArgs(C.Structure):
    """openfish_b200_norm_t."""
    _fields_ = ([("dtype", C.c_int), ("kind", C.c_int), ("width", C.c_int), ("eps", C.c_float), ("residual_scale", C.c_float),
                 ("rows", C.c_longlong)]
                + [(n, C.c_void_p) for n in ("x", "residual", "weight", "bias", "out", "q", "q_scale")]
                + [(n, C.c_longlong) for n in ("x_stride", "residual_stride", "out_stride", "q_stride")])


def declare(L):
    """The argument types of the encoder's entry points in the loaded library."""
    for name, args in (("attention", AttentionArgs), ("matmul_i8", MatmulI8Args), ("norm", NormArgs)):
        f = getattr(L, "openfish_b200_" + name)
        f.restype, f.argtypes = None, [C.c_void_p, C.POINTER(args)]
        if name != "norm":
            f = getattr(L, "openfish_b200_%s_workspace" % name)
            f.restype, f.argtypes = C.c_size_t, [C.POINTER(args)]
    L.openfish_b200_encoder_wait.restype, L.openfish_b200_encoder_wait.argtypes = None, [C.c_void_p]


def _lib():
    from . import lib
    return lib()


def _check():
    from . import _check
    _check()


def _code(dtype):
    import torch
    if dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("float16 or bfloat16, not %s" % dtype)
    return 0 if dtype == torch.float16 else 1


def _want(name, x, dims, dtype, device, shape=None):
    """Checks that x is a CUDA tensor of this kind whose last dimension is contiguous; its address."""
    import torch
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dim() != dims or x.dtype != dtype:
        raise TypeError("%s must be a CUDA %s tensor of %d dimensions" % (name, dtype, dims))
    if x.device != device:
        raise ValueError("%s is on %s, not on %s" % (name, x.device, device))
    if shape is not None and tuple(x.shape) != tuple(shape):
        raise ValueError("%s has shape %s, not %s" % (name, tuple(x.shape), tuple(shape)))
    if x.shape[-1] > 1 and x.stride(-1) != 1:
        raise ValueError("%s: the elements of a row must lie next to each other" % name)
    return x.data_ptr()


def _optional(name, x, *args):
    return None if x is None else _want(name, x, *args)


@contextlib.contextmanager
def _on(device, stream):
    """The device current, and the stream that the call goes to (allocations made meanwhile belong to it)."""
    import torch
    if stream is None:
        if device.index == torch.cuda.current_device():
            yield torch.cuda.current_stream(device).cuda_stream
        else:
            with torch.cuda.device(device):
                yield torch.cuda.current_stream(device).cuda_stream
    else:
        if stream.device != device:
            raise ValueError("the stream is on %s, the tensors on %s" % (stream.device, device))
        with torch.cuda.stream(stream):
            yield stream.cuda_stream


def _workspace(given, need, device):
    """(address, bytes) of the given workspace, or of a new one that the stream's allocator takes back in order."""
    import torch
    if given is not None:
        return _want("workspace", given, 1, torch.uint8, device), given.numel(), given
    if not need:
        return None, 0, None
    own = torch.empty(need, dtype=torch.uint8, device=device)
    return own.data_ptr(), need, own


def _is_tensor(name, x, dims):
    import torch
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dim() != dims:
        raise TypeError("%s must be a CUDA tensor of %d dimensions" % (name, dims))


def attention_args(q, k, v, q_start, k_start, max_q, max_k, out, q_used=None, k_used=None, causal=False, window=None, scale=None):
    """The arguments of openfish_b200_attention for these tensors, checked; without a workspace."""
    import torch
    for name, x in (("q", q), ("k", k), ("v", v)):
        _is_tensor(name, x, 3)
    dt, dev = q.dtype, q.device
    a = AttentionArgs(dtype=_code(dt))
    a.q_rows, a.q_heads, a.head_dim = q.shape
    a.k_rows, a.kv_heads, _ = k.shape
    a.q = _want("q", q, 3, dt, dev)
    a.k = _want("k", k, 3, dt, dev, (k.shape[0], k.shape[1], q.shape[2]))
    a.v = _want("v", v, 3, dt, dev, k.shape)
    a.out = _want("out", out, 3, dt, dev, q.shape)
    if not isinstance(q_start, torch.Tensor) or q_start.numel() < 1:
        raise TypeError("q_start must be a CUDA int32 tensor of at least one element")
    a.sequences = q_start.numel() - 1
    for name, x, n in (("q_start", q_start, a.sequences + 1), ("k_start", k_start, a.sequences + 1), ("q_used", q_used, a.sequences),
                       ("k_used", k_used, a.sequences)):
        if x is not None or name.endswith("start"):
            setattr(a, name, _want(name, x, 1, torch.int32, dev, (n,)))
    a.max_q, a.max_k = int(max_q), int(max_k)
    left, right = (-1, -1) if window is None else window
    if causal:
        right = 0 if right < 0 else min(right, 0)
    a.window_left, a.window_right = int(left), int(right)
    a.scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else scale
    for name, x in (("q", q), ("k", k), ("v", v), ("out", out)):
        setattr(a, name + "_stride_row", x.stride(0))
        setattr(a, name + "_stride_head", x.stride(1))
    return a


def attention(q, k, v, q_start, k_start, max_q, max_k, q_used=None, k_used=None, causal=False, window=None, scale=None, out=None,
              workspace=None, stream=None):
    """openfish_b200_attention: q [q_rows][q_heads][head_dim], k and v [k_rows][kv_heads][head_dim]; sequence s has the rows
    q_start[s]:q_start[s+1] and k_start[s]:k_start[s+1] (int32 on the device), or the first q_used[s] / k_used[s] of them.
    max_q, max_k: at least the longest sequence's.  window (left, right): how many keys before and behind its own place a
    query sees, -1 for all; causal: none behind.  scale: 1/sqrt(head_dim) by default.  Returns out (rows behind a sequence's
    used queries are not written).  workspace: a uint8 tensor of attention_workspace_bytes; made where it is not given."""
    import torch
    _is_tensor("q", q, 3)
    with _on(q.device, stream) as at:
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        a = attention_args(q, k, v, q_start, k_start, max_q, max_k, out, q_used, k_used, causal, window, scale)
        need = 0 if workspace is not None else _lib().openfish_b200_attention_workspace(C.byref(a))
        a.workspace, a.workspace_bytes, _keep = _workspace(workspace, need, q.device)
        _lib().openfish_b200_attention(at, C.byref(a))
    _check()
    return out


def attention_workspace_bytes(args):
    """openfish_b200_attention_workspace of what attention_args gives."""
    n = _lib().openfish_b200_attention_workspace(C.byref(args))
    _check()
    return n


def matmul_i8_args(x, x_scale, w, w_scale, out, bias=None):
    """The arguments of openfish_b200_matmul_i8 for these tensors, checked; without a workspace."""
    import torch
    _is_tensor("x", x, 2)
    _is_tensor("w", w, 2)
    _is_tensor("out", out, 2)
    dev = x.device
    a = MatmulI8Args(dtype=_code(out.dtype))
    (a.rows, a.depth), a.cols = x.shape, w.shape[0]
    a.x = _want("x", x, 2, torch.int8, dev)
    a.w = _want("w", w, 2, torch.int8, dev, (w.shape[0], x.shape[1]))
    a.x_scale = _want("x_scale", x_scale, 1, torch.float32, dev, (x.shape[0],))
    a.w_scale = _want("w_scale", w_scale, 1, torch.float32, dev, (w.shape[0],))
    a.bias = _optional("bias", bias, 1, out.dtype, dev, (w.shape[0],))
    a.out = _want("out", out, 2, out.dtype, dev, (x.shape[0], w.shape[0]))
    a.x_stride, a.w_stride, a.out_stride = x.stride(0), w.stride(0), out.stride(0)
    return a


def matmul_i8(x, x_scale, w, w_scale, bias=None, dtype=None, out=None, workspace=None, stream=None):
    """openfish_b200_matmul_i8: x [rows][depth] and w [cols][depth] int8 (as quantize_i8 gives them), x_scale [rows] and
    w_scale [cols] float32, bias [cols] of the result's type.  Returns out [rows][cols] (dtype: float16 by default)."""
    import torch
    _is_tensor("x", x, 2)
    _is_tensor("w", w, 2)
    with _on(x.device, stream) as at:
        if out is None:
            out = torch.empty((x.shape[0], w.shape[0]), dtype=dtype or torch.float16, device=x.device)
        elif dtype is not None and dtype != out.dtype:
            raise TypeError("out is %s, not %s" % (out.dtype, dtype))
        a = matmul_i8_args(x, x_scale, w, w_scale, out, bias)
        need = 0 if workspace is not None else _lib().openfish_b200_matmul_i8_workspace(C.byref(a))
        a.workspace, a.workspace_bytes, _keep = _workspace(workspace, need, x.device)
        _lib().openfish_b200_matmul_i8(at, C.byref(a))
    _check()
    return out


def norm(x, kind, weight=None, bias=None, eps=1e-5, residual=None, residual_scale=1.0, out=None, quantize=False, stream=None):
    """openfish_b200_norm of the rows of x [rows][width] + residual_scale * residual; kind "layer", "rms" or "none".  Returns
    out, or (out, q, q_scale) with quantize=True: the rows in 8 bits (int8 [rows][width], each row on a 16-byte boundary as
    matmul_i8 wants it) and their scales.  out=False: no result in 16 bits (None in its place).  out may be x or residual."""
    import torch
    if kind not in NORM_KINDS:
        raise ValueError("kind must be one of %s" % ", ".join(NORM_KINDS))
    _is_tensor("x", x, 2)
    dt, dev, shape = x.dtype, x.device, tuple(x.shape)
    a = NormArgs(dtype=_code(dt), kind=NORM_KINDS[kind], eps=eps, residual_scale=residual_scale)
    a.rows, a.width = shape
    a.x, a.x_stride = _want("x", x, 2, dt, dev), x.stride(0)
    if residual is not None:
        a.residual, a.residual_stride = _want("residual", residual, 2, dt, dev, shape), residual.stride(0)
    a.weight = _optional("weight", weight, 1, dt, dev, shape[1:])
    a.bias = _optional("bias", bias, 1, dt, dev, shape[1:])
    with _on(dev, stream) as at:
        if out is None:
            out = torch.empty(shape, dtype=dt, device=dev)
        if out is not False:
            a.out, a.out_stride = _want("out", out, 2, dt, dev, shape), out.stride(0)
        if quantize:
            q = torch.empty((shape[0], (shape[1] + 15) // 16 * 16), dtype=torch.int8, device=dev)[:, : shape[1]]
            q_scale = torch.empty(shape[0], dtype=torch.float32, device=dev)
            a.q, a.q_stride, a.q_scale = q.data_ptr(), q.stride(0), q_scale.data_ptr()
        _lib().openfish_b200_norm(at, C.byref(a))
    _check()
    out = None if out is False else out
    return (out, q, q_scale) if quantize else out


def quantize_i8(x, stream=None):
    """The rows of x [rows][width] in 8 bits: (q, scale), x ~ q * scale[:, None] (norm of kind "none").  For tokens, and once
    for the weights of a product."""
    return norm(x, "none", out=False, quantize=True, stream=stream)[1:]


def encoder_wait(stream=None):
    """openfish_b200_encoder_wait: waits for the stream (default: the current one) and raises if a kernel of these operators has given up."""
    import torch
    _lib().openfish_b200_encoder_wait((stream or torch.cuda.current_stream()).cuda_stream)
    _check()
