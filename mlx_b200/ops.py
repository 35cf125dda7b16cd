"""Host-side mirror of the reference operator front-end for the quantized path.

Same names, argument meaning and error behaviour as ``mlx.core.quantize``,
``dequantize``, ``quantized_matmul`` and ``gather_qmm`` (reference: mlx/ops.cpp:4784-4834
quantized_matmul, :5208-5245 quantize, :5465-5517 dequantize, :5553-5629 gather_qmm;
validation helpers :110-181, :4704-4754) in the affine mode.  ``quantize``, ``dequantize`` and ``qqmm`` have the
microscaled 4-bit modes ``mxfp4`` and ``nvfp4`` too; ``grouped_mm`` and ``grouped_qqmm`` are products of rows that are
already sorted by expert, with one size per expert; ``route_experts``, ``dispatch_rows`` and ``combine_rows`` bring tokens
there and back, ``group_rows`` and ``add_adapters`` put low-rank adapters beside a shared projection.  Arrays are ``torch`` CUDA tensors: torch only
supplies device memory and streams, every computation is a call into libb200q.so.
Invalid arguments raise ``ValueError`` (the reference's std::invalid_argument).
"""
from __future__ import annotations

import ctypes
import operator
import os
import threading
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib

_lib.load()   # with its symbols present, and its message if it is not built
from . import _front  # noqa: E402  (the native form of the ordinary calls: csrc/front.cpp)

_SCRATCH_OPS = {"qmm": 0, "gather": 1, "grouped": 2}
_DT = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_MODES = ("affine", "mxfp4", "mxfp8", "nvfp4")
_FP4 = {"mxfp4": (_lib.MXFP4, 32), "nvfp4": (_lib.NVFP4, 16)}   # mode -> (its code, its group size)


def _ptr(t: Optional[torch.Tensor]):
    return ctypes.c_void_p(t.data_ptr()) if t is not None and t.numel() > 0 else ctypes.c_void_p(0)


def _stream(t: torch.Tensor):
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _require_cuda(tag: str, *ts: torch.Tensor) -> torch.device:
    dev = ts[0].device
    for t in ts:
        if not t.is_cuda:
            raise RuntimeError(f"[{tag}] tensors must live on a CUDA device: there is no CPU fallback")
        if t.device != dev:
            raise ValueError(f"[{tag}] all tensors must be on the same device")
    return dev


def _as_u32(w: torch.Tensor, tag: str) -> torch.Tensor:
    if w.dtype == torch.uint32:
        return w
    raise ValueError(f"[{tag}] The weight matrix should be uint32 but received {w.dtype}")


class _Workspaces:
    """One zero-initialised scratch buffer per (device, stream, operator); it only grows.

    quantized_matmul, gather_qmm and the grouped products keep separate buffers: the matmul kernels rely on
    counters that start at zero and are left at zero (those of the grouped products lie elsewhere than
    quantized_matmul's), while gather_qmm uses its buffer as plain scratch (sorted indices, tile table, gathered rows).

    A buffer that has become too small is kept: a CUDA graph captured before goes on using it.
    Every new one is at least twice as large, so that the old ones never add up to more than it."""

    def __init__(self):
        self._bufs = {}
        self._outgrown = []   # (key, buffer)
        self._making = threading.RLock()   # one buffer at a time: of two made at once the native form could keep the one that is dropped

    def get(self, dev: torch.device, nbytes: int, op: str) -> torch.Tensor:
        key = (dev.index, torch.cuda.current_stream(dev).cuda_stream, op)
        buf = self._bufs.get(key)
        if buf is not None and buf.numel() >= nbytes:
            return buf
        with self._making:
            buf = self._bufs.get(key)
            if buf is None or buf.numel() < nbytes:
                nbytes = max(nbytes, 256)
                if buf is not None:
                    self._outgrown.append((key, buf))
                    nbytes = max(nbytes, 2 * buf.numel())
                with torch.cuda.device(dev):
                    buf = torch.zeros(nbytes, dtype=torch.uint8, device=dev)
                self._bufs[key] = buf
                _front.scratch(dev.index, key[1], _SCRATCH_OPS[op], buf.data_ptr(), buf.numel())
            return buf

    def all(self):
        """Every (key, buffer) that a kernel may still be using."""
        return list(self._bufs.items()) + self._outgrown


_workspaces = _Workspaces()

_STATUS_TEXT = {
    1: "gather index out of range (that output was zeroed)",
    2: "bounded wait expired in the bulk-copy ring of a decode kernel",
    3: "bounded wait expired in the tcgen05 prefill kernel",
    4: "bounded wait expired in the tcgen05 decode kernel",
    5: "bounded wait expired in the TMA ring of the stream decode kernel",
    6: "bounded wait for a peer GPU's completion flag expired: the gathered output is incomplete",
    7: "bounded wait expired in the row-owning decode kernel",
    8: "bounded wait expired in the grouped tensor-core kernel",
    9: "a group size was negative, or the groups reach past the last row (they end there)",
}


class DeviceStatusError(RuntimeError):
    """A kernel of this library gave up on a bounded wait (or met a bad gather index) and said so
    in the status word of its workspace: the outputs of that call are not valid."""

    def __init__(self, code: int, words, where: str):
        self.code, self.words = int(code), tuple(int(w) for w in words)
        super().__init__(f"b200q device status {self.code} ({_STATUS_TEXT.get(self.code, 'unknown')}) in the "
                         f"{where} workspace; status words {self.words}")


def read_workspace_status(ws: torch.Tensor, stream_ptr: int, where: str = "caller") -> None:
    """Synchronises the stream, reads and clears the status word at the end of `ws`, and raises
    DeviceStatusError if it is non-zero, after zeroing the whole workspace again (an aborted
    kernel leaves counters and partial sums behind that would corrupt every later call)."""
    lib = _lib.load()
    st = (ctypes.c_uint32 * 4)()
    sp = ctypes.c_void_p(stream_ptr)
    with torch.cuda.device(ws.device):
        _lib.check(lib.b200q_read_status(ctypes.c_void_p(ws.data_ptr()), ws.numel(), sp, st))
        if st[0] != 0:
            _lib.check(lib.b200q_workspace_init(ctypes.c_void_p(ws.data_ptr()), ws.numel(), sp))
            raise DeviceStatusError(st[0], list(st), where)


def check_status(device: Optional[torch.device] = None) -> None:
    """Checked mode on request: synchronises every stream this module has launched on (for
    `device`, or all devices) and raises DeviceStatusError if any kernel reported a failure since
    the last check.  The operators themselves never synchronise; call this where the results are
    about to be consumed on the host, or set B200Q_CHECK_STATUS=1 to have every operator call do
    it before it returns (debugging: it serialises host and device)."""
    for (dev_index, stream_ptr, op), ws in _workspaces.all():
        if device is not None and torch.device(device).index not in (None, dev_index):
            continue
        read_workspace_status(ws, stream_ptr, op)


def _checked() -> bool:
    import os
    return os.environ.get("B200Q_CHECK_STATUS", "0") == "1"


def _mode_params(mode: str, group_size, bits, tag: str) -> Tuple[int, int]:
    if mode not in _MODES:
        raise ValueError(f"[{tag}] Invalid quantization mode '{mode}'.")
    if mode != "affine":
        raise NotImplementedError(f"[{tag}] only the affine mode is built; '{mode}' is out of scope"
                                  + ("" if mode not in _FP4 else " (quantize, dequantize, qqmm and grouped_qqmm have it)"))
    return (64 if group_size is None else int(group_size), 4 if bits is None else int(bits))


def _validate_mode_with_type(tag, scales, biases, out_type):
    # mlx/ops.cpp:4704-4754
    if out_type is not None and not out_type.is_floating_point:
        raise ValueError(f"[{tag}] Only real floating types are supported but output dtype == {out_type}.")
    if biases is None:
        raise ValueError(f"[{tag}] Biases must be provided for affine quantization.")
    dtype = torch.promote_types(scales.dtype, biases.dtype)
    if not dtype.is_floating_point:
        raise ValueError(
            f"[{tag}] Only real floating types are supported but scales.dtype() == {scales.dtype} "
            f"and biases.dtype() == {biases.dtype}."
        )
    return out_type if out_type is not None else dtype


def _validate_quantized_input(tag, w, scales, group_size, bits, biases):
    # mlx/ops.cpp:110-150
    _as_u32(w, tag)
    if biases is not None and scales.shape != biases.shape:
        raise ValueError(
            f"[{tag}] Scales and biases should have the same shape. Received scales with shape "
            f"{tuple(scales.shape)} and biases with {tuple(biases.shape)}"
        )
    if w.ndim < 2 or scales.ndim != w.ndim or tuple(w.shape[:-2]) != tuple(scales.shape[:-2]):
        raise ValueError(
            f"[{tag}] Weight and scales should have the same batch shape. Received weight with shape "
            f"{tuple(w.shape)}, scales with {tuple(scales.shape)}."
        )
    if w.shape[-1] * 32 // bits != scales.shape[-1] * group_size:
        raise ValueError(
            f"[{tag}] The shapes of the weight and scales are incompatible based on bits and group_size. "
            f"w.shape() == {tuple(w.shape)} and scales.shape() == {tuple(scales.shape)} "
            f"with group_size={group_size} and bits={bits}"
        )


def _extract_dims(tag, x, w, scales, biases, transpose, group_size, bits):
    # mlx/ops.cpp:152-181
    _validate_quantized_input(tag, w, scales, group_size, bits, biases)
    if x.ndim < 1:
        raise ValueError(f"[{tag}] x must have at least one dimension")
    x_inner = x.shape[-1]
    w_inner = w.shape[-1] * 32 // bits if transpose else w.shape[-2]
    w_outer = w.shape[-2] if transpose else w.shape[-1] * 32 // bits
    if w_inner != x_inner:
        raise ValueError(
            f"[{tag}] Last dimension of first input with shape (..., {x_inner}) does not match the expanded "
            f"quantized matrix ({w_inner}, {w_outer}) computed from shape {tuple(w.shape)} with "
            f"group_size={group_size}, bits={bits} and transpose={transpose}"
        )
    return w_inner, w_outer


# --------------------------------------------------------------------------- quantize
def quantize(w: torch.Tensor, group_size: Optional[int] = None, bits: Optional[int] = None,
             mode: str = "affine", global_scale: Optional[torch.Tensor] = None):
    """-> (w_q uint32 [..., K*bits/32], scales [..., K/g], biases [..., K/g]); mlx/ops.cpp:5208.

    mode "mxfp4" (groups of 32) or "nvfp4" (groups of 16): -> (w_q uint32 [..., K/8], scales uint8 [..., K/g]), 4-bit
    floating-point codes under a power of two or an E4M3 number per group; see b200q_fp4_quantize in include/b200q.h for
    the rounding.  global_scale (nvfp4): what every scale is relative to, a float32 tensor with one element or one per
    matrix of a stack; largest magnitude / (448 * 6) is the usual choice."""
    if mode in _FP4:
        return _fp4_quantize(w, group_size, bits, mode, global_scale)
    if global_scale is not None:
        raise ValueError(f"[quantize] a global scale belongs to the nvfp4 mode, not to '{mode}'.")
    q = _front.quantize(w, group_size, bits, mode)
    if q is not None:
        return q
    group_size, bits = _mode_params(mode, group_size, bits, "quantize")
    if not w.dtype.is_floating_point or w.dtype not in _DT:
        raise ValueError(f"[quantize] Only real floating types can be quantized but w has type {w.dtype}.")
    if w.ndim < 2:
        raise ValueError(
            f"[quantize] The matrix to be quantized must have at least 2 dimension but it has only {w.ndim}."
        )
    if group_size not in (32, 64, 128):
        raise ValueError(
            f"[quantize] The requested group size {group_size} is not supported. "
            "The supported group sizes are 32, 64, and 128."
        )
    if bits < 2 or bits > 8 or bits == 7:
        raise ValueError(
            f"[quantize] The requested number of bits {bits} is not supported. "
            "The supported bits are 2, 3, 4, 5, 6 and 8."
        )
    if w.shape[-1] % group_size != 0:
        raise ValueError(
            f"[quantize] The last dimension of the matrix needs to be divisible by the quantization group "
            f"size {group_size}. However the provided matrix has shape {tuple(w.shape)}"
        )
    dev = _require_cuda("quantize", w)
    w = w.contiguous()
    K = w.shape[-1]
    rows = w.numel() // K if K else 0
    lead = tuple(w.shape[:-1])
    with torch.cuda.device(dev):
        wq = torch.empty(lead + (K * bits // 32,), dtype=torch.uint32, device=dev)
        scales = torch.empty(lead + (K // group_size,), dtype=w.dtype, device=dev)
        biases = torch.empty_like(scales)
        rc = _lib.load().b200q_quantize(_ptr(w), _DT[w.dtype], rows, K, group_size, bits, _ptr(wq),
                                        _ptr(scales), _ptr(biases), _stream(w))
    _lib.check(rc)
    return wq, scales, biases


def dequantize(w: torch.Tensor, scales: torch.Tensor, biases: Optional[torch.Tensor] = None,
               group_size: Optional[int] = None, bits: Optional[int] = None, mode: str = "affine",
               dtype: Optional[torch.dtype] = None, global_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """mlx/ops.cpp:5465-5517 (+ affine_dequantize :5258-5340).  The microscaled modes have no biases; their values come
    in `dtype`, bfloat16 if it is not given."""
    if mode in _FP4:
        return _fp4_dequantize(w, scales, biases, group_size, bits, mode, dtype, global_scale)
    if global_scale is not None:
        raise ValueError(f"[dequantize] a global scale belongs to the nvfp4 mode, not to '{mode}'.")
    if dtype is None or dtype == scales.dtype:
        out = _front.dequantize(w, scales, biases, group_size, bits, mode)
        if out is not None:
            return out
    group_size, bits = _mode_params(mode, group_size, bits, "dequantize")
    out_type = _validate_mode_with_type("dequantize", scales, biases, dtype)
    if bits <= 0:
        raise ValueError(f"[dequantize] Invalid value for bits: {bits}")
    if group_size <= 0:
        raise ValueError(f"[dequantize] Invalid value for group_size: {group_size}")
    if w.dtype != torch.uint32:
        raise ValueError("[dequantize] The matrix should be given as a uint32")
    if w.ndim < 2:
        raise ValueError(
            f"[dequantize] The matrix to be dequantized must have at least 2 dimension but it has only {w.ndim}."
        )
    if (w.ndim != scales.ndim or w.ndim != biases.ndim or tuple(w.shape[:-1]) != tuple(scales.shape[:-1])
            or tuple(w.shape[:-1]) != tuple(biases.shape[:-1])):
        raise ValueError("[dequantize] Shape of scales and biases does not match the matrix")
    K = w.shape[-1] * 32 // bits
    if K != scales.shape[-1] * group_size or scales.shape != biases.shape:
        raise ValueError(
            "[dequantize] Shape of scales and biases does not match the matrix given the quantization "
            f"parameters. Provided matrix of shape {tuple(w.shape)} and scales/biases of shape "
            f"{tuple(scales.shape)} with group_size={group_size} and bits={bits}."
        )
    if scales.dtype not in _DT or scales.dtype != biases.dtype:
        ct = torch.promote_types(scales.dtype, biases.dtype)
        scales, biases = scales.to(ct), biases.to(ct)
    dev = _require_cuda("dequantize", w, scales, biases)
    w, scales, biases = w.contiguous(), scales.contiguous(), biases.contiguous()
    rows = w.numel() // w.shape[-1] if w.shape[-1] else 0
    with torch.cuda.device(dev):
        out = torch.empty(tuple(w.shape[:-1]) + (K,), dtype=scales.dtype, device=dev)
        rc = _lib.load().b200q_dequantize(_ptr(w), _ptr(scales), _ptr(biases), _DT[scales.dtype], rows, K,
                                          group_size, bits, _ptr(out), _stream(w))
    _lib.check(rc)
    return out if out.dtype == out_type else out.to(out_type)


# ------------------------------------------------------------------- microscaled 4-bit modes
def _fp4_params(tag, mode, group_size, bits):
    if mode not in _MODES:
        raise ValueError(f"[{tag}] Invalid quantization mode '{mode}'.")
    if mode not in _FP4:
        raise NotImplementedError(f"[{tag}] mode '{mode}' is not built; 'mxfp4' and 'nvfp4' are")
    code, group = _FP4[mode]
    if (group if group_size is None else group_size) != group or (4 if bits is None else bits) != 4:
        raise ValueError(f"[{tag}] mode '{mode}' has 4 bits in groups of {group}, not {bits} in groups of {group_size}.")
    return code, group


def _fp4_global(tag, mode, g, counts, dev):
    """A global scale as a contiguous float32 tensor on `dev`, or None; `counts`: how many elements it may have."""
    if g is None:
        return None
    if mode != "nvfp4":
        raise ValueError(f"[{tag}] a global scale belongs to the nvfp4 mode, not to '{mode}'.")
    if not isinstance(g, torch.Tensor) or not g.dtype.is_floating_point or g.numel() not in counts:
        raise ValueError(f"[{tag}] a global scale is a floating-point tensor of {' or '.join(str(c) for c in sorted(set(counts)))} element(s).")
    if g.device != dev:
        raise ValueError(f"[{tag}] all tensors must be on the same device")
    return g.detach().to(torch.float32).contiguous()


def _fp4_weights(tag, w, scales, group):
    _as_u32(w, tag)
    if scales.dtype != torch.uint8:
        raise ValueError(f"[{tag}] The scales should be uint8 but received {scales.dtype}")
    if w.ndim < 2 or scales.ndim != w.ndim or w.shape[:-1] != scales.shape[:-1] or w.shape[-1] * 8 != scales.shape[-1] * group:
        raise ValueError(f"[{tag}] The shapes of the weight and scales are incompatible: w.shape() == {tuple(w.shape)} and "
                         f"scales.shape() == {tuple(scales.shape)} with 4 bits in groups of {group}")


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """Contiguous and on a 16-byte boundary."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _matrices(shape) -> int:
    return torch.Size(shape[:-2]).numel()


def _fp4_quantize(w, group_size, bits, mode, global_scale):
    q = _front.fp4_quantize(w, group_size, bits, mode, global_scale)
    if q is not None:
        return q
    code, group = _fp4_params("quantize", mode, group_size, bits)
    if w.dtype not in _DT:
        raise ValueError(f"[quantize] Only real floating types can be quantized but w has type {w.dtype}.")
    if w.ndim < 2:
        raise ValueError(f"[quantize] The matrix to be quantized must have at least 2 dimension but it has only {w.ndim}.")
    if w.shape[-1] % group != 0:
        raise ValueError("[quantize] The last dimension of the matrix needs to be divisible by the quantization group "
                         f"size {group}. However the provided matrix has shape {tuple(w.shape)}")
    dev = _require_cuda("quantize", w)
    n_mat = _matrices(w.shape)
    g = _fp4_global("quantize", mode, global_scale, (1, max(n_mat, 1)), dev)
    w = w.detach().contiguous()
    K, rows, lead = w.shape[-1], torch.Size(w.shape[:-1]).numel(), tuple(w.shape[:-1])
    with torch.cuda.device(dev):
        wq = torch.empty(lead + (K // 8,), dtype=torch.uint32, device=dev)
        scales = torch.empty(lead + (K // group,), dtype=torch.uint8, device=dev)
        per = max(rows if g is None or g.numel() == 1 else w.shape[-2], 1)
        rc = _lib.load().b200q_fp4_quantize(_ptr(w), _DT[w.dtype], rows, K, code, _ptr(g), per, _ptr(wq), _ptr(scales), _stream(w))
    _lib.check(rc)
    return wq, scales


def _fp4_dequantize(w, scales, biases, group_size, bits, mode, dtype, global_scale):
    if biases is None:
        v = _front.fp4_dequantize(w, scales, group_size, bits, mode, _DT.get(torch.bfloat16 if dtype is None else dtype, -1), global_scale)
        if v is not None:
            return v
    code, group = _fp4_params("dequantize", mode, group_size, bits)
    if biases is not None:
        raise ValueError(f"[dequantize] Biases must be null for quantization mode '{mode}'.")
    dtype = torch.bfloat16 if dtype is None else dtype
    if dtype not in _DT:
        raise ValueError(f"[dequantize] Only real floating types are supported but output dtype == {dtype}.")
    _fp4_weights("dequantize", w, scales, group)
    dev = _require_cuda("dequantize", w, scales)
    g = _fp4_global("dequantize", mode, global_scale, (1, max(_matrices(w.shape), 1)), dev)
    w, scales = _aligned(w), scales.contiguous()
    K, rows = w.shape[-1] * 8, torch.Size(w.shape[:-1]).numel()
    with torch.cuda.device(dev):
        out = torch.empty(tuple(w.shape[:-1]) + (K,), dtype=dtype, device=dev)
        per = max(rows if g is None or g.numel() == 1 else w.shape[-2], 1)
        rc = _lib.load().b200q_fp4_dequantize(_ptr(w), _ptr(scales), code, _ptr(g), per, _DT[dtype], rows, K, _ptr(out), _stream(w))
    _lib.check(rc)
    return out


def quantized_embedding(ids: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor,
                        group_size: Optional[int] = None, bits: Optional[int] = None,
                        mode: str = "affine") -> torch.Tensor:
    """QuantizedEmbedding.__call__ (python/mlx/nn/layers/quantized.py:149-158):
    dequantize(w[ids], scales[ids], biases[ids]) as one kernel.  ids: any integer tensor;
    out: ids.shape + [K] in the dtype of scales."""
    group_size, bits = _mode_params(mode, group_size, bits, "quantized_embedding")
    _validate_mode_with_type("quantized_embedding", scales, biases, None)
    if w.dtype != torch.uint32:
        raise ValueError("[quantized_embedding] The matrix should be given as a uint32")
    if w.ndim != 2 or scales.ndim != 2 or biases.shape != scales.shape or scales.shape[0] != w.shape[0]:
        raise ValueError("[quantized_embedding] Shape of scales and biases does not match the matrix")
    K = w.shape[-1] * 32 // bits
    if K != scales.shape[-1] * group_size:
        raise ValueError(
            "[quantized_embedding] Shape of scales and biases does not match the matrix given the quantization "
            f"parameters. Provided matrix of shape {tuple(w.shape)} and scales/biases of shape "
            f"{tuple(scales.shape)} with group_size={group_size} and bits={bits}."
        )
    if ids.dtype.is_floating_point or ids.dtype == torch.bool:
        raise ValueError("[quantized_embedding] ids must be integral.")
    if scales.dtype not in _DT or scales.dtype != biases.dtype:
        ct = torch.promote_types(scales.dtype, biases.dtype)
        scales, biases = scales.to(ct), biases.to(ct)
    dev = _require_cuda("quantized_embedding", w, scales, biases)
    w, scales, biases = w.contiguous(), scales.contiguous(), biases.contiguous()
    ids64 = ids.to(device=dev, dtype=torch.int64).contiguous().reshape(-1)
    ids64 = torch.where(ids64 < 0, ids64 + w.shape[0], ids64)  # negative ids count from the end, as indexing does
    ids32 = ids64.to(torch.int32)  # uint32 bit pattern
    with torch.cuda.device(dev):
        out = torch.empty(tuple(ids.shape) + (K,), dtype=scales.dtype, device=dev)
        rc = _lib.load().b200q_dequantize_rows(_ptr(w), _ptr(scales), _ptr(biases), _ptr(ids32), ids32.numel(),
                                               _DT[scales.dtype], w.shape[0], K, group_size, bits, _ptr(out),
                                               _stream(w))
    _lib.check(rc)
    return out


# ------------------------------------------------------------------- quantized_matmul
_weights_constant = os.environ.get("B200Q_WEIGHTS_CONSTANT", "") == "1"


def set_weights_constant(on: bool) -> None:
    """The caller's promise that packed weights, scales and biases are not written by whatever
    precedes a matmul on its stream (b200q_set_weights_constant): the decode kernel may then request
    them before the previous kernel has finished.  quantized_matmul suspends the promise for a call
    in which it had to cast or copy one of the three itself (that copy IS the preceding kernel)."""
    global _weights_constant
    _weights_constant = bool(on)
    _lib.load().b200q_set_weights_constant(int(_weights_constant))


def quantized_matmul(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor,
                     biases: Optional[torch.Tensor] = None, transpose: bool = True,
                     group_size: Optional[int] = None, bits: Optional[int] = None,
                     mode: str = "affine") -> torch.Tensor:
    """mlx/ops.cpp:4784-4834.  x [..., M, K] (or [K]); w [..., N, K*bits/32] when transposed."""
    y = _front.qmm(x, w, scales, biases, transpose, group_size, bits, mode)
    if y is not None:
        return y
    group_size, bits = _mode_params(mode, group_size, bits, "quantized_matmul")
    dtype = _validate_mode_with_type("quantized_matmul", scales, biases, None)
    _, w_outer = _extract_dims("quantized_matmul", x, w, scales, biases, transpose, group_size, bits)
    dtype = torch.promote_types(x.dtype, dtype)
    if not dtype.is_floating_point or dtype not in _DT:
        raise ValueError(f"[quantized_matmul] Only real floating types are supported but x.dtype() == {x.dtype}.")
    dev = _require_cuda("quantized_matmul", x, w, scales, biases)
    given = (w, scales, biases)
    x, scales, biases = x.to(dtype), scales.to(dtype), biases.to(dtype)

    vector = x.ndim == 1
    if vector:
        x = x.unsqueeze(0)
    K = x.shape[-1]
    M = x.shape[-2]
    if x.ndim > 2 and w.ndim > 2:
        # both batched: broadcast the batch dimensions (mlx/ops.cpp:4823-4825)
        bshape = torch.broadcast_shapes(x.shape[:-2], w.shape[:-2])
        x = x.expand(bshape + x.shape[-2:]).contiguous()
        w = w.expand(bshape + w.shape[-2:]).contiguous()
        scales = scales.expand(bshape + scales.shape[-2:]).contiguous()
        biases = biases.expand(bshape + biases.shape[-2:]).contiguous()
        batch, w_stride, out_lead = x.numel() // max(M * K, 1), 1, tuple(bshape)
    elif w.ndim > 2:
        # 2-D x against a stack of matrices
        bshape = tuple(w.shape[:-2])
        x = x.expand(bshape + x.shape[-2:]).contiguous()
        w, scales, biases = w.contiguous(), scales.contiguous(), biases.contiguous()
        batch, w_stride, out_lead = w.numel() // max(w.shape[-1] * w.shape[-2], 1), 1, bshape
    else:
        x, w, scales, biases = x.contiguous(), w.contiguous(), scales.contiguous(), biases.contiguous()
        out_lead = tuple(x.shape[:-2])
        batch, w_stride = (x.numel() // max(M * K, 1) if M * K else 0), 0
        if M * K == 0:
            batch = 1
            for d in out_lead:
                batch *= d
    N = w_outer
    lib = _lib.load()
    with torch.cuda.device(dev):
        y = torch.empty(out_lead + (M, N), dtype=dtype, device=dev)
        need = lib.b200q_qmm_workspace_bytes(_DT[dtype], batch, M, N, K, group_size, bits, int(transpose))
        ws = _workspaces.get(dev, need, "qmm")
        # a weight operand this function has just cast or copied was written by the kernel right
        # before the matmul on this stream: no early weight loads for this call
        fresh = _weights_constant and any(a.data_ptr() != b.data_ptr() for a, b in zip((w, scales, biases), given))
        if fresh:
            lib.b200q_set_weights_constant(0)
        try:
            rc = lib.b200q_qmm(_ptr(x), _ptr(w), _ptr(scales), _ptr(biases), _ptr(y), _DT[dtype], batch, M, N, K,
                               group_size, bits, int(transpose), w_stride, _ptr(ws), ws.numel(), _stream(x))
        finally:
            if fresh:
                lib.b200q_set_weights_constant(1)
    _lib.check(rc)
    if _checked():
        read_workspace_status(ws, torch.cuda.current_stream(dev).cuda_stream, "qmm")
    return y.squeeze(-2) if vector else y


# -------------------------------------------------------------------------- gather_qmm
def gather_qmm(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, biases: Optional[torch.Tensor] = None,
               lhs_indices: Optional[torch.Tensor] = None, rhs_indices: Optional[torch.Tensor] = None,
               transpose: bool = True, group_size: Optional[int] = None, bits: Optional[int] = None,
               mode: str = "affine", sorted_indices: bool = False) -> torch.Tensor:
    """mlx/ops.cpp:5553-5629.  out shape = broadcast(lhs, rhs).shape + [M, N]."""
    if lhs_indices is None and rhs_indices is None:
        return quantized_matmul(x, w, scales, biases, transpose, group_size, bits, mode)
    y = _front.gather(x, w, scales, biases, lhs_indices, rhs_indices, transpose, group_size, bits, mode)
    if y is not None:
        return y
    group_size, bits = _mode_params(mode, group_size, bits, "gather_qmm")
    out_type = _validate_mode_with_type("gather_qmm", scales, biases, None)
    _, w_outer = _extract_dims("gather_qmm", x, w, scales, biases, transpose, group_size, bits)
    out_type = torch.promote_types(x.dtype, out_type)
    if not out_type.is_floating_point or out_type not in _DT:
        raise ValueError(f"[gather_qmm] Only real floating types are supported but x.dtype() == {x.dtype}.")
    if x.ndim < 2:
        raise ValueError("[gather_qmm] x must have at least two dimensions")
    for idx, name in ((lhs_indices, "lhs_indices"), (rhs_indices, "rhs_indices")):
        if idx is not None and (idx.dtype.is_floating_point or idx.dtype == torch.bool):
            raise ValueError(f"[gather_qmm] Got {name} with invalid dtype. Indices must be integral.")
    dev = _require_cuda("gather_qmm", x, w, scales, biases)

    def default_idx(t):  # indices_or_default, mlx/ops.cpp:79-108
        shape = tuple(t.shape[:-2])
        n = 1
        for d in shape:
            n *= d
        return torch.arange(n, dtype=torch.int64, device=dev).reshape(shape)

    lhs = default_idx(x) if lhs_indices is None else lhs_indices.to(device=dev, dtype=torch.int64)
    rhs = default_idx(w) if rhs_indices is None else rhs_indices.to(device=dev, dtype=torch.int64)
    lhs, rhs = torch.broadcast_tensors(lhs, rhs)
    idx_shape = tuple(lhs.shape)
    lhs32 = lhs.contiguous().reshape(-1).to(torch.int32)  # bit pattern of uint32 indices
    rhs32 = rhs.contiguous().reshape(-1).to(torch.int32)

    x, scales, biases = x.to(out_type).contiguous(), scales.to(out_type).contiguous(), biases.to(out_type).contiguous()
    w = w.contiguous()
    M, K = x.shape[-2], x.shape[-1]
    x_batch = x.numel() // max(M * K, 1) if M * K else 0
    E = w.numel() // max(w.shape[-1] * w.shape[-2], 1) if w.shape[-1] * w.shape[-2] else 0
    N = w_outer
    n_idx = lhs32.numel()
    flags = (1 if (sorted_indices and rhs_indices is None) else 0) | (2 if (sorted_indices and lhs_indices is None) else 0)
    lib = _lib.load()
    with torch.cuda.device(dev):
        y = torch.empty(idx_shape + (M, N), dtype=out_type, device=dev)
        need = lib.b200q_gather_qmm_workspace_bytes(_DT[out_type], n_idx, x_batch, E, M, N, K, group_size, bits,
                                                    int(transpose))
        ws = _workspaces.get(dev, need, "gather")
        rc = lib.b200q_gather_qmm(_ptr(x), _ptr(w), _ptr(scales), _ptr(biases), _ptr(lhs32), _ptr(rhs32), n_idx,
                                  _ptr(y), _DT[out_type], x_batch, E, M, N, K, group_size, bits, int(transpose),
                                  flags, _ptr(ws), ws.numel(), _stream(x))
    _lib.check(rc)
    if _checked():
        read_workspace_status(ws, torch.cuda.current_stream(dev).cuda_stream, "gather")
    return y


def qmm_kernel_name(dtype: torch.dtype, M: int, N: int, K: int, group_size: int = 64, bits: int = 4,
                    transpose: bool = True, batch: int = 1) -> str:
    """Which kernel family quantized_matmul launches for this problem."""
    return _lib.load().b200q_qmm_kernel_name(_DT[dtype], batch, M, N, K, group_size, bits, int(transpose)).decode()


def gather_qmm_chain(x: torch.Tensor, w1: torch.Tensor, scales1: torch.Tensor, biases1: torch.Tensor,
                     w2: torch.Tensor, scales2: torch.Tensor, biases2: torch.Tensor,
                     rhs_indices: torch.Tensor, lhs_indices: Optional[torch.Tensor] = None,
                     group_size: Optional[int] = None, bits: Optional[int] = None) -> torch.Tensor:
    """gather_qmm(gather_qmm(x, w1, ...), w2, ...) over the same index pairs with one sort by expert
    (the reference composes the two calls, benchmarks/python/gather_qmm_bench.py:52-63).
    x [B, M, K1] bf16; w1 [E, N1, K1*bits/32]; w2 [E, N2, N1*bits/32]; out: idx_shape + [M, N2]."""
    group_size, bits = _mode_params("affine", group_size, bits, "gather_qmm_chain")
    _validate_quantized_input("gather_qmm_chain", w1, scales1, group_size, bits, biases1)
    _validate_quantized_input("gather_qmm_chain", w2, scales2, group_size, bits, biases2)
    if x.dtype != torch.bfloat16 or x.ndim < 2:
        raise ValueError("[gather_qmm_chain] x must be bfloat16 with at least two dimensions")
    dev = _require_cuda("gather_qmm_chain", x, w1, scales1, biases1, w2, scales2, biases2)
    M, K1 = x.shape[-2], x.shape[-1]
    N1, N2 = w1.shape[-2], w2.shape[-2]
    if w1.shape[-1] * 32 // bits != K1 or w2.shape[-1] * 32 // bits != N1 or w1.shape[:-2] != w2.shape[:-2]:
        raise ValueError("[gather_qmm_chain] w1 must map K1 -> N1 and w2 N1 -> N2 for the same experts")
    x_batch = x.numel() // max(M * K1, 1)
    E = w1.numel() // max(w1.shape[-1] * N1, 1)
    rhs = rhs_indices.to(device=dev, dtype=torch.int64)
    lhs = (torch.arange(x_batch, device=dev).reshape(tuple(x.shape[:-2])) if lhs_indices is None
           else lhs_indices.to(device=dev, dtype=torch.int64))
    lhs, rhs = torch.broadcast_tensors(lhs, rhs)
    idx_shape = tuple(lhs.shape)
    lhs32, rhs32 = lhs.contiguous().reshape(-1).to(torch.int32), rhs.contiguous().reshape(-1).to(torch.int32)
    n_idx = lhs32.numel()
    x = x.contiguous()
    c = lambda t: t.to(torch.bfloat16).contiguous()
    scales1, biases1, scales2, biases2 = c(scales1), c(biases1), c(scales2), c(biases2)
    w1, w2 = w1.contiguous(), w2.contiguous()
    lib = _lib.load()
    with torch.cuda.device(dev):
        y = torch.empty(idx_shape + (M, N2), dtype=torch.bfloat16, device=dev)
        need = lib.b200q_gather_qmm_chain_workspace_bytes(n_idx, E, M, N1, K1)
        ws = _workspaces.get(dev, need, "gather")
        rc = lib.b200q_gather_qmm_chain(_ptr(x), _ptr(w1), _ptr(scales1), _ptr(biases1), _ptr(w2), _ptr(scales2),
                                        _ptr(biases2), _ptr(lhs32), _ptr(rhs32), n_idx, _ptr(y), _lib.BF16, x_batch, E, M,
                                        N1, K1, N2, group_size, bits, _ptr(ws), ws.numel(), _stream(x))
    _lib.check(rc)
    return y


def gather_qmm_swiglu(x: torch.Tensor, gate, up, down, rhs_indices: torch.Tensor,
                      lhs_indices: Optional[torch.Tensor] = None, group_size: Optional[int] = None,
                      bits: Optional[int] = None) -> torch.Tensor:
    """Gated expert MLP: gather_qmm(silu(gather_qmm(x, *gate)) * gather_qmm(x, *up), *down) over the same
    index pairs with one sort (three mlx/ops.cpp:5553-5629 calls and the activation in the reference).
    gate, up, down: (w, scales, biases) triples; gate/up [E, H, K1*bits/32], down [E, N2, H*bits/32];
    x [B, M, K1] bf16; out: idx_shape + [M, N2]."""
    y = _front.swiglu(x, gate, up, down, rhs_indices, lhs_indices, group_size, bits)
    if y is not None:
        return y
    group_size, bits = _mode_params("affine", group_size, bits, "gather_qmm_swiglu")
    for t in (gate, up, down):
        _validate_quantized_input("gather_qmm_swiglu", t[0], t[1], group_size, bits, t[2])
    if x.dtype != torch.bfloat16 or x.ndim < 2:
        raise ValueError("[gather_qmm_swiglu] x must be bfloat16 with at least two dimensions")
    M, K1 = x.shape[-2], x.shape[-1]
    H, N2 = gate[0].shape[-2], down[0].shape[-2]
    if (gate[0].shape != up[0].shape or gate[0].shape[-1] * 32 // bits != K1 or down[0].shape[-1] * 32 // bits != H
            or gate[0].shape[:-2] != down[0].shape[:-2]):
        raise ValueError("[gather_qmm_swiglu] gate and up must map K1 -> H and down H -> N2 for the same experts")
    dev = _require_cuda("gather_qmm_swiglu", x, *gate, *up, *down)
    x_batch = x.numel() // max(M * K1, 1)
    E = gate[0].numel() // max(gate[0].shape[-1] * H, 1)
    rhs = rhs_indices.to(device=dev, dtype=torch.int64)
    lhs = (torch.arange(x_batch, device=dev).reshape(tuple(x.shape[:-2])) if lhs_indices is None
           else lhs_indices.to(device=dev, dtype=torch.int64))
    lhs, rhs = torch.broadcast_tensors(lhs, rhs)
    idx_shape = tuple(lhs.shape)
    lhs32, rhs32 = lhs.contiguous().reshape(-1).to(torch.int32), rhs.contiguous().reshape(-1).to(torch.int32)
    n_idx = lhs32.numel()
    x = x.contiguous()
    trip = lambda t: (t[0].contiguous(), t[1].to(torch.bfloat16).contiguous(), t[2].to(torch.bfloat16).contiguous())
    gate, up, down = trip(gate), trip(up), trip(down)
    lib = _lib.load()
    with torch.cuda.device(dev):
        y = torch.empty(idx_shape + (M, N2), dtype=torch.bfloat16, device=dev)
        need = lib.b200q_gather_qmm_swiglu_workspace_bytes(n_idx, E, M, H, K1)
        ws = _workspaces.get(dev, need, "gather")
        rc = lib.b200q_gather_qmm_swiglu(_ptr(x), *[_ptr(t) for t in gate], *[_ptr(t) for t in up], *[_ptr(t) for t in down],
                                         _ptr(lhs32), _ptr(rhs32), n_idx, _ptr(y), _lib.BF16, x_batch, E, M, H, K1, N2,
                                         group_size, bits, _ptr(ws), ws.numel(), _stream(x))
    _lib.check(rc)
    return y


# ------------------------------------------------------------------- microscaled products, products grouped by expert
def _group_sizes(tag, sizes, E, dev):
    if sizes.dtype.is_floating_point or sizes.dtype.is_complex or sizes.dtype == torch.bool:
        raise ValueError(f"[{tag}] Group sizes must be integral but are {sizes.dtype}.")
    if sizes.ndim != 1 or sizes.shape[0] != E:
        raise ValueError(f"[{tag}] One group size per expert is needed: sizes.shape() == {tuple(sizes.shape)} with {E} experts.")
    if sizes.device != dev:
        raise ValueError(f"[{tag}] all tensors must be on the same device")
    return (sizes if sizes.dtype in (torch.int32, torch.int64) else sizes.to(torch.int64)).contiguous()


def _qqmm(tag, x, w, scales, sizes, group_size, bits, mode, gx, gw):
    code, group = _fp4_params(tag, mode, group_size, bits)
    if x.dtype not in _DT:
        raise ValueError(f"[{tag}] Only real floating types are supported but x.dtype() == {x.dtype}.")
    _fp4_weights(tag, w, scales, group)
    if sizes is None and (w.ndim != 2 or x.ndim < 1):
        raise ValueError(f"[{tag}] x must have at least one dimension and w two, but they have {x.ndim} and {w.ndim}.")
    if sizes is not None and (w.ndim != 3 or x.ndim != 2):
        raise ValueError(f"[{tag}] x must have two dimensions and w three, but they have {x.ndim} and {w.ndim}.")
    E, N, K = (1 if w.ndim == 2 else w.shape[0]), w.shape[-2], w.shape[-1] * 8
    if x.shape[-1] != K:
        raise ValueError(f"[{tag}] Last dimension of first input with shape (..., {x.shape[-1]}) does not match the expanded "
                         f"quantized matrix ({K}, {N}) computed from shape {tuple(w.shape)}")
    dev = _require_cuda(tag, x, w, scales)
    if sizes is not None:
        sizes = _group_sizes(tag, sizes, E, dev)
    gx, gw = _fp4_global(tag, mode, gx, (1,), dev), _fp4_global(tag, mode, gw, (1, max(E, 1)), dev)
    x, w, scales = x.detach().contiguous(), _aligned(w), scales.contiguous()
    T = torch.Size(x.shape[:-1]).numel()
    lib = _lib.load()
    with torch.cuda.device(dev):
        y = torch.empty(tuple(x.shape[:-1]) + (N,), dtype=x.dtype, device=dev)
        ws = _workspaces.get(dev, lib.b200q_grouped_qqmm_workspace_bytes(T, E, N, K, code), "grouped")
        rc = lib.b200q_grouped_qqmm(_ptr(x), _ptr(w), _ptr(scales), _ptr(sizes), 0 if sizes is None else sizes.element_size(), _ptr(y),
                                    _DT[x.dtype], T, E, N, K, code, _ptr(gx), _ptr(gw), int(gw is not None and gw.numel() > 1),
                                    _ptr(ws), ws.numel(), _stream(x))
    _lib.check(rc)
    if _checked():
        read_workspace_status(ws, torch.cuda.current_stream(dev).cuda_stream, "grouped")
    return y


def qqmm(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, group_size: Optional[int] = None, bits: Optional[int] = None,
         mode: str = "nvfp4", global_scale_x: Optional[torch.Tensor] = None,
         global_scale_w: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [..., K] times the transpose of a quantized matrix (w uint32 [N, K/8], scales uint8 [N, K/g]), both in 4-bit
    floating point: x is quantized on the way, as quantize(x, mode=mode, global_scale=global_scale_x) does, and the codes of
    both are multiplied with their scales, by the 4-bit tensor cores or (up to 8 rows, where that is faster) as float16, which
    holds them exactly.  Sums in float32, the result [..., N] in x's type.
    global_scale_w: what `w` was quantized with.  (QQMatmul of the reference, mlx/backend/cuda/quantized/qqmm.cpp.)"""
    y = _front.qqmm(x, w, scales, None, group_size, bits, mode, global_scale_x, global_scale_w)
    return y if y is not None else _qqmm("qqmm", x, w, scales, None, group_size, bits, mode, global_scale_x, global_scale_w)


def grouped_qqmm(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, sizes: torch.Tensor, group_size: Optional[int] = None,
                 bits: Optional[int] = None, mode: str = "nvfp4", global_scale_x: Optional[torch.Tensor] = None,
                 global_scale_w: Optional[torch.Tensor] = None) -> torch.Tensor:
    """qqmm of rows sorted by expert: of x [T, K] the first sizes[0] rows multiply w[0] [N, K/8], the next sizes[1] rows w[1]
    and so on.  sizes: integers on the device, never read by the host; rows past their sum give zeros.  global_scale_w: one
    element, or one per expert."""
    y = _front.qqmm(x, w, scales, sizes, group_size, bits, mode, global_scale_x, global_scale_w)
    return y if y is not None else _qqmm("grouped_qqmm", x, w, scales, sizes, group_size, bits, mode, global_scale_x, global_scale_w)


def qqmm_kernel_name(M: int, N: int, K: int, mode: str = "nvfp4", experts: Optional[int] = None) -> str:
    """Which kernel qqmm (experts: grouped_qqmm) launches for M rows of x and operands on 16-byte boundaries."""
    code, _ = _fp4_params("qqmm_kernel_name", mode, None, None)
    return _lib.load().b200q_grouped_qqmm_kernel_name(M, 1 if experts is None else experts, N, K, code, int(experts is not None)).decode()


def _grouped_operands(tag, x, w, sizes, transpose):
    if x.dtype not in (torch.float16, torch.bfloat16) or w.dtype != x.dtype:
        raise ValueError(f"[{tag}] x and w must both be float16 or bfloat16 but are {x.dtype} and {w.dtype}.")
    if x.ndim != 2 or w.ndim != 3:
        raise ValueError(f"[{tag}] x must have two dimensions and w three, but they have {x.ndim} and {w.ndim}.")
    E, N, K = w.shape[0], w.shape[1 if transpose else 2], w.shape[2 if transpose else 1]
    if x.shape[1] != K:
        raise ValueError(f"[{tag}] Last dimension of first input with shape {tuple(x.shape)} does not match the matrices "
                         f"({K}, {N}) of w with shape {tuple(w.shape)} and transpose={transpose}")
    dev = _require_cuda(tag, x, w)
    return dev, _group_sizes(tag, sizes, E, dev), E, N, K


def grouped_mm(x: torch.Tensor, w: torch.Tensor, sizes: torch.Tensor, transpose: bool = True) -> torch.Tensor:
    """Rows sorted by expert through 16-bit weights: of x [T, K] the first sizes[0] rows multiply the transpose of w[0]
    (w [E, N, K]; transpose=False: w[0] of w [E, K, N]), the next sizes[1] rows that of w[1] and so on; out [T, N].  sizes:
    integers on the device, never read by the host; rows past their sum give zeros.  bfloat16 and float16, sums in float32.
    grad.grouped_mm is the same with gradients."""
    y = _front.grouped_mm(x, w, sizes, transpose)
    if y is not None:
        return y
    transpose = bool(transpose)
    dev, sizes, E, N, K = _grouped_operands("grouped_mm", x, w, sizes, transpose)
    x, w = _aligned(x.detach()), _aligned(w.detach())
    T = x.shape[0]
    lib = _lib.load()
    with torch.cuda.device(dev):
        y = torch.empty((T, N), dtype=x.dtype, device=dev)
        ws = _workspaces.get(dev, lib.b200q_grouped_mm_workspace_bytes(T, E, N, K, int(transpose)), "grouped")
        rc = lib.b200q_grouped_mm(_ptr(x), _ptr(w), _ptr(sizes), sizes.element_size(), _ptr(y), _DT[x.dtype], T, E, N, K,
                                  int(transpose), _ptr(ws), ws.numel(), _stream(x))
    _lib.check(rc)
    if _checked():
        read_workspace_status(ws, torch.cuda.current_stream(dev).cuda_stream, "grouped")
    return y


def grouped_mm_dw(dy: torch.Tensor, x: torch.Tensor, sizes: torch.Tensor, transpose: bool = True) -> torch.Tensor:
    """The gradient of grouped_mm with respect to w, in w's layout: for every expert the sum over its rows of dy[t]^T x[t]
    ([E, N, K]; transpose=False: x[t]^T dy[t], [E, K, N]).  An expert without rows gets zeros."""
    dw = _front.grouped_mm_dw(dy, x, sizes, transpose)
    if dw is not None:
        return dw
    if x.dtype not in (torch.float16, torch.bfloat16) or dy.dtype != x.dtype:
        raise ValueError(f"[grouped_mm_dw] dy and x must both be float16 or bfloat16 but are {dy.dtype} and {x.dtype}.")
    if x.ndim != 2 or dy.ndim != 2 or x.shape[0] != dy.shape[0]:
        raise ValueError(f"[grouped_mm_dw] dy and x must be matrices with as many rows, but have shapes {tuple(dy.shape)} and {tuple(x.shape)}.")
    dev = _require_cuda("grouped_mm_dw", dy, x)
    if sizes.ndim != 1:
        raise ValueError(f"[grouped_mm_dw] sizes must have one dimension but has shape {tuple(sizes.shape)}.")
    E, T = sizes.shape[0], x.shape[0]
    sizes = _group_sizes("grouped_mm_dw", sizes, E, dev)
    dy, x = _aligned(dy.detach()), _aligned(x.detach())
    a, b = (dy, x) if transpose else (x, dy)
    N, K = a.shape[1], b.shape[1]
    lib = _lib.load()
    with torch.cuda.device(dev):
        dw = torch.empty((E, N, K), dtype=x.dtype, device=dev)
        ws = _workspaces.get(dev, lib.b200q_grouped_mm_dw_workspace_bytes(T, N, K), "grouped")
        rc = lib.b200q_grouped_mm_dw(_ptr(a), _ptr(b), _ptr(sizes), sizes.element_size(), _ptr(dw), _DT[x.dtype], T, E, N, K, _ptr(ws),
                                     ws.numel(), _stream(x))
    _lib.check(rc)
    if _checked():
        read_workspace_status(ws, torch.cuda.current_stream(dev).cuda_stream, "grouped")
    return dw


# ------------------------------------------------------------------- routing, rows between tokens and experts, adapters
class Routing(NamedTuple):
    """What route_experts decides; pair p = token * top + choice.  weights float32 and experts int32 [..., top] (-1: no expert),
    sizes int32 [E]: pairs per expert, as the grouped products take them; places int32 [..., top]: where a pair stands in the experts'
    order (-1: nowhere); order int32 [tokens * top]: the pair at every place, behind the last one -1 - p of the pairs without an expert."""
    weights: torch.Tensor
    experts: torch.Tensor
    sizes: torch.Tensor
    places: torch.Tensor
    order: torch.Tensor


class RowGroups(NamedTuple):
    """Rows sorted by group, as group_rows leaves them: sizes int32 [n], starts int32 [n + 1], order int32 [rows] (rows without a group last,
    as -1 - row) and the table of tiles that add_adapters reads."""
    sizes: torch.Tensor
    starts: torch.Tensor
    order: torch.Tensor
    tiles: torch.Tensor


_SCORING = {"softmax": _lib.SOFTMAX, "sigmoid": _lib.SIGMOID}


def _scratch(nbytes: int, dev: torch.device) -> torch.Tensor:
    """Plain scratch of one call: the allocator keeps it apart from every other call's, captured ones included."""
    return torch.empty(max(nbytes, 1), dtype=torch.uint8, device=dev)


def _route_args(tag, logits, top, scoring, groups, top_groups, group_best):
    if logits.dtype not in _DT:
        raise ValueError(f"[{tag}] Only real floating types are supported but logits.dtype() == {logits.dtype}.")
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise ValueError(f"[{tag}] logits must have a last dimension of experts but have shape {tuple(logits.shape)}.")
    if scoring not in _SCORING:
        raise ValueError(f"[{tag}] scoring is 'softmax' or 'sigmoid', not '{scoring}'.")
    E = logits.shape[-1]
    top, groups = operator.index(top), operator.index(groups)
    top_groups = groups if top_groups is None else operator.index(top_groups)
    if groups < 1 or E % groups != 0 or not 1 <= top_groups <= groups:
        raise ValueError(f"[{tag}] cannot take {top_groups} of {groups} groups of {E} experts.")
    if not 1 <= top <= E // groups * top_groups:
        raise ValueError(f"[{tag}] cannot take {top} experts out of {top_groups} groups of {E // groups}.")
    if group_best not in (1, 2):
        raise ValueError(f"[{tag}] a group is ranked by its best 1 or 2 experts, not {group_best}.")
    return E, top, groups, top_groups


def route_experts(logits: torch.Tensor, top: int, scoring: str = "softmax", bias: Optional[torch.Tensor] = None, groups: int = 1,
                  top_groups: Optional[int] = None, group_best: int = 1, renormalize: bool = False, scale: float = 1.0) -> Routing:
    """Chooses `top` experts for every token from its router logits [..., E], and sorts the pairs by expert.

    Scores are the logits' softmax or sigmoid.  Experts are taken by falling logit, or by falling score + bias where there is a bias
    (float [E], which balances the experts' load and does not enter the weights), ties to the lowest index; the order is that of 64-bit
    arithmetic.  groups > 1: of the groups of E / groups consecutive experts only the top_groups best stay, ranked by the sum of their
    group_best (1 or 2) best.  Weights are the scores, renormalized to a sum of 1 over the experts taken if asked for, times scale.
    An expert with a logit (or bias) of -inf is off and never taken: a token with too few experts on has pairs without one (expert
    -1, weight 0, place -1), a token of padding none at all.  grad.route_experts is the same with the weights' gradient."""
    r = _front.route(logits, top, scoring, bias, groups, top_groups, group_best, renormalize, scale)
    if r is not None:
        return r
    tag = "route_experts"
    E, top, groups, top_groups = _route_args(tag, logits, top, scoring, groups, top_groups, group_best)
    if bias is not None and (not bias.dtype.is_floating_point or tuple(bias.shape) != (E,)):
        raise ValueError(f"[{tag}] the bias is a floating-point tensor of {E} elements.")
    dev = _require_cuda(tag, logits) if bias is None else _require_cuda(tag, logits, bias)
    logits = logits.detach().contiguous()
    bias = None if bias is None else bias.detach().to(torch.float32).contiguous()
    lead, T = tuple(logits.shape[:-1]), torch.Size(logits.shape[:-1]).numel()
    lib = _lib.load()
    with torch.cuda.device(dev):
        new = lambda *shape: torch.empty(shape, dtype=torch.int32, device=dev)
        weights = torch.empty(lead + (top,), dtype=torch.float32, device=dev)
        experts, sizes, places, order = new(*lead, top), new(E), new(*lead, top), new(T * top)
        need = lib.b200q_route_workspace_bytes(T, E, top)
        ws = _scratch(need, dev) if need else None
        rc = lib.b200q_route(_ptr(logits), _DT[logits.dtype], T, E, top, _SCORING[scoring], _ptr(bias), groups, top_groups, group_best,
                             int(bool(renormalize)), float(scale), _ptr(weights), _ptr(experts), _ptr(sizes), _ptr(places), _ptr(order),
                             _ptr(ws), need, _stream(logits))
    _lib.check(rc)
    return Routing(weights, experts, sizes, places, order)


def route_dlogits(dw: torch.Tensor, logits: torch.Tensor, experts: torch.Tensor, scoring: str = "softmax", renormalize: bool = False,
                  scale: float = 1.0) -> torch.Tensor:
    """The gradient with respect to the logits, in their type, of a loss whose gradient with respect to route_experts' weights is dw."""
    tag = "route_dlogits"
    if logits.dtype not in _DT or scoring not in _SCORING:
        raise ValueError(f"[{tag}] unsupported logits.dtype() == {logits.dtype} or scoring '{scoring}'.")
    if experts.dtype != torch.int32 or experts.ndim != logits.ndim or experts.shape[:-1] != logits.shape[:-1] or dw.shape != experts.shape:
        raise ValueError(f"[{tag}] dw and experts (int32) must have one entry per pair, but have shapes {tuple(dw.shape)} and "
                         f"{tuple(experts.shape)} with logits {tuple(logits.shape)}.")
    dev = _require_cuda(tag, logits, dw, experts)
    logits, dw, experts = logits.detach().contiguous(), dw.detach().to(torch.float32).contiguous(), experts.contiguous()
    with torch.cuda.device(dev):
        dl = torch.empty_like(logits)
        rc = _lib.load().b200q_route_dlogits(_ptr(dw), _ptr(logits), _DT[logits.dtype], _ptr(experts), torch.Size(logits.shape[:-1]).numel(),
                                             logits.shape[-1], experts.shape[-1], _SCORING[scoring], int(bool(renormalize)), float(scale),
                                             _ptr(dl), _stream(logits))
    _lib.check(rc)
    return dl


def _plan(tag, places, order):
    if places.dtype != torch.int32 or order.dtype != torch.int32 or places.ndim < 1 or tuple(order.shape) != (places.numel(),):
        raise ValueError(f"[{tag}] places and order are int32, with one entry per pair each, but have shapes {tuple(places.shape)} and {tuple(order.shape)}.")
    return places.contiguous(), order.contiguous()


def dispatch_rows(x: torch.Tensor, routing: Routing) -> torch.Tensor:
    """The tokens' rows x [..., D] in the experts' order, [tokens * top, D]: the rows that grouped_mm and grouped_qqmm take with routing.sizes.
    Rows behind the last pair with an expert are zeros."""
    xs = _front.dispatch(x, routing)
    if xs is not None:
        return xs
    tag = "dispatch_rows"
    if x.dtype not in _DT:
        raise ValueError(f"[{tag}] Only real floating types are supported but x.dtype() == {x.dtype}.")
    places, order = _plan(tag, routing.places, routing.order)
    if x.ndim < 1 or x.shape[:-1] != places.shape[:-1]:
        raise ValueError(f"[{tag}] x {tuple(x.shape)} does not have a row for every token of the routing {tuple(places.shape)}.")
    dev = _require_cuda(tag, x, places, order)
    x = x.detach().contiguous()
    with torch.cuda.device(dev):
        xs = torch.empty((order.shape[0], x.shape[-1]), dtype=x.dtype, device=dev)
        rc = _lib.load().b200q_dispatch_rows(_ptr(x), _DT[x.dtype], torch.Size(x.shape[:-1]).numel(), places.shape[-1], x.shape[-1], _ptr(places),
                                             _ptr(order), _ptr(xs), _stream(x))
    _lib.check(rc)
    return xs


def _combine(tag, y, places, order, weights):
    if y.dtype not in _DT:
        raise ValueError(f"[{tag}] Only real floating types are supported but y.dtype() == {y.dtype}.")
    places, order = _plan(tag, places, order)
    if y.ndim != 2 or y.shape[0] != order.shape[0]:
        raise ValueError(f"[{tag}] y {tuple(y.shape)} does not have a row for every pair of the routing {tuple(places.shape)}.")
    if weights is not None and (not weights.dtype.is_floating_point or weights.shape != places.shape):
        raise ValueError(f"[{tag}] the weights must be one floating-point number per pair but have shape {tuple(weights.shape)}.")
    dev = _require_cuda(tag, y, places, order) if weights is None else _require_cuda(tag, y, places, order, weights)
    return dev, y.detach().contiguous(), places, order, None if weights is None else weights.detach().to(torch.float32).contiguous()


def combine_rows(y: torch.Tensor, routing: Routing, weighted: bool = True) -> torch.Tensor:
    """The experts' results y [tokens * top, D], in their order, back to the tokens: out[t] = sum of weights[t, j] y[places[t, j]], [..., D];
    weighted=False: the plain sum, which is the gradient of dispatch_rows.  Sums in float32, in the order of the choices."""
    out = _front.combine(y, routing, weighted)
    if out is not None:
        return out
    dev, y, places, _, weights = _combine("combine_rows", y, routing.places, routing.order, routing.weights if weighted else None)
    with torch.cuda.device(dev):
        out = torch.empty(tuple(places.shape[:-1]) + (y.shape[1],), dtype=y.dtype, device=dev)
        rc = _lib.load().b200q_combine_rows(_ptr(y), _DT[y.dtype], torch.Size(places.shape[:-1]).numel(), places.shape[-1], y.shape[1], _ptr(places),
                                            _ptr(weights), _ptr(out), _stream(y))
    _lib.check(rc)
    return out


def combine_rows_grad(dy: torch.Tensor, y: torch.Tensor, routing: Routing, for_y: bool = True, for_weights: bool = True):
    """-> gradients of combine_rows with respect to y and to the weights (None where not asked for)."""
    tag = "combine_rows_grad"
    if dy.dtype != y.dtype or y.ndim != 2 or tuple(dy.shape) != tuple(routing.places.shape[:-1]) + (y.shape[1],):
        raise ValueError(f"[{tag}] dy {tuple(dy.shape)} ({dy.dtype}) does not match the result of combine_rows.")
    dev, y, places, order, weights = _combine(tag, y, routing.places, routing.order, routing.weights)
    _require_cuda(tag, y, dy)
    dy = dy.detach().contiguous()
    with torch.cuda.device(dev):
        dys = torch.empty_like(y) if for_y else None
        dw = torch.empty_like(weights) if for_weights else None
        rc = _lib.load().b200q_combine_rows_grad(_ptr(dy), _ptr(y), _DT[y.dtype], torch.Size(places.shape[:-1]).numel(), places.shape[-1], y.shape[1],
                                                 _ptr(places), _ptr(order), _ptr(weights), _ptr(dys), _ptr(dw), _stream(y))
    _lib.check(rc)
    return dys, dw


def group_rows(ids: torch.Tensor, n: int) -> RowGroups:
    """Rows sorted by group: ids, any integers, name every row's group (adapter); outside [0, n): none.  Computed once for a batch
    and used beside all its projections."""
    g = _front.group_rows(ids, n)
    if g is not None:
        return g
    tag = "group_rows"
    if ids.dtype.is_floating_point or ids.dtype.is_complex or ids.dtype == torch.bool:
        raise ValueError(f"[{tag}] ids must be integral but are {ids.dtype}.")
    n = operator.index(n)
    if n < 0:
        raise ValueError(f"[{tag}] there cannot be {n} groups.")
    dev = _require_cuda(tag, ids)
    ids = (ids if ids.dtype in (torch.int32, torch.int64) else ids.to(torch.int64)).contiguous()
    T = ids.numel()
    lib = _lib.load()
    with torch.cuda.device(dev):
        new = lambda *shape: torch.empty(shape, dtype=torch.int32, device=dev)
        sizes, starts, order, tiles = new(n), new(n + 1), new(T), new(lib.b200q_group_rows_tiles(T, n), 4)
        need = lib.b200q_group_rows_workspace_bytes(T, n)
        ws = _scratch(need, dev) if need else None
        rc = lib.b200q_group_rows(_ptr(ids), ids.element_size(), T, n, _ptr(sizes), _ptr(starts), _ptr(order), _ptr(tiles), _ptr(ws), need, _stream(ids))
    _lib.check(rc)
    return RowGroups(sizes, starts, order, tiles)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    end = lambda t: t.data_ptr() + t.numel() * t.element_size()
    return a.data_ptr() < end(b) and b.data_ptr() < end(a)


def _adapter_args(tag, y, x, a, b, groups, scales):
    if x.dtype not in (torch.float16, torch.bfloat16) or any(t.dtype != x.dtype for t in (y, a, b)):
        raise ValueError(f"[{tag}] y, x, a and b must all be float16 or bfloat16 but are {y.dtype}, {x.dtype}, {a.dtype} and {b.dtype}.")
    if a.ndim != 3 or b.ndim != 3 or x.ndim < 1 or y.ndim < 1:
        raise ValueError(f"[{tag}] a and b must have three dimensions and x and y one at least, but they have {a.ndim}, {b.ndim}, {x.ndim} and {y.ndim}.")
    L, r, K, N = *a.shape, b.shape[1]
    if b.shape[0] != L or b.shape[2] != r or x.shape[-1] != K or y.shape[-1] != N or x.shape[:-1] != y.shape[:-1]:
        raise ValueError(f"[{tag}] The shapes of y {tuple(y.shape)}, x {tuple(x.shape)}, a {tuple(a.shape)} and b {tuple(b.shape)} do not match: "
                         "[..., N], [..., K], [adapters, rank, K] and [adapters, N, rank] are needed")
    T = torch.Size(x.shape[:-1]).numel()
    if any(t.dtype != torch.int32 for t in groups) or tuple(groups.sizes.shape) != (L,) or tuple(groups.starts.shape) != (L + 1,) or \
            tuple(groups.order.shape) != (T,) or tuple(groups.tiles.shape) != (_lib.load().b200q_group_rows_tiles(T, L), 4):
        raise ValueError(f"[{tag}] the groups are not those of group_rows for {T} rows and {L} adapters.")
    if scales is not None and (not scales.dtype.is_floating_point or tuple(scales.shape) != (L,)):
        raise ValueError(f"[{tag}] the scales are one floating-point number per adapter.")
    dev = _require_cuda(tag, y, x, a, b, *groups, *(() if scales is None else (scales,)))
    scales = None if scales is None else scales.detach().to(torch.float32).contiguous()
    return dev, T, L, N, K, r, RowGroups(*(t.contiguous() for t in groups)), scales


def _inner(T: int, rank: int) -> Tuple[int, int, int]:
    return T, 3, (rank + 15) // 16 * 16


def add_adapters(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, groups: RowGroups, scales: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Low-rank adapters of many requests at once beside a shared projection: y [..., N], what the projection (quantized_matmul, qqmm, ...)
    made of x [..., K], plus scales[l] b[l] (a[l] x[t]) for every row t with an adapter l.  a [adapters, rank, K], b [adapters, N, rank],
    scales [adapters] (None: 1); groups: group_rows of the rows' adapters.  bfloat16 and float16; sums and inner products in
    float32, the result rounded once.  out: where the sum goes, y itself for a sum in place.  grad.add_adapters is the same with gradients."""
    return _add_adapters(y, x, a, b, groups, scales, out)[0]


def _add_adapters(y, x, a, b, groups, scales=None, out=None):
    """-> add_adapters' result and the inner products, three bfloat16 parts per value [rows, 3, rank in whole 16s] in the order of the groups."""
    r = _front.add_adapters(y, x, a, b, groups, scales, out)
    if r is not None:
        return r
    tag = "add_adapters"
    dev, T, L, N, K, rank, groups, scales = _adapter_args(tag, y, x, a, b, groups, scales)
    if out is not None:
        if out.dtype != y.dtype or out.shape != y.shape or out.device != y.device or not out.is_contiguous():
            raise ValueError(f"[{tag}] out must be a contiguous tensor like y.")
        if out.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"[{tag}] out must not be part of a graph.")
        if any(_overlap(out, t) for t in (x, a, b)) or (_overlap(out, y) and (out.data_ptr() != y.data_ptr() or not y.is_contiguous())):
            raise ValueError(f"[{tag}] out must be y itself or not overlap the operands.")
    into = out
    y, x, a, b = (t.detach().contiguous() for t in (y, x, a, b))
    with torch.cuda.device(dev):
        out = torch.empty_like(y) if out is None else out
        h = torch.empty(_inner(T, rank), dtype=torch.bfloat16, device=dev)
        rc = _lib.load().b200q_add_adapters(_ptr(y), _ptr(x), _ptr(a), _ptr(b), _DT[x.dtype], T, L, N, K, rank, _ptr(groups.order), _ptr(groups.tiles),
                                            _ptr(scales), _ptr(h), _ptr(out), _stream(x))
    _lib.check(rc)
    if into is not None:
        torch.autograd.graph.increment_version(into)   # whoever has kept it for a gradient hears of it
    return out, h


def add_adapters_grad(dy: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, groups: RowGroups, h: Optional[torch.Tensor] = None,
                      scales: Optional[torch.Tensor] = None, for_x: bool = True, for_a: bool = True, for_b: bool = True):
    """-> gradients of add_adapters with respect to x, a and b (None where not asked for; that of y is dy).  h: the inner products, as the
    forward pass leaves them for b's gradient; None: computed again where that is asked for."""
    tag = "add_adapters_grad"
    dev, T, L, N, K, rank, groups, scales = _adapter_args(tag, dy, x, a, b, groups, scales)
    if h is None and for_b:
        h = _add_adapters(dy, x, a, b, groups, scales)[1]
    if h is not None and (h.dtype != torch.bfloat16 or tuple(h.shape) != _inner(T, rank)):
        raise ValueError(f"[{tag}] h must be bfloat16 {_inner(T, rank)}.")
    _require_cuda(tag, x, *(() if h is None else (h,)))
    dy, x, a, b = (t.detach().contiguous() for t in (dy, x, a, b))
    h = None if h is None else _aligned(h)
    with torch.cuda.device(dev):
        dx, da, db = (torch.empty_like(t) if wanted else None for t, wanted in ((x, for_x), (a, for_a), (b, for_b)))
        g = torch.empty(_inner(T, rank), dtype=torch.bfloat16, device=dev) if for_x or for_a else None
        rc = _lib.load().b200q_add_adapters_grad(_ptr(dy), _ptr(x), _ptr(a), _ptr(b), _DT[x.dtype], T, L, N, K, rank, _ptr(groups.order),
                                                 _ptr(groups.starts), _ptr(groups.tiles), _ptr(scales), _ptr(h), _ptr(g), _ptr(dx), _ptr(da), _ptr(db),
                                                 _stream(x))
    _lib.check(rc)
    return dx, da, db
