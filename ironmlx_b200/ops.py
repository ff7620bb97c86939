"""Host-side mirror of the reference's quantized-op wrappers
(mlx/src/ops.rs:630-727): same names, argument order and meaning, errors
raised as `IronMLXError` the way the reference returns `Error::Mlx`.

Tensors are torch CUDA tensors used as plain device buffers; every op is one
call into the C ABI on the given stream.  There is no fallback path.

Packed weights are int32 (the bits of MLX's uint32 words), affine
scales/biases bf16, mxfp8/nvfp4 scales uint8.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import IronMLXError, QTensor, check, lib, resolve_format

_OUT_DTYPES = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def stream_ptr(stream=None) -> int:
    """cudaStream_t of a torch stream (default: the current stream)."""
    s = torch.cuda.current_stream() if stream is None else stream
    return s.cuda_stream


def _require_cuda(*tensors):
    for t in tensors:
        if t is not None and (not t.is_cuda or not t.is_contiguous()):
            raise IronMLXError(_lib.ERR_INVALID, "tensors must be contiguous CUDA tensors")


def qtensor(w, scales, biases=None, global_scale: Optional[float] = None) -> QTensor:
    return QTensor(_ptr(w), _ptr(scales), _ptr(biases), 1.0 if global_scale is None else float(global_scale))


def _packed_cols(in_dim: int, bits: int) -> int:
    return in_dim * bits // 32


def dequantize(w, scales, biases=None, group_size=None, bits=None, mode: str = "affine",
               stream=None, dtype=torch.bfloat16, global_scale=None) -> torch.Tensor:
    """`ops::dequantize` (mlx/src/ops.rs:653-686): packed [.., out, in*bits/32] -> [.., out, in]."""
    g, b, m = resolve_format(group_size, bits, mode)
    _require_cuda(w, scales, biases)
    in_dim = w.shape[-1] * 32 // b
    rows = w.numel() // w.shape[-1]
    out = torch.empty(*w.shape[:-1], in_dim, dtype=dtype, device=w.device)
    qt = qtensor(w, scales, biases, global_scale)
    check(lib().imx_dequantize(C.byref(qt), rows, in_dim, g, b, m, _OUT_DTYPES[dtype], out.data_ptr(),
                               stream_ptr(stream)))
    return out


def quantized_matmul(x, w, scales, biases=None, transpose: bool = True, group_size=None, bits=None,
                     mode: str = "affine", stream=None, global_scale=None) -> torch.Tensor:
    """`ops::quantized_matmul` (mlx/src/ops.rs:695-727): `x @ dequantize(w)^T`
    (transpose=True, how every layer of the path calls it) or `x @ dequantize(w)`."""
    g, b, m = resolve_format(group_size, bits, mode)
    _require_cuda(x, w, scales, biases)
    if x.dtype != torch.bfloat16:
        raise IronMLXError(_lib.ERR_INVALID, "quantized_matmul: x must be bfloat16")
    if w.dim() != 2:
        raise IronMLXError(_lib.ERR_INVALID, "quantized_matmul: w must be 2-D [out, in*bits/32]")
    n_out, in_dim = w.shape[0], w.shape[1] * 32 // b
    inner = in_dim if transpose else n_out
    if x.shape[-1] != inner:
        raise IronMLXError(_lib.ERR_INVALID,
                           f"quantized_matmul: last dimension of x ({x.shape[-1]}) does not match {inner}")
    m_rows = x.numel() // inner
    x = x.contiguous()
    y = torch.empty(*x.shape[:-1], n_out if transpose else in_dim, dtype=torch.bfloat16, device=x.device)
    qt = qtensor(w, scales, biases, global_scale)
    if transpose:
        # the layers' form: on the expert kernels where they take the shape (scratch cached per device and size)
        nb = C.c_size_t(0)
        check(lib().imx_quantized_matmul_scratch_bytes(m_rows, n_out, in_dim, g, b, m, C.byref(nb)))
        ws = scratch(x.device, nb.value)
        check(lib().imx_quantized_matmul_ws(x.data_ptr(), m_rows, C.byref(qt), n_out, in_dim, g, b, m, y.data_ptr(),
                                            ws.data_ptr(), ws.numel(), stream_ptr(stream)))
        return y
    check(lib().imx_quantized_matmul(x.data_ptr(), m_rows, C.byref(qt), n_out, in_dim, 0,
                                     g, b, m, y.data_ptr(), stream_ptr(stream)))
    return y


_SCRATCH = {}


def scratch(device, nbytes: int) -> torch.Tensor:
    """A zero-filled device buffer of at least nbytes, kept per device (the layer calls' scratch; one stream of
    calls at a time per device)."""
    key = (device.type, device.index)
    buf = _SCRATCH.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _SCRATCH[key] = buf
    return buf


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Dense `x @ W^T (+ b)` (mlx/src/nn/linear.rs:170-177), bf16 in and out, fp32 accumulation."""
    _require_cuda(x, weight, bias)
    if x.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise IronMLXError(_lib.ERR_INVALID, "linear: x [.., in] and weight [out, in] must be bfloat16")
    x = x.contiguous()
    n_out, in_dim = weight.shape
    y = torch.empty(*x.shape[:-1], n_out, dtype=torch.bfloat16, device=x.device)
    check(lib().imx_linear(x.data_ptr(), x.numel() // in_dim, in_dim, weight.data_ptr(), n_out, _ptr(bias), y.data_ptr(),
                           stream_ptr(stream)))
    return y


def expert_forward(x: torch.Tensor, gate_up_w, gate_up_s, gate_up_b, down_w, down_s, down_b, group_size=None, bits=None,
                   mode: str = "affine", stream=None, gate_up_scale=None, down_scale=None) -> torch.Tensor:
    """`down(silu(gate(x)) * up(x))` for one expert over all rows of x (mlx/src/nn/moe.rs:26-32,
    mlx/src/nn/mlp.rs:27-33).  gate_up_*: [2I, .] with the gate rows first; down_*: [H, .]."""
    g, b, m = resolve_format(group_size, bits, mode)
    _require_cuda(x, gate_up_w, gate_up_s, gate_up_b, down_w, down_s, down_b)
    hidden = x.shape[-1]
    inter = gate_up_w.shape[-2] // 2
    if x.dtype != torch.bfloat16 or down_w.shape[-2] != hidden:
        raise IronMLXError(_lib.ERR_INVALID, "expert_forward: x must be bfloat16 [.., hidden] matching down [hidden, .]")
    x = x.contiguous()
    rows = x.numel() // hidden
    y = torch.empty_like(x)
    cfg = _lib.MoEConfig(hidden, 1, 1, inter, 0, 1, m, b, g, 0)
    nb = C.c_size_t(0)
    check(lib().imx_expert_scratch_bytes(C.byref(cfg), rows, C.byref(nb)))
    ws = scratch(x.device, nb.value)
    gu, dn = qtensor(gate_up_w, gate_up_s, gate_up_b, gate_up_scale), qtensor(down_w, down_s, down_b, down_scale)
    check(lib().imx_expert_forward(C.byref(cfg), C.byref(gu), C.byref(dn), x.data_ptr(), rows, y.data_ptr(), ws.data_ptr(),
                                   ws.numel(), stream_ptr(stream)))
    return y


def quantize(w, group_size=None, bits=None, mode: str = "affine", stream=None, global_scale=None):
    """Quantize float weights [.., out, in] -> (packed int32, scales, biases-or-None).
    For nvfp4 the fp32 tensor scale is taken from `global_scale`, or derived
    from the tensor's absolute maximum, and returned as a fourth element."""
    g, b, m = resolve_format(group_size, bits, mode)
    w = w.to(torch.float32).contiguous()
    _require_cuda(w)
    in_dim = w.shape[-1]
    rows = w.numel() // in_dim
    if in_dim % g or (in_dim * b) % 32:
        raise IronMLXError(_lib.ERR_INVALID, f"quantize: last dimension {in_dim} does not fit group {g} / {b} bits")
    packed = torch.empty(*w.shape[:-1], _packed_cols(in_dim, b), dtype=torch.int32, device=w.device)
    sdtype = torch.bfloat16 if mode == "affine" else torch.uint8
    scales = torch.empty(*w.shape[:-1], in_dim // g, dtype=sdtype, device=w.device)
    biases = torch.empty_like(scales) if mode == "affine" else None
    gs = 1.0
    if mode == "nvfp4":
        gs = float(global_scale) if global_scale is not None else max(float(w.abs().max()), 1e-30) / (6.0 * 448.0)
    check(lib().imx_quantize(w.data_ptr(), rows, in_dim, g, b, m, gs, packed.data_ptr(), scales.data_ptr(),
                             _ptr(biases), stream_ptr(stream)))
    if mode == "nvfp4":
        return packed, scales, None, gs
    return packed, scales, biases


def gather_qmm(x, w, scales, biases, lhs_indices, rhs_indices, group_size=None, bits=None,
               mode: str = "affine", stream=None, global_scale=None) -> torch.Tensor:
    """y[j] = x[lhs_indices[j]] @ dequantize(w[rhs_indices[j]])^T: the per-row
    form of the reference's take_axis + quantized_matmul per expert
    (mlx/src/nn/moe.rs:124-130).  w: [E, out, in*bits/32]."""
    g, b, m = resolve_format(group_size, bits, mode)
    _require_cuda(x, w, scales, biases, lhs_indices, rhs_indices)
    if x.dtype != torch.bfloat16 or w.dim() != 3:
        raise IronMLXError(_lib.ERR_INVALID, "gather_qmm: x must be bfloat16 and w 3-D [E, out, in*bits/32]")
    n_out, in_dim = w.shape[1], w.shape[2] * 32 // b
    n_rows = rhs_indices.numel()
    y = torch.empty(n_rows, n_out, dtype=torch.bfloat16, device=x.device)
    qt = qtensor(w, scales, biases, global_scale)
    lhs = None if lhs_indices is None else lhs_indices.to(torch.int32)
    check(lib().imx_gather_qmm(x.data_ptr(), _ptr(lhs), C.byref(qt), rhs_indices.to(torch.int32).data_ptr(),
                               n_rows, n_out, in_dim, g, b, m, y.data_ptr(), stream_ptr(stream)))
    return y


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float, stream=None) -> torch.Tensor:
    """`fast::rms_norm` (mlx/src/fast.rs:37-49): x * rsqrt(mean(x^2) + eps) * weight over the last
    axis; bf16 in and out."""
    _require_cuda(x, weight)
    if x.dtype != torch.bfloat16 or (weight is not None and weight.dtype != torch.bfloat16):
        raise IronMLXError(_lib.ERR_INVALID, "rms_norm: x and weight must be bfloat16")
    h = x.shape[-1]
    if weight is not None and weight.numel() != h:
        raise IronMLXError(_lib.ERR_INVALID, f"rms_norm: weight has {weight.numel()} elements, rows have {h}")
    x = x.contiguous()
    y = torch.empty_like(x)
    check(lib().imx_rms_norm(x.data_ptr(), x.numel() // h, h, None if weight is None else weight.data_ptr(),
                             float(eps), y.data_ptr(), stream_ptr(stream)))
    return y


class Mxfp8Rows(NamedTuple):
    """Activation rows in mxfp8, laid out as `quantize(..., mode="mxfp8")` lays out weights: e4m3 codes as int32 words
    [.., in/4] and ue8m0 scales uint8 [.., in/32]."""
    packed: torch.Tensor
    scales: torch.Tensor


def _on(x: torch.Tensor, stream):
    """The device of x, and the given stream, made current: what is allocated within belongs to that stream, and the
    launches go to that device."""
    if stream is None:
        return torch.cuda.device(x.device)
    if stream.device_index != x.get_device():
        raise IronMLXError(_lib.ERR_INVALID, f"a stream of device {stream.device_index} cannot take work on {x.device}")
    return torch.cuda.stream(stream)


def _elsewhere(x: torch.Tensor, stream) -> bool:
    """Whether a call on x has to switch stream or device first (`_on`)."""
    return stream is not None or x.get_device() != _current_device()


# The current device, and its current stream's handle: a call of a few microseconds would spend three on the Stream object.
_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _require_same_device(name, first, *tensors):
    if not first.is_cuda or not first.is_contiguous():
        raise IronMLXError(_lib.ERR_INVALID, f"{name}: tensors must be contiguous CUDA tensors")
    device = first.get_device()
    for t in tensors:
        if t is not None and (t.get_device() != device or not t.is_contiguous()):
            if not t.is_cuda or not t.is_contiguous():
                raise IronMLXError(_lib.ERR_INVALID, f"{name}: tensors must be contiguous CUDA tensors")
            raise IronMLXError(_lib.ERR_INVALID, f"{name}: tensors on {first.device} and {t.device}")


def _row_count(name: str, x: torch.Tensor, length: int) -> int:
    n = x.numel() // length
    if n > 0x7fffffff:
        raise IronMLXError(_lib.ERR_INVALID, f"{name}: {n} rows, at most 2^31 - 1")
    return n


def _count(name: str, what: str, value: int) -> None:
    """Refuses a dimension that the C ABI's int does not hold (ctypes would cut it off)."""
    if value > 0x7fffffff:
        raise IronMLXError(_lib.ERR_INVALID, f"{name}: {what} of {value}, at most 2^31 - 1")


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: Optional[torch.Tensor], eps: float,
                 out: str = "bf16", stream=None):
    """`h = x + residual` and `rms_norm(h)` in one pass, sums in fp32, each output rounded once.

    Returns (h, y, rows): y bf16 for out="bf16" or "both" (None otherwise), rows an `Mxfp8Rows` that `mxfp8_matmul` reads
    for out="mxfp8" or "both" (None otherwise).  Without a residual h is x itself."""
    _require_same_device("add_rms_norm", x, residual, weight)
    if out not in ("bf16", "mxfp8", "both"):
        raise IronMLXError(_lib.ERR_INVALID, f"add_rms_norm: out must be bf16, mxfp8 or both, not {out!r}")
    shape = x.shape
    bf16 = torch.bfloat16
    if x.dtype != bf16 or (residual is not None and residual.dtype != bf16) or (weight is not None and weight.dtype != bf16):
        raise IronMLXError(_lib.ERR_INVALID, "add_rms_norm: x, residual and weight must be bfloat16")
    if len(shape) == 0 or shape[-1] == 0:
        raise IronMLXError(_lib.ERR_INVALID, "add_rms_norm: x has no last dimension")
    hidden = shape[-1]
    if residual is not None and residual.shape != shape:
        raise IronMLXError(_lib.ERR_INVALID, f"add_rms_norm: residual {tuple(residual.shape)} and x {tuple(shape)} differ")
    if weight is not None and weight.numel() != hidden:
        raise IronMLXError(_lib.ERR_INVALID, f"add_rms_norm: weight has {weight.numel()} elements, rows have {hidden}")
    if out != "bf16" and hidden % 32:
        raise IronMLXError(_lib.ERR_INVALID, f"add_rms_norm: 8-bit rows need a row length ({hidden}) that is a multiple of 32")
    if _elsewhere(x, stream):
        with _on(x, stream):
            return add_rms_norm(x, residual, weight, eps, out)
    n = _row_count("add_rms_norm", x, hidden)
    _count("add_rms_norm", "a row length", hidden)
    h, y, rows = x, None, None
    residual_at = h_at = y_at = q_at = scales_at = None
    if residual is not None:
        h = torch.empty_like(x)
        residual_at, h_at = residual.data_ptr(), h.data_ptr()
    if out != "mxfp8":
        y = torch.empty_like(x)
        y_at = y.data_ptr()
    if out != "bf16":
        lead, device = shape[:-1], x.device
        q = torch.empty(*lead, hidden // 4, dtype=torch.int32, device=device)
        scales = torch.empty(*lead, hidden // 32, dtype=torch.uint8, device=device)
        rows = Mxfp8Rows(q, scales)
        q_at, scales_at = q.data_ptr(), scales.data_ptr()
    check(lib().imx_add_rms_norm(x.data_ptr(), residual_at, n, hidden, None if weight is None else weight.data_ptr(), eps, h_at, y_at,
                                 q_at, scales_at, _raw_stream(x.get_device())))
    return h, y, rows


_STATUS = {}


def _status_block(index: int) -> int:
    """The address of the status block that the `mxfp8_matmul` and `low_rank_add` calls of a device, the current one, share: the
    library's own, which kernels only ever set, so that a captured call's replays are reported like any call."""
    at = _STATUS.get(index)
    if at is None:
        block = C.c_void_p()
        check(lib().imx_status_block(C.byref(block)))
        at = _STATUS[index] = block.value
    return at


def check_status(device=None, stream=None) -> None:
    """Raises if a bounded wait ran out in an `mxfp8_matmul` or `low_rank_add` call on the device (default: the current one),
    replayed ones among them, since the last check; synchronises the stream."""
    index = torch.device("cuda" if device is None else device).index
    index = torch.cuda.current_device() if index is None else index
    if index not in _STATUS:                     # no such call yet
        return
    if stream is not None and stream.device_index != index:
        raise IronMLXError(_lib.ERR_INVALID, f"a stream of device {stream.device_index} cannot take work on cuda:{index}")
    with torch.cuda.device(index) if stream is None else torch.cuda.stream(stream):
        check(lib().imx_moe_status(_STATUS[index], stream_ptr()))


def mxfp8_matmul(rows, w: torch.Tensor, scales: torch.Tensor, stream=None) -> torch.Tensor:
    """`dequantize(rows) @ dequantize(w)^T` with both operands in mxfp8, bf16 out: rows as `add_rms_norm` or `quantize`
    left them ((packed, scales), an `Mxfp8Rows`), w [out, in/4] int32 and scales [out, in/32] uint8."""
    x, xs = rows[0], rows[1]
    _require_same_device("mxfp8_matmul", x, xs, w, scales)
    if x.dtype != torch.int32 or w.dtype != torch.int32 or xs.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise IronMLXError(_lib.ERR_INVALID, "mxfp8_matmul: packed values must be int32 words, scales uint8")
    shape, wshape = x.shape, w.shape
    if len(wshape) != 2 or len(shape) == 0 or wshape[1] % 8 or w.numel() == 0:
        raise IronMLXError(_lib.ERR_INVALID, "mxfp8_matmul: w must be [out, in/4] and scales [out, in/32], in a multiple of 32")
    n_out, words = wshape
    if shape[-1] != words:
        raise IronMLXError(_lib.ERR_INVALID, f"mxfp8_matmul: rows have {shape[-1] * 4} values, the weight takes {words * 4}")
    lead = tuple(shape)[:-1]
    if scales.shape != (n_out, words // 8) or xs.shape != (*lead, words // 8):
        raise IronMLXError(_lib.ERR_INVALID, "mxfp8_matmul: one scale per 32 values is needed for the rows and the weight")
    if _elsewhere(x, stream):
        with _on(x, stream):
            return mxfp8_matmul(rows, w, scales)
    n = _row_count("mxfp8_matmul", x, words)
    if max(words * 4, n_out) > 0x7fffffff:
        _count("mxfp8_matmul", "an input dimension", words * 4)
        _count("mxfp8_matmul", "an output dimension", n_out)
    index = x.get_device()
    y = torch.empty(*lead, n_out, dtype=torch.bfloat16, device=x.device)
    qt = QTensor(w.data_ptr(), scales.data_ptr(), None, 1.0)
    check(lib().imx_mxfp8_matmul(x.data_ptr(), xs.data_ptr(), n, C.byref(qt), n_out, words * 4, y.data_ptr(),
                                 _status_block(index), 256, _raw_stream(index)))
    return y


def low_rank_add(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, ids: torch.Tensor,
                 scale: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """`y[t] + scale[j] * (x[t] @ a[j]^T) @ b[j]^T` with j = ids[t], the adapter of row t (none where it is outside
    [0, count): the row is y's): the adapters of many requests beside a shared projection y = W x.

    y [.., out_dim], x [.., in], a [count, rank, in], b [count, out_dim, rank] bf16; ids int32, one per row; scale fp32
    [count].  `out` may be y itself; a new tensor by default."""
    _require_same_device("low_rank_add", y, x, a, b, ids, scale, out)
    if y.dtype != torch.bfloat16 or x.dtype != torch.bfloat16 or a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16:
        raise IronMLXError(_lib.ERR_INVALID, "low_rank_add: y, x, a and b must be bfloat16")
    ashape, bshape, xshape, yshape = a.shape, b.shape, x.shape, y.shape
    if len(ashape) != 3 or len(bshape) != 3 or ashape[0] != bshape[0] or ashape[1] != bshape[2] or a.numel() == 0 or b.numel() == 0:
        raise IronMLXError(_lib.ERR_INVALID, "low_rank_add: a must be [count, rank, in] and b [count, out, rank]")
    count, rank, in_dim = ashape
    n_out = bshape[1]
    if len(xshape) == 0 or len(yshape) == 0 or xshape[-1] != in_dim or yshape[-1] != n_out or xshape[:-1] != yshape[:-1]:
        raise IronMLXError(_lib.ERR_INVALID,
                           f"low_rank_add: x {tuple(xshape)} and y {tuple(yshape)} do not match adapters {in_dim} -> {n_out}")
    rows = _row_count("low_rank_add", x, in_dim)
    if max(in_dim, n_out, rank, count) > 0x7fffffff:
        for what, value in (("an input dimension", in_dim), ("an output dimension", n_out), ("a rank", rank), ("a number of adapters", count)):
            _count("low_rank_add", what, value)
    if ids.dtype != torch.int32 or ids.numel() != rows:
        raise IronMLXError(_lib.ERR_INVALID, f"low_rank_add: ids must be int32, one for each of the {rows} rows")
    if scale is not None and (scale.dtype != torch.float32 or scale.numel() != count):
        raise IronMLXError(_lib.ERR_INVALID, f"low_rank_add: scale must be float32, one for each of the {count} adapters")
    if out is not None and (out.shape != yshape or out.dtype != torch.bfloat16):
        raise IronMLXError(_lib.ERR_INVALID, "low_rank_add: out must have y's shape and type")
    if _elsewhere(x, stream):
        with _on(x, stream):
            return low_rank_add(y, x, a, b, ids, scale, out)
    if out is None:
        out = torch.empty_like(y)
    ad = _lib.Adapters(a.data_ptr(), b.data_ptr(), None if scale is None else scale.data_ptr(), count, rank)
    index = x.get_device()
    check(lib().imx_low_rank_add(y.data_ptr(), x.data_ptr(), rows, in_dim, C.byref(ad), ids.data_ptr(), n_out, out.data_ptr(),
                                 _status_block(index), 256, _raw_stream(index)))
    return out
