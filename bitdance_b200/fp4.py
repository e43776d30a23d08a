"""Microscaled 4-bit floating point: quantiser, dequantiser and the W4A4 GEMM, tensor-level
entry points over the C ABI (NVFP4 and MXFP4 operands, tcgen05 kind::mxf4nvf4 / kind::mxf4).

Where ``ops.w4a6_gemm`` spends its time turning 4-bit weights into 6-bit operands on chip, the
products here take both operands in 4 bits as they are: coarser activations, and twice the
tensor-core rate. Weights quantised once by ``ops.quantize_nvfp4`` serve both paths.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from ._lib import call
from .ops import EPILOGUES, _OUT, _need, quantize_nvfp4, tensor_scale_of

FP4_FORMATS = {"nvfp4": _lib.BD_FP4_NVFP4, "mxfp4": _lib.BD_FP4_MXFP4}
_BLOCK = {"nvfp4": 16, "mxfp4": 32}
_IN4 = {torch.float32: _lib.BD_IN_F32, torch.bfloat16: _lib.BD_IN_BF16,
        torch.float16: _lib.BD_IN_F16}


@dataclass
class Fp4Operand:
    """A (rows, K) matrix in microscaled 4-bit floating point, either operand of ``w4a4_gemm``
    (activations: rows are tokens; weights: rows are outputs). Its values are
    code * block scale * (row_scale[row] * tensor_scale)."""
    codes: torch.Tensor   # (rows, K/2) u8, element 2j in the low nibble of byte j
    scales: torch.Tensor  # scale tiles (flat u8): [ceil(rows/128)][ceil(scales per row/4)][512]
    rows: int
    K: int
    fmt: str              # "nvfp4": E4M3 per 16 elements; "mxfp4": E8M0 per 32
    row_scale: Optional[torch.Tensor] = None  # (rows,) fp32
    tensor_scale: float = 1.0


def _fmt(fmt: str) -> int:
    if fmt not in FP4_FORMATS:
        raise ValueError(f"unknown 4-bit format {fmt!r}: 'nvfp4' or 'mxfp4'")
    return FP4_FORMATS[fmt]


def _scale_bytes(rows: int, K: int, fmt: str) -> int:
    return (rows + 127) // 128 * ((K // _BLOCK[fmt] + 3) // 4) * 512


# These entry points serve single tokens, where a call's time is the host's: addresses go to the
# library as integers, and the current stream and device come from torch's C layer, as do new tensors
# where it has a call for them (0.8 us; torch.empty reads its arguments for another 0.8, and for 1.5
# and 2.3 more where the sizes are a tuple or a torch.Size).
_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else \
    torch.cuda.current_device
try:
    from torch._C._dynamo.guards import _empty_strided_cuda as _alloc
except ImportError:
    _alloc = None


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _stream_ptr(stream) -> int:
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(_device())
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)


def _empty(stream, dtype, device, *shape):
    """A new tensor of one or two dimensions that belongs to the stream the kernels run on (its memory
    is reused in that stream's order), on the current device (``device``: the arguments were checked
    to be there)."""
    if stream is None:
        if _alloc is not None:
            return _alloc(shape, (shape[1], 1) if len(shape) == 2 else (1,), dtype)
        return torch.empty(*shape, dtype=dtype, device=device)
    if not hasattr(stream, "cuda_stream"):
        stream = torch.cuda.ExternalStream(int(stream), device=device)
    with torch.cuda.stream(stream):
        return torch.empty(*shape, dtype=dtype, device=device)


def _have(t, dtype, what: str, numel: int, dev: int) -> None:
    """``ops._need`` with its common case first: on device dev, the current one."""
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == dev
            and t.is_contiguous() and t.numel() >= numel):
        _need(t, dtype, what, numel)


def _check_x4(x: torch.Tensor):
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError("x must be a 2-D tensor (M, K)")
    if x.dtype not in _IN4:
        raise TypeError(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    if not (x.is_cuda and x.is_contiguous() and x.get_device() == _device()):
        _need(x, x.dtype, "x")
    M, K = x.shape
    if K == 0 or K % 32:
        raise ValueError(f"K must be a positive multiple of 32, got {K}")
    return M, K


def _check_operand(op: Fp4Operand, what: str, dev: Optional[int] = None) -> int:
    """The operand's device, the current one (dev: already known)."""
    _fmt(op.fmt)
    if dev is None:
        if not (isinstance(op.codes, torch.Tensor) and op.codes.is_cuda):
            _need(op.codes, torch.uint8, f"{what}.codes")
        dev = _device()
    if op.rows < 0 or op.K <= 0 or op.K % 32:
        raise ValueError(f"{what}: K must be a positive multiple of 32, got {op.K}")
    _have(op.codes, torch.uint8, f"{what}.codes", op.rows * op.K // 2, dev)
    _have(op.scales, torch.uint8, f"{what}.scales", _scale_bytes(op.rows, op.K, op.fmt), dev)
    if op.row_scale is not None:
        _have(op.row_scale, torch.float32, f"{what}.row_scale", op.rows, dev)
    return dev


def quantize_fp4(x: torch.Tensor, fmt: str = "nvfp4", stream=None,
                 overlap_prev: bool = False) -> Fp4Operand:
    """x (M, K) fp32 / bf16 / fp16 -> Fp4Operand in one launch, K % 32 == 0. "nvfp4": E4M3 scales
    per 16 elements under an fp32 scale per row (a token's codes do not depend on the rest of the
    batch); "mxfp4": E8M0 scales per 32. A NaN or Inf sets BD_DEVERR_NONFINITE in the device error
    word and leaves its row undefined."""
    code = _fmt(fmt)
    M, K = _check_x4(x)
    device = x.device
    codes = _empty(stream, torch.uint8, device, M, K // 2)
    scales = _empty(stream, torch.uint8, device, _scale_bytes(M, K, fmt))
    row_scale = _empty(stream, torch.float32, device, M) if fmt == "nvfp4" else None
    call("bd_quantize_fp4", x.data_ptr(), _IN4[x.dtype], code, codes.data_ptr(), None,
         scales.data_ptr(), _ptr(row_scale), M, K,
         _lib.BD_GEMM_OVERLAP_PREV if overlap_prev else 0, _stream_ptr(stream))
    return Fp4Operand(codes, scales, M, K, fmt, row_scale)


def quantize_mxfp4(x: torch.Tensor, stream=None):
    """x (M, K) fp32 / bf16 / fp16 -> (codes (M, K/2) packed E2M1 nibbles, E8M0 (M, K/32) u8):
    ``quantize_fp4(x, "mxfp4")`` in the natural layout (the reference's quantize(x, E8M0, E2M1),
    vector_quant_error.py:283-319)."""
    M, K = _check_x4(x)
    codes = _empty(stream, torch.uint8, x.device, M, K // 2)
    e8m0 = _empty(stream, torch.uint8, x.device, M, K // 32)
    call("bd_quantize_fp4", x.data_ptr(), _IN4[x.dtype], _lib.BD_FP4_MXFP4, codes.data_ptr(),
         e8m0.data_ptr(), None, None, M, K, 0, _stream_ptr(stream))
    return codes, e8m0


def pack_fp4(codes: torch.Tensor, scales: torch.Tensor, fmt: str = "nvfp4",
             tensor_scale: float = 1.0, row_scale: Optional[torch.Tensor] = None,
             stream=None) -> Fp4Operand:
    """Natural codes (rows, K/2) and block scales ((rows, K/16) E4M3 or (rows, K/32) E8M0 bytes) ->
    Fp4Operand. The codes are the operand as they are (not copied); only the scales are re-laid."""
    code = _fmt(fmt)
    if codes.dim() != 2:
        raise ValueError("codes must be 2-D (rows, K/2)")
    rows, K = codes.shape[0], 2 * codes.shape[1]
    if K == 0 or K % 32:
        raise ValueError(f"K must be a positive multiple of 32, got {K}")
    _need(codes, torch.uint8, "codes")
    _need(scales, torch.uint8, "scales", rows * (K // _BLOCK[fmt]))
    if row_scale is not None:
        _need(row_scale, torch.float32, "row_scale", rows)
    tiled = _empty(stream, torch.uint8, codes.device, _scale_bytes(rows, K, fmt))
    call("bd_tile_scales_fp4", scales.data_ptr(), tiled.data_ptr(), rows, K, code,
         _stream_ptr(stream))
    return Fp4Operand(codes, tiled, rows, K, fmt, row_scale, float(tensor_scale))


def quantize_weights_fp4(w: torch.Tensor, fmt: str = "nvfp4", stream=None) -> Fp4Operand:
    """Weights w (N, K) fp32 / bf16 -> Fp4Operand. "nvfp4": the codes of ``quantize_nvfp4`` (one
    fp32 scale for the tensor, read back to the host once); "mxfp4": ``quantize_fp4``."""
    if _fmt(fmt) == _lib.BD_FP4_MXFP4:
        return quantize_fp4(w, fmt, stream)
    if stream is not None:  # quantize_nvfp4 allocates on the current stream
        with torch.cuda.stream(stream if hasattr(stream, "cuda_stream") else
                               torch.cuda.ExternalStream(int(stream), device=w.device)):
            return quantize_weights_fp4(w, fmt)
    codes, scales, tstat = quantize_nvfp4(w)
    return pack_fp4(codes, scales, fmt, tensor_scale_of(tstat))


def dequantize_fp4(op: Fp4Operand, out_dtype=torch.float32, out: Optional[torch.Tensor] = None,
                   stream=None) -> torch.Tensor:
    """The values of an operand, (rows, K) in out_dtype (fp32, bf16 or fp16)."""
    dev = _check_operand(op, "operand")
    if out_dtype not in _OUT:
        raise TypeError(f"unsupported output dtype {out_dtype}")
    if out is None:
        out = _empty(stream, out_dtype, op.codes.device, op.rows, op.K)
    else:
        _have(out, out_dtype, "out", op.rows * op.K, dev)
    call("bd_dequantize_fp4", op.codes.data_ptr(), op.scales.data_ptr(), _ptr(op.row_scale),
         float(op.tensor_scale), out.data_ptr(), _OUT[out_dtype], FP4_FORMATS[op.fmt], op.rows,
         op.K, 0, _stream_ptr(stream))
    return out


def _epilogue(epilogue: str, bias, N: int, dev: int) -> int:
    if epilogue not in EPILOGUES:
        raise ValueError(f"unknown epilogue {epilogue!r}")
    epi = EPILOGUES[epilogue]
    if bias is not None:
        _have(bias, torch.bfloat16, "bias", N, dev)
    if epi != _lib.BD_EPI_NONE and bias is None:
        raise ValueError(f"epilogue {epilogue!r} needs a bias")
    return epi


def _output(out, M: int, N: int, out_dtype, device, dev: int, stream):
    if out_dtype not in _OUT:
        raise TypeError(f"unsupported output dtype {out_dtype}")
    if out is None:
        return _empty(stream, out_dtype, device, M, N)
    _have(out, out_dtype, "out", M * N, dev)
    return out


def w4a4_gemm(acts: Fp4Operand, weights: Fp4Operand, bias: Optional[torch.Tensor] = None,
              out_dtype=torch.bfloat16, epilogue: str = "none",
              out: Optional[torch.Tensor] = None, stream=None, overlap_prev: bool = False,
              weights_static: bool = False) -> torch.Tensor:
    """C[M, N] = act(A . B^T + bias) of two 4-bit operands of one format on the tensor cores (any
    M and N, K % 32 == 0; no workspace). bias (N,) bf16 is added by the epilogues "bias", "bias_relu",
    "bias_silu" and "bias_gelu" ("none" leaves it unread). overlap_prev, weights_static: as in
    ``w4a6_gemm``."""
    if acts.fmt != weights.fmt:
        raise ValueError(f"format mismatch: activations {acts.fmt}, weights {weights.fmt}")
    if acts.K != weights.K:
        raise ValueError(f"K mismatch: activations {acts.K}, weights {weights.K}")
    dev = _check_operand(acts, "acts")
    _check_operand(weights, "weights", dev)
    M, N, K = acts.rows, weights.rows, acts.K
    epi = _epilogue(epilogue, bias, N, dev)
    out = _output(out, M, N, out_dtype, acts.codes.device, dev, stream)
    flags = (_lib.BD_GEMM_OVERLAP_PREV if overlap_prev else 0) | \
        (_lib.BD_GEMM_WEIGHTS_STATIC if weights_static else 0)
    call("bd_w4a4_gemm", out.data_ptr(), acts.codes.data_ptr(), acts.scales.data_ptr(),
         _ptr(acts.row_scale), weights.codes.data_ptr(), weights.scales.data_ptr(),
         _ptr(weights.row_scale), float(acts.tensor_scale) * float(weights.tensor_scale),
         _ptr(bias), M, N, K, FP4_FORMATS[acts.fmt], _OUT[out_dtype], epi, flags,
         _stream_ptr(stream))
    return out


def w4a4_linear(x: torch.Tensor, weights: Fp4Operand, bias: Optional[torch.Tensor] = None,
                out_dtype=torch.bfloat16, epilogue: str = "none",
                out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """C = act(quantize_fp4(x) . W^T + bias) from raw activations x (M, K) fp32 / bf16 / fp16, in
    the weights' format: the quantiser, then the W4A4 GEMM, which for few tokens streams its first
    weights while the quantiser runs. bias, epilogue: as in ``w4a4_gemm``."""
    M, K = _check_x4(x)
    if weights.K != K:
        raise ValueError(f"K mismatch: activations {K}, weights {weights.K}")
    dev = _check_operand(weights, "weights", x.get_device())
    N = weights.rows
    epi = _epilogue(epilogue, bias, N, dev)
    out = _output(out, M, N, out_dtype, x.device, dev, stream)
    if M == 0:
        return out
    nbytes = _linear_workspace(M, K, weights.fmt)
    ws = _empty(stream, torch.uint8, x.device, nbytes)
    call("bd_w4a4_linear", out.data_ptr(), x.data_ptr(), _IN4[x.dtype], weights.codes.data_ptr(),
         weights.scales.data_ptr(), _ptr(weights.row_scale), float(weights.tensor_scale),
         _ptr(bias), M, N, K, FP4_FORMATS[weights.fmt], _OUT[out_dtype], epi, ws.data_ptr(),
         nbytes, _stream_ptr(stream))
    return out


def _linear_workspace(M: int, K: int, fmt: str) -> int:
    """bd_query_w4a4_linear_workspace without the call."""
    def up(v):
        return (v + 255) // 256 * 256
    return up(M * K // 2) + up(_scale_bytes(M, K, fmt)) + up(4 * M)
