"""Mixture-of-experts layer for a few tokens on NVFP4 expert weights: tensor-level entry points
over the C ABI (bd_moe_layer, bd_moe_experts; two kernels each)."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from ._lib import call
from .fp4 import _device, _empty, _have, _ptr, _stream_ptr
from .ops import _OUT, _need, quantize_nvfp4

MOE_MAX_TOKENS, MOE_MAX_EXPERTS, MOE_MAX_TOP_K = 64, 512, 16
SCORINGS = {"softmax": _lib.BD_MOE_SOFTMAX, "sigmoid": _lib.BD_MOE_SIGMOID}
_IN_MOE = {torch.bfloat16: _lib.BD_IN_BF16, torch.float16: _lib.BD_IN_F16,
           torch.float32: _lib.BD_IN_F32}


@dataclass
class MoeWeights:
    """Expert weights in NVFP4, natural layout: what ``quantize_nvfp4`` gives, stacked over the E
    experts. gate_up holds the I gate rows, then the I up rows."""
    gate_up: torch.Tensor               # (E, 2I, H/2) u8: packed E2M1 codes
    gate_up_scales: torch.Tensor        # (E, 2I, H/16) u8: E4M3
    gate_up_tensor_scale: torch.Tensor  # (E,) fp32
    down: torch.Tensor                  # (E, H, I/2) u8
    down_scales: torch.Tensor           # (E, H, I/16) u8
    down_tensor_scale: torch.Tensor     # (E,) fp32


def quantize_moe_weights(gate_up: torch.Tensor, down: torch.Tensor, stream=None) -> MoeWeights:
    """gate_up (E, 2I, H) and down (E, H, I), fp32 or bf16 on the GPU -> MoeWeights (each expert's
    matrix by ``quantize_nvfp4``, its own tensor scale)."""
    if gate_up.dim() != 3 or down.dim() != 3:
        raise ValueError("gate_up must be (E, 2I, H) and down (E, H, I)")
    E, two_i, H = gate_up.shape
    if two_i % 2 or down.shape != (E, H, two_i // 2):
        raise ValueError(f"gate_up {tuple(gate_up.shape)} and down {tuple(down.shape)} do not match")
    if stream is not None:  # quantize_nvfp4 allocates on the current stream
        with torch.cuda.stream(stream if hasattr(stream, "cuda_stream") else
                               torch.cuda.ExternalStream(int(stream), device=gate_up.device)):
            return quantize_moe_weights(gate_up, down)
    parts = []
    for w in (gate_up, down):
        q = [quantize_nvfp4(w[e]) for e in range(E)]
        parts += [torch.stack([c for c, _, _ in q]), torch.stack([s for _, s, _ in q]),
                  torch.stack([t[:1].view(torch.float32)[0] for _, _, t in q])]
    return MoeWeights(*parts)


def _check(x: torch.Tensor, w: MoeWeights, top_k: int):
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError("x must be a 2-D tensor (tokens, H)")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"x must be bfloat16 or float16, got {x.dtype}")
    if not (x.is_cuda and x.is_contiguous() and x.get_device() == _device()):
        _need(x, x.dtype, "x")
    dev = x.get_device()
    T, H = x.shape
    if w.gate_up.dim() != 3 or w.down.dim() != 3:
        raise ValueError("expert weights must be (E, rows, K/2)")
    E, two_i, half = w.gate_up.shape
    inter = two_i // 2
    if two_i % 2 or half * 2 != H or w.down.shape != (E, H, inter // 2):
        raise ValueError(f"x has {H} columns, gate_up {tuple(w.gate_up.shape)}, down "
                         f"{tuple(w.down.shape)}: expected (E, 2I, H/2) and (E, H, I/2)")
    if H == 0 or inter == 0 or H % 128 or inter % 128:
        raise ValueError(f"H and I must be positive multiples of 128, got {H} and {inter}")
    if T > MOE_MAX_TOKENS:
        raise ValueError(f"at most {MOE_MAX_TOKENS} tokens, got {T}")
    if not 1 <= E <= MOE_MAX_EXPERTS:
        raise ValueError(f"1 to {MOE_MAX_EXPERTS} experts, got {E}")
    if not 1 <= top_k <= min(MOE_MAX_TOP_K, E):
        raise ValueError(f"top_k must be in 1..{min(MOE_MAX_TOP_K, E)}, got {top_k}")
    _have(w.gate_up, torch.uint8, "gate_up", 0, dev)
    _have(w.gate_up_scales, torch.uint8, "gate_up_scales", E * two_i * (H // 16), dev)
    _have(w.gate_up_tensor_scale, torch.float32, "gate_up_tensor_scale", E, dev)
    _have(w.down, torch.uint8, "down", 0, dev)
    _have(w.down_scales, torch.uint8, "down_scales", E * H * (inter // 16), dev)
    _have(w.down_tensor_scale, torch.float32, "down_tensor_scale", E, dev)
    return T, H, inter, E, dev


def _workspace_bytes(T: int, H: int, inter: int, E: int, top_k: int) -> int:
    """bd_query_moe_workspace without the call."""
    def up(v):
        return (v + 255) // 256 * 256
    if T == 0:
        return 0
    pairs = T * top_k
    return up(4 * (5 + 2 * E)) + up(4 * pairs) + up(4 * T) + up(T * ((H + 255) // 256) * 1152) + \
        up(4 * pairs * inter) + up(pairs * ((inter + 255) // 256) * 1152) + 4 * H * max(pairs, 256)


def _out_tensor(out, x: torch.Tensor, T: int, H: int, out_dtype, dev: int, stream):
    dtype = x.dtype if out_dtype is None else out_dtype
    if dtype not in _OUT:
        raise TypeError(f"unsupported output dtype {dtype}")
    if out is None:
        return _empty(stream, dtype, x.device, T, H)
    _have(out, dtype, "out", T * H, dev)
    return out


def _weight_args(w: MoeWeights):
    return (w.gate_up.data_ptr(), w.gate_up_scales.data_ptr(), w.gate_up_tensor_scale.data_ptr(),
            w.down.data_ptr(), w.down_scales.data_ptr(), w.down_tensor_scale.data_ptr())


def moe_experts(x: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor,
                experts: MoeWeights, out_dtype=None, out: Optional[torch.Tensor] = None,
                stream=None) -> torch.Tensor:
    """y[t] = sum over s of topk_weights[t, s] * expert topk_ids[t, s] (x[t]), each expert
    Wd (silu(Wg x) * (Wu x)). x (T, H) bf16 / fp16, T <= 64; topk_ids (T, k) int32, -1 for an empty
    slot (a token with none gets zeros), any other id outside the experts sets BD_DEVERR_RANGE and
    counts as -1; topk_weights (T, k) fp32. Returns (T, H) in x's dtype or out_dtype."""
    if topk_ids.dim() != 2 or topk_ids.shape[0] != x.shape[0] or \
            topk_weights.shape != topk_ids.shape:
        raise ValueError("topk_ids and topk_weights must be (tokens, top_k)")
    top_k = topk_ids.shape[1]
    T, H, inter, E, dev = _check(x, experts, top_k)
    _have(topk_ids, torch.int32, "topk_ids", 0, dev)
    _have(topk_weights, torch.float32, "topk_weights", 0, dev)
    out = _out_tensor(out, x, T, H, out_dtype, dev, stream)
    nbytes = _workspace_bytes(T, H, inter, E, top_k)
    ws = _empty(stream, torch.uint8, x.device, nbytes)
    call("bd_moe_experts", out.data_ptr(), x.data_ptr(), _IN_MOE[x.dtype], topk_ids.data_ptr(),
         topk_weights.data_ptr(), *_weight_args(experts), T, H, inter, E, top_k, _OUT[out.dtype],
         ws.data_ptr(), nbytes, _stream_ptr(stream))
    return out


def moe_layer(x: torch.Tensor, router: torch.Tensor, experts: MoeWeights, top_k: int,
              scoring: str = "softmax", renormalize: bool = True,
              selection_bias: Optional[torch.Tensor] = None, routed_scale: float = 1.0,
              out_dtype=None, out: Optional[torch.Tensor] = None, return_routing: bool = False,
              stream=None):
    """A whole mixture-of-experts layer for x (T, H) bf16 / fp16, T <= 64, in two kernels: router
    (E, H) in x's dtype or fp32 -> scores ("softmax" over the experts or "sigmoid"), the top_k
    experts by score (+ selection_bias (E,) fp32, for the selection only; ties to the lowest
    index), weights = score, divided by their sum if renormalize, times routed_scale; then
    ``moe_experts``. Returns y, or (y, ids (T, k) int32, weights (T, k) fp32) with
    return_routing, best expert first."""
    if scoring not in SCORINGS:
        raise ValueError(f"unknown scoring {scoring!r}: 'softmax' or 'sigmoid'")
    T, H, inter, E, dev = _check(x, experts, top_k)
    if router.shape != (E, H):
        raise ValueError(f"router must be ({E}, {H}), got {tuple(router.shape)}")
    if router.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"router must be {x.dtype} or float32, got {router.dtype}")
    _have(router, router.dtype, "router", 0, dev)
    if selection_bias is not None:
        _have(selection_bias, torch.float32, "selection_bias", E, dev)
    out = _out_tensor(out, x, T, H, out_dtype, dev, stream)
    nbytes = _workspace_bytes(T, H, inter, E, top_k)
    if return_routing:
        ids = _empty(stream, torch.int32, x.device, T, top_k)
        weights = _empty(stream, torch.float32, x.device, T, top_k)
        ws = _empty(stream, torch.uint8, x.device, nbytes)
        ids_at, weights_at = ids.data_ptr(), weights.data_ptr()
    else:  # behind the workspace
        ws = _empty(stream, torch.uint8, x.device, nbytes + 8 * T * top_k)
        ids_at = ws.data_ptr() + nbytes
        weights_at = ids_at + 4 * T * top_k
    call("bd_moe_layer", out.data_ptr(), ids_at, weights_at, x.data_ptr(), _IN_MOE[x.dtype],
         router.data_ptr(), _IN_MOE[router.dtype], _ptr(selection_bias), SCORINGS[scoring],
         1 if renormalize else 0, float(routed_scale), *_weight_args(experts), T, H, inter, E,
         top_k, _OUT[out.dtype], ws.data_ptr(), nbytes, _stream_ptr(stream))
    return (out, ids, weights) if return_routing else out
