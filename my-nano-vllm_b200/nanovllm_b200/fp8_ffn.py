"""The feed-forward half of an FP8 layer around the block-scaled linear layer of ``fp8_linear``.

``add_rms_norm_fp8(x, residual, weight, eps)``  residual addition and RMS norm, the result written in
    e4m3 with one bf16 scale per row and 128 columns: the operand of ``fp8_block_gemm`` (in place of
    RMSNorm.forward, nanovllm/layers/layernorm.py:28-50, and then ``fp8_dyn_quant``).
``silu_mul_fp8(gate_up)``  SiLU(gate) * up in the same form (SiluAndMul, nanovllm/layers/
    activation.py:8-11, and then ``fp8_dyn_quant``).
``fp8_moe(...)``  a whole mixture-of-experts layer for a few tokens, experts' weights block-scaled
    as ``fp8_block_linear``'s (no counterpart in the reference, whose model is dense).

A dense block, with the weights of ``fp8_block_linear``:

    xq, xs, residual, _ = add_rms_norm_fp8(x, residual, norm_weight, eps)
    hq, hs = silu_mul_fp8(fp8_block_gemm(xq, xs, gate_up_weight, gate_up_scale))
    x = fp8_block_gemm(hq, hs, down_weight, down_scale)

and a mixture of experts:

    xq, xs, residual, y = add_rms_norm_fp8(x, residual, norm_weight, eps, return_norm=True)
    x = fp8_moe(y, xq, xs, router_weight, gate_up_weight, gate_up_scale, down_weight, down_scale, 8)

All launch on ``torch.cuda.current_stream()`` of the tensors' device, allocate outputs and scratch
with ``torch.empty`` and never synchronise, so they can be captured into CUDA graphs.  A device wait of
``fp8_moe`` that gives up is recorded in a word of the library's own (``fp8_attention.device_error``).
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from .fp8_attention import _MOE_DEVICES
from .fp8_linear import BLOCK_SIZE

_DTYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16}
_BF16, _E4M3 = torch.bfloat16, torch.float8_e4m3fn
MAX_TOKENS = 1024       # tokens in one fp8_moe call
MAX_SLOTS = 8192        # tokens * top_k in one fp8_moe call

# The kernels of a decoded token take 2 to 25 us, so the host side counts: raw stream handles and
# empty_strided cost 0.1 and 1.4 us a call where current_stream() and empty() cost 2.2 and 2.4, and a
# helper's call 0.3.
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_empty = torch.empty_strided
_norm_quant = _lib.lib.fp8attn_add_rms_norm_quant
_silu_quant = _lib.lib.fp8attn_silu_mul_quant
_moe = _lib.lib.fp8attn_fp8_moe


def add_rms_norm_fp8(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor,
                     eps: float, return_norm: bool = False):
    """s = x + residual (x alone without one), y = s / sqrt(mean(s^2) + eps) * weight, in fp32.

    Args:
        x, residual: bf16 or fp16 [M, K] (rows may be strided); K a multiple of 128 up to 16384
        weight: [K], of x's type
    Returns (xq, x_scale, residual_out, norm): y as e4m3 [M, K] with scales bf16 [M, K / 128]; s and,
    with ``return_norm``, y, both rounded to x's type (else None; residual_out is None without a
    residual).
    """
    dtype, device = x.dtype, x.get_device()
    code = _DTYPES.get(dtype)
    assert code is not None and device >= 0, "x must be a bf16 or fp16 CUDA tensor"
    assert x.dim() == 2 and x.stride(1) == 1
    if device != _current_device():
        with torch.cuda.device(device):
            return add_rms_norm_fp8(x, residual, weight, eps, return_norm)
    M, K = x.shape
    assert weight.get_device() == device and weight.dtype == dtype and weight.is_contiguous()
    assert weight.numel() == K and K % BLOCK_SIZE == 0 and K > 0
    dev = x.device
    # the row stride of a single row is never used, and torch leaves it arbitrary
    x_stride = x.stride(0) if M > 1 else K
    res = y = None
    res_in = res_stride = res_out = y_out = 0
    if residual is not None:
        assert residual.get_device() == device and residual.dtype == dtype
        assert residual.shape == x.shape and residual.stride(1) == 1
        res_stride = residual.stride(0) if M > 1 else K
        res = _empty((M, K), (K, 1), dtype=dtype, device=dev)
        res_in, res_out = residual.data_ptr(), res.data_ptr()
    if return_norm:
        y = _empty((M, K), (K, 1), dtype=dtype, device=dev)
        y_out = y.data_ptr()
    groups = K // BLOCK_SIZE
    xq = _empty((M, K), (K, 1), dtype=_E4M3, device=dev)
    xs = _empty((M, groups), (groups, 1), dtype=_BF16, device=dev)
    if M > 0:
        rc = _norm_quant(x.data_ptr(), x_stride, res_in, res_stride, weight.data_ptr(), eps,
                         xq.data_ptr(), xs.data_ptr(), res_out, y_out, M, K, code,
                         _raw_stream(device))
        if rc:
            _lib.check(rc)
    return xq, xs, res, y


def silu_mul_fp8(gate_up: torch.Tensor):
    """gate_up: bf16 or fp16 [M, 2 I] (rows may be strided), gate columns first; I a multiple of 128 up
    to 2^20.  Returns (hq, h_scale): gate / (1 + exp(-gate)) * up as e4m3 [M, I] with scales bf16
    [M, I / 128]."""
    device = gate_up.get_device()
    code = _DTYPES.get(gate_up.dtype)
    assert code is not None and device >= 0, "gate_up must be a bf16 or fp16 CUDA tensor"
    assert gate_up.dim() == 2 and gate_up.stride(1) == 1
    if device != _current_device():
        with torch.cuda.device(device):
            return silu_mul_fp8(gate_up)
    M, columns = gate_up.shape
    assert columns % (2 * BLOCK_SIZE) == 0 and columns > 0
    inner, dev = columns // 2, gate_up.device
    groups = inner // BLOCK_SIZE
    hq = _empty((M, inner), (inner, 1), dtype=_E4M3, device=dev)
    hs = _empty((M, groups), (groups, 1), dtype=_BF16, device=dev)
    if M > 0:
        rc = _silu_quant(gate_up.data_ptr(), gate_up.stride(0) if M > 1 else columns, hq.data_ptr(),
                         hs.data_ptr(), M, inner, code, _raw_stream(device))
        if rc:
            _lib.check(rc)
    return hq, hs


@functools.lru_cache(maxsize=1024)
def _moe_scratch_bytes(device: int, T: int, H: int, I: int, E: int, top_k: int) -> int:
    """By the current device's number of SMs, which ``device`` stands for."""
    return _lib.lib.fp8attn_fp8_moe_workspace_bytes(T, H, I, E, top_k)


def _check_experts(w: torch.Tensor, scale: torch.Tensor, device: int, e: int, n: int, k: int):
    assert w.get_device() == device and w.dtype == _E4M3 and w.is_contiguous()
    assert scale.get_device() == device and scale.dtype == _BF16 and scale.is_contiguous()
    assert w.shape == (e, n, k) and scale.shape == (e, n // BLOCK_SIZE, k // BLOCK_SIZE)


def fp8_moe(x: torch.Tensor, xq: torch.Tensor, x_scale: torch.Tensor, router_weight: torch.Tensor,
            gate_up_weight: torch.Tensor, gate_up_scale: torch.Tensor, down_weight: torch.Tensor,
            down_scale: torch.Tensor, top_k: int, renormalize: bool = True,
            return_router: bool = False):
    """Router, top-k, the experts' two products and their weighted sum, for up to 1024 tokens.

    Args:
        x: bf16 [T, H], what the router reads; xq, x_scale: the same quantised, e4m3 [T, H] and bf16
            [T, H / 128] (``add_rms_norm_fp8`` with ``return_norm``, or ``fp8_dyn_quant``)
        router_weight: bf16 [E, H]
        gate_up_weight: e4m3 [E, 2 I, H], gate rows first; gate_up_scale: bf16 [E, 2 I / 128, H / 128]
        down_weight: e4m3 [E, H, I]; down_scale: bf16 [E, H / 128, I / 128]
        top_k: experts per token, by softmax probability (ties: the lower expert first)
        renormalize: divide the chosen probabilities by their sum
    Returns bf16 [T, H], or with ``return_router`` (out, weights fp32 [T, top_k], ids int32
    [T, top_k]).
    """
    device = x.get_device()
    assert device >= 0 and x.dtype == _BF16, "x must be a bf16 CUDA tensor"
    assert x.dim() == 2 and x.stride(1) == 1
    if device != _current_device():
        with torch.cuda.device(device):
            return fp8_moe(x, xq, x_scale, router_weight, gate_up_weight, gate_up_scale, down_weight,
                           down_scale, top_k, renormalize, return_router)
    T, H = x.shape
    assert xq.get_device() == device and xq.dtype == _E4M3
    assert xq.shape == x.shape and xq.stride(1) == 1 and H % BLOCK_SIZE == 0 and H > 0
    assert x_scale.get_device() == device and x_scale.dtype == _BF16 and x_scale.is_contiguous()
    assert x_scale.shape == (T, H // BLOCK_SIZE)
    assert router_weight.get_device() == device and router_weight.dtype == _BF16
    assert router_weight.is_contiguous() and router_weight.dim() == 2 and router_weight.shape[1] == H
    E, I = router_weight.shape[0], down_weight.shape[-1]
    assert I % BLOCK_SIZE == 0 and I > 0
    _check_experts(gate_up_weight, gate_up_scale, device, E, 2 * I, H)
    _check_experts(down_weight, down_scale, device, E, H, I)
    dev = x.device
    out = _empty((T, H), (H, 1), dtype=_BF16, device=dev)
    weights = ids = None
    weights_out = ids_out = 0
    if return_router:
        weights = _empty((T, top_k), (top_k, 1), dtype=torch.float32, device=dev)
        ids = _empty((T, top_k), (top_k, 1), dtype=torch.int32, device=dev)
        weights_out, ids_out = weights.data_ptr(), ids.data_ptr()
    if T > 0:
        _MOE_DEVICES.add(device)
        nbytes = _moe_scratch_bytes(device, T, H, I, E, top_k)
        # scratch of this call alone: calls on other streams and captured graphs share none
        scratch = _empty((max(nbytes, 0),), (1,), dtype=torch.uint8, device=dev)
        # the row stride of a single row is never used, and torch leaves it arbitrary
        rc = _moe(x.data_ptr(), x.stride(0) if T > 1 else H, xq.data_ptr(),
                  xq.stride(0) if T > 1 else H, x_scale.data_ptr(), router_weight.data_ptr(),
                  gate_up_weight.data_ptr(), gate_up_scale.data_ptr(), down_weight.data_ptr(),
                  down_scale.data_ptr(), out.data_ptr(), H, weights_out, ids_out, T, H, I, E, top_k,
                  1 if renormalize else 0, scratch.data_ptr(), nbytes, 0, _raw_stream(device))
        if rc:
            _lib.check(rc)
    return (out, weights, ids) if return_router else out
