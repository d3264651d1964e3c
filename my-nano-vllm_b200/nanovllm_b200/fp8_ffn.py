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
with ``torch.empty`` and never synchronise, so they can be captured into CUDA graphs.
"""
from __future__ import annotations

import torch

from . import _lib
from .fp8_attention import _stream, workspace
from .fp8_linear import BLOCK_SIZE

_DTYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16}
MAX_TOKENS = 1024       # tokens in one fp8_moe call
MAX_SLOTS = 8192        # tokens * top_k in one fp8_moe call


def _call(device: torch.device, fn, *args) -> None:
    """fn(*args, stream) on the current stream of ``device``, which is made the current device for
    the launch where it is not."""
    if device.index == torch.cuda.current_device():
        _lib.check(fn(*args, _stream(device)))
    else:
        with torch.cuda.device(device):
            _lib.check(fn(*args, _stream(device)))


def _rows(t: torch.Tensor) -> int:
    """Row stride in elements; that of a single row is never used, and torch leaves it arbitrary."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _check_rows(t: torch.Tensor, device: torch.device, dtype: torch.dtype):
    assert t.device == device and t.dtype == dtype and t.dim() == 2
    assert t.stride(1) == 1 or t.shape[1] <= 1


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
    assert x.is_cuda and x.dtype in _DTYPES, "x must be a bf16 or fp16 CUDA tensor"
    _check_rows(x, x.device, x.dtype)
    M, K = x.shape
    assert weight.device == x.device and weight.dtype == x.dtype and weight.is_contiguous()
    assert weight.numel() == K and K % BLOCK_SIZE == 0 and K > 0
    if residual is not None:
        _check_rows(residual, x.device, x.dtype)
        assert residual.shape == x.shape
    xq = torch.empty((M, K), dtype=torch.float8_e4m3fn, device=x.device)
    xs = torch.empty((M, K // BLOCK_SIZE), dtype=torch.bfloat16, device=x.device)
    res = torch.empty((M, K), dtype=x.dtype, device=x.device) if residual is not None else None
    y = torch.empty((M, K), dtype=x.dtype, device=x.device) if return_norm else None
    if M == 0:
        return xq, xs, res, y
    _call(x.device, _lib.lib.fp8attn_add_rms_norm_quant, x.data_ptr(), _rows(x),
          residual.data_ptr() if residual is not None else 0,
          _rows(residual) if residual is not None else 0, weight.data_ptr(), float(eps),
          xq.data_ptr(), xs.data_ptr(), res.data_ptr() if res is not None else 0,
          y.data_ptr() if y is not None else 0, M, K, _DTYPES[x.dtype])
    return xq, xs, res, y


def silu_mul_fp8(gate_up: torch.Tensor):
    """gate_up: bf16 or fp16 [M, 2 I] (rows may be strided), gate columns first; I a multiple of 128.
    Returns (hq, h_scale): gate / (1 + exp(-gate)) * up as e4m3 [M, I] with scales bf16 [M, I / 128]."""
    assert gate_up.is_cuda and gate_up.dtype in _DTYPES, "gate_up must be a bf16 or fp16 CUDA tensor"
    _check_rows(gate_up, gate_up.device, gate_up.dtype)
    M, I2 = gate_up.shape
    assert I2 % (2 * BLOCK_SIZE) == 0 and I2 > 0
    hq = torch.empty((M, I2 // 2), dtype=torch.float8_e4m3fn, device=gate_up.device)
    hs = torch.empty((M, I2 // 2 // BLOCK_SIZE), dtype=torch.bfloat16, device=gate_up.device)
    if M == 0:
        return hq, hs
    _call(gate_up.device, _lib.lib.fp8attn_silu_mul_quant, gate_up.data_ptr(), _rows(gate_up),
          hq.data_ptr(), hs.data_ptr(), M, I2 // 2, _DTYPES[gate_up.dtype])
    return hq, hs


def _check_experts(w: torch.Tensor, scale: torch.Tensor, device: torch.device, shape):
    assert w.device == device and w.dtype == torch.float8_e4m3fn and w.is_contiguous()
    assert scale.device == device and scale.dtype == torch.bfloat16 and scale.is_contiguous()
    e, n, k = shape
    assert tuple(w.shape) == (e, n, k), (tuple(w.shape), shape)
    assert tuple(scale.shape) == (e, n // BLOCK_SIZE, k // BLOCK_SIZE)


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
    assert x.is_cuda and x.dtype == torch.bfloat16, "x must be a bf16 CUDA tensor"
    dev = x.device
    _check_rows(x, dev, torch.bfloat16)
    _check_rows(xq, dev, torch.float8_e4m3fn)
    T, H = x.shape
    assert xq.shape == x.shape and H % BLOCK_SIZE == 0 and H > 0
    assert x_scale.device == dev and x_scale.dtype == torch.bfloat16 and x_scale.is_contiguous()
    assert tuple(x_scale.shape) == (T, H // BLOCK_SIZE)
    assert router_weight.device == dev and router_weight.dtype == torch.bfloat16
    assert router_weight.is_contiguous() and router_weight.dim() == 2 and router_weight.shape[1] == H
    E = router_weight.shape[0]
    I = down_weight.shape[-1]
    assert I % BLOCK_SIZE == 0 and I > 0
    _check_experts(gate_up_weight, gate_up_scale, dev, (E, 2 * I, H))
    _check_experts(down_weight, down_scale, dev, (E, H, I))
    out = torch.empty((T, H), dtype=torch.bfloat16, device=dev)
    weights = ids = None
    if return_router:
        weights = torch.empty((T, top_k), dtype=torch.float32, device=dev)
        ids = torch.empty((T, top_k), dtype=torch.int32, device=dev)
    if T > 0:
        nbytes = _lib.lib.fp8attn_fp8_moe_workspace_bytes(T, H, I, E, top_k)
        # scratch of this call alone: calls on other streams and captured graphs share none
        scratch = torch.empty(max(nbytes, 0), dtype=torch.uint8, device=dev)
        _call(dev, _lib.lib.fp8attn_fp8_moe, x.data_ptr(), _rows(x), xq.data_ptr(), _rows(xq),
              x_scale.data_ptr(), router_weight.data_ptr(), gate_up_weight.data_ptr(),
              gate_up_scale.data_ptr(), down_weight.data_ptr(), down_scale.data_ptr(),
              out.data_ptr(), H, weights.data_ptr() if return_router else 0,
              ids.data_ptr() if return_router else 0, T, H, I, E, int(top_k),
              1 if renormalize else 0, scratch.data_ptr(), nbytes,
              workspace(dev, 4).data_ptr() + _lib.WS_ERROR_OFFSET)
    return (out, weights, ids) if return_router else out
