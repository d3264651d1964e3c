"""Rotary positions: all of a head or part of it, by halves or interleaved pairs, any table.

``apply_rope(q, k, positions, cos_sin_cache)``  turns q and k by their tokens' positions
    (RotaryEmbedding.forward, nanovllm/layers/rotary_embedding.py:37-47, is the case of whole heads by
    halves).  For models without the q/k norm of ``qk_epilogue.qk_norm_rope_store``, and before
    ``int4_cache.store_kvcache_int4``.
``rope_table(...)``  the table of cos and sin, with the usual ways of scaling it for long contexts.

``apply_rope`` launches on ``torch.cuda.current_stream()`` of the tensors' device and never
synchronises, so it can be captured into CUDA graphs.
"""
from __future__ import annotations

import math

import torch

from . import _lib

_DTYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16}
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_empty = torch.empty_strided
_rope = _lib.lib.fp8attn_rope


def apply_rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor,
               cos_sin_cache: torch.Tensor, interleaved: bool = False, inplace: bool = False):
    """(x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin) for the pairs of each head's first R values, in fp32.

    Args:
        q, k: bf16 or fp16 [N, heads, D] (tokens and heads may be strided); k may be None; D even
        positions: int64 [N]; outside the table its first or last row is taken
        cos_sin_cache: fp32 [max_position, (1,) R], cos of R / 2 angles, then sin; R even, up to D
        interleaved: pairs are (2 i, 2 i + 1) in place of (i, i + R / 2)
        inplace: turn q and k where they lie (then no two of their rows may share memory)
    Returns (q, k): contiguous copies, or with ``inplace`` the tensors themselves; k is None without one.
    """
    dtype, device = q.dtype, q.get_device()
    code = _DTYPES.get(dtype)
    assert code is not None and device >= 0, "q must be a bf16 or fp16 CUDA tensor"
    assert q.dim() == 3
    if device != _current_device():
        with torch.cuda.device(device):
            return apply_rope(q, k, positions, cos_sin_cache, interleaved, inplace)
    N, heads, D = q.shape
    q_ts, q_hs, unit = q.stride()
    assert unit == 1
    assert positions.get_device() == device and positions.dtype == torch.int64
    assert positions.is_contiguous() and positions.numel() == N
    assert cos_sin_cache.get_device() == device and cos_sin_cache.dtype == torch.float32
    R, size = cos_sin_cache.shape[-1], cos_sin_cache.numel()
    assert size > 0 and cos_sin_cache.is_contiguous()
    assert D % 2 == 0 and D > 0 and R % 2 == 0 and R <= D
    on = q.device
    kv_heads = k_ptr = k_ts = k_hs = k_out_ptr = 0
    k_out = None
    if k is not None:
        assert k.get_device() == device and k.dtype == dtype and k.dim() == 3
        k_tokens, kv_heads, k_width = k.shape
        k_ts, k_hs, unit = k.stride()
        assert k_tokens == N and k_width == D and unit == 1
        if heads == 0:  # all there is to turn is k
            return (q if inplace else torch.empty_like(q),
                    apply_rope(k, None, positions, cos_sin_cache, interleaved, inplace)[0])
        k_out = k if inplace else _empty((N, kv_heads, D), (kv_heads * D, D, 1), dtype=dtype, device=on)
        k_ptr, k_out_ptr = k.data_ptr(), k_out.data_ptr()
    q_out = q if inplace else _empty((N, heads, D), (heads * D, D, 1), dtype=dtype, device=on)
    if N > 0 and heads > 0:
        out = (q_ts, q_hs, k_ts, k_hs) if inplace else (heads * D, D, kv_heads * D, D)
        rc = _rope(q.data_ptr(), q_ts, q_hs, k_ptr, k_ts, k_hs, positions.data_ptr(),
                   cos_sin_cache.data_ptr(), size // R, q_out.data_ptr(), out[0], out[1], k_out_ptr,
                   out[2], out[3], N, heads, kv_heads, D, R, 1 if interleaved else 0, code,
                   _raw_stream(device))
        if rc:
            _lib.check(rc)
    return q_out, k_out


def rope_table(max_position: int, rotary_dim: int, base: float = 10000.0, scaling: str | None = None,
               factor: float = 1.0, original_max_position: int | None = None, beta_fast: float = 32.0,
               beta_slow: float = 1.0, low_freq_factor: float = 1.0, high_freq_factor: float = 4.0,
               attention_factor: float | None = None, device="cuda") -> torch.Tensor:
    """cos and sin of position * base^(-2 i / R) as ``apply_rope`` reads them, fp32 [max_position, R];
    angles are computed in 64 bits and rounded after their cos and sin.

    ``scaling`` stretches ``original_max_position`` positions by ``factor``:
      None         as trained
      "linear"     every position divided by factor
      "ntk"        the base raised to base * factor^(R / (R - 2)), so that the slowest angle is divided by
                   factor and the fastest is not
      "yarn"       angles that turn less than beta_slow times over the original length are divided by factor,
                   those that turn more than beta_fast times are not, a ramp between them; cos and sin times
                   attention_factor (0.1 ln(factor) + 1 where it is not given)
      "wavelength" the same by wavelength: longer than original / low_freq_factor divided, shorter than
                   original / high_freq_factor not, interpolated between them
    """
    assert max_position > 0 and rotary_dim > 0 and rotary_dim % 2 == 0 and factor >= 1.0
    if scaling in ("yarn", "wavelength"):
        assert original_max_position, f"{scaling} needs original_max_position"
    power = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
    times = 1.0
    if scaling == "ntk":
        assert rotary_dim > 2
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freq = base ** -power
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        # index of the pair that turns n times over the original length
        pair = lambda n: (rotary_dim * math.log(original_max_position / (n * 2 * math.pi))  # noqa: E731
                          / (2 * math.log(base)))
        lo = max(math.floor(pair(beta_fast)), 0)
        hi = min(math.ceil(pair(beta_slow)), rotary_dim - 1)
        ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        freq = freq * (1 - ramp) + freq / factor * ramp
        times = attention_factor if attention_factor is not None else \
            0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    elif scaling == "wavelength":
        assert high_freq_factor > low_freq_factor
        share = ((original_max_position * freq / (2 * math.pi) - low_freq_factor)
                 / (high_freq_factor - low_freq_factor)).clamp(0, 1)  # 1: as trained
        freq = freq * share + freq / factor * (1 - share)
    else:
        assert scaling in (None, "ntk"), f"unknown scaling {scaling!r}"
    angle = torch.arange(max_position, dtype=torch.float64, device=device)[:, None] * freq.to(device)
    return torch.cat([angle.cos() * times, angle.sin() * times], 1).float()
