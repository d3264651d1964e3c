"""A paged key/value cache of 4-bit codes, and the attention that reads it: about half the bytes of the
e4m3 cache of ``attention`` and ``fp8_attention``, so twice the context in the same memory.

``new_kvcache_int4(num_blocks, block_size, num_kv_heads)``          the three tensors of a cache
``store_kvcache_int4(key, value, *cache, slot_mapping)``            quantises rows as it writes them
``load_kvcache_int4(*cache, slot_mapping)``                         reads rows back as bf16
``int4_decode_attention(q, *cache, block_tables, context_lens, softmax_scale)``
``int4_prefill_attention(q, *cache, block_tables, cu_seqlens_q, cu_seqlens_k, max_seqlen_q,
    max_seqlen_k, softmax_scale)``

A row (one token of one kv head, 128 values) is held as its lowest value, a step (both bf16) and 128
codes of 4 bits, and stands for low + step * code; include/fp8attn.h has the layout.  The arguments are
those of ``store_kvcache``, ``fp8_decode_attention`` and ``fp8_prefill_attention`` with the cache
(k_cache, v_cache, kv_scale) in place of theirs; the reference has an e4m3 cache only
(nanovllm/layers/attention.py:11-40, nanovllm/kernels/fp8_attention.py:173-207, :314-353).  One layer of a
step:

    q, k = apply_rope(q, k, positions, cos_sin_cache)
    store_kvcache_int4(k, v, *cache, slot_mapping)
    o = int4_decode_attention(q, *cache, block_tables, context_lens, softmax_scale)

and of a model with q/k norms, the first call without a cache of its own:

    q, k = qk_norm_rope_store(qkv, positions, q_norm_weight, k_norm_weight, eps, cos_sin_cache, num_heads,
                              num_kv_heads, None, None, None, return_k=True)
    store_kvcache_int4(k, v, *cache, slot_mapping)

All launch on ``torch.cuda.current_stream()`` of the tensors' device, allocate outputs and scratch with
``torch.empty`` (scratch is one call's own) and never synchronise or read device memory on the host, so
they can be captured into CUDA graphs.  A device wait of the attention that gives up is recorded in a word
of the library's own (``fp8_attention.device_error``).
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from .fp8_attention import _INT4_DEVICES

HEAD_DIM = 128
_BF16, _U8, _I32 = torch.bfloat16, torch.uint8, torch.int32

_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_empty = torch.empty_strided
_store = _lib.lib.fp8attn_int4_store
_load = _lib.lib.fp8attn_int4_load
_decode = _lib.lib.fp8attn_int4_decode
_prefill = _lib.lib.fp8attn_int4_prefill


def new_kvcache_int4(num_blocks: int, block_size: int, num_kv_heads: int, device="cuda"):
    """(k_cache, v_cache, kv_scale): uint8 [num_blocks, num_kv_heads, block_size, 64] twice and bf16
    [num_blocks, num_kv_heads, block_size, 4] (k step, k low, v step, v low), all zeros."""
    assert num_blocks > 0 and num_kv_heads > 0 and block_size > 0 and block_size % 16 == 0
    shape = (num_blocks, num_kv_heads, block_size)
    return (torch.zeros(*shape, HEAD_DIM // 2, dtype=_U8, device=device),
            torch.zeros(*shape, HEAD_DIM // 2, dtype=_U8, device=device),
            torch.zeros(*shape, 4, dtype=_BF16, device=device))


def _check_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, kv_scale: torch.Tensor, device: int):
    assert k_cache.get_device() == device and v_cache.get_device() == device
    assert kv_scale.get_device() == device
    assert k_cache.dtype == _U8 and v_cache.dtype == _U8 and kv_scale.dtype == _BF16
    shape = k_cache.shape
    assert len(shape) == 4 and shape[3] == HEAD_DIM // 2 and v_cache.shape == shape
    assert kv_scale.shape == (*shape[:3], 4)
    assert k_cache.is_contiguous() and v_cache.is_contiguous() and kv_scale.is_contiguous()
    return shape


def store_kvcache_int4(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                       v_cache: torch.Tensor, kv_scale: torch.Tensor,
                       slot_mapping: torch.Tensor) -> None:
    """Quantises row i of ``key`` and ``value`` (bf16 [N, num_kv_heads, 128], tokens and heads may be
    strided) into slot ``slot_mapping[i]`` (int32 [N]; page * block_size + place).  Slots that are -1 or
    outside the cache are skipped; the others must differ.  A row with a NaN or an infinity reads as NaN."""
    device = key.get_device()
    assert device >= 0 and key.dtype == _BF16, "key must be a bf16 CUDA tensor"
    assert value.get_device() == device and value.dtype == _BF16
    assert key.dim() == 3
    if device != _current_device():
        with torch.cuda.device(device):
            return store_kvcache_int4(key, value, k_cache, v_cache, kv_scale, slot_mapping)
    num_blocks, kv_heads, block_size, _ = _check_cache(k_cache, v_cache, kv_scale, device)
    shape = key.shape
    N = shape[0]
    assert shape[1] == kv_heads and shape[2] == HEAD_DIM and value.shape == shape
    (k_ts, k_hs, k_unit), (v_ts, v_hs, v_unit) = key.stride(), value.stride()
    assert k_unit == 1 and v_unit == 1
    assert slot_mapping.get_device() == device and slot_mapping.dtype == _I32
    assert slot_mapping.is_contiguous() and slot_mapping.numel() == N
    rc = _store(key.data_ptr(), k_ts, k_hs, value.data_ptr(), v_ts, v_hs, k_cache.data_ptr(),
                v_cache.data_ptr(), kv_scale.data_ptr(), slot_mapping.data_ptr(), N, kv_heads,
                HEAD_DIM, num_blocks, block_size, _raw_stream(device))
    if rc:
        _lib.check(rc)


def load_kvcache_int4(k_cache: torch.Tensor, v_cache: torch.Tensor, kv_scale: torch.Tensor,
                      slot_mapping: torch.Tensor):
    """(key, value) bf16 [N, num_kv_heads, 128]: low + step * code of the rows at ``slot_mapping`` (int32 [N],
    any order, repeats allowed), rounded once; zeros for slots that are -1 or outside the cache."""
    device = k_cache.get_device()
    assert device >= 0, "the cache must be CUDA tensors"
    if device != _current_device():
        with torch.cuda.device(device):
            return load_kvcache_int4(k_cache, v_cache, kv_scale, slot_mapping)
    num_blocks, kv_heads, block_size, _ = _check_cache(k_cache, v_cache, kv_scale, device)
    assert slot_mapping.get_device() == device and slot_mapping.dtype == _I32
    assert slot_mapping.is_contiguous() and slot_mapping.dim() == 1
    N = slot_mapping.shape[0]
    shape, strides = (N, kv_heads, HEAD_DIM), (kv_heads * HEAD_DIM, HEAD_DIM, 1)
    on = k_cache.device
    key = _empty(shape, strides, dtype=_BF16, device=on)
    value = _empty(shape, strides, dtype=_BF16, device=on)
    rc = _load(k_cache.data_ptr(), v_cache.data_ptr(), kv_scale.data_ptr(), slot_mapping.data_ptr(),
               key.data_ptr(), value.data_ptr(), N, kv_heads, HEAD_DIM, num_blocks, block_size,
               _raw_stream(device))
    if rc:
        _lib.check(rc)
    return key, value


@functools.lru_cache(maxsize=1024)
def _scratch_bytes(device: int, num_seqs: int, heads: int, kv_heads: int, max_q: int) -> int:
    """On the current device, which ``device`` stands for.  A failure is raised, and so not remembered."""
    nbytes = _lib.lib.fp8attn_int4_workspace_bytes(num_seqs, heads, kv_heads, max_q)
    if nbytes < 0:
        _lib.check(_lib.EINVAL)
    return nbytes


def int4_decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                          kv_scale: torch.Tensor, block_tables: torch.Tensor,
                          context_lens: torch.Tensor, softmax_scale: float) -> torch.Tensor:
    """
    Args:
        q: [batch_size, num_heads, 128] bf16 (rows may be strided)
        k_cache, v_cache, kv_scale: the cache; num_heads a multiple of its num_kv_heads
        block_tables: [batch_size, max_num_blocks] int32 (-1 padded; positions in pages that are not
            in the cache are masked)
        context_lens: [batch_size] int32, each sequence's positions (its new token's included)
        softmax_scale: attention scaling factor (1/sqrt(128))
    Returns:
        [batch_size, num_heads, 128] attention output (bf16); zeros where nothing is seen
    """
    device = q.get_device()
    assert device >= 0 and q.dtype == _BF16, "q must be a bf16 CUDA tensor"
    if device != _current_device():
        with torch.cuda.device(device):
            return int4_decode_attention(q, k_cache, v_cache, kv_scale, block_tables, context_lens,
                                         softmax_scale)
    assert q.dim() == 3
    batch, heads, dim = q.shape
    row, head, unit = q.stride()
    assert dim == HEAD_DIM and unit == 1 and (head == HEAD_DIM or heads == 1)
    num_blocks, kv_heads, block_size, _ = _check_cache(k_cache, v_cache, kv_scale, device)
    assert block_tables.get_device() == device and block_tables.dtype == _I32 and block_tables.dim() == 2
    sequences, columns = block_tables.shape
    table_row, unit = block_tables.stride()
    assert sequences >= batch and unit == 1
    assert context_lens.get_device() == device and context_lens.dtype == _I32
    assert context_lens.is_contiguous() and context_lens.numel() >= batch
    width = heads * HEAD_DIM
    on = q.device
    out = _empty((batch, heads, HEAD_DIM), (width, HEAD_DIM, 1), dtype=_BF16, device=on)
    if batch == 0:
        return out
    _INT4_DEVICES.add(device)
    nbytes = _scratch_bytes(device, batch, heads, kv_heads, 1)
    scratch = _empty((nbytes,), (1,), dtype=_U8, device=on)
    # the row stride of a single row is never used, and torch leaves it arbitrary
    rc = _decode(out.data_ptr(), q.data_ptr(), row if batch > 1 else width, k_cache.data_ptr(),
                 v_cache.data_ptr(), kv_scale.data_ptr(), block_tables.data_ptr(),
                 table_row if batch > 1 else columns, columns, context_lens.data_ptr(),
                 batch, heads, kv_heads, HEAD_DIM, num_blocks, block_size, softmax_scale,
                 scratch.data_ptr(), nbytes, _raw_stream(device))
    if rc:
        _lib.check(rc)
    return out


def int4_prefill_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                           kv_scale: torch.Tensor, block_tables: torch.Tensor,
                           cu_seqlens_q: torch.Tensor, cu_seqlens_k: torch.Tensor, max_seqlen_q: int,
                           max_seqlen_k: int, softmax_scale: float) -> torch.Tensor:
    """Causal attention of each sequence's new tokens (the last of its positions, stored in the cache
    before) over all of its positions in the cache: chunked prefill, prompts, speculative verification.

    Args:
        q: [num_tokens, num_heads, 128] bf16 (rows may be strided), the sequences' new tokens one after another
        k_cache, v_cache, kv_scale, block_tables: as ``int4_decode_attention``'s
        cu_seqlens_q, cu_seqlens_k: [num_seqs + 1] int32, new tokens and positions before each sequence
        max_seqlen_q: the most new tokens of a sequence; max_seqlen_k is not used
    Returns bf16 [num_tokens, num_heads, 128]; rows that see nothing are zeros, rows behind the last
    sequence's are not written.
    """
    device = q.get_device()
    assert device >= 0 and q.dtype == _BF16, "q must be a bf16 CUDA tensor"
    if device != _current_device():
        with torch.cuda.device(device):
            return int4_prefill_attention(q, k_cache, v_cache, kv_scale, block_tables, cu_seqlens_q,
                                          cu_seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale)
    assert q.dim() == 3
    tokens, heads, dim = q.shape
    row, head, unit = q.stride()
    assert dim == HEAD_DIM and unit == 1 and (head == HEAD_DIM or heads == 1)
    num_blocks, kv_heads, block_size, _ = _check_cache(k_cache, v_cache, kv_scale, device)
    for cu in (cu_seqlens_q, cu_seqlens_k):
        assert cu.get_device() == device and cu.dtype == _I32 and cu.is_contiguous()
    num_seqs = cu_seqlens_q.numel() - 1
    assert cu_seqlens_k.numel() >= num_seqs + 1
    assert block_tables.get_device() == device and block_tables.dtype == _I32 and block_tables.dim() == 2
    sequences, columns = block_tables.shape
    table_row, unit = block_tables.stride()
    assert sequences >= num_seqs and unit == 1
    width = heads * HEAD_DIM
    on = q.device
    out = _empty((tokens, heads, HEAD_DIM), (width, HEAD_DIM, 1), dtype=_BF16, device=on)
    if tokens == 0 or num_seqs <= 0:
        return out
    # no sequence has more new tokens than there are rows
    max_q = min(int(max_seqlen_q), tokens)
    _INT4_DEVICES.add(device)
    nbytes = _scratch_bytes(device, num_seqs, heads, kv_heads, max_q)
    scratch = _empty((nbytes,), (1,), dtype=_U8, device=on)
    rc = _prefill(out.data_ptr(), q.data_ptr(), row if tokens > 1 else width,
                  k_cache.data_ptr(), v_cache.data_ptr(), kv_scale.data_ptr(),
                  block_tables.data_ptr(), table_row if num_seqs > 1 else columns, columns,
                  cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(), num_seqs, max_q, heads, kv_heads,
                  HEAD_DIM, num_blocks, block_size, softmax_scale, scratch.data_ptr(), nbytes,
                  _raw_stream(device))
    if rc:
        _lib.check(rc)
    return out
