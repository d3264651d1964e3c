"""Calls of the rotary operators and of attention over the 4-bit cache that the documentation allows and that are easily
forgotten."""
import pytest
import torch

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _randn(*shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16)


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _filled(blocks, block, kv, seed):
    from nanovllm_b200.int4_cache import new_kvcache_int4, store_kvcache_int4
    cache = new_kvcache_int4(blocks, block, kv)
    n = blocks * block
    store_kvcache_int4(_randn(n, kv, 128, seed=seed), _randn(n, kv, 128, seed=seed + 1), *cache,
                       torch.arange(n, dtype=torch.int32, device="cuda"))
    return cache


@pytest.mark.parametrize("news,lens", [([1], [3000]), ([5, 1], [900, 40]), ([300, 40, 0], [3000, 800, 16]),
                                       ([700], [700])], ids=str)
def test_workspace_may_hold_anything(news, lens):
    """The joining kernel goes by what the attention kernels have written, whatever stood there."""
    from nanovllm_b200 import _lib
    block, kv, heads = 16, 2, 8
    blocks = sum(-(-n // block) for n in lens)
    cache = _filled(blocks, block, kv, 1)
    table = torch.full((len(lens), max(-(-n // block) for n in lens)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(lens):
        pages = -(-n // block)
        table[i, :pages] = torch.arange(at, at + pages, device="cuda")
        at += pages
    q = _randn(sum(news), heads, 128, seed=3)
    cum = lambda v: _ints(*[sum(v[:i]) for i in range(len(v) + 1)])  # noqa: E731
    cq, ck = cum(news), cum(lens)
    nbytes = _lib.lib.fp8attn_int4_workspace_bytes(len(news), heads, kv, max(news))
    outs = []
    for fill in (0, 255, 127, 1):
        work = torch.full((nbytes,), fill, dtype=torch.uint8, device="cuda")
        out = torch.empty_like(q)
        assert _lib.lib.fp8attn_int4_prefill(
            out.data_ptr(), q.data_ptr(), q.stride(0), *(t.data_ptr() for t in cache), table.data_ptr(), table.stride(0),
            table.shape[1], cq.data_ptr(), ck.data_ptr(), len(news), max(news), heads, kv, 128, blocks, block, SCALE,
            work.data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream) == 0
        outs.append(out)
    assert all(torch.equal(o, outs[0]) for o in outs) and torch.isfinite(outs[0]).all()


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("tokens", [0, 1, 300])
def test_rope_of_keys_alone(tokens, inplace):
    """q without heads: k is turned all the same."""
    from nanovllm_b200.rope import apply_rope, rope_table
    table, pos = rope_table(500, 128), torch.arange(tokens, device="cuda")
    k = _randn(tokens, 4, 128, seed=5)
    want, none = apply_rope(k, None, pos, table)
    assert none is None
    q, given = torch.empty(tokens, 0, 128, dtype=torch.bfloat16, device="cuda"), k.clone()
    torch.full_like(k, 7.0)  # freed at once: an output that nobody writes would hold it
    got_q, got = apply_rope(q, given, pos, table, inplace=inplace)
    assert got_q.shape == q.shape and torch.equal(got, want)
    assert not inplace or got is given


def test_block_table_without_columns():
    """Nothing is seen, as with a table of -1."""
    from nanovllm_b200.int4_cache import int4_decode_attention, int4_prefill_attention
    cache, table = _filled(2, 16, 2, 6), torch.empty(3, 0, dtype=torch.int32, device="cuda")
    out = int4_decode_attention(_randn(3, 8, 128, seed=7), *cache, table, _ints(0, 5, 0), SCALE)
    assert out.shape == (3, 8, 128) and torch.all(out == 0)
    for new in (2, 100):
        out = int4_prefill_attention(_randn(3 * new, 8, 128, seed=8), *cache, table, _ints(0, new, 2 * new, 3 * new),
                                     _ints(0, 0, 30, 30), new, 30, SCALE)
        assert torch.all(out == 0)


def test_a_layer_with_norms():
    """The fused epilogue without a cache of its own, the store and the attention one after another: a prompt, then a token,
    against a float64 layer on the rows as the cache holds them."""
    from nanovllm_b200.int4_cache import (int4_decode_attention, int4_prefill_attention, load_kvcache_int4,
                                          new_kvcache_int4, store_kvcache_int4)
    from nanovllm_b200.qk_epilogue import qk_norm_rope_store
    from nanovllm_b200.rope import rope_table
    heads, kv, n = 8, 2, 100
    qkv, w = _randn(n, (heads + 2 * kv) * 128, seed=9), _randn(128, seed=10)
    table, cache = rope_table(200, 128), new_kvcache_int4(8, 16, kv)
    pages = torch.tensor([[3, 1, 7, 0, 2, 6, 4]], dtype=torch.int32, device="cuda")

    def layer(lo, hi):
        pos = torch.arange(lo, hi, device="cuda")
        q, k = qk_norm_rope_store(qkv[lo:hi], pos, w, w, 1e-6, table, heads, kv, None, None, None, return_k=True)
        slots = (pages[0].long()[pos // 16] * 16 + pos % 16).to(torch.int32)
        store_kvcache_int4(k, qkv[lo:hi, (heads + kv) * 128:].unflatten(1, (kv, 128)), *cache, slots)
        if hi - lo == 1:
            return q, int4_decode_attention(q, *cache, pages, _ints(hi), SCALE)
        return q, int4_prefill_attention(q, *cache, pages, _ints(0, hi - lo), _ints(0, hi), hi - lo, hi, SCALE)

    for lo, hi in ((0, n - 1), (n - 1, n)):
        q, out = layer(lo, hi)
        at = torch.arange(hi, device="cuda")
        k, v = (x.double() for x in load_kvcache_int4(*cache, (pages[0].long()[at // 16] * 16 + at % 16).to(torch.int32)))
        for h in range(heads):
            s = q[:, h].double() @ k[:, h // 4].T * SCALE
            s = s.masked_fill(at[None] > torch.arange(lo, hi, device="cuda")[:, None], -float("inf"))
            want = torch.softmax(s, -1) @ v[:, h // 4]
            # rows read back are rounded to bf16 (2^-9 in the mean square, in the scores and in the values), the output too
            assert (out[:, h].double() - want).norm() <= 2.0 ** -6 * want.norm()
