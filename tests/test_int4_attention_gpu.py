"""int4_decode_attention and int4_prefill_attention against the 64-bit restatement (oracle/int4.py), whose
bounds follow from the kernels' arithmetic; the output's rounding adds 2^-8 of the value."""
import math

import pytest
import torch

from oracle import int4

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _cache(blocks, block, kv, seed, spread=1.0):
    from nanovllm_b200.int4_cache import new_kvcache_int4
    g = _gen(seed)
    cache = new_kvcache_int4(blocks, block, kv)
    for j in range(2):
        x = torch.randn(blocks, kv, block, 128, generator=g, device="cuda")
        x = x * torch.exp2(torch.randint(-2, 3, (blocks, kv, block, 1), generator=g, device="cuda") * spread)
        code, step, low = int4.quantise(x.to(torch.bfloat16))
        cache[j].copy_(int4.pack(code))
        cache[2][..., 2 * j].copy_(step)
        cache[2][..., 2 * j + 1].copy_(low)
    return cache


def _tables(lens, block, seed, extra=0, more=0):
    """Scattered pages; ``extra`` columns of -1, ``more`` pages that nobody uses."""
    counts = [max(0, -(-n // block)) for n in lens]
    page = torch.randperm(sum(counts) + more, generator=torch.Generator().manual_seed(seed))
    table = torch.full((len(lens), max(counts + [1]) + extra), -1, dtype=torch.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = page[at:at + c].to(torch.int32)
        at += c
    return table.cuda(), max(sum(counts) + more, 1)


def _poison(cache, table, lens):
    """NaN in every row that no sequence sees: pages of nobody, rows behind a context."""
    used = torch.zeros(cache[2].shape[0] * cache[2].shape[2], dtype=torch.bool, device="cuda")
    block = cache[2].shape[2]
    for i, n in enumerate(lens):
        at = torch.arange(max(n, 0), device="cuda")
        page = table[i].long()[at // block]
        ok = (page >= 0) & (page < cache[2].shape[0])
        used[(page * block + at % block)[ok]] = True
    hidden = ~used.view(-1, block)
    scale = cache[2].permute(0, 2, 1, 3)
    scale[hidden] = math.nan
    cache[2].copy_(scale.permute(0, 2, 1, 3))


def _assert_near(got, ref, bound, what=""):
    far = (got.double() - ref).abs()
    room = bound + 2.0 ** -8 * (ref.abs() + bound)
    bad = ~(far <= room)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, first at "
                           f"{bad.nonzero()[0].tolist()}: {got[bad][0]} for {ref[bad][0]}, "
                           f"{float((far / room).nan_to_num(math.inf).max()):.2f} of the bound")


def _check_decode(q, cache, table, lens, scale=SCALE):
    from nanovllm_b200.int4_cache import int4_decode_attention
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = int4_decode_attention(q, *cache, table, ctx, scale)
    assert out.shape == q.shape and out.dtype == torch.bfloat16 and out.is_contiguous()
    for i, n in enumerate(lens):
        ref, bound = int4.attention(q[i:i + 1], *cache, table[i], n, scale)
        _assert_near(out[i:i + 1], ref, bound, f"sequence {i} of {n} positions")
    return out


def _check_chunk(q, cache, table, news, lens, scale=SCALE, max_q=None):
    from nanovllm_b200.int4_cache import int4_prefill_attention
    cum = lambda v: torch.tensor([sum(v[:i]) for i in range(len(v) + 1)], dtype=torch.int32,  # noqa: E731
                                 device="cuda")
    out = int4_prefill_attention(q, *cache, table, cum(news), cum(lens), max_q or max(news), max(lens), scale)
    at = 0
    for i, (m, n) in enumerate(zip(news, lens)):
        rows = m * (q.shape[1] // cache[0].shape[1])  # more than 32: the kernel for long chunks
        ref, bound = int4.attention(q[at:at + m], *cache, table[i], n, scale, in_f16=m > 1 and rows > 32)
        _assert_near(out[at:at + m], ref, bound, f"sequence {i}: {m} of {n} positions")
        at += m
    return out


def _q(n, heads, seed, sd=1.5):
    return (torch.randn(n, heads, 128, generator=_gen(seed), device="cuda") * sd).to(torch.bfloat16)


LENS = [[1], [16], [31, 33], [127, 128, 129], [700], [0, 5, 0, 1], [3000, 1, 64, 257, 0, 1029]]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("heads,kv,block", [(32, 8, 256), (8, 8, 16), (16, 2, 48), (5, 1, 64), (32, 2, 16),
                                            (40, 2, 32), (64, 1, 128), (3, 3, 16)])
def test_decode(lens, heads, kv, block):
    table, blocks = _tables(lens, block, 1, extra=2, more=3)
    cache = _cache(blocks, block, kv, 2)
    _poison(cache, table, lens)
    _check_decode(_q(len(lens), heads, 3), cache, table, lens)


@pytest.mark.parametrize("heads,kv", [(32, 8), (8, 1)])
def test_decode_many_sequences(heads, kv):
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 200, (700,), generator=g).tolist()
    table, blocks = _tables(lens, 16, 6)
    cache = _cache(blocks, 16, kv, 7)
    _check_decode(_q(len(lens), heads, 8), cache, table, lens)


def test_decode_thousands_of_sequences():
    lens = [(7 * i) % 40 for i in range(5000)]
    table, blocks = _tables(lens, 16, 6)
    cache = _cache(blocks, 16, 1, 7)
    from nanovllm_b200.int4_cache import int4_decode_attention
    q = _q(len(lens), 2, 8)
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = int4_decode_attention(q, *cache, table, ctx, SCALE)
    for i in list(range(0, 5000, 61)) + [4999]:
        ref, bound = int4.attention(q[i:i + 1], *cache, table[i], lens[i], SCALE)
        _assert_near(out[i:i + 1], ref, bound, f"sequence {i}")


def test_decode_long_context_with_late_peaks():
    """Cuts of one sequence over all CTAs; maxima that grow late, in rows of the largest steps."""
    n = 131071
    table, blocks = _tables([n], 256, 9)
    cache = _cache(blocks, 256, 2, 10)
    q = _q(1, 8, 11)
    for pos in (20000, 90001, 131070):
        page = int(table[0, pos // 256])
        row = (q[0, 0].float() * (1 + pos / 60000)).to(torch.bfloat16)
        code, step, low = int4.quantise(row)
        cache[0][page, 0, pos % 256] = int4.pack(code)
        cache[2][page, 0, pos % 256, 0], cache[2][page, 0, pos % 256, 1] = step, low
    _check_decode(q, cache, table, [n])


def test_decode_pages_that_are_not_there():
    lens = [600, 300]
    table, blocks = _tables(lens, 48, 12)
    table[0, 3], table[0, 7], table[1, 0] = -1, blocks + 5, -2
    cache = _cache(blocks, 48, 2, 13)
    _poison(cache, table, lens)
    _check_decode(_q(2, 8, 14), cache, table, lens)
    table[:] = -1
    out = _check_decode(_q(2, 8, 14), cache, table, lens)
    assert torch.all(out == 0)


def test_decode_context_past_the_table_and_negative():
    table, blocks = _tables([64, 64, 64], 16, 15)
    cache = _cache(blocks, 16, 2, 16)
    q = _q(3, 4, 17)
    out = _check_decode(q, cache, table, [64, 1000, -3])
    assert torch.all(out[2] == 0)


def test_decode_nan_row_reaches_its_head_only():
    lens = [200, 200]
    table, blocks = _tables(lens, 32, 18)
    cache = _cache(blocks, 32, 2, 19)
    page = int(table[1, 2])
    cache[2][page, 1, 7, 2] = math.nan          # a step of V, kv head 1 of sequence 1
    from nanovllm_b200.int4_cache import int4_decode_attention
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = _q(2, 4, 20)
    out = int4_decode_attention(q, *cache, table, ctx, SCALE)
    assert torch.isnan(out[1, 2:]).all() and torch.isfinite(out[0]).all() and torch.isfinite(out[1, :2]).all()
    cache[2][page, 1, 7, 2], cache[2][page, 1, 7, 0] = 0.1, math.nan   # a step of K
    out = int4_decode_attention(q, *cache, table, ctx, SCALE)
    assert torch.isnan(out[1, 2:]).all() and torch.isfinite(out[0]).all() and torch.isfinite(out[1, :2]).all()


@pytest.mark.parametrize("sd,spread", [(0.0, 1.0), (1e-30, 1.0), (40.0, 1.0), (1.5, 5.0)])
def test_decode_ranges(sd, spread):
    """q of zeros, tiny and large; steps that differ by 2^20."""
    lens = [500, 77]
    table, blocks = _tables(lens, 64, 21)
    cache = _cache(blocks, 64, 2, 22, spread)
    _check_decode(_q(2, 8, 23, sd), cache, table, lens)


def test_decode_strided_q_and_wide_table():
    lens = [100, 333]
    table, blocks = _tables(lens, 16, 24)
    cache = _cache(blocks, 16, 2, 25)
    wide = torch.randn(2, 20 * 128, generator=_gen(26), device="cuda").to(torch.bfloat16)
    big = torch.full((2, table.shape[1] + 9), -1, dtype=torch.int32, device="cuda")
    big[:, :table.shape[1]] = table
    _check_decode(wide[:, 512:512 + 8 * 128].view(2, 8, 128), cache, big[:, :table.shape[1]], lens)


def test_decode_far_pages():
    """Byte offsets past 2^32."""
    blocks, block, kv = 41000, 256, 8
    from nanovllm_b200.int4_cache import new_kvcache_int4
    cache = new_kvcache_int4(blocks, block, kv)
    small = _cache(3, block, kv, 27)
    for t, s in zip(cache, small):
        t[-3:] = s
    table = torch.tensor([[blocks - 1, blocks - 3, blocks - 2]], dtype=torch.int32, device="cuda")
    _check_decode(_q(1, 32, 28), cache, table, [700])


def test_decode_same_bits_again_and_in_graphs():
    from nanovllm_b200.int4_cache import int4_decode_attention
    lens = [4000, 3, 900, 1200, 0]
    table, blocks = _tables(lens, 64, 29)
    cache = _cache(blocks, 64, 4, 30)
    q, ctx = _q(5, 16, 31), torch.tensor(lens, dtype=torch.int32, device="cuda")
    call = lambda: int4_decode_attention(q, *cache, table, ctx, SCALE)  # noqa: E731
    first = call()
    assert all(torch.equal(call(), first) for _ in range(5))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):  # two graphs, replayed at once on two streams
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = call()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], first) and torch.equal(outs[1], first) and torch.equal(eager, first)
    # other lengths in the same graph
    ctx.copy_(torch.tensor([17, 0, 900, 1, 0], dtype=torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], call())


CHUNKS = [([1], [1]), ([5], [700]), ([5, 1, 3], [64, 1, 500]), ([9, 2], [9, 300]), ([16], [1000]),
          ([33, 100], [33, 1000]), ([130], [130]), ([257, 1, 40], [600, 900, 40])]


@pytest.mark.parametrize("news,lens", CHUNKS, ids=str)
@pytest.mark.parametrize("heads,kv,block", [(32, 8, 256), (4, 4, 16), (16, 2, 48), (5, 1, 64), (24, 1, 32)])
def test_chunk(news, lens, heads, kv, block):
    table, blocks = _tables(lens, block, 32, extra=1, more=2)
    cache = _cache(blocks, block, kv, 33)
    _poison(cache, table, lens)
    _check_chunk(_q(sum(news), heads, 34), cache, table, news, lens)


def test_chunk_is_decode_for_single_tokens():
    from nanovllm_b200.int4_cache import int4_decode_attention
    lens = [900, 33, 5]
    table, blocks = _tables(lens, 16, 35)
    cache = _cache(blocks, 16, 2, 36)
    q = _q(3, 8, 37)
    out = _check_chunk(q, cache, table, [1, 1, 1], lens)
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    assert torch.equal(out, int4_decode_attention(q, *cache, table, ctx, SCALE))


@pytest.mark.parametrize("news,lens", [([3, 0, 4], [100, 50, 9]), ([5, 2], [3, 2]), ([4], [0]), ([200, 150], [100, 7])],
                         ids=str)
def test_chunk_empty_and_rows_that_see_nothing(news, lens):
    """Sequences without new tokens; more new tokens than positions: the first rows see nothing."""
    table, blocks = _tables(lens, 16, 38)
    cache = _cache(blocks, 16, 2, 39)
    _poison(cache, table, lens)
    _check_chunk(_q(sum(news), 8, 40), cache, table, news, lens)


def test_chunk_pages_that_are_not_there():
    news, lens = [7, 150], [300, 700]
    table, blocks = _tables(lens, 16, 41)
    table[0, 2], table[1, 5], table[1, 30] = -1, blocks + 1, -1
    cache = _cache(blocks, 16, 2, 42)
    _poison(cache, table, lens)
    _check_chunk(_q(sum(news), 8, 43), cache, table, news, lens)


@pytest.mark.parametrize("news,lens,heads,kv", [([3, 1], [70, 20], 48, 1), ([300], [300], 48, 1), ([1, 5, 64], [9, 150, 64], 28, 4),
                                                ([260, 3], [261, 700], 3, 1), ([6], [5000], 3, 3), ([11], [400], 2, 1)],
                         ids=str)
def test_chunk_groups(news, lens, heads, kv):
    """Groups that divide no tile, and more query heads of a kv head than a row group has rows."""
    table, blocks = _tables(lens, 32, 46)
    cache = _cache(blocks, 32, kv, 47)
    _poison(cache, table, lens)
    _check_chunk(_q(sum(news), heads, 48), cache, table, news, lens)


@pytest.mark.parametrize("news,lens", [([300], [9000]), ([40, 1, 700], [6000, 3000, 700]), ([16], [20000]), ([129] * 3, [4000] * 3)],
                         ids=str)
@pytest.mark.parametrize("spread", [1.0, 5.0])
def test_chunk_cut_over_ctas(news, lens, spread):
    """Items of many tiles in several CTAs, whose parts are joined; steps that differ by 2^20."""
    table, blocks = _tables(lens, 64, 49)
    cache = _cache(blocks, 64, 1, 50, spread)
    _check_chunk(_q(sum(news), 4, 51), cache, table, news, lens)


@pytest.mark.parametrize("new", [1, 2, 5])
def test_long_pieces(new):
    """So much work that a CTA has thousands of positions of a pair: sums put aside on the way, where a row has seen
    nothing yet, where its maximum and V's largest step come after that."""
    from nanovllm_b200.int4_cache import int4_decode_attention, int4_prefill_attention
    seqs, n, block, kv, heads = 40, 20000, 64, 8, 32
    pages = -(-n // block)
    cache = _cache(3 * pages, block, kv, 71)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(seqs, 1)  # all but two share their pages
    table[3] += pages
    table[5] += 2 * pages
    table[3, :170] = -1                                      # sees nothing in its first 10,880 positions
    cache[2][2 * pages + 180:, :, :, 2:] *= 2.0 ** 12        # V's steps and lowest values grow late
    q = _q(seqs * new, heads, 72)
    late = int(table[5, 250])
    for h in range(kv):                                      # and the rows' maxima
        code, step, low = int4.quantise((q[5 * new, 4 * h].float() * 1.5).to(torch.bfloat16))
        cache[0][late, h, 7] = int4.pack(code)
        cache[2][late, h, 7, 0], cache[2][late, h, 7, 1] = step, low
    cum = lambda m: torch.arange(seqs + 1, dtype=torch.int32, device="cuda") * m  # noqa: E731
    if new == 1:
        out = int4_decode_attention(q, *cache, table, torch.full((seqs,), n, dtype=torch.int32, device="cuda"), SCALE)
    else:
        out = int4_prefill_attention(q, *cache, table, cum(new), cum(n), new, n, SCALE)
    for i in (0, 3, 5, 17, seqs - 1):
        at = slice(i * new, (i + 1) * new)
        ref, bound = int4.attention(q[at], *cache, table[i], n, SCALE)
        _assert_near(out[at], ref, bound, f"sequence {i}")


def test_chunk_many_sequences():
    g = torch.Generator().manual_seed(52)
    news = torch.randint(0, 4, (600,), generator=g).tolist()
    for i in (3, 77, 400):
        news[i] = 70
    lens = [m + int(x) for m, x in zip(news, torch.randint(0, 150, (600,), generator=g))]
    table, blocks = _tables(lens, 16, 53)
    cache = _cache(blocks, 16, 2, 54)
    _check_chunk(_q(sum(news), 8, 55), cache, table, news, lens)


@pytest.mark.parametrize("scale", [-0.1, 0.0, 1.0])
@pytest.mark.parametrize("news,lens", [([1, 3], [200, 90]), ([150], [333])], ids=str)
def test_scales(news, lens, scale):
    table, blocks = _tables(lens, 16, 56)
    cache = _cache(blocks, 16, 2, 57)
    _check_chunk(_q(sum(news), 8, 58, 0.5), cache, table, news, lens, scale)


@pytest.mark.parametrize("column,value", [(0, math.nan), (1, math.nan), (2, math.nan), (3, math.nan), (2, math.inf),
                                          (3, -math.inf)])
@pytest.mark.parametrize("new,heads", [(2, 4), (6, 4), (9, 4), (150, 8)])
def test_chunk_bad_row_reaches_rows_that_see_it(new, heads, column, value):
    """A step or lowest value that is no number, in a row among the new tokens: queries before it and other kv heads
    keep their bits."""
    from nanovllm_b200.int4_cache import int4_prefill_attention
    lens, at = [400, 300], new - 2
    table, blocks = _tables(lens, 32, 59)
    cache = _cache(blocks, 32, 2, 60)
    q = _q(new + 3, heads, 61)
    cu = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    call = lambda: int4_prefill_attention(q, *cache, table, cu(0, new, new + 3), cu(0, 400, 700), max(new, 3), 400,
                                          SCALE)  # noqa: E731
    clean = call()
    pos = 400 - new + at
    cache[2][int(table[0, pos // 32]), 1, pos % 32, column] = value
    out = call()
    half = heads // 2
    assert torch.equal(out[new:], clean[new:]) and torch.equal(out[:, :half], clean[:, :half])
    assert torch.equal(out[:at], clean[:at])
    assert not torch.isfinite(out[at:new, half:]).any()


def test_infinite_and_nan_queries_stay_in_their_rows():
    from nanovllm_b200.int4_cache import int4_prefill_attention
    news, lens = [5, 140], [300, 400]
    table, blocks = _tables(lens, 16, 62)
    cache = _cache(blocks, 16, 2, 63)
    q = _q(145, 8, 64)
    cu = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    call = lambda: int4_prefill_attention(q, *cache, table, cu(0, 5, 145), cu(0, 300, 700), 140, 400, SCALE)  # noqa: E731
    clean = call()
    for row, head, value in ((1, 2, math.nan), (3, 7, math.inf), (60, 0, math.nan), (100, 5, -math.inf)):
        q[row, head, 17] = value
    out = call()
    hit = torch.zeros(145, 8, dtype=torch.bool, device="cuda")
    for row, head in ((1, 2), (3, 7), (60, 0), (100, 5)):
        hit[row, head] = True
    assert torch.equal(out[~hit], clean[~hit]) and not torch.isfinite(out[hit]).any()


def test_chunk_same_bits_again_in_graphs_and_on_streams():
    from nanovllm_b200.int4_cache import int4_prefill_attention
    news, lens = [500, 1, 7, 90], [3000, 5000, 800, 90]
    table, blocks = _tables(lens, 64, 65)
    cache = _cache(blocks, 64, 2, 66)
    q = _q(sum(news) + 9, 8, 67)
    cum = lambda v: torch.tensor([sum(v[:i]) for i in range(len(v) + 1)], dtype=torch.int32, device="cuda")  # noqa: E731
    cq, ck = cum(news), cum(lens)
    call = lambda: int4_prefill_attention(q, *cache, table, cq, ck, 500, 5000, SCALE)[:sum(news)]  # noqa: E731
    first = call()
    assert all(torch.equal(call(), first) for _ in range(3))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = call()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], first) and torch.equal(outs[1], first) and torch.equal(eager, first)
    # other lengths in the same graph: the batch is padded by sequences without new tokens
    cq.copy_(torch.tensor([0, 3, 40, 40, 40], dtype=torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0][:40], call()[:40])


def test_chunk_rows_behind_the_last_sequence_are_left():
    """Through the C interface, whose caller owns the output: rows of no sequence keep what they held, also where a
    chunk ends inside a tile of rows."""
    from nanovllm_b200 import _lib
    for news, lens in (([5], [70]), ([131], [200]), ([300, 2], [300, 40])):
        table, blocks = _tables(lens, 16, 68)
        cache = _cache(blocks, 16, 2, 69)
        n = sum(news)
        q = _q(n, 8, 70)
        cum = lambda v: torch.tensor([sum(v[:i]) for i in range(len(v) + 1)], dtype=torch.int32, device="cuda")  # noqa: E731
        cq, ck = cum(news), cum(lens)
        out = torch.full((n + 300, 8, 128), 7.0, dtype=torch.bfloat16, device="cuda")
        nbytes = _lib.lib.fp8attn_int4_workspace_bytes(len(news), 8, 2, max(news))
        work = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
        args = lambda size: (out.data_ptr(), q.data_ptr(), q.stride(0), *(t.data_ptr() for t in cache), table.data_ptr(),  # noqa: E731
                             table.stride(0), table.shape[1], cq.data_ptr(), ck.data_ptr(), len(news), max(news), 8, 2, 128,
                             blocks, 16, SCALE, work.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
        assert _lib.lib.fp8attn_int4_prefill(*args(nbytes - 1)) != 0
        assert "workspace" in _lib.lib.fp8attn_last_error().decode()
        assert torch.all(out == 7)
        assert _lib.lib.fp8attn_int4_prefill(*args(nbytes)) == 0
        assert torch.all(out[n:] == 7) and not torch.any(torch.all(out[:n] == 7, -1))


def test_first_call_of_a_process_inside_a_capture():
    code = """
import torch
from nanovllm_b200.int4_cache import int4_prefill_attention, new_kvcache_int4, store_kvcache_int4
cache = new_kvcache_int4(8, 16, 2)
kv = torch.randn(100, 2, 128, device="cuda").to(torch.bfloat16)
slots = torch.arange(100, dtype=torch.int32, device="cuda")
q = torch.randn(100, 8, 128, device="cuda").to(torch.bfloat16)
table = torch.arange(8, dtype=torch.int32, device="cuda")[None]
cu = torch.tensor([0, 100], dtype=torch.int32, device="cuda")
call = lambda: (store_kvcache_int4(kv, kv, *cache, slots), int4_prefill_attention(q, *cache, table, cu, cu, 100, 100, 0.1))[1]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = call()
g.replay()
assert torch.equal(out, call()) and torch.isfinite(out).all()
print("same")
"""
    import os
    import subprocess
    import sys
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                          env={**os.environ, "PYTHONPATH": os.pathsep.join(sys.path)})
    assert done.returncode == 0 and "same" in done.stdout, done.stderr


def test_no_wait_has_run_out():
    from nanovllm_b200 import fp8_attention
    assert fp8_attention.device_error() == 0


def test_a_layer_of_steps():
    """Rotary, store and attention one after another, as a server calls them: a prompt in two chunks, then single
    tokens, and the same through a captured graph."""
    from nanovllm_b200.int4_cache import (int4_decode_attention, int4_prefill_attention, load_kvcache_int4,
                                          new_kvcache_int4, store_kvcache_int4)
    from nanovllm_b200.rope import apply_rope, rope_table
    heads, kv, block, prompt, steps = 8, 2, 16, 150, 5
    g = _gen(44)
    cache = new_kvcache_int4(20, block, kv)
    cos_sin = rope_table(400, 128, base=1e6, scaling="yarn", factor=4.0, original_max_position=100)
    table = torch.randperm(20, generator=torch.Generator().manual_seed(45))[:12].to(torch.int32).cuda()[None]
    total = prompt + steps
    qkv = torch.randn(total, heads + 2 * kv, 128, generator=g, device="cuda").to(torch.bfloat16)

    def layer(rows, positions, slots, ctx, attend):
        q, k = apply_rope(rows[:, :heads], rows[:, heads:heads + kv], positions, cos_sin)
        store_kvcache_int4(k, rows[:, heads + kv:], *cache, slots)
        return q, attend(q, ctx)

    slot = lambda pos: (table[0].long()[pos // block] * block + pos % block).to(torch.int32)  # noqa: E731
    seen = []
    for lo, hi in ((0, 100), (100, prompt)):
        pos = torch.arange(lo, hi, device="cuda")
        cu = lambda n: torch.tensor([0, n], dtype=torch.int32, device="cuda")  # noqa: E731
        q, out = layer(qkv[lo:hi], pos, slot(pos), None, lambda q, _: int4_prefill_attention(
            q, *cache, table, cu(hi - lo), cu(hi), hi - lo, hi, SCALE))
        ref, bound = int4.attention(q, *cache, table[0], hi, SCALE, in_f16=True)
        _assert_near(out, ref, bound, f"chunk to {hi}")
        seen.append(q)
    rows, pos = qkv[prompt:prompt + 1].clone(), torch.tensor([prompt], device="cuda")
    slots, ctx = slot(pos), torch.tensor([prompt + 1], dtype=torch.int32, device="cuda")
    attend = lambda q, c: int4_decode_attention(q, *cache, table, c, SCALE)  # noqa: E731
    layer(rows, pos, slots, ctx, attend)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, out = layer(rows, pos, slots, ctx, attend)
    for i in range(steps):
        rows.copy_(qkv[prompt + i:prompt + i + 1])
        pos.fill_(prompt + i)
        slots.copy_(slot(pos))
        ctx.fill_(prompt + i + 1)
        graph.replay()
        torch.cuda.synchronize()
        ref, bound = int4.attention(q, *cache, table[0], prompt + i + 1, SCALE)
        _assert_near(out, ref, bound, f"token {i}")
    # the cache holds the turned keys, each within half a step
    k, _ = load_kvcache_int4(*cache, slot(torch.arange(total, device="cuda")))
    want = apply_rope(qkv[:, heads:heads + kv], None, torch.arange(total, device="cuda"), cos_sin)[0].double()
    step = (want.amax(-1, keepdim=True) - want.amin(-1, keepdim=True)) / 15
    assert torch.all((k.double() - want).abs() <= step * 0.54 + k.double().abs() * 2.0 ** -8)
