"""Attention over the 4-bit cache at the ends of bf16's range and between rows of very different size, held to the 2-norm
of each output row (oracle/int4.py, ``attention_norm``)."""
import math

import pytest
import torch

from oracle import int4

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(*shape, seed):
    return torch.randn(*shape, generator=_gen(seed), device="cuda", dtype=torch.float64)


def _cum(v):
    return torch.tensor([sum(v[:i]) for i in range(len(v) + 1)], dtype=torch.int32, device="cuda")


def _filled(key, value, block):
    """A cache that holds the rows of key and value [positions, kv_heads, 128] of one sequence, its pages in any order, and
    the sequence's table."""
    from nanovllm_b200.int4_cache import new_kvcache_int4
    n, kv, _ = key.shape
    pages = -(-n // block)
    cache = new_kvcache_int4(pages + 1, block, kv)
    table = (torch.randperm(pages, generator=torch.Generator().manual_seed(n)) + 1).to(torch.int32).cuda()
    at = torch.arange(n, device="cuda")
    int4.store(key.to(torch.bfloat16), value.to(torch.bfloat16), *cache,
               (table[at // block] * block + at % block).to(torch.int32))
    return cache, table


def _attend(q, cache, table, n, scale=SCALE):
    """The last rows of one sequence: a single token through decode, more as a chunk."""
    from nanovllm_b200.int4_cache import int4_decode_attention, int4_prefill_attention
    if q.shape[0] == 1:
        return int4_decode_attention(q, *cache, table[None], torch.tensor([n], dtype=torch.int32, device="cuda"), scale)
    return int4_prefill_attention(q, *cache, table[None], _cum([q.shape[0]]), _cum([n]), q.shape[0], n, scale)


def _check(q, cache, table, n, rows=slice(None), scale=SCALE):
    out = _attend(q, cache, table, n, scale)
    ref, room = int4.attention_norm(q, *cache, table, n, scale)
    far = (out.double() - ref).norm(dim=-1)
    bad = ~(far <= room)[rows]
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} rows off, first at {bad.nonzero()[0].tolist()}, "
                           f"{float((far / room)[rows].nan_to_num(math.inf).max()):.2f} of what they may be")
    return out


# query rows of one token (the split-context kernel), of a few, and of a long chunk
NEWS = [1, 5, 150]


@pytest.mark.parametrize("new", NEWS)
@pytest.mark.parametrize("n", [300, 200000])
def test_sums_over_a_long_context_stay_finite(new, n):
    """Values of 2^111: the sum over all positions of p v, before it is divided by the sum of p, passes fp32's range,
    the parts' own sums do not."""
    kv, heads = 1, 4
    key, value = _randn(n, kv, 128, seed=1), (2 + 0.2 * _randn(n, kv, 128, seed=2)) * 2.0 ** 110
    q = (0.1 * _randn(new, heads, 128, seed=3)).to(torch.bfloat16)
    _check(q, *_filled(key, value, 64), n)


# powers of two of K's and V's rows, and q's, such that scores are ordinary numbers
POWERS = [(0, 113), (0, 120), (0, 125), (0, -115), (0, -126), (113, 0), (125, 0), (-100, 0), (-115, 0), (112, 126), (-112, -120)]


@pytest.mark.parametrize("new", [33, 150])
@pytest.mark.parametrize("k_power,v_power", POWERS, ids=str)
def test_chunk_over_bf16s_range(new, k_power, v_power):
    n, kv, heads = 333, 2, 8
    key, value = (_randn(n, kv, 128, seed=s).clamp(-3, 3) * 2.0 ** (p - 1) for s, p in ((4, k_power), (5, v_power)))
    q = (1.5 * _randn(new, heads, 128, seed=6) * 2.0 ** (1 - k_power)).to(torch.bfloat16)
    out = _check(q, *_filled(key, value, 16), n)
    assert torch.isfinite(out).all()


def _ordinary(n, kv, heads, new, seed=7):
    return _randn(n, kv, 128, seed=seed), _randn(n, kv, 128, seed=seed + 1), 1.5 * _randn(new, heads, 128, seed=seed + 2)


@pytest.mark.parametrize("new,n", [(150, 400), (40, 9000)])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("power", [5, 10, 14, 20, 60, 100, -20, -100])
def test_chunk_beside_a_row_of_another_size(new, n, which, power):
    """The last token's row of K or V, which the queries before it do not see."""
    key, value, q = _ordinary(n, 1, 4, new)
    (key if which == "k" else value)[-1] *= 2.0 ** power
    _check(q.to(torch.bfloat16), *_filled(key, value, 64), n, slice(0, -1))


def _peaks(key, q, places):
    """Makes query row r of head 0 look at positions places[r], by a key along it."""
    for r, at in enumerate(places):
        key[at, 0] = q[r, 0] * 3


@pytest.mark.parametrize("new", [40, 150])
@pytest.mark.parametrize("powers", [{0: -9}, {0: -40, 500: 5}, {3: 12}, {0: 40, 130: -40, 700: 3}, {5: "zero"},
                                    {130: -20, 131: 20, 300: 0, 600: -20}], ids=str)
def test_chunk_values_of_many_sizes(new, powers):
    """Rows of V whose sizes differ by far more than f16 holds: queries that look at one of them alone, at an ordinary one,
    or at all; tiles with such a row and without take turns."""
    n = 1000
    key, value, q = _ordinary(n, 1, 4, new)
    for at, power in powers.items():
        value[at] *= 0.0 if power == "zero" else 2.0 ** power
    _peaks(key, q, list(powers) + [1, 129, 400, 801])
    _check(q.to(torch.bfloat16), *_filled(key, value, 16), n)


@pytest.mark.parametrize("new", [40, 150])
def test_chunk_keys_of_many_sizes(new):
    n = 700
    key, value, q = _ordinary(n, 1, 4, new)
    key *= torch.exp2(torch.randint(-25, 2, (n, 1, 1), generator=_gen(10), device="cuda").double())
    key[5], key[300:303] = 0, 0
    _check(q.to(torch.bfloat16), *_filled(key, value, 16), n)


@pytest.mark.parametrize("new", [40, 150])
def test_chunk_rows_of_any_size_at_all(new):
    """Every row of V with a power of its own, 2^-120 to 2^120, over several tiles and CTAs."""
    for n in (200, 5000):
        key, value, q = _ordinary(n, 2, 4, new)
        value *= torch.exp2(torch.randint(-120, 120, (n, 2, 1), generator=_gen(11), device="cuda").double())
        _peaks(key, q, range(0, n, max(1, n // 30)))
        _check(q.to(torch.bfloat16), *_filled(key, value, 32), n)


# ------------------------------------------------------------ the split-context kernel: up to 32 rows of a kv head
@pytest.mark.parametrize("new,heads", [(1, 4), (1, 8), (3, 4), (5, 4), (8, 4)])
@pytest.mark.parametrize("k_power,v_power", POWERS, ids=str)
def test_few_rows_over_bf16s_range(new, heads, k_power, v_power):
    n, kv = 333, 1
    key, value = (_randn(n, kv, 128, seed=s).clamp(-3, 3) * 2.0 ** (p - 1) for s, p in ((4, k_power), (5, v_power)))
    q = (1.5 * _randn(new, heads, 128, seed=6) * 2.0 ** (1 - k_power)).to(torch.bfloat16)
    out = _check(q, *_filled(key, value, 16), n)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("new,n", [(2, 400), (5, 9000), (8, 40000)])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("power", [5, 10, 14, 20, 60, 100, -20, -100])
def test_few_rows_beside_a_row_of_another_size(new, n, which, power):
    key, value, q = _ordinary(n, 1, 4, new)
    (key if which == "k" else value)[-1] *= 2.0 ** power
    _check(q.to(torch.bfloat16), *_filled(key, value, 64), n, slice(0, -1))


@pytest.mark.parametrize("new,heads", [(1, 4), (1, 32), (8, 4)])
@pytest.mark.parametrize("powers", [{0: -9}, {0: -40, 500: 5}, {3: 12}, {0: 40, 130: -40, 700: 3}, {5: "zero"},
                                    {130: -20, 131: 20, 300: 0, 600: -20}, {0: "zero", 1: "zero", 2: -126, 600: 126}], ids=str)
@pytest.mark.parametrize("n", [1000, 30000])
def test_few_rows_values_of_many_sizes(new, heads, powers, n):
    """Every query row looks at one position; tiles with a row of another size and without take turns."""
    key, value, q = _ordinary(n, 1, heads, new)
    value.clamp_(-1, 1)
    for at, power in powers.items():
        value[at] *= 0.0 if power == "zero" else 2.0 ** power
    places = list(powers) + [1, 129, 400, 801, n - 9]
    for i in range(new * heads):
        key[places[i % len(places)], 0] = q.view(-1, 128)[i] * 3
    _check(q.to(torch.bfloat16), *_filled(key, value, 16), n)


@pytest.mark.parametrize("new,heads", [(1, 4), (5, 4), (8, 4)])
@pytest.mark.parametrize("n", [200, 5000, 300000])
def test_few_rows_of_any_size_at_all(new, heads, n):
    key, value, q = _ordinary(n, 1, heads, new)
    value *= torch.exp2(torch.randint(-120, 120, (n, 1, 1), generator=_gen(11), device="cuda").double())
    step = max(1, n // 30)
    for i in range(new * heads):
        key[i % 30 * step, 0] = q.view(-1, 128)[i] * 3
    _check(q.to(torch.bfloat16), *_filled(key, value, 32), n)


def test_few_rows_constant_rows_and_none():
    """Steps of zero beside others, and a cache of zeros."""
    key, value, q = _ordinary(500, 1, 4, 1)
    value[::3] = value[::3, :, :1]
    _check(q.to(torch.bfloat16), *_filled(key, value, 32), 500)
    value[:] = 0
    out = _check(q.to(torch.bfloat16), *_filled(key, value, 32), 500)
    assert torch.all(out == 0)


def test_few_rows_huge_constant_rows():
    """Steps of zero all through, and lowest values whose sum passes fp32's range."""
    key, value, q = _ordinary(5000, 1, 4, 1)
    value = value[:, :, :1].abs().clamp(1, 2).expand(-1, -1, 128) * 2.0 ** 120
    _check((0.1 * q).to(torch.bfloat16), *_filled(key, value, 32), 5000)


def _sum_of_sizes(q, cache, table, n):
    """sum p |v| of query rows that see nearly all of n positions."""
    (kc, ks, kl), (vc, vs, vl), _ = int4.sequence(*cache, table, n)
    group = q.shape[1] // kc.shape[1]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    for h in range(q.shape[1]):
        g = h // group
        p = torch.softmax(q[:, h].double() @ (kl[:, g] + ks[:, g] * kc[:, g]).T * SCALE, -1)
        out[:, h] = p @ (vl[:, g] + vs[:, g] * vc[:, g]).abs()
    return out


@pytest.mark.parametrize("new,instructions", [(1, 64), (5, 128)])
def test_few_rows_cuts_do_not_grow_with_the_context(new, instructions):
    """So many sequences (on the same pages) that a CTA has all units of a pair: beside the output's rounding, what the tensor
    cores cut off.  Each instruction cuts up to 17 terms at 2^-24 of the largest, 2^-25 on average; between two times
    that sums are put aside there are 64 or 128 instructions, on sums that grow from zero: 64 * 17 * 2^-25 / 2 = 2^-15.9 of
    sum p |v| in all, or twice that."""
    from nanovllm_b200.int4_cache import int4_decode_attention, int4_prefill_attention
    n, kv, heads, seqs, block = 32768, 8, 32, 64, 256
    key, value = _randn(n, kv, 128, seed=21), _randn(n, kv, 128, seed=22)
    q = (1.5 * _randn(seqs * new, heads, 128, seed=23)).to(torch.bfloat16)
    cache, table = _filled(key, value, block)
    tables = table.repeat(seqs, 1)
    if new == 1:
        out = int4_decode_attention(q, *cache, tables, torch.full((seqs,), n, dtype=torch.int32, device="cuda"), SCALE)
    else:
        out = int4_prefill_attention(q, *cache, tables, _cum([new] * seqs), _cum([n] * seqs), new, n, SCALE)
    far, rounding, room = 0.0, 0.0, 0.0
    for i in (0, 31, 63):
        at = slice(i * new, (i + 1) * new)
        ref, _ = int4.attention_norm(q[at], *cache, table, n, SCALE)
        far += float((out[at].double() - ref).square().sum())
        rounding += float((ref.to(torch.bfloat16).double() - ref).square().sum())
        room += float(_sum_of_sizes(q[at], cache, table, n).square().sum())
    assert (far - rounding) ** 0.5 <= instructions * 17 * 2.0 ** -26 * room ** 0.5


@pytest.mark.parametrize("new", [1, 3, 5, 8])
@pytest.mark.parametrize("from_unit", [0, 40])
def test_few_rows_of_many_sizes_in_long_pieces(new, from_unit):
    """So many sequences (on the same pages) that a CTA has a whole pair, whose sums are put aside many times while its query
    rows have powers of their own: from its first unit of 128 positions on, or from a later one."""
    from nanovllm_b200.int4_cache import int4_decode_attention, int4_prefill_attention
    n, kv, heads, seqs = 20000, 2, 8, 220
    key, value = _randn(n, kv, 128, seed=31), _randn(n, kv, 128, seed=32)
    powers = torch.randint(-30, 30, (n, kv, 1), generator=_gen(33), device="cuda").double()
    powers[:128 * from_unit] = 0
    value *= torch.exp2(powers)
    q = 1.5 * _randn(seqs * new, heads, 128, seed=34)
    checked = (0, 7, 219)
    for x, i in enumerate(checked):  # rows that look at one position each, early, late and small ones among them
        for r in range(new * heads):
            key[(r * 613 + 97 * x) % (n - new), r % heads // 4] = 2 * q[i * new + r // heads, r % heads]
    q = q.to(torch.bfloat16)
    cache, table = _filled(key, value, 32)
    tables = table.repeat(seqs, 1)
    if new == 1:
        out = int4_decode_attention(q, *cache, tables, torch.full((seqs,), n, dtype=torch.int32, device="cuda"), SCALE)
    else:
        out = int4_prefill_attention(q, *cache, tables, _cum([new] * seqs), _cum([n] * seqs), new, n, SCALE)
    for i in checked:
        at = slice(i * new, (i + 1) * new)
        ref, room = int4.attention_norm(q[at], *cache, table, n, SCALE)
        far = (out[at].double() - ref).norm(dim=-1)
        assert torch.all(far <= room), f"sequence {i}: {float((far / room).nan_to_num(math.inf).max()):.2f}"


@pytest.mark.parametrize("new,heads", [(2, 4), (6, 4), (8, 4), (150, 4)])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_row_that_is_no_number_beside_rows_of_many_sizes(new, heads, which, bad):
    """It reaches the queries that see it, and those before it get what they see.  (As it is stored: with a step that is no
    number, whatever its values were.)"""
    n = 900
    key, value, q = _ordinary(n, 1, heads, new)
    value *= torch.exp2(torch.randint(-40, 40, (n, 1, 1), generator=_gen(41), device="cuda").double())
    (key if which == "k" else value)[n - 2, 0, 17] = bad
    cache, table = _filled(key, value, 32)
    q = q.to(torch.bfloat16)
    out = _attend(q, cache, table, n)
    ref, room = int4.attention_norm(q[:new - 2], *cache, table, n - 2, SCALE)
    assert torch.all((out[:new - 2].double() - ref).norm(dim=-1) <= room)
    assert not torch.isfinite(out[new - 2:]).any()


@pytest.mark.parametrize("new", [1, 5, 150])
def test_rows_of_many_sizes_give_the_same_bits_in_a_graph(new):
    n = 5000
    key, value, q = _ordinary(n, 1, 4, new)
    value *= torch.exp2(torch.randint(-60, 60, (n, 1, 1), generator=_gen(42), device="cuda").double())
    cache, table = _filled(key, value, 32)
    q = q.to(torch.bfloat16)
    first = _attend(q, cache, table, n)
    ctx, tables = torch.tensor([n], dtype=torch.int32, device="cuda"), table[None].contiguous()
    cq, ck = _cum([new]), _cum([n])
    from nanovllm_b200.int4_cache import int4_decode_attention, int4_prefill_attention
    call = lambda: (int4_decode_attention(q, *cache, tables, ctx, SCALE) if new == 1 else  # noqa: E731
                    int4_prefill_attention(q, *cache, tables, cq, ck, new, n, SCALE))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first) and torch.equal(call(), first)


def test_no_wait_has_run_out():
    from nanovllm_b200 import fp8_attention
    assert fp8_attention.device_error() == 0
