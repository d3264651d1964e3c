"""Attention over the 4-bit cache held to the 2-norm of each output row (oracle/int4.py, ``attention_norm``; tests/test_int4_cpu.py
shows what that tells apart), with inputs in which every page, tile and part of a cut counts for some row."""
import math

import pytest
import torch

from oracle import int4

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _cum(v):
    return torch.tensor([sum(v[:i]) for i in range(len(v) + 1)], dtype=torch.int32, device="cuda")


def _cache(lens, kv, block, seed, spread=0.0):
    """Caches of several sequences, their pages mixed; keys, for the tests that put something into them."""
    from nanovllm_b200.int4_cache import new_kvcache_int4
    counts = [-(-n // block) for n in lens]
    page = torch.randperm(sum(counts), generator=torch.Generator().manual_seed(seed)).to(torch.int32).cuda()
    table = torch.full((len(lens), max(counts)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = page[at:at + c]
        at += c
    n, g = sum(counts) * block, _gen(seed)
    rows = [torch.randn(n, kv, 128, generator=g, device="cuda") *
            torch.exp2(spread * torch.randn(n, kv, 1, generator=g, device="cuda")) for _ in range(2)]
    cache = new_kvcache_int4(sum(counts), block, kv)
    int4.store(rows[0].to(torch.bfloat16), rows[1].to(torch.bfloat16), *cache,
               torch.arange(n, dtype=torch.int32, device="cuda"))
    return cache, table


def _look_at(cache, table, places, q):
    """The key at places[r] of a sequence along q[r] (one kv head)."""
    block = cache[0].shape[2]
    for row, at in zip(q, places):
        code, step, low = int4.quantise((row.float() * 2).to(torch.bfloat16))
        page = int(table[at // block])
        cache[0][page, 0, at % block] = int4.pack(code)
        cache[2][page, 0, at % block, 0], cache[2][page, 0, at % block, 1] = step, low


def _check(out, q, cache, table, n, what, scale=SCALE):
    ref, room = int4.attention_norm(q, *cache, table, n, scale)
    far = (out.double() - ref).norm(dim=-1)
    bad = ~(far <= room)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} rows off, first at {bad.nonzero()[0].tolist()}, "
                           f"{float((far / room).nan_to_num(math.inf).max()):.2f} of what they may be")


def _run(q, cache, table, news, lens, scale=SCALE):
    from nanovllm_b200.int4_cache import int4_decode_attention, int4_prefill_attention
    if all(m == 1 for m in news):
        out = int4_decode_attention(q, *cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), scale)
    else:
        out = int4_prefill_attention(q, *cache, table, _cum(news), _cum(lens), max(news), max(lens), scale)
    at = 0
    for i, (m, n) in enumerate(zip(news, lens)):
        _check(out[at:at + m], q[at:at + m], cache, table[i], n, f"sequence {i}, {m} of {n}", scale)
        at += m


def _q(n, heads, seed, sd=1.5):
    return (torch.randn(n, heads, 128, generator=_gen(seed), device="cuda") * sd).to(torch.bfloat16)


@pytest.mark.parametrize("news,lens", [([1], [1]), ([1], [33]), ([1] * 3, [127, 128, 700]), ([1] * 2, [3000, 9]),
                                       ([2, 5], [500, 90]), ([8], [4000]), ([40], [40]), ([33, 100], [33, 1000]),
                                       ([257, 1, 40], [600, 900, 40]), ([129] * 3, [4000] * 3)], ids=str)
@pytest.mark.parametrize("heads,kv,block", [(32, 8, 256), (4, 4, 16), (16, 2, 48), (5, 1, 64), (24, 1, 32)])
@pytest.mark.parametrize("spread", [0.0, 1.0])
def test_rows(news, lens, heads, kv, block, spread):
    cache, table = _cache(lens, kv, block, 1, spread)
    _run(_q(sum(news), heads, 2), cache, table, news, lens)


@pytest.mark.parametrize("news,lens", [([1] * 40, [20000] * 40), ([5] * 8, [20000] * 8), ([150], [30000])], ids=str)
def test_long_contexts(news, lens):
    n, block = lens[0], 64
    cache, one = _cache([n], 1, block, 3)
    table = one.repeat(len(lens), 1)  # all on the same pages
    _run(_q(sum(news), 4, 4), cache, table, news, lens)


@pytest.mark.parametrize("new,heads,n,block", [(1, 1, 20000, 64), (1, 8, 20000, 64), (4, 8, 9000, 16), (150, 4, 30000, 64),
                                               (300, 2, 9000, 16)])
def test_every_page_counts_for_a_row(new, heads, n, block):
    """Query rows that look at one position each, spread over all pages: nothing of the context can be left out, taken twice
    or joined with a wrong weight without a row that shows it."""
    pages = n // block
    per_seq = new * heads
    seqs = -(-pages // per_seq) if new < 100 else 1
    cache, one = _cache([n], 1, block, 5)
    q = _q(seqs * new, heads, 6)
    rows = q.view(-1, 128)
    places = [int((i + 0.5) * n / rows.shape[0]) for i in range(rows.shape[0])]
    if new > 1:  # all of them behind what the first query sees
        places = [min(p, n - new) for p in places]
    _look_at(cache, one[0], places, rows)
    _run(q, cache, one.repeat(seqs, 1), [new] * seqs, [n] * seqs)


@pytest.mark.parametrize("sd,scale", [(0.0, SCALE), (1e-30, SCALE), (10.0, SCALE), (0.5, -0.1), (0.5, 0.0), (0.3, 1.0)])
@pytest.mark.parametrize("news,lens", [([1, 1], [500, 77]), ([3], [400]), ([150], [333])], ids=str)
def test_scales_of_scores(sd, scale, news, lens):
    cache, table = _cache(lens, 2, 16, 7)
    _run(_q(sum(news), 8, 8, sd), cache, table, news, lens, scale)


@pytest.mark.parametrize("seed", range(32))
def test_drawn(seed):
    """Heads, pages, lengths, sizes of rows, missing pages and rows of zeros as they come."""
    import random
    rng = random.Random(seed)
    kv, group = rng.choice([1, 2, 3]), rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16, 32, 40])
    seqs, kind = rng.choice([1, 2, 5]), rng.choice(["one", "few", "chunk", "mixed"])
    lens = [max(1, int(math.exp(rng.uniform(0, math.log(3000))))) for _ in range(seqs)]
    news = [min(n, {"one": 1, "few": rng.randint(1, 8), "chunk": rng.randint(1, 300),
                    "mixed": rng.choice([0, 1, 5, 200])}[kind]) for n in lens]
    news[0] = max(news[0], 1)
    cache, table = _cache(lens, kv, rng.choice([16, 32, 48, 64, 128, 256]), seed)
    shape, scale, g = cache[2].shape[:3], cache[2], _gen(seed)
    randn = lambda: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    spread = rng.choice([0.0, 0.5, 3.0, 10.0, 30.0])
    size = torch.exp2((spread * randn()).round().clamp(-100, 100))
    if rng.random() < 0.5:
        size = torch.where(randn() > 2.3, size, 1.0)
    scale[..., 2:] = (scale[..., 2:].float() * size[..., None]).to(torch.bfloat16)
    if rng.random() < 0.5:  # smaller keys: scores stay numbers
        size = torch.exp2((min(spread, 3.0) * randn()).round().clamp(-60, 2))
        scale[..., :2] = (scale[..., :2].float() * size[..., None]).to(torch.bfloat16)
    if rng.random() < 0.3:
        scale[..., 2:][randn() > 2.0] = 0
    if rng.random() < 0.3:
        table[0, rng.randrange(table.shape[1])] = -1
    _run(_q(sum(news), kv * group, seed + 1, rng.choice([0.1, 1.5, 3.0])), cache, table, news, lens)
