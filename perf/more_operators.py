"""The operators of a 4-bit key/value cache, as cases that can be measured.

A cache row (one token of one kv head, 128 values) is held as 128 codes of 4 bits with a step and a
lowest value in bf16: x ~ low + step * code.

``rope``    rotary positions of q and k: halves or interleaved pairs, all of the head or part of it;
``cache``   new tokens' keys and values quantised into a paged cache as they are written, and read back;
``decode``  attention of one new token per sequence over the paged 4-bit cache;
``chunk``   causal attention of a chunk of new tokens per sequence over the paged 4-bit cache.

``run`` computes a case with elementary torch operations, or, where ``own`` is set, with the
framework's kernels; ``exact`` computes it from the definitions in 64 bits.
"""
import math
import os
import random
import sys

import torch

sys.path.append(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                             "my-nano-vllm_b200"))     # where the package lies

own = False

D = 128                      # values in a cache row
SCALE = D ** -0.5            # of the attention scores
ROW_BYTES = D // 2 + 4       # codes, step and lowest value of one row
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decoded token of a 32-head model, the whole head rotated by halves
        dict(name="rope_decode_1", op="rope", tokens=1, heads=32, kv_heads=8, dim=128, rotary=128,
             interleaved=False, dtype="bf16"),
        # a ragged chunk, half of each head rotated by interleaved pairs, fp16
        dict(name="rope_partial_fp16", op="rope", tokens=1237, heads=40, kv_heads=8, dim=128,
             rotary=64, interleaved=True, dtype="fp16"),
        # a whole prefill budget
        dict(name="rope_prefill_8192", op="rope", tokens=8192, heads=32, kv_heads=8, dim=128,
             rotary=128, interleaved=False, dtype="bf16"),
        # the new rows of a decode batch
        dict(name="cache_decode_64", op="cache", tokens=64, kv_heads=8, block=256),
        # the new rows of a whole prefill budget, some of them padding
        dict(name="cache_prefill_8192", op="cache", tokens=8192, kv_heads=8, block=256),
        # one short conversation, small pages
        dict(name="decode_one_short", op="decode", seqs=1, shortest=700, longest=700, heads=16,
             kv_heads=8, block=16),
        # one long document: the work of a single token spread over the GPU
        dict(name="decode_one_long", op="decode", seqs=1, shortest=131071, longest=131071, heads=32,
             kv_heads=8, block=256),
        # a large batch of uneven contexts
        dict(name="decode_batch_256", op="decode", seqs=256, shortest=512, longest=4096, heads=32,
             kv_heads=8, block=256),
        # long contexts of a larger model: the largest of the decode cases
        dict(name="decode_long_64", op="decode", seqs=64, shortest=32768, longest=32768, heads=64,
             kv_heads=8, block=256),
        # speculative verification: 1 + 4 rows of each sequence
        dict(name="chunk_verify_192", op="chunk", seqs=192, fewest=5, most=5, shortest=512,
             longest=4096, heads=32, kv_heads=8, block=256),
        # prompts of uneven lengths, some with a prefix that is in the cache already
        dict(name="chunk_prompts_7", op="chunk", seqs=7, fewest=33, most=1500, shortest=33,
             longest=2500, heads=32, kv_heads=8, block=64),
        # one chunk of a long document
        dict(name="chunk_long_2048", op="chunk", seqs=1, fewest=2048, most=2048, shortest=32768,
             longest=32768, heads=32, kv_heads=8, block=256),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "cache", "decode", "chunk"])
    if op == "rope":
        dim = rng.choice([64, 80, 96, 128, 192, 256])
        kv = rng.choice([1, 2, 4, 8, 16])
        heads = kv * rng.randint(1, 8)
        tokens = _log_int(rng, 1, min(16384, 8192 * 40 * 128 // ((heads + kv) * dim)))
        return dict(op=op, tokens=tokens, heads=heads, kv_heads=kv, dim=dim,
                    rotary=dim if rng.random() < 0.5 else 2 * rng.randint(8, dim // 2),
                    interleaved=rng.random() < 0.5, dtype=rng.choice(["bf16", "fp16"]))
    kv = rng.choice([1, 2, 4, 8, 16])
    block = rng.choice([16, 32, 48, 64, 128, 256])
    if op == "cache":
        return dict(op=op, tokens=_log_int(rng, 1, min(16384, 8192 * 8 // kv)), kv_heads=kv,
                    block=block)
    group = rng.choice([1, 2, 4, 5, 7, 8, 12, 16])
    if op == "decode":
        longest = _log_int(rng, 1, 131072)
        seqs = _log_int(rng, 1, max(1, min(512, 64 * 32768 * 8 // (longest * kv))))
        return dict(op=op, seqs=seqs, shortest=max(1, int(longest * rng.uniform(0.1, 1))),
                    longest=longest, heads=kv * group, kv_heads=kv, block=block)
    # a chunk of up to 2048 tokens, scores of at most 2048 x 32768 for 32 heads in all, and a plain
    # form's dequantised cache of at most 2^26 rows
    longest = _log_int(rng, 1, 32768)
    most = _log_int(rng, 1, min(longest, 2048))
    room = min(2048 * 32768 * 32 // (most * longest * kv * group), 2 ** 26 // (8 * longest * kv))
    if room < 1:
        group = max(1, min(group, 2048 * 32768 * 32 // (most * longest * kv)))
    seqs = _log_int(rng, 1, max(1, min(192, room)))
    fewest = max(1, int(most * rng.uniform(0.2, 1)))
    return dict(op=op, seqs=seqs, fewest=fewest, most=most,
                shortest=max(1, int(longest * rng.uniform(0.2, 1))), longest=longest,
                heads=kv * group, kv_heads=kv, block=block)


def _lengths(case):
    """Contexts (and, for chunks, how many of their last tokens are new), by the case alone."""
    rng = random.Random("%d %d %d" % (case["seqs"], case["shortest"], case["longest"]))
    lens = [rng.randint(case["shortest"], case["longest"]) for _ in range(case["seqs"])]
    if case["op"] == "decode":
        return lens, None
    news = [min(n, rng.randint(case["fewest"], case["most"])) for n in lens]
    return lens, news


# ------------------------------------------------------------------------------------ inputs
def _quantise(x):
    """Rows [..., 128] -> (codes uint8 [..., 128], (step, lowest) bf16 [..., 2])."""
    low, high = x.amin(-1).float(), x.amax(-1).float()
    step = ((high - low) / 15).to(torch.bfloat16)
    # which code is nearest is a comparison with a border: 64 bits
    wide = step.double()[..., None]
    code = torch.round((x.double() - low.double()[..., None]) / torch.where(wide > 0, wide, 1))
    code = torch.where(wide > 0, code.clamp(0, 15), 0).to(torch.uint8)
    return code, torch.stack([step, low.to(torch.bfloat16)], -1)


def _pack(code):
    """Values 2 i and 2 i + 1 of a row in the low and high half of byte i."""
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _cache(blocks, block, kv_heads, gen):
    """A paged cache [blocks, kv_heads, block, ...] as a running program has it: quantised keys (some
    channels stand out, as keys' do) and values."""
    shape = (blocks, kv_heads, block)
    caches = [torch.empty(*shape, D // 2, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scale = torch.empty(*shape, 4, dtype=torch.bfloat16, device="cuda")
    spread = 1 + 3 * (torch.rand(kv_heads, 1, D, generator=gen, device="cuda") > 0.95)
    part = max(1, 2 ** 26 // (kv_heads * block * D))
    for i in range(0, blocks, part):
        n = min(part, blocks - i)
        for j in range(2):
            x = torch.randn(n, *shape[1:], D, generator=gen, device="cuda")
            code, sl = _quantise((x * spread if j == 0 else x).to(torch.bfloat16))
            caches[j][i:i + n] = _pack(code)
            scale[i:i + n, ..., 2 * j:2 * j + 2] = sl
    return caches[0], caches[1], scale


def _tables(lens, block, gen):
    """Every sequence's pages, scattered over the cache; -1 behind a sequence's last."""
    counts = [-(-n // block) for n in lens]
    page = torch.randperm(sum(counts), generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(counts)), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(max(counts), device="cuda") < torch.tensor(counts, device="cuda")[:, None]] = page
    return table, sum(counts)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    s = {"case": case}
    if case["op"] == "rope":
        n, h, kv, dim, r = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "rotary"))
        # q and k lie side by side, as a projection leaves them
        qkv = randn(n, (h + 2 * kv) * dim).to(DTYPES[case["dtype"]])
        s["q"] = qkv[:, :h * dim].view(n, h, dim)
        s["k"] = qkv[:, h * dim:(h + kv) * dim].view(n, kv, dim)
        s["positions"] = torch.randint(0, 32768, (n,), generator=gen, device="cuda")
        # positions stretched by four beyond the lengths trained on
        angle = torch.arange(32768, device="cuda").double()[:, None] / 4 * (
            1e6 ** (-torch.arange(0, r, 2, device="cuda").double() / r))
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float()
    elif case["op"] == "cache":
        n, kv, block = case["tokens"], case["kv_heads"], case["block"]
        blocks = -(-5 * n // (4 * block)) + 1
        s["key"] = (randn(n, kv, D) * (1 + 3 * (torch.rand(kv, D, generator=gen, device="cuda") >
                                                0.95))).to(torch.bfloat16)
        s["value"] = randn(n, kv, D).to(torch.bfloat16)
        s["k_cache"], s["v_cache"], s["kv_scale"] = _cache(blocks, block, kv, gen)
        # tokens follow one another within a page, pages are scattered; one row in 16 is padding
        page = torch.randperm(blocks, generator=gen, device="cuda")
        at = torch.arange(n, device="cuda")
        slot = page[at // block] * block + at % block
        s["slots"] = torch.where(at % 16 == 15, -1, slot).to(torch.int32)
    else:
        lens, news = _lengths(case)
        s["tables"], pages = _tables(lens, case["block"], gen)
        s["k_cache"], s["v_cache"], s["kv_scale"] = _cache(pages, case["block"], case["kv_heads"], gen)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        if news is None:
            s["q"] = (1.5 * randn(case["seqs"], case["heads"], D)).to(torch.bfloat16)
        else:
            s["q"] = (1.5 * randn(sum(news), case["heads"], D)).to(torch.bfloat16)
            s["most"], s["longest"] = max(news), max(lens)
            cumulated = lambda v: torch.tensor([sum(v[:i]) for i in range(len(v) + 1)],  # noqa: E731
                                               dtype=torch.int32, device="cuda")
            s["cu_q"], s["cu_k"] = cumulated(news), cumulated(lens)
    return s


# ------------------------------------------------------------------- plain forms, 32 bits
def _rope_plain(s):
    c = s["case"]
    r, half = c["rotary"], c["rotary"] // 2
    cos, sin = s["cos_sin"][s["positions"]][:, None].chunk(2, -1)

    def turn(x):
        y = x[..., :r].float()
        a, b = (y[..., 0::2], y[..., 1::2]) if c["interleaved"] else (y[..., :half], y[..., half:])
        a, b = a * cos - b * sin, b * cos + a * sin
        y = torch.stack([a, b], -1).flatten(-2) if c["interleaved"] else torch.cat([a, b], -1)
        return torch.cat([y.to(x.dtype), x[..., r:]], -1)

    return turn(s["q"]), turn(s["k"])


def _unpack(cache, scale):
    """Rows' codes and (step, lowest) -> the values that they stand for, fp32."""
    code = torch.stack([cache & 15, cache >> 4], -1).flatten(-2)
    return torch.addcmul(scale[..., 1:].float(), code.float(), scale[..., :1].float())


def _cache_plain(s):
    block = s["case"]["block"]
    slot = s["slots"].long()
    kept = slot >= 0
    page, place = slot // block, slot % block
    out = []
    for j, (rows, cache) in enumerate([(s["key"], s["k_cache"]), (s["value"], s["v_cache"])]):
        code, sl = _quantise(rows[kept])
        cache[page[kept], :, place[kept]] = _pack(code)
        both = s["kv_scale"][..., 2 * j:2 * j + 2]
        both[page[kept], :, place[kept]] = sl
        back = _unpack(cache[page, :, place], both[page, :, place])
        out.append(torch.where(kept[:, None, None], back, 0).to(torch.bfloat16))
    return out[0], out[1], s["kv_scale"]


def _history(s):
    """Keys and values [seqs, kv_heads, positions, 128] in fp32, padded to the longest context."""
    pages = s["tables"].clamp(min=0).long()
    scale = s["kv_scale"][pages]
    rows = lambda cache, sl: _unpack(cache[pages], sl).transpose(1, 2).flatten(2, 3)  # noqa: E731
    return rows(s["k_cache"], scale[..., :2]), rows(s["v_cache"], scale[..., 2:])


def _attend(q, k, v, seen):
    """q [seqs, kv_heads, rows, 128]; seen [seqs, 1, rows or 1, positions]."""
    score = torch.matmul(q, k.transpose(-1, -2)).mul_(SCALE)
    score.masked_fill_(~seen, -math.inf)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    return torch.matmul(score, v) / score.sum(-1, keepdim=True)


def _decode_plain(s):
    b, h, kv = s["case"]["seqs"], s["case"]["heads"], s["case"]["kv_heads"]
    k, v = _history(s)
    seen = torch.arange(k.shape[2], device="cuda") < s["lens"][:, None, None, None]
    q = s["q"].float().view(b, kv, h // kv, D)
    return _attend(q, k, v, seen).view(b, h, D).to(torch.bfloat16)


def _chunk_plain(s):
    h, kv, most = s["case"]["heads"], s["case"]["kv_heads"], s["most"]
    k, v = _history(s)
    news = (s["cu_q"][1:] - s["cu_q"][:-1])[:, None]
    row = torch.arange(most, device="cuda")
    real = row < news
    q = torch.zeros(len(news), most, h, D, device="cuda")
    q[real] = s["q"].float()
    # row i of a chunk sees the positions up to its own; rows of padding see the first
    last = torch.where(real, row + s["lens"][:, None] - news, 0)
    seen = torch.arange(k.shape[2], device="cuda") <= last[:, None, :, None]
    seen = seen.repeat_interleave(h // kv, 2)
    q = q.view(len(news), most, kv, h // kv, D).permute(0, 2, 1, 3, 4).flatten(2, 3)
    out = _attend(q, k, v, seen).view(len(news), kv, most, h // kv, D)
    return out.permute(0, 2, 1, 3, 4).flatten(2, 3)[real].to(torch.bfloat16)


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        from nanovllm_b200 import int4_cache, rope
        if op == "rope":
            return rope.apply_rope(s["q"], s["k"], s["positions"], s["cos_sin"],
                                   interleaved=s["case"]["interleaved"])
        caches = s["k_cache"], s["v_cache"], s["kv_scale"]
        if op == "cache":
            int4_cache.store_kvcache_int4(s["key"], s["value"], *caches, s["slots"])
            return (*int4_cache.load_kvcache_int4(*caches, s["slots"]), s["kv_scale"])
        if op == "decode":
            return int4_cache.int4_decode_attention(s["q"], *caches, s["tables"], s["lens"], SCALE)
        return int4_cache.int4_prefill_attention(s["q"], *caches, s["tables"], s["cu_q"], s["cu_k"],
                                                 s["most"], s["longest"], SCALE)
    return {"rope": _rope_plain, "cache": _cache_plain, "decode": _decode_plain,
            "chunk": _chunk_plain}[op](state)


# ------------------------------------------------------------------------------------- floors
def work(case):
    if case["op"] == "rope":
        n, both = case["tokens"], case["heads"] + case["kv_heads"]
        return {"bytes": n * (4 * both * case["dim"] + 4 * case["rotary"] + 8),
                "flops": 3 * n * both * case["rotary"]}
    if case["op"] == "cache":
        n = case["tokens"] - case["tokens"] // 16          # rows that are not padding
        rows = 2 * n * case["kv_heads"]
        # written from 16 bits, read back into 16 bits; zeros for the padding
        return {"bytes": rows * 2 * (2 * D + ROW_BYTES) + 4 * (case["tokens"] - n) *
                case["kv_heads"] * D + 8 * case["tokens"], "flops": rows * D * 7}
    lens, news = _lengths(case)
    rows, h = (news or [1] * len(lens)), case["heads"]
    seen = sum(m * (n - m) + m * (m + 1) // 2 for m, n in zip(rows, lens))
    return {"bytes": sum(lens) * 2 * case["kv_heads"] * ROW_BYTES + 4 * sum(rows) * h * D +
            4 * sum(-(-n // case["block"]) for n in lens), "flops": 4 * seen * h * D}


# --------------------------------------------------------------------- definitions, 64 bits
def _bf16_nearest(v):
    """Nearest value with 8 significant bits (ties to even), in float64."""
    grid = torch.exp2(torch.frexp(v)[1].double() - 8)
    return torch.round(v / grid) * grid


def _rows_exact(x):
    """What reading a row back gives, and its step and lowest value."""
    x = x.double()
    low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    step = _bf16_nearest((high - low) / 15)
    code = torch.round((x - low) / step.clamp(min=1e-300)).clamp(0, 15)
    return low + code * step, torch.cat([step, low], -1)


def _sequence_exact(s, i, n):
    """Keys and values [kv_heads, n, 128] of sequence i."""
    block = s["case"]["block"]
    at = torch.arange(n, device="cuda")
    page, place = s["tables"][i].long()[at // block], at % block
    got = []
    for j, cache in enumerate((s["k_cache"], s["v_cache"])):
        byte = cache[page, :, place].double()
        high = torch.floor(byte / 16)
        code = torch.stack([byte - 16 * high, high], -1).reshape(*byte.shape[:-1], D)
        sl = s["kv_scale"][page, :, place].double()
        got.append((sl[..., 2 * j + 1, None] + code * sl[..., 2 * j, None]).transpose(0, 1))
    return got


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        r = case["rotary"]
        table = s["cos_sin"].double()[s["positions"]]
        turn = torch.complex(table[:, :r // 2], table[:, r // 2:])[:, None]
        out = []
        for x in (s["q"].double(), s["k"].double()):
            y = x.clone()
            if case["interleaved"]:
                z = torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], r // 2, 2).contiguous())
                y[..., :r] = torch.view_as_real(z * turn).reshape(*x.shape[:-1], r)
            else:
                z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * turn
                y[..., :r] = torch.cat([z.real, z.imag], -1)
            out.append(y)
        return out[0], out[1]
    if case["op"] == "cache":
        scale = s["kv_scale"].double()
        slot = s["slots"].long()
        out = []
        for j, x in enumerate((s["key"], s["value"])):
            y, sl = _rows_exact(x)
            y[slot < 0] = 0
            out.append(y)
            keep = (slot >= 0).nonzero()[:, 0]
            scale[slot[keep] // case["block"], :, slot[keep] % case["block"],
                  2 * j:2 * j + 2] = sl[keep]
        return out[0], out[1], scale
    lens, news = _lengths(case)
    h, kv = case["heads"], case["kv_heads"]
    q, first, out = s["q"].double(), 0, []
    for i, n in enumerate(lens):
        m = news[i] if news else 1
        k, v = _sequence_exact(s, i, n)
        rows = q[first:first + m].view(m, kv, h // kv, D)
        last = torch.arange(n - m, n, device="cuda")
        hidden = torch.arange(n, device="cuda") > last[:, None]
        part = torch.empty(m, kv, h // kv, D, dtype=torch.float64, device="cuda")
        for g in range(kv):
            for e in range(h // kv):
                score = rows[:, g, e] @ k[g].T * SCALE
                score[hidden] = -math.inf
                part[:, g, e] = torch.softmax(score, -1) @ v[g]
        out.append(part.view(m, h, D))
        first += m
    return torch.cat(out)
