"""The rotary and 4-bit cache entry points without a GPU: refusals come before any device is touched; the
rotary tables against their formulas; the restatement of the cache against itself."""
import math

import pytest
import torch

from nanovllm_b200 import _lib, int4_cache, rope
from oracle import int4

P = 4096  # an aligned address that nothing reads


def _message():
    return _lib.lib.fp8attn_last_error().decode()


def _rope(**over):
    a = dict(q=P, qt=4096, qh=128, k=P, kt=1024, kh=128, pos=P, cs=P, maxp=100, qo=2 * P, qot=4096, qoh=128,
             ko=3 * P, kot=1024, koh=128, n=4, heads=32, kv=8, d=128, r=128, inter=0, dtype=0, stream=None)
    assert set(over) <= set(a)
    a.update(over)
    return _lib.lib.fp8attn_rope(*a.values())


@pytest.mark.parametrize("bad,msg", [
    (dict(dtype=2), "dtype"), (dict(d=127), "head_dim"), (dict(d=0), "head_dim"), (dict(d=4098), "head_dim"),
    (dict(r=63), "rotary_dim"), (dict(r=130), "rotary_dim"), (dict(r=0), "rotary_dim"), (dict(n=-1), "sizes"),
    (dict(heads=0), "sizes"), (dict(maxp=0), "sizes"), (dict(q=None), "null"), (dict(k=None), "null"),
    (dict(pos=None), "null"), (dict(q=P + 1), "aligned"), (dict(cs=P + 4), "aligned"), (dict(pos=P + 4), "aligned"),
    (dict(qot=0), "overlap"), (dict(qoh=127), "overlap"), (dict(koh=0), "overlap"), (dict(qot=4095), "overlap"),
    (dict(qo=P * 2, ko=P * 2), "same memory"), (dict(n=1 << 40), "2^32"), (dict(n=1 << 21), "2^32"),
])
def test_rope_refusals(bad, msg):
    assert _rope(**bad) == _lib.EINVAL
    assert msg in _message()


def test_rope_without_tokens():
    assert _rope(n=0, q=None) == _lib.OK


def _store(**over):
    a = dict(key=P, kt=1024, kh=128, value=P, vt=1024, vh=128, kc=P, vc=P, sc=P, slots=P, n=4, kv=8, d=128, nb=10,
             bs=16, stream=None)
    assert set(over) <= set(a)
    a.update(over)
    return _lib.lib.fp8attn_int4_store(*a.values())


def _load(**over):
    a = dict(kc=P, vc=P, sc=P, slots=P, ko=P, vo=P, n=4, kv=8, d=128, nb=10, bs=16, stream=None)
    assert set(over) <= set(a)
    a.update(over)
    return _lib.lib.fp8attn_int4_load(*a.values())


CACHE = [(dict(d=64), "head_dim"), (dict(bs=24), "block_size"), (dict(bs=0), "block_size"), (dict(nb=0), "num_blocks"),
         (dict(nb=1 << 27), "num_blocks"), (dict(kc=None), "null"), (dict(sc=None), "null"), (dict(vc=P + 8), "aligned"),
         (dict(sc=P + 8), "aligned"), (dict(kv=0), "num_kv_heads")]
ROWS = [(dict(n=-1), "num_tokens"), (dict(n=1 << 29), "num_tokens"), (dict(kv=4097), "num_tokens"),
        (dict(slots=None), "null")]


@pytest.mark.parametrize("bad,msg", CACHE + ROWS + [(dict(key=None), "null"), (dict(value=P + 1), "aligned")])
def test_store_refusals(bad, msg):
    assert _store(**bad) == _lib.EINVAL
    assert msg in _message()


@pytest.mark.parametrize("bad,msg", CACHE + ROWS + [(dict(ko=None), "null"), (dict(vo=P + 8), "aligned")])
def test_load_refusals(bad, msg):
    assert _load(**bad) == _lib.EINVAL
    assert msg in _message()


def test_no_rows():
    assert _store(n=0, key=None, slots=None) == _lib.OK and _load(n=0, ko=None) == _lib.OK


def _decode(**over):
    a = dict(out=P, q=P, qs=4096, kc=P, vc=P, sc=P, bt=P, bts=4, mb=4, ctx=P, seqs=2, heads=32, kv=8, d=128, nb=10,
             bs=256, scale=0.088, ws=P, wsb=1 << 30, stream=None)
    assert set(over) <= set(a)
    a.update(over)
    return _lib.lib.fp8attn_int4_decode(*a.values())


def _prefill(**over):
    a = dict(out=P, q=P, qs=4096, kc=P, vc=P, sc=P, bt=P, bts=4, mb=4, cq=P, ck=P, seqs=2, mq=8, heads=32, kv=8, d=128,
             nb=10, bs=256, scale=0.088, ws=P, wsb=1 << 30, stream=None)
    assert set(over) <= set(a)
    a.update(over)
    return _lib.lib.fp8attn_int4_prefill(*a.values())


ATTENTION = CACHE + [(dict(heads=30), "multiple"), (dict(heads=0), "multiple"), (dict(seqs=65536), "num_seqs"),
                     (dict(seqs=-1), "num_seqs"), (dict(q=None), "null"), (dict(bt=None), "null"),
                     (dict(q=P + 8), "aligned"), (dict(qs=4000), "aligned"), (dict(qs=4100), "aligned"),
                     (dict(bts=3), "block table"), (dict(mb=-1), "block table"),
                     (dict(mb=1 << 16, bts=1 << 16), "2^24"),
                     (dict(seqs=60000, mb=(1 << 16) - 1, bts=1 << 16), "too much")]


@pytest.mark.parametrize("bad,msg", ATTENTION + [(dict(ctx=None), "null")])
def test_decode_refusals(bad, msg):
    assert _decode(**bad) == _lib.EINVAL
    assert msg in _message()


@pytest.mark.parametrize("bad,msg", ATTENTION + [(dict(cq=None), "null"), (dict(ck=None), "null"),
                                                 (dict(mq=-1), "max_seqlen_q")])
def test_prefill_refusals(bad, msg):
    assert _prefill(**bad) == _lib.EINVAL
    assert msg in _message()


def test_nothing_to_attend():
    assert _decode(seqs=0, ctx=None) == _lib.OK and _prefill(mq=0) == _lib.OK
    assert _lib.lib.fp8attn_int4_workspace_bytes(4, 30, 8, 1) == -1
    assert _lib.lib.fp8attn_int4_workspace_bytes(-1, 32, 8, 1) == -1


def test_python_checks():
    cache = int4_cache.new_kvcache_int4(2, 16, 2, device="cpu")
    assert [tuple(t.shape) for t in cache] == [(2, 2, 16, 64), (2, 2, 16, 64), (2, 2, 16, 4)]
    x = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    slots = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: int4_cache.store_kvcache_int4(x, x, *cache, slots),
                 lambda: int4_cache.load_kvcache_int4(*cache, slots),
                 lambda: int4_cache.int4_decode_attention(x, *cache, slots[None], slots, 1.0),
                 lambda: int4_cache.int4_prefill_attention(x, *cache, slots[None], slots, slots, 1, 1, 1.0),
                 lambda: rope.apply_rope(x, x, slots.long(), torch.zeros(4, 128))):
        with pytest.raises(AssertionError, match="CUDA"):
            call()
    with pytest.raises(AssertionError):
        int4_cache.new_kvcache_int4(2, 24, 2, device="cpu")


# ------------------------------------------------------------------------------- rotary tables
def _angles(freq, n):
    return torch.tensor([[p * f for f in freq] for p in range(n)], dtype=torch.float64)


def _check_table(table, freq, times=1.0):
    angle = _angles(freq, table.shape[0])
    want = torch.cat([angle.cos(), angle.sin()], 1) * times
    # an angle below 2^10 in 64 bits is within 2^-43 of the formula's, cos and sin round to fp32 once
    assert table.dtype == torch.float32
    assert torch.all((table.double() - want).abs() <= 2.0 ** -24 * want.abs() + 2.0 ** -42)


def test_table_plain_linear_and_ntk():
    r, base, n = 64, 10000.0, 700
    freq = [base ** (-2 * i / r) for i in range(r // 2)]
    _check_table(rope.rope_table(n, r, base, device="cpu"), freq)
    _check_table(rope.rope_table(n, r, base, scaling="linear", factor=4.0, device="cpu"), [f / 4 for f in freq])
    table = rope.rope_table(n, r, base, scaling="ntk", factor=4.0, device="cpu")
    high = base * 4.0 ** (r / (r - 2))
    _check_table(table, [high ** (-2 * i / r) for i in range(r // 2)])
    assert high ** (-(r - 2) / r) == pytest.approx(freq[-1] / 4, rel=1e-12)   # the slowest is divided by 4


def test_table_yarn():
    r, base, factor, length = 128, 1e6, 4.0, 32768
    freq = [base ** (-2 * i / r) for i in range(r // 2)]
    turns = [length * f / (2 * math.pi) for f in freq]
    table = rope.rope_table(300, r, base, scaling="yarn", factor=factor, original_max_position=length, device="cpu")
    times = 0.1 * math.log(factor) + 1
    at = lambda n: r * math.log(length / (n * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    lo, hi = math.floor(at(32)), math.ceil(at(1))
    want = []
    for i, f in enumerate(freq):
        ramp = min(max((i - lo) / (hi - lo), 0), 1)
        want.append(f * (1 - ramp) + f / factor * ramp)
        if turns[i] > 33:
            assert ramp < 0.1
        if turns[i] < 0.9:
            assert want[-1] == f / factor
    _check_table(table, want, times)
    half = rope.rope_table(300, r, base, scaling="yarn", factor=factor, original_max_position=length,
                           attention_factor=0.5, device="cpu")
    _check_table(half, want, 0.5)
    _check_table(rope.rope_table(300, r, base, scaling="yarn", factor=1.0, original_max_position=length,
                                 device="cpu"), freq)


def test_table_by_wavelength():
    r, base, factor, length = 128, 500000.0, 8.0, 8192
    want = []
    for i in range(r // 2):
        f = base ** (-2 * i / r)
        wave = 2 * math.pi / f
        if wave < length / 4:
            want.append(f)
        elif wave > length / 1:
            want.append(f / factor)
        else:
            s = (length / wave - 1) / (4 - 1)
            want.append((1 - s) * f / factor + s * f)
    _check_table(rope.rope_table(300, r, base, scaling="wavelength", factor=factor, original_max_position=length,
                                 device="cpu"), want)


@pytest.mark.parametrize("kw", [dict(rotary_dim=63), dict(max_position=0), dict(scaling="other"), dict(scaling="yarn"),
                                dict(factor=0.5), dict(scaling="ntk", rotary_dim=2)])
def test_table_refusals(kw):
    with pytest.raises(AssertionError):
        rope.rope_table(**{"max_position": 10, "rotary_dim": 64, "device": "cpu", **kw})


# ------------------------------------------------------------------------------- the restatement
def test_restated_rows_are_within_half_a_step():
    x = torch.randn(500, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    code, step, low = int4.quantise(x)
    assert torch.equal(int4.unpack(int4.pack(code)), code)
    y = low.double()[:, None] + step.double()[:, None] * code.double()
    real = (x.double().amax(-1) - x.double().amin(-1)) / 15
    assert torch.all((x.double() - y).abs() <= real[:, None] * (0.5 + 15 * 2.0 ** -9))
    assert torch.all((step.double() - real).abs() <= real * 2.0 ** -8)


def test_restated_attention_is_softmax_of_the_rows():
    g = torch.Generator().manual_seed(2)
    n, kv, block = 40, 2, 16
    cache = int4_cache.new_kvcache_int4(3, block, kv, device="cpu")
    k, v = (torch.randn(n, kv, 128, generator=g).to(torch.bfloat16) for _ in range(2))
    table = torch.tensor([2, 0, 1], dtype=torch.int32)
    at = torch.arange(n)
    int4.store(k, v, *cache, table[at // block] * block + (at % block).to(torch.int32))
    q = torch.randn(5, 4, 128, generator=g).to(torch.bfloat16)
    out, bound = int4.attention(q, *cache, table, n, 0.1)
    (kc, ks, kl), (vc, vs, vl), _ = int4.sequence(*cache, table, n)
    for h in range(4):
        s = q[:, h].double() @ (kl + ks * kc)[:, h // 2].T * 0.1
        s = s.masked_fill(torch.arange(n)[None] > torch.arange(n - 5, n)[:, None], -math.inf)
        assert torch.allclose(out[:, h], torch.softmax(s, -1) @ (vl + vs * vc)[:, h // 2], rtol=1e-12, atol=1e-13)
    assert torch.all(bound > 0) and torch.all(bound < 0.02)


def test_a_failed_size_is_asked_for_again(monkeypatch):
    """What the workspace needs is remembered, that it could not be had is not."""
    answers, asked = [-1, -1, 4096], []

    class Lib:
        def fp8attn_int4_workspace_bytes(self, *args):
            asked.append(args)
            return answers[len(asked) - 1]

        fp8attn_last_error = _lib.lib.fp8attn_last_error

    monkeypatch.setattr(_lib, "lib", Lib())
    int4_cache._scratch_bytes.cache_clear()
    for _ in range(2):
        with pytest.raises(RuntimeError):
            int4_cache._scratch_bytes(0, 3, 8, 2, 1)
    assert int4_cache._scratch_bytes(0, 3, 8, 2, 1) == 4096 == int4_cache._scratch_bytes(0, 3, 8, 2, 1)
    assert len(asked) == 3
    int4_cache._scratch_bytes.cache_clear()


@pytest.mark.parametrize("args,msg", [((-1, 32, 8, 1), "num_seqs"), ((65536, 32, 8, 1), "num_seqs"),
                                      ((4, 30, 8, 1), "multiple"), ((4, 32, 0, 1), "multiple")])
def test_workspace_refusals_say_why(args, msg):
    assert _lib.lib.fp8attn_int4_workspace_bytes(*args) == -1
    assert msg in _message()


def _filled_cpu(n, kv, block, seed, spread=0.0):
    g = torch.Generator().manual_seed(seed)
    cache = int4_cache.new_kvcache_int4(-(-n // block), block, kv, device="cpu")
    k, v = (torch.randn(n, kv, 128, generator=g) * torch.exp2(spread * torch.randn(n, kv, 1, generator=g)) for _ in range(2))
    slots = torch.arange(n, dtype=torch.int32)
    int4.store(k.to(torch.bfloat16), v.to(torch.bfloat16), *cache, slots)
    return cache, torch.arange(-(-n // block), dtype=torch.int32), torch.randn(3, 4 * kv, 128, generator=g).to(torch.bfloat16)


@pytest.mark.parametrize("n,block,spread", [(50, 16, 0.0), (2000, 16, 0.0), (2000, 16, 1.0), (20000, 64, 0.0)])
def test_the_norm_tells_wrong_outputs(n, block, spread):
    """What ``attention_norm`` allows is far less than what zeros, a page left out, a scale 1 % off, values 1 % off (3 % where
    scores are large), or rows one place off make of an output.  (With rows of many sizes some queries look at one position alone: neither the
    scale nor another page changes those.)"""
    all_or_some = torch.all if spread == 0 else torch.any
    cache, table, q = _filled_cpu(n, 1, block, 3, spread)
    ref, room = int4.attention_norm(q, *cache, table, n, 0.09)
    off = lambda out: ((out - ref).norm(dim=-1) / room)  # noqa: E731
    assert torch.all(off(ref.to(torch.bfloat16).double()) < 1)       # the rounding alone
    assert torch.all(off(torch.zeros_like(ref)) > 20)
    assert all_or_some(off(int4.attention_norm(q, *cache, table, n, 0.09 * 1.01)[0]) > 1)
    assert torch.all(off(ref * (1.01 if spread == 0 else 1.03)) > 1)
    assert torch.all(off(ref.roll(1, 0)) > 20) and torch.all(off(ref.roll(1, 1)) > 20)
    for page in (0, table.numel() // 2, table.numel() - 2) if spread == 0 else ():
        without = table.clone()
        without[page] = -1
        worst = off(int4.attention_norm(q, *cache, without, n, 0.09)[0])
        assert torch.all(worst > 1), f"page {page}"
