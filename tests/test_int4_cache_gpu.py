"""store_kvcache_int4 and load_kvcache_int4 against the 64-bit restatement (oracle/int4.py): codes, steps and
lowest values are equal in every bit, values read back are one rounding from low + step * code."""
import math

import pytest
import torch

from oracle import int4

pytestmark = pytest.mark.gpu


def _randn(shape, seed, sd=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * sd).to(torch.bfloat16)


def _filled(blocks, block, kv, seed):
    """A cache with something in every byte."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    code = lambda: torch.randint(0, 256, (blocks, kv, block, 64), generator=g, device="cuda",  # noqa: E731
                                 dtype=torch.int32).to(torch.uint8)
    return code(), code(), torch.randn(blocks, kv, block, 4, generator=g, device="cuda").to(torch.bfloat16)


def _slots(n, total, seed):
    g = torch.Generator().manual_seed(seed)
    s = torch.randperm(total, generator=g)[:n].to(torch.int32)
    s[3::7] = -1
    s[5::11] = total + 3
    return s.cuda()


def _check_store(key, value, cache, slots):
    from nanovllm_b200.int4_cache import store_kvcache_int4
    want = [t.clone() for t in cache]
    int4.store(key, value, *want, slots)
    store_kvcache_int4(key, value, *cache, slots)
    for got, ref in zip(cache[:2], want[:2]):
        assert torch.equal(got, ref), f"{int((got != ref).sum())} bytes of codes differ"
    nan = torch.isnan(want[2])
    assert torch.equal(torch.isnan(cache[2]), nan)
    assert torch.equal(cache[2][~nan], want[2][~nan])


def _check_load(cache, slots):
    from nanovllm_b200.int4_cache import load_kvcache_int4
    blocks, kv, block, _ = cache[0].shape
    key, value = load_kvcache_int4(*cache, slots)
    ok = (slots >= 0) & (slots < blocks * block)
    at = slots.long().clamp(0, blocks * block - 1)
    for got, codes, j in ((key, cache[0], 0), (value, cache[1], 2)):
        assert got.shape == (slots.numel(), kv, 128) and got.is_contiguous()
        assert torch.all(got[~ok] == 0)
        c, step, low = int4.rows(codes[at // block, :, at % block],
                                 cache[2][at // block, :, at % block, j:j + 2])
        ref = (low + step * c)[ok]
        far = (got[ok].double() - ref).abs()
        # one rounding to 8 bits after one in fp32; 2^-134 is half a step of bf16's smallest numbers
        room = ref.abs() * 2.0 ** -8 * (1 + 2.0 ** -15) + 2.0 ** -134
        assert torch.equal(torch.isnan(got[ok]), torch.isnan(ref))
        fine = torch.isfinite(ref) & (ref.abs() < 3.38e38)
        assert torch.all((far <= room)[fine])
    return key, value


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 33, 500, 4097])
@pytest.mark.parametrize("kv,block", [(8, 256), (1, 16), (3, 48), (2, 64)])
def test_write_and_read_back(n, kv, block):
    blocks = 2 * n // block + 2
    cache = _filled(blocks, block, kv, n)
    key, value = _randn((n, kv, 128), 1), _randn((n, kv, 128), 2, 3.0)
    slots = _slots(n, blocks * block, n + kv)
    _check_store(key, value, cache, slots)
    k, v = _check_load(cache, slots)
    # a value is half a step from the one written, and what the step's rounding (2^-9) adds over 15 steps
    ok = (slots >= 0) & (slots < blocks * block)
    for x, y in ((key, k), (value, v)):
        x, y = x[ok].double(), y[ok].double()
        step = (x.amax(-1, keepdim=True) - x.amin(-1, keepdim=True)) / 15
        assert torch.all((x - y).abs() <= step * (0.5 + 15 * 2.0 ** -9) * (1 + 2.0 ** -8) + y.abs() * 2.0 ** -8)


@pytest.mark.parametrize("make", ["tokens", "heads", "odd", "headmajor", "expanded"])
def test_strided_rows(make):
    n, kv, block = 77, 4, 32
    if make == "tokens":  # as a fused projection leaves them
        wide = _randn((n, 3 * kv * 128), 3)
        key, value = wide[:, 512:1024].view(n, kv, 128), wide[:, 1024:].view(n, kv, 128)
    elif make == "heads":
        wide = _randn((n, kv, 2, 128), 4)
        key, value = wide[:, :, 0], wide[:, :, 1]
    elif make == "odd":   # no 16-byte accesses
        flat = _randn((n * (kv * 128 + 3) + 8,), 5)
        key = torch.as_strided(flat, (n, kv, 128), (kv * 128 + 3, 128, 1), 1)
        value = torch.as_strided(flat, (n, kv, 128), (kv * 128 + 3, 128, 1), 4)
    elif make == "headmajor":
        key, value = _randn((kv, n, 128), 6).transpose(0, 1), _randn((kv, n, 128), 7).transpose(0, 1)
    else:
        key, value = _randn((1, kv, 128), 8).expand(n, kv, 128), _randn((n, 1, 128), 9).expand(n, kv, 128)
    cache = _filled(8, block, kv, 1)
    _check_store(key, value, cache, _slots(n, 8 * block, 2))


def _special_rows():
    g = torch.Generator().manual_seed(11)
    rand = lambda: torch.randn(128, generator=g)  # noqa: E731
    ints = lambda top: torch.randint(0, top, (128,), generator=g).float()  # noqa: E731
    rows = [torch.zeros(128), torch.full((128,), -3.25), rand() * 1e-38, rand() * 1e-40, rand() * 3e37,
            ints(31) / 2, ints(16), ints(31) - 15, ints(61) / 4 - 7,       # quotients on borders
            torch.where(torch.arange(128) < 64, 1.0, 1.0078125),          # one step of bf16 apart
            torch.where(torch.arange(128) == 5, 1e30, 0.0) + 0.0, rand() + 1000.0,
            torch.tensor([0.0, -0.0] * 64), torch.tensor([9.2e-41, 0.0] * 64),
            torch.tensor([1.3e-39, 0.0, 4e-40, 9e-41] * 32), torch.tensor([3e38, -3e38] + [0.0] * 126),
            torch.tensor([-4.0, 1e-5, 0.0, 11.0] * 32), torch.tensor([2.0 ** 60, 2.0 ** -60, -1.0, 0.0] * 32)]
    nan, inf = rand(), rand()
    nan[17], inf[100] = math.nan, -math.inf
    both = rand()
    both[0], both[127] = math.inf, -math.inf
    rows += [nan, inf, both, torch.full((128,), math.inf), torch.full((128,), math.nan)]
    for i in range(30):  # rows on a grid, where many quotients are borders
        low, step = float(torch.randn((), generator=g)), 2.0 ** float(torch.randint(-6, 6, (), generator=g))
        x = torch.tensor(low).to(torch.bfloat16).float() + step * ints(31) / 2
        rows.append(x)
    return torch.stack(rows).to(torch.bfloat16)


def test_borders_extremes_and_nan():
    x = _special_rows().cuda()
    n = x.shape[0]
    key = torch.stack([x, x.flip(0)], 1)     # two heads
    value = torch.stack([x.flip(0), x], 1)
    cache = _filled(4, 32, 2, 3)
    slots = torch.randperm(128, generator=torch.Generator().manual_seed(1))[:n].to(torch.int32).cuda()
    _check_store(key, value, cache, slots)
    k, _ = _check_load(cache, slots)
    bad = ~torch.isfinite(x.float()).all(-1) | (x.float().amax(-1) - x.float().amin(-1) > 3.4e38)
    assert bad.sum() == 6
    assert torch.equal(torch.isnan(k[:, 0]).all(-1), bad) and torch.equal(torch.isnan(k[:, 0]).any(-1), bad)
    const = ~bad & (x.float().amax(-1) == x.float().amin(-1))
    assert torch.equal(k[:, 0][const].float(), x[const].float())


def test_every_border_of_many_grids():
    """Rows whose values lie on the halves between codes for every step's mantissa: ties go to even."""
    rows = []
    for mantissa in range(128, 256, 3):
        step = mantissa * 2.0 ** -7
        for low in (0.0, -1.0, 3.0, -4.0):
            x = low + step * torch.arange(31, dtype=torch.float64) / 2
            rows.append(torch.cat([x, x, x, x, x[:4]]).to(torch.bfloat16))
    x = torch.stack(rows)[:, None].cuda()
    cache = _filled(x.shape[0] // 16 + 1, 16, 1, 4)
    slots = torch.arange(x.shape[0], dtype=torch.int32, device="cuda")
    _check_store(x, x.flip(0), cache, slots)


def test_repeated_reads_and_empty_calls():
    from nanovllm_b200.int4_cache import load_kvcache_int4, new_kvcache_int4, store_kvcache_int4
    cache = _filled(3, 16, 2, 5)
    _check_load(cache, torch.tensor([5, 5, 47, 0, -1, 48, 5, -7], dtype=torch.int32, device="cuda"))
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    k, v = load_kvcache_int4(*cache, none)
    assert k.shape == (0, 2, 128) and v.shape == (0, 2, 128)
    before = [t.clone() for t in cache]
    empty = torch.empty(0, 2, 128, dtype=torch.bfloat16, device="cuda")
    store_kvcache_int4(empty, empty, *cache, none)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, before))
    k, v = load_kvcache_int4(*new_kvcache_int4(2, 16, 3), torch.arange(32, dtype=torch.int32, device="cuda"))
    assert torch.all(k == 0) and torch.all(v == 0)


def test_slots_far_into_a_large_cache():
    """Byte offsets past 2^32."""
    from nanovllm_b200.int4_cache import new_kvcache_int4
    blocks, block, kv = 41000, 256, 8       # 5.4 GB of codes for K
    cache = new_kvcache_int4(blocks, block, kv)
    n = 40
    g = torch.Generator().manual_seed(1)
    slots = (blocks * block - 1 - torch.randperm(200, generator=g)[:n]).to(torch.int32).cuda()
    from nanovllm_b200.int4_cache import store_kvcache_int4
    key, value = _randn((n, kv, 128), 1), _randn((n, kv, 128), 2)
    store_kvcache_int4(key, value, *cache, slots)
    _check_load(cache, slots)
    page, place = slots.long() // block, slots.long() % block
    code, step, low = int4.quantise(key)
    assert torch.equal(cache[0][page, :, place], int4.pack(code))
    assert torch.equal(cache[2][page, :, place, 0], step) and torch.equal(cache[2][page, :, place, 1], low)
    assert int(cache[0][:blocks - 1].count_nonzero()) == 0


def test_captured_on_another_stream():
    from nanovllm_b200.int4_cache import load_kvcache_int4, store_kvcache_int4
    n, kv = 50, 4
    cache = _filled(8, 16, kv, 6)
    key, value, slots = _randn((n, kv, 128), 1), _randn((n, kv, 128), 2), _slots(n, 128, 3)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        store_kvcache_int4(key, value, *cache, slots)
        load_kvcache_int4(*cache, slots)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        store_kvcache_int4(key, value, *cache, slots)
        k, v = load_kvcache_int4(*cache, slots)
    for seed in range(3):
        key.copy_(_randn((n, kv, 128), 10 + seed))
        slots.copy_(_slots(n, 128, 20 + seed))
        graph.replay()
        torch.cuda.synchronize()
        want = load_kvcache_int4(*cache, slots)
        assert torch.equal(k, want[0]) and torch.equal(v, want[1])
        code, step, low = int4.quantise(key)
        ok = (slots >= 0) & (slots < 128)
        at = slots[ok].long()
        assert torch.equal(cache[0][at // 16, :, at % 16], int4.pack(code)[ok])
