"""apply_rope against the definition in 64 bits on the same table.

Tolerance: two products and a sum in fp32, each within half a step of its own result: at most 2^-23 of
|x1 cos| + |x2 sin|; then one rounding to the type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def _randn(shape, seed, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _table(positions, r, seed=3):
    from nanovllm_b200.rope import rope_table
    return rope_table(positions, r, base=1e6)


def _turned(x, positions, table, interleaved):
    """(value, magnitude of its two products) in float64."""
    r = table.shape[-1]
    row = table.double()[positions.clamp(0, table.shape[0] - 1)]
    c, s = row[:, None, :r // 2], row[:, None, r // 2:]
    y, size = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    first = slice(0, r, 2) if interleaved else slice(0, r // 2)
    second = slice(1, r, 2) if interleaved else slice(r // 2, r)
    a, b = x.double()[..., first], x.double()[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first], size[..., second] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, size


def _check(got, x, positions, table, interleaved):
    ref, size = _turned(x, positions, table, interleaved)
    half = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps / 2
    assert got.shape == x.shape and got.dtype == x.dtype
    far = (got.double() - ref).abs()
    assert torch.all(far <= half * (ref.abs() + 2.0 ** -23 * size) + 2.0 ** -23 * size + tiny)
    r = table.shape[-1]
    assert torch.equal(got[..., r:], x[..., r:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,heads,kv,d,r", [(1, 32, 8, 128, 128), (7, 3, 1, 128, 64), (300, 40, 8, 128, 128),
                                            (5, 4, 4, 80, 80), (6, 2, 2, 80, 32), (9, 5, 1, 64, 20),
                                            (4, 2, 1, 96, 90), (3, 1, 1, 2, 2), (11, 7, 7, 192, 64),
                                            (2, 16, 16, 256, 256), (2000, 9, 2, 128, 96), (3, 2, 1, 6, 4),
                                            (900, 9, 2, 80, 34), (800, 10, 1, 96, 44)])
def test_against_definition(n, heads, kv, d, r, interleaved, dtype):
    from nanovllm_b200.rope import apply_rope
    q, k = _randn((n, heads, d), n, dtype), _randn((n, kv, d), n + 1, dtype)
    table = _table(5000, r)
    g = torch.Generator(device="cuda").manual_seed(n)
    positions = torch.randint(0, 5000, (n,), generator=g, device="cuda")
    got = apply_rope(q, k, positions, table, interleaved=interleaved)
    for y, x in zip(got, (q, k)):
        assert y.is_contiguous()
        _check(y, x, positions, table, interleaved)
    again = q.clone(), k.clone()
    res = apply_rope(*again, positions, table, interleaved=interleaved, inplace=True)
    assert res[0] is again[0] and res[1] is again[1]
    assert torch.equal(res[0], got[0]) and torch.equal(res[1], got[1])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("make", ["fused", "headmajor", "odd", "even", "expanded"])
def test_strides(make, interleaved):
    from nanovllm_b200.rope import apply_rope
    n, heads, kv, d, dtype = 37, 6, 2, 128, torch.bfloat16
    if make == "fused":
        wide = _randn((n, (heads + 2 * kv) * d), 1, dtype)
        q, k = wide[:, :heads * d].view(n, heads, d), wide[:, heads * d:(heads + kv) * d].view(n, kv, d)
    elif make == "headmajor":
        q, k = _randn((heads, n, d), 1, dtype).transpose(0, 1), _randn((kv, n, d), 2, dtype).transpose(0, 1)
    elif make in ("odd", "even"):
        step = 3 if make == "odd" else 2
        flat = _randn((n * (heads * d + step) + 200,), 3, dtype)
        q = torch.as_strided(flat, (n, heads, d), (heads * d + step, d, 1), step)
        k = torch.as_strided(_randn((n * (kv * d + step) + 200,), 4, dtype), (n, kv, d), (kv * d + step, d, 1), step)
    else:
        q, k = _randn((1, heads, d), 5, dtype).expand(n, heads, d), _randn((n, 1, d), 6, dtype).expand(n, kv, d)
    table = _table(1000, 64)
    positions = torch.arange(n, device="cuda") * 17
    got = apply_rope(q, k, positions, table, interleaved=interleaved)
    _check(got[0], q, positions, table, interleaved)
    _check(got[1], k, positions, table, interleaved)
    if make != "expanded":
        around = None if make not in ("odd", "even") else flat.clone()
        res = apply_rope(q, k, positions, table, interleaved=interleaved, inplace=True)
        assert torch.equal(res[0], got[0]) and torch.equal(res[1], got[1])
        if around is not None:   # what lies between the rows stays
            back = torch.as_strided(around, q.shape, q.stride(), q.storage_offset())
            back.copy_(q)
            assert torch.equal(around, flat)


def test_in_place_rows_that_share_memory_are_refused():
    from nanovllm_b200._lib import Fp8AttnError
    from nanovllm_b200.rope import apply_rope
    q = _randn((4, 1, 128), 1, torch.bfloat16).expand(4, 3, 128)
    positions = torch.arange(4, device="cuda")
    with pytest.raises(Fp8AttnError, match="overlap"):
        apply_rope(q, None, positions, _table(10, 128), inplace=True)
    x = _randn((4, 2, 128), 1, torch.bfloat16)
    with pytest.raises(Fp8AttnError, match="same memory"):
        apply_rope(x, x, positions, _table(10, 128), inplace=True)


def test_positions_outside_the_table_and_no_k():
    from nanovllm_b200.rope import apply_rope
    q = _randn((5, 2, 128), 1, torch.bfloat16)
    table = _table(100, 128).view(100, 1, 128)
    positions = torch.tensor([-1, 0, 99, 100, 1 << 40], device="cuda")
    got, none = apply_rope(q, None, positions, table)
    assert none is None
    _check(got, q, positions, table.view(100, 128), False)
    empty = apply_rope(q[:0], q[:0], positions[:0], table)
    assert empty[0].shape == (0, 2, 128) and empty[1].shape == (0, 2, 128)


def test_nan_and_infinity_stay_in_their_pair():
    from nanovllm_b200.rope import apply_rope
    q = _randn((1, 2, 128), 1, torch.bfloat16)
    q[0, 0, 3] = float("nan")
    q[0, 1, 70] = float("inf")
    got, _ = apply_rope(q, None, torch.tensor([5], device="cuda"), _table(100, 128))
    bad = ~torch.isfinite(got)
    assert bad.nonzero().tolist() == [[0, 0, 3], [0, 0, 67], [0, 1, 6], [0, 1, 70]]


def test_matches_the_fused_epilogue():
    """With unit norm weights the fused epilogue's q and k are those of apply_rope on its normalised rows."""
    from nanovllm_b200.qk_epilogue import qk_norm_rope_store
    from nanovllm_b200.rope import apply_rope
    n, heads, kv = 33, 8, 2
    qkv = _randn((n, (heads + 2 * kv) * 128), 1, torch.bfloat16)
    w = _randn((128,), 2, torch.bfloat16)
    positions, table = torch.arange(n, device="cuda") * 5, _table(400, 128)
    turned = qk_norm_rope_store(qkv, positions, w, w, 1e-6, table, heads, kv, None, None, None, return_k=True)
    plain = qk_norm_rope_store(qkv, positions * 0, w, w, 1e-6, table, heads, kv, None, None, None, return_k=True)
    got = apply_rope(*plain, positions, table)   # position 0 turns nothing
    assert torch.equal(got[0], turned[0]) and torch.equal(got[1], turned[1])


def test_captured():
    from nanovllm_b200.rope import apply_rope
    q, k = _randn((20, 8, 128), 1, torch.float16), _randn((20, 2, 128), 2, torch.float16)
    positions, table = torch.arange(20, device="cuda"), _table(1000, 128)
    apply_rope(q, k, positions, table)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = apply_rope(q, k, positions, table)
    positions += 300
    graph.replay()
    torch.cuda.synchronize()
    _check(got[0], q, positions, table, False)
    _check(got[1], k, positions, table, False)
