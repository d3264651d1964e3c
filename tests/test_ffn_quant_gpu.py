"""add_rms_norm_fp8 and silu_mul_fp8 against 64-bit restatements (oracle/ffn.py).

Tolerances, from the arithmetic: the norm's fp32 sum runs over at most 32 terms in a thread, 5 in a warp
and 16 warps, so it is off by at most 53 2^-24, its inverse root by half of that and 2 ulps, and three
more products by half an ulp each: under 2^-18.  SiLU: exp within 2 ulps, an addition, a division and a
product: under 2^-20, and where 1 + exp(-g) is above 2^126 (g < -87.3), whose inverse is below fp32's
normal numbers, the result is 0 for a true |h| of at most 87.4 2^-126 |u|, below 2^-119 |u|.  Outputs in 8 and 16 bits are then the rounding of a value within that of the definition's.
"""
import pytest
import torch

from oracle import ffn

pytestmark = pytest.mark.gpu
EPS = 1e-6
NORM_REL = 2.0 ** -18
SILU_REL = 2.0 ** -20
DTYPES = [torch.bfloat16, torch.float16]


def _randn(shape, seed, dtype, sd=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * sd).to(dtype)


def _norm_inputs(m, k, dtype, seed, residual=True):
    x = _randn((m, k), seed, dtype)
    r = _randn((m, k), seed + 1, dtype, 3.0) if residual else None
    w = _randn((k,), seed + 2, dtype, 0.3) + 1
    return x, r, w.to(dtype)


def _check_norm(x, r, w, eps=EPS, return_norm=True):
    from nanovllm_b200.fp8_ffn import add_rms_norm_fp8
    q, d, res, y = add_rms_norm_fp8(x, r, w, eps, return_norm=return_norm)
    m, k = x.shape
    assert q.shape == (m, k) and q.dtype == torch.float8_e4m3fn and q.is_contiguous()
    assert d.shape == (m, k // 128) and d.dtype == torch.bfloat16 and d.is_contiguous()
    s64, y64 = ffn.norm(x, r, w, eps)
    ffn.assert_quantised(q, d, y64, NORM_REL)
    if r is None:
        assert res is None
    else:
        ffn.assert_within(res, s64, s64.abs() * 2.0 ** -23, ffn.dtype_round(x.dtype), "residual")
    if return_norm:
        ffn.assert_within(y, y64, y64.abs() * NORM_REL, ffn.dtype_round(x.dtype), "norm")
    else:
        assert y is None
    return q, d, res, y


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("m,k", [(1, 128), (1, 4096), (3, 256), (5, 384), (7, 512), (2, 640), (9, 1152),
                                 (33, 2048), (4, 2176), (17, 4096), (6, 4224), (3, 5120), (2, 8192),
                                 (5, 8320), (2, 16384), (1000, 1024)])
def test_norm(m, k, residual, dtype):
    _check_norm(*_norm_inputs(m, k, dtype, 3 * m + k, residual))


def test_norm_without_the_unquantised_output():
    _check_norm(*_norm_inputs(11, 1024, torch.bfloat16, 5), return_norm=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_edges(dtype):
    x, r, w = _norm_inputs(8, 1024, dtype, 21)
    x[0], r[0] = 0, 0                       # an all-zero row: scale 1, zeros
    r[1] = -x[1]                            # cancels
    x[2, :128], r[2, :128] = 0, 0           # an all-zero group
    w[256:384] = 0                          # a group that the weight empties
    x[3], r[3] = 2.0 ** -13, 2.0 ** -14     # tiny: eps counts
    x[4, 7] = 60000.0                       # one value over all others
    q, d, res, y = _check_norm(x, r, w)
    assert bool((d[0] == 1).all()) and bool((q[0].float() == 0).all())
    assert float(d[2, 0]) == 1 and float(d[5, 2]) == 1


def test_norm_nan_and_infinity_stay_in_their_row():
    x, r, w = _norm_inputs(5, 512, torch.bfloat16, 31)
    x[1, 100] = float("nan")
    x[3, 200] = float("inf")
    from nanovllm_b200.fp8_ffn import add_rms_norm_fp8
    q, d, res, y = add_rms_norm_fp8(x, r, w, EPS, return_norm=True)
    v = ffn.dequantise(q, d)
    assert bool(torch.isnan(v[1]).all()) and bool(torch.isnan(y[1]).all())
    assert bool(torch.isnan(y[3, 200])) and bool((y[3, :100] == 0).all())  # x / inf
    keep = [0, 2, 4]
    s64, y64 = ffn.norm(x[keep], r[keep], w, EPS)
    ffn.assert_quantised(q[keep], d[keep], y64, NORM_REL)


def test_norm_strided_rows_and_single_rows():
    x, r, w = _norm_inputs(13, 640, torch.bfloat16, 41)
    wide = torch.zeros(13, 2000, dtype=torch.bfloat16, device="cuda")
    wide[:, 8:648] = x
    wide_r = torch.zeros(26, 640, dtype=torch.bfloat16, device="cuda")
    wide_r[::2] = r
    a = _check_norm(x, r, w)
    b = _check_norm(wide[:, 8:648], wide_r[::2], w)
    for s, t in zip(a, b):
        assert torch.equal(s.view(torch.uint8), t.view(torch.uint8))
    _check_norm(wide[3:4, 8:648], wide_r[4:5], w)
    _check_norm(x[2:3].t().contiguous().t(), r[2:3], w)     # one row, column-major strides


def test_norm_in_place_residual_through_the_c_abi():
    from nanovllm_b200 import _lib
    x, r, w = _norm_inputs(300, 2048, torch.bfloat16, 51)
    from nanovllm_b200.fp8_ffn import add_rms_norm_fp8
    q, d, res, _ = add_rms_norm_fp8(x, r, w, EPS)
    q2, d2, r2 = torch.empty_like(q), torch.empty_like(d), r.clone()
    _lib.check(_lib.lib.fp8attn_add_rms_norm_quant(
        x.data_ptr(), 2048, r2.data_ptr(), 2048, w.data_ptr(), EPS, q2.data_ptr(), d2.data_ptr(),
        r2.data_ptr(), 0, 300, 2048, _lib.BF16, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(res, r2) and torch.equal(d, d2)
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8))


@pytest.mark.parametrize("m,k", [(1, 128), (3, 1152), (5, 16384)])
def test_norm_writes_its_rows_only(m, k):
    """Outputs between guard rows, through the C-ABI."""
    from nanovllm_b200 import _lib
    x, r, w = _norm_inputs(m, k, torch.bfloat16, 61)
    bufs = [torch.full(((m + 2) * n,), 0x5A, dtype=torch.uint8, device="cuda")
            for n in (k, 2 * k // 128 * 8, 2 * k, 2 * k)]
    row = [k, 2 * k // 128, 2 * k, 2 * k]
    ptr = [b.data_ptr() + (n + 15) // 16 * 16 for b, n in zip(bufs, row)]
    _lib.check(_lib.lib.fp8attn_add_rms_norm_quant(
        x.data_ptr(), k, r.data_ptr(), k, w.data_ptr(), EPS, ptr[0], ptr[1], ptr[2], ptr[3], m, k,
        _lib.BF16, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    for b, n in zip(bufs, row):
        lo = (n + 15) // 16 * 16
        assert bool((b[:lo] == 0x5A).all()) and bool((b[lo + m * n:] == 0x5A).all())


# ------------------------------------------------------------------------------------------ silu
def _check_silu(gu):
    from nanovllm_b200.fp8_ffn import silu_mul_fp8
    q, d = silu_mul_fp8(gu)
    m, i = gu.shape[0], gu.shape[1] // 2
    assert q.shape == (m, i) and d.shape == (m, i // 128)
    assert q.is_contiguous() and d.is_contiguous() and d.dtype == torch.bfloat16
    h = ffn.silu_mul(gu[:, :i], gu[:, i:])
    top = float(torch.nan_to_num(gu[:, i:].double(), posinf=0, neginf=0).abs().max()) if m else 0
    ffn.assert_quantised(q, d, h, SILU_REL, absolute=2.0 ** -119 * max(1.0, top))
    return q, d


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,i", [(1, 128), (1, 12288), (3, 256), (17, 384), (5, 1152), (2, 25600),
                                 (333, 640), (1000, 768), (64, 4096)])
def test_silu(m, i, dtype):
    _check_silu(_randn((m, 2 * i), m + i, dtype, 2.0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_silu_edges(dtype):
    gu = _randn((6, 1024), 71, dtype, 2.0)
    gu[0] = 0                                # all zero: scale 1
    gu[1, :512] = -200.0                     # exp(-g) overflows: h is 0 in fp32
    gu[2, :512] = 200.0                      # sigmoid is 1
    gu[3, 640:768] = 0                       # a group of zero ups
    gu[4, 3] = 30000.0
    gu[4, 515] = 2.0
    q, d = _check_silu(gu)
    assert bool((d[0] == 1).all()) and bool((q[0].float() == 0).all())
    assert float(d[3, 1]) == 1


def test_silu_nan_and_infinity():
    gu = _randn((3, 512), 81, torch.bfloat16)
    gu[0, 5] = float("nan")                  # gate: that value alone
    gu[1, 256 + 130] = float("nan")          # up
    gu[2, 7] = float("inf")                  # the group's scale is infinite
    from nanovllm_b200.fp8_ffn import silu_mul_fp8
    q, d = silu_mul_fp8(gu)
    f = q.float()
    assert bool(torch.isnan(f[0, 5])) and int(torch.isnan(f[0]).sum()) == 1
    assert bool(torch.isnan(f[1, 130])) and int(torch.isnan(f[1]).sum()) == 1
    clean = gu.clone()
    clean[0, 5] = 0
    clean[1, 256 + 130] = 0
    cq, cd = silu_mul_fp8(clean)
    assert torch.equal(d[:2], cd[:2])
    keep = ~torch.isnan(f[:2])
    assert torch.equal(f[:2][keep], cq.float()[:2][keep])
    assert float(d[2, 0]) == float("inf") and bool(torch.isfinite(d[2, 1]))


def test_silu_strided_rows():
    gu = _randn((9, 768), 91, torch.bfloat16)
    wide = torch.zeros(18, 1000, dtype=torch.bfloat16, device="cuda")
    wide[::2, 16:784] = gu
    a, b = _check_silu(gu), _check_silu(wide[::2, 16:784])
    assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])


def test_long_inputs_pass_32_bit_offsets():
    """More than 2^31 elements in: rows at both ends."""
    from nanovllm_b200.fp8_ffn import add_rms_norm_fp8, silu_mul_fp8
    m, i = 90_001, 12288                                    # 2.2e9 values of gate_up
    gu = torch.zeros((m, 2 * i), dtype=torch.bfloat16, device="cuda")
    rows = [0, 1, m // 2, m - 1]
    gu[rows] = _randn((len(rows), 2 * i), 7, torch.bfloat16, 2.0)
    q, d = silu_mul_fp8(gu)
    h = ffn.silu_mul(gu[rows][:, :i], gu[rows][:, i:])
    ffn.assert_quantised(q[rows], d[rows], h, SILU_REL, 2.0 ** -110)
    assert bool((d[2:m // 2] == 1).all())
    x = gu.view(-1)[:m * 2 * i // 16384 * 16384].view(-1, 16384)
    w = _randn((16384,), 8, torch.bfloat16)
    q, d, _, _ = add_rms_norm_fp8(x, None, w, EPS)
    ends = [0, x.shape[0] - 1]
    _, y64 = ffn.norm(x[ends], None, w, EPS)
    ffn.assert_quantised(q[ends], d[ends], y64, NORM_REL)


# ---------------------------------------------------------------------- as a program uses them
def test_empty_batches():
    from nanovllm_b200.fp8_ffn import add_rms_norm_fp8, silu_mul_fp8
    x = torch.empty((0, 512), dtype=torch.bfloat16, device="cuda")
    w = torch.ones(512, dtype=torch.bfloat16, device="cuda")
    q, d, res, y = add_rms_norm_fp8(x, x, w, EPS, return_norm=True)
    assert q.shape == (0, 512) and d.shape == (0, 4) and res.shape == y.shape == (0, 512)
    q, d = silu_mul_fp8(x)
    assert q.shape == (0, 256) and d.shape == (0, 2)


def test_dense_block_as_a_layer_runs_it():
    """norm -> gate_up product -> SiLU -> down product: the operands are what the product's own
    quantisation makes of the same values, to within its midpoints."""
    from nanovllm_b200.fp8_ffn import add_rms_norm_fp8, silu_mul_fp8
    from nanovllm_b200.fp8_linear import fp8_block_gemm, fp8_dyn_quant
    m, h, i = 37, 1024, 1536
    x, r, w = _norm_inputs(m, h, torch.bfloat16, 101)
    w13 = _randn((2 * i, h), 1, torch.float32, 100.0).clamp(-448, 448).to(torch.float8_e4m3fn)
    w2 = _randn((h, i), 2, torch.float32, 100.0).clamp(-448, 448).to(torch.float8_e4m3fn)
    s13 = (torch.rand(2 * i // 128, h // 128, device="cuda") * 3e-4).to(torch.bfloat16)
    s2 = (torch.rand(h // 128, i // 128, device="cuda") * 3e-4).to(torch.bfloat16)
    xq, xs, res, y = add_rms_norm_fp8(x, r, w, EPS, return_norm=True)
    gu = fp8_block_gemm(xq, xs, w13, s13)
    hq, hs = silu_mul_fp8(gu)
    out = fp8_block_gemm(hq, hs, w2, s2)
    # each stage from the stage before it, in 64 bits
    gu64 = ffn.dequantise(xq, xs) @ ffn.weight_values(w13, s13).t()
    bound = ffn.dequantise(xq, xs).abs() @ ffn.weight_values(w13, s13).abs().t() * 2.0 ** -16
    ffn.assert_within(gu, gu64, bound, ffn.bf16, "gate_up")
    ffn.assert_quantised(hq, hs, ffn.silu_mul(gu[:, :i], gu[:, i:]), SILU_REL, 2.0 ** -110)
    hv, v2 = ffn.dequantise(hq, hs), ffn.weight_values(w2, s2)
    ffn.assert_within(out, hv @ v2.t(), hv.abs() @ v2.abs().t() * 2.0 ** -16, ffn.bf16, "down")
    # the stand-alone quantisation of the bf16 norm sees values half a bf16 step away at most
    q2, d2 = fp8_dyn_quant(y)
    a, b = ffn.dequantise(xq, xs), ffn.dequantise(q2, d2)
    step = ffn.spread(ffn.group_scale(a)) * 2.0 ** -9 + a.abs() * (2.0 ** -3 + 2.0 ** -7)
    assert bool(((a - b).abs() <= step).all())


def test_captured_and_replayed_with_new_inputs():
    from nanovllm_b200.fp8_ffn import add_rms_norm_fp8, silu_mul_fp8
    x, r, w = _norm_inputs(19, 2048, torch.bfloat16, 111)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        add_rms_norm_fp8(x, r, w, EPS)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q, d, res, y = add_rms_norm_fp8(x, r, w, EPS, return_norm=True)
        hq, hs = silu_mul_fp8(y)
    for seed in (1, 2):
        nx, nr, _ = _norm_inputs(19, 2048, torch.bfloat16, seed)
        x.copy_(nx)
        r.copy_(nr)
        g.replay()
        s64, y64 = ffn.norm(x, r, w, EPS)
        ffn.assert_quantised(q, d, y64, NORM_REL)
        ffn.assert_quantised(hq, hs, ffn.silu_mul(y[:, :1024], y[:, 1024:]), SILU_REL, 2.0 ** -110)


def test_another_stream_and_repeated_calls_agree():
    from nanovllm_b200.fp8_ffn import add_rms_norm_fp8, silu_mul_fp8
    x, r, w = _norm_inputs(65, 4096, torch.float16, 121)
    a = add_rms_norm_fp8(x, r, w, EPS, return_norm=True)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b = add_rms_norm_fp8(x, r, w, EPS, return_norm=True)
        hb = silu_mul_fp8(b[3])
    ha = silu_mul_fp8(a[3])
    torch.cuda.synchronize()
    for p, q in zip((*a, *ha), (*b, *hb)):
        assert torch.equal(p.view(torch.uint8), q.view(torch.uint8))


def test_refusals():
    from nanovllm_b200._lib import Fp8AttnError
    from nanovllm_b200.fp8_ffn import add_rms_norm_fp8, silu_mul_fp8
    x, r, w = _norm_inputs(4, 512, torch.bfloat16, 131)
    for bad in [lambda: add_rms_norm_fp8(x.float(), r, w, EPS),
                lambda: add_rms_norm_fp8(x.cpu(), r, w, EPS),
                lambda: add_rms_norm_fp8(x, r.half(), w, EPS),
                lambda: add_rms_norm_fp8(x, r[:3], w, EPS),
                lambda: add_rms_norm_fp8(x, r, w[:256], EPS),
                lambda: add_rms_norm_fp8(x, r, w.float(), EPS),
                lambda: add_rms_norm_fp8(x[:, :200], r[:, :200], w[:200], EPS),
                lambda: add_rms_norm_fp8(x.t(), r.t(), w[:4], EPS),
                lambda: silu_mul_fp8(x[:, :384]), lambda: silu_mul_fp8(x.float()),
                lambda: silu_mul_fp8(x.cpu()), lambda: silu_mul_fp8(x[0])]:
        with pytest.raises(AssertionError):
            bad()
    wide = torch.zeros(4, 700, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(Fp8AttnError):                       # rows 700 apart: not 16-byte aligned
        add_rms_norm_fp8(wide[:, :512], None, w, EPS)
    with pytest.raises(Fp8AttnError):                       # a row that starts 2 bytes off
        silu_mul_fp8(torch.zeros(4, 720, dtype=torch.bfloat16, device="cuda")[:, 1:513])
    with pytest.raises(Fp8AttnError):                       # too many columns
        add_rms_norm_fp8(torch.zeros(2, 16512, dtype=torch.bfloat16, device="cuda"), None,
                         torch.ones(16512, dtype=torch.bfloat16, device="cuda"), EPS)
