"""The FP8 feed-forward operators at the ends of their documented ranges: the widest rows, many tokens on few
experts, rows so far apart that offsets pass 32 bits.  Tolerances as in test_ffn_quant_gpu and test_moe_gpu."""
import pytest
import torch

from oracle import ffn
from test_ffn_quant_gpu import DTYPES, _check_norm, _check_silu, _norm_inputs, _randn
from test_moe_gpu import _check, _inputs, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,i", [(1, 1 << 20), (3, (1 << 20) - 128)])
def test_widest_silu(m, i, dtype):
    _check_silu(_randn((m, 2 * i), m, dtype, 2.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(512, 16384), (513, 16384), (512, 8192), (513, 8192), (513, 5248),
                                 (514, 4096), (700, 128)])
def test_norm_on_both_sides_of_its_rules(m, k, dtype):
    _check_norm(*_norm_inputs(m, k, dtype, m + k))


@pytest.mark.parametrize("T,H,I,E,k", [
    (3, 16384, 128, 4, 2), (3, 128, 16384, 4, 2), (2, 16384, 16384, 2, 1),
    (33, 16384, 256, 3, 3),
    (1024, 1024, 512, 8, 2),        # 256 tokens to an expert
    (1024, 256, 256, 1, 1),         # all of them to one
    (1024, 128, 128, 16, 8),
    (256, 256, 384, 32, 32),        # every expert, the largest top_k
    (193, 512, 256, 16, 1)])        # 12 tokens to an expert and a little more
def test_moe_at_its_ends(T, H, I, E, k):
    _check(_inputs(T, H, I, E, T + H + I + E), k)


def _far_apart(t, stride):
    """The rows of t, `stride` elements apart, in a buffer that is never written between them."""
    buf = torch.empty((t.shape[0] - 1) * stride + t.shape[1], dtype=torch.uint8 if t.element_size() == 1
                      else t.dtype, device="cuda")
    rows = buf.as_strided(t.shape, (stride, 1))
    rows.copy_(t.view(torch.uint8) if t.element_size() == 1 else t)
    return rows.view(t.dtype) if t.element_size() == 1 else rows


def test_rows_far_apart():
    """Offsets past 2^31 elements, and 2^32 bytes, in every strided input."""
    from nanovllm_b200.fp8_ffn import add_rms_norm_fp8, silu_mul_fp8
    stride = 1 << 26
    x, r, w = _norm_inputs(40, 512, torch.bfloat16, 3)
    want = add_rms_norm_fp8(x, r, w, 1e-6, return_norm=True)
    got = add_rms_norm_fp8(_far_apart(x, stride), r, w, 1e-6, return_norm=True)
    for p, q in zip(want, got):
        assert torch.equal(p.view(torch.uint8), q.view(torch.uint8))
    got = add_rms_norm_fp8(x, _far_apart(r, stride), w, 1e-6, return_norm=True)
    for p, q in zip(want, got):
        assert torch.equal(p.view(torch.uint8), q.view(torch.uint8))
    for p, q in zip(silu_mul_fp8(x), silu_mul_fp8(_far_apart(x, stride))):
        assert torch.equal(p.view(torch.uint8), q.view(torch.uint8))
    a = _inputs(40, 256, 128, 8, 4)
    want = _run(a, 3)
    b = dict(a, x=_far_apart(a["x"], stride))
    for p, q in zip(want, _run(b, 3)):
        assert torch.equal(p, q)
    b = dict(a, xq=_far_apart(a["xq"], 2 * stride))
    for p, q in zip(want, _run(b, 3)):
        assert torch.equal(p, q)


def test_logits_of_every_size():
    """Tokens from 2^-60 to 2^20: the order and the weights of the experts hold for each."""
    a = _inputs(41, 512, 128, 24, 5)
    scale = torch.exp2(torch.arange(41, device="cuda").float() * 2 - 60)
    from nanovllm_b200.fp8_linear import fp8_dyn_quant
    a["x"] = (a["x"].float() * scale[:, None]).to(torch.bfloat16)
    a["xq"], a["x_scale"] = fp8_dyn_quant(a["x"])
    _, c, ids = _run(a, 5)
    want, want_ids = ffn.route(a["x"], a["router"], 5, True)
    assert torch.equal(ids.long(), want_ids)
    few = scale <= 16                                     # beyond, weights fall below fp32's numbers
    assert bool(((c.double() - want).abs() <= want * ffn.route_rel(a["x"], a["router"]))[few].all())
