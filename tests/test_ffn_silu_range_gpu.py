"""SiLU * up of gates so far below zero that 1 + exp(-g) nearly leaves fp32's range."""
import pytest
import torch

from oracle import ffn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_silu_of_gates_down_to_the_end_of_fp32_s_powers(dtype):
    """1 + exp(-g) is a number of fp32 down to g = -88.7.  There h is the definition's, to the relative
    error of the rest (2^-20) and half a step of the smallest fp32 numbers in each of the two products."""
    from nanovllm_b200.fp8_ffn import silu_mul_fp8
    g = torch.linspace(-88.5, -84.0, 40, device="cuda").to(dtype).unique()
    g = g[g >= -88.5]
    for scale in (1.0, 2.0 ** 14):
        gen = torch.Generator(device="cuda").manual_seed(5)
        u = torch.randn(len(g), 256, generator=gen, device="cuda")
        u = ((u.sign() + (u == 0)) * (0.5 + u.abs().clamp(max=3)) * scale).to(dtype)
        gu = torch.cat([g[:, None].expand(len(g), 256), u], 1).contiguous()
        q, d = silu_mul_fp8(gu)
        h = ffn.silu_mul(gu[:, :256], gu[:, 256:])
        tiny = 2.0 ** -150 * (1 + float(u.double().abs().max()))
        dd = ffn.group_scale(h)
        ffn.assert_within(d, dd, dd * (2.0 ** -20 + 2.0 ** -23) + tiny / 448 + 2.0 ** -150, ffn.bf16, "scale")
        assert bool((d.double() < 1).all())                   # no group taken for an empty one
        if scale > 1:                                         # scales are normal numbers here
            ffn.assert_quantised(q, d, h, 2.0 ** -20, tiny)


def test_silu_below_the_end_of_fp32_s_powers_is_zero():
    from nanovllm_b200.fp8_ffn import silu_mul_fp8
    gu = torch.ones(3, 512, dtype=torch.bfloat16, device="cuda")
    gu[0, :256], gu[1, :256], gu[2, :256] = -89.5, -1000.0, -3.0e38
    q, d = silu_mul_fp8(gu)
    assert bool((d == 1).all()) and bool((q.float() == 0).all())
