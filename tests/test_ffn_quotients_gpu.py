"""The 8-bit values of the feed-forward operators are quotients rounded to nearest in fp32, then to e4m3."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quotients_are_divisions(dtype):
    """SiLU of a large gate is the gate, so gate 256 makes h = 256 u exactly, for u of every fraction
    against a largest value of every fraction: e4m3(h / (a / 448)), both divisions in fp32, byte for
    byte."""
    from nanovllm_b200.fp8_ffn import silu_mul_fp8
    steps = 128 if dtype == torch.bfloat16 else 1024
    step = max(1, steps // 128)
    f = 1 + torch.arange(0, steps, step, device="cuda").float() / steps
    groups = []
    for shift in (1.0, 0.5, 0.25, 2.0 ** -6):                  # values of several magnitudes under the largest
        groups.append((f * shift).expand(len(f), len(f)))
    u = torch.cat(groups, 0)                                   # [4 x 128, 128] values
    top = (2 * f).repeat(4)                                    # each row's largest, of every fraction
    u = torch.cat([u, u], 1)
    u[:, 127] = top
    u[:, 255] = -top
    gu = torch.cat([torch.full_like(u, 256.0), u], 1).to(dtype)
    q, d = silu_mul_fp8(gu)
    h = 256.0 * u.to(dtype).float()
    a = h.view(len(u), 2, 128).abs().amax(-1)
    want_d = a / torch.full_like(a, 448.0)   # (a number as divisor: torch multiplies by its inverse)
    want = (h.view(len(u), 2, 128) / want_d[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    assert torch.equal(d, want_d.to(torch.bfloat16))
    got = q.view(torch.uint8)
    want = want.view(len(u), 256).view(torch.uint8)
    assert int((got != want).sum()) == 0
