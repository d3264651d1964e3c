"""fp8_moe chooses the experts of the definition, whose logits are sums in 64 bits, also where two logits are
closer than sums in 32 bits can tell."""
import pytest
import torch

from oracle import ffn

pytestmark = pytest.mark.gpu


def _router_case(T, H, E, seed):
    """Experts 2 i and 2 i + 1 have the same rows but in column 0, where the odd one's product is 2^-28
    larger: less than half of fp32's step at the logits' size, far more than fp64's."""
    from nanovllm_b200.fp8_linear import fp8_dyn_quant
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, H, generator=gen, device="cuda").to(torch.bfloat16)
    x[:, 0] = 2.0 ** -20
    router = (4 * torch.randn(E, H, generator=gen, device="cuda") / H ** 0.5).to(torch.bfloat16)
    router[1::2] = router[0::2][:E // 2]
    router[:, 0] = 0
    router[1::2, 0] = 2.0 ** -8
    w13 = torch.zeros(E, 256, H, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    w2 = torch.zeros(E, H, 128, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    s13 = torch.ones(E, 2, H // 128, dtype=torch.bfloat16, device="cuda")
    s2 = torch.ones(E, H // 128, 1, dtype=torch.bfloat16, device="cuda")
    xq, xs = fp8_dyn_quant(x)
    return x, xq, xs, router, w13, s13, w2, s2


@pytest.mark.parametrize("T,H,E,k", [
    (1, 2048, 16, 4), (1, 128, 2, 1), (3, 128, 2, 2), (8, 1152, 60, 6), (9, 2048, 128, 8),
    (17, 2048, 128, 7),             # a pair on both sides of the last place
    (64, 512, 129, 3), (250, 256, 40, 32), (5, 4096, 512, 31), (2, 16384, 300, 8)])
def test_experts_whose_logits_all_but_tie(T, H, E, k):
    from nanovllm_b200.fp8_ffn import fp8_moe
    a = _router_case(T, H, E, 7 * T + H + E)
    want_c, want = ffn.route(a[0], a[3], k, True)
    even, first = want % 2 == 0, want.new_zeros(T, k)
    for place in range(1, k):
        first[:, place] = ((want[:, place - 1] == want[:, place] + 1) & even[:, place]).long()
    assert k == 1 or bool(first.any())                # pairs that are chosen, the odd one first
    out, c, ids = fp8_moe(*a, k, return_router=True)
    assert torch.equal(ids.long(), want)
    assert bool(((c.double() - want_c).abs() <= want_c * ffn.route_rel(a[0], a[3])).all())
    assert bool((out == 0).all())


def test_equal_rows_still_go_to_the_lower_expert():
    """Rows that are equal bit for bit, among others: their sums are equal in any precision."""
    from nanovllm_b200.fp8_ffn import fp8_moe
    a = list(_router_case(20, 1024, 48, 11))
    a[3][1::2] = a[3][0::2]
    want = ffn.route(a[0], a[3], 7, True)[1]
    # matrix products may sum two equal rows differently: order equal rows by hand
    low = want - want % 2
    assert bool((low[:, 0::2][:, :3] == low[:, 1::2]).all())
    want = torch.stack([low[:, p] + p % 2 for p in range(7)], 1)
    assert torch.equal(fp8_moe(*a, 7, return_router=True)[2].long(), want)
