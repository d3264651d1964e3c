"""The oracle's bound on the router's weights lets the kernel's arithmetic pass and mistakes not: both are
imitated here, in 64 bits."""
import pytest
import torch

from oracle import ffn

SIZES = [(16, 2048, 128, 8), (25, 1152, 60, 6), (5, 4096, 8, 2), (3, 128, 7, 3)]


def _inputs(T, H, E, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, generator=gen).to(torch.bfloat16)
    return x, (torch.randn(E, H, generator=gen) * 1.5 / H ** 0.5).to(torch.bfloat16)


def _truncate(v, bits):
    """To `bits` significant bits, towards zero."""
    step = torch.exp2(torch.frexp(v)[1].double() - bits)
    return torch.trunc(v / step) * step


def _kernel_logits(x, w, bits=24, group_sums=True):
    """Sums of 16 products, truncated, two of them chained, then 64 bits and one rounding to fp32; without
    group_sums one chain through all columns."""
    total = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64)
    chain = torch.zeros_like(total)
    for c in range(0, x.shape[1], 32):
        for half in ffn.router_halves(c):
            chain = _truncate(chain + x[:, half].double() @ w[:, half].double().t(), bits)
        if group_sums:
            total, chain = total + chain, torch.zeros_like(total)
    return (total + chain).float().double()


def _weights(logits, ids, renormalize):
    c = torch.softmax(logits, -1).gather(1, ids)
    return c / c.sum(-1, keepdim=True) if renormalize else c


def _worst(x, w, k, renormalize, **how):
    """Largest error of the weights, in units of the bound."""
    want, ids = ffn.route(x, w, k, renormalize)
    got = _weights(_kernel_logits(x, w, **how), ids, renormalize)
    return float(((got - want).abs() / (want * ffn.route_rel(x, w))).max())


@pytest.mark.parametrize("T,H,E,k", SIZES)
def test_the_bound_is_a_few_times_what_the_arithmetic_does(T, H, E, k):
    x, w = _inputs(T, H, E, T + H)
    assert float(ffn.route_rel(x, w).max()) < 2.0 ** -16
    assert _worst(x, w, k, True) < 1 and _worst(x, w, k, False) < 1


@pytest.mark.parametrize("T,H,E,k", SIZES)
def test_lost_bits_are_outside(T, H, E, k):
    x, w = _inputs(T, H, E, T + H)
    assert _worst(x, w, k, False, bits=16) > 1            # sums of 16 bits
    want, ids = ffn.route(x, w, k, False)
    logits = x.double() @ w.double().t()
    short = _truncate(logits, 14)                         # logits of 14 bits
    assert bool(((_weights(short, ids, False) - want).abs() > want * ffn.route_rel(x, w)).any())
    coarse = torch.softmax(logits, -1).gather(1, ids) * (1 + 2.0 ** -15)   # a coarse exponential
    assert bool(((coarse - want).abs() > want * ffn.route_rel(x, w)).all())


def test_a_chain_through_all_columns_is_outside():
    x, w = _inputs(64, 16384, 8, 9)
    x, w = x.abs(), w.abs()                               # terms of one sign: logits of several hundred
    assert _worst(x, w, 2, False, group_sums=False) > 1


def test_zeros_and_single_terms():
    x, w = _inputs(4, 256, 8, 3)
    assert bool((ffn.route_rel(torch.zeros_like(x), w) == 2.0 ** -19).all())
    x[:, 1:] = 0
    assert float(ffn.route_rel(x, w).max()) < 2.0 ** -16
