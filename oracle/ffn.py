"""The FP8 feed-forward operators in 64 bits, from their definitions, with bounds on what 32-bit
arithmetic may change (test infrastructure only).

Quantised results are checked as intervals: an fp32 result y' with |y' - y| <= err rounds to an e4m3
(or bf16, fp16) value between the roundings of y - err and y + err, since rounding is monotone.
"""
from __future__ import annotations

import torch

GROUP = 128
E4M3_MAX = 448.0


def round_to(v: torch.Tensor, mantissa: int, min_exponent: int, largest: float) -> torch.Tensor:
    """float64 -> nearest value (ties to even) with ``mantissa`` fraction bits and steps no finer than
    2^(min_exponent - mantissa); magnitudes past ``largest`` saturate to it (infinities stay)."""
    e = torch.frexp(v)[1].double() - 1
    step = torch.exp2(e.clamp(min=min_exponent) - mantissa)
    r = torch.round(v / step) * step
    r = torch.where(r.abs() > largest, torch.copysign(torch.full_like(r, largest), r), r)
    return torch.where(torch.isfinite(v), r, v)


def e4m3(v):
    return round_to(v.clamp(-E4M3_MAX, E4M3_MAX), 3, -6, E4M3_MAX)


def bf16(v):
    return round_to(v, 7, -126, 3.3895313892515355e38)


def fp16(v):
    return round_to(v, 10, -14, 65504.0)


def dtype_round(dtype):
    return {torch.bfloat16: bf16, torch.float16: fp16}[dtype]


def group_scale(y: torch.Tensor) -> torch.Tensor:
    """[M, K] -> [M, K / 128] scales before their rounding; NaN left out, 1 for an all-zero group."""
    g = torch.nan_to_num(y.abs(), nan=0.0, posinf=float("inf")).view(y.shape[0], -1, GROUP)
    d = g.amax(-1) / E4M3_MAX
    return torch.where(d > 0, d, torch.ones_like(d))


def spread(d: torch.Tensor) -> torch.Tensor:
    return d.repeat_interleave(GROUP, -1)


def norm(x, residual, weight, eps):
    """(s, y) in float64."""
    s = x.double() + (residual.double() if residual is not None else 0)
    return s, s / torch.sqrt(s.square().mean(-1, keepdim=True) + eps) * weight.double()


def silu_mul(g, u):
    return g.double() * torch.sigmoid(g.double()) * u.double()


def assert_within(got, ref, err, rounding, what):
    """got (any float type) between rounding(ref - err) and rounding(ref + err), elementwise; NaN
    exactly where ref is NaN."""
    got = got.double()
    nan = torch.isnan(ref)
    assert bool((torch.isnan(got) == nan).all()), (what, "NaN", int((torch.isnan(got) != nan).sum()))
    lo, hi = rounding(ref - err), rounding(ref + err)
    bad = ~nan & ((got < lo) | (got > hi))
    if bool(bad.any()):
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; first {i}: "
                             f"{got[i].item()!r} not in [{lo[i].item()!r}, {hi[i].item()!r}]")


def assert_quantised(q, scale, y, rel, absolute=0.0):
    """(q, scale) of an fp32 y' with |y' - y| <= rel |y| + absolute: the scale within that of the
    group's largest, the quotient within twice that and the two divisions' half ulps.  A group whose
    largest is at most ``absolute`` may be all zero in fp32, which has scale 1 and zeros."""
    d = group_scale(y)
    empty = (d * E4M3_MAX <= absolute) & (scale == 1) & (q.float().view(*d.shape, GROUP) == 0).all(-1)
    d, y = torch.where(empty, torch.ones_like(d), d), torch.where(spread(empty), torch.zeros_like(y), y)
    assert_within(scale, d, d * (rel + 2.0 ** -23) + absolute / E4M3_MAX, bf16, "scale")
    v = y / spread(d)
    assert_within(q, v, v.abs() * (2 * rel + 2.0 ** -22) + absolute / spread(d) * 2, e4m3, "values")


def dequantise(q, scale):
    return q.double() * spread(scale.double())


def weight_values(w, scale):
    """e4m3 [N, K] with bf16 block scales -> float64."""
    return w.double() * spread(scale.double()).repeat_interleave(GROUP, 0)


def route(x, router, top_k, renormalize):
    """(weights float64 [T, k], ids [T, k]): ties to the lower expert, NaN last."""
    logits = x.double() @ router.double().t()
    p = torch.softmax(logits, -1)
    key = torch.where(torch.isnan(logits), torch.full_like(logits, float("-inf")), logits)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :top_k]
    c = p.gather(1, order)
    return (c / c.sum(-1, keepdim=True) if renormalize else c), order


def router_halves(c):
    """The columns of each of the two products that the router chains, of the 32 from c on."""
    return [[c + i for i in range(32) if i % 8 < 4], [c + i for i in range(32) if i % 8 >= 4]]


def route_rel(x, router):
    """[T, 1]: how far, relatively, the router's weights may be off.

    A logit is an fp64 sum over groups of 32 columns, rounded to fp32 once (2^-24 of it); a group is two
    tensor-core sums of 16 products, one on top of the other.  Such a sum truncates at 2^-23 of the
    largest of its terms and partial sums, m.  Rounding errors of different groups have the signs of
    different sums, so they add up as squares; eight times that, two sums a group and a factor of four.
    (The worst case, 32 additions of 2^-23 of a group's absolute terms, all of one sign, is used where
    it is smaller.)  A weight is a ratio of exponentials of differences of logits: twice a logit's
    error, the rounded difference, and a few ulps of the exponentials and the fp32 sums of up to 512 of them."""
    x, router = x.double(), router.double()
    logits, squares = x.new_zeros(x.shape[0], router.shape[0]), x.new_zeros(x.shape[0], router.shape[0])
    for c in range(0, x.shape[1], 32):
        a, b = [x[:, half] @ router[:, half].t() for half in router_halves(c)]
        term = (x[:, None, c:c + 32] * router[None, :, c:c + 32]).abs().amax(-1)
        squares += torch.maximum(term, torch.maximum(a.abs(), (a + b).abs())).square()
        logits += a + b
    worst = (x.abs() @ router.abs().t()) * 32 * 2.0 ** -23
    off = torch.minimum(8 * 2.0 ** -23 * squares.sqrt(), worst) + logits.abs() * 2.0 ** -24
    spread_ = (logits.amax(-1) - logits.amin(-1))[:, None]
    return 2 * off.amax(-1, keepdim=True) + spread_ * 2.0 ** -24 + 2.0 ** -19


def moe(x, xq, x_scale, router, w13, w13_scale, w2, w2_scale, top_k, renormalize):
    """(out float64 [T, H], err [T, H], weights, ids).  ``err`` bounds what fp32 sums may change
    before the last rounding:

    * a dot product's n fp32 additions are off by at most n 2^-24 of its terms' absolute sum (128
      columns, then the blocks and two scale products): rel_g of that sum A for g and for u;
    * h = silu(g) u then moves by at most 1.1 |u| err_g + |silu(g)| err_u (|silu'| <= 1.1) and a few
      ulps; its scale and quotient follow, and a quotient that may cross a midpoint between two e4m3
      values moves its dequantised value by up to the distance of the interval's two roundings;
    * the second product adds its own n 2^-24, the router's weights route_rel.
    """
    c, ids = route(x, router, top_k, renormalize)
    rel_c = torch.nan_to_num(route_rel(x, router), posinf=0.0)
    T, H = x.shape
    I = w2.shape[-1]
    out = torch.zeros(T, H, dtype=torch.float64, device=x.device)
    err = torch.zeros_like(out)
    xv = dequantise(xq, x_scale)
    rel1 = (GROUP + H // GROUP + 4) * 2.0 ** -24
    rel2 = (GROUP + I // GROUP + 4) * 2.0 ** -24
    for e in range(router.shape[0]):
        t, place = (ids == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        v13 = weight_values(w13[e], w13_scale[e])
        gu, a = xv[t] @ v13.t(), xv[t].abs() @ v13.abs().t()
        g, u = gu[:, :I], gu[:, I:]
        eg, eu = rel1 * a[:, :I], rel1 * a[:, I:]
        sg = g * torch.sigmoid(g)
        h = sg * u
        eh = 1.1 * (u.abs() + eu) * eg + sg.abs() * eu + h.abs() * 2.0 ** -20
        eh = torch.nan_to_num(eh, nan=0.0)
        d = group_scale(h)
        top = torch.nan_to_num(eh, posinf=0.0).view(len(t), -1, GROUP).amax(-1)
        ed = top / E4M3_MAX + d * 2.0 ** -23
        dv = spread(d)
        q = e4m3(h / dv)
        eq = eh / dv + (h / dv).abs() * spread(ed / d) * 1.01 + (h / dv).abs() * 2.0 ** -22
        moved = torch.maximum(e4m3(h / dv + eq) - q, q - e4m3(h / dv - eq))
        ds = bf16(d)
        eds = torch.maximum(bf16(d + ed) - ds, ds - bf16(d - ed))
        hv = q * spread(ds)
        ehv = moved * spread(ds + eds) + q.abs() * spread(eds)
        v2 = weight_values(w2[e], w2_scale[e])
        y = hv @ v2.t()
        ey = torch.nan_to_num(ehv) @ v2.abs().t() + rel2 * (hv.abs() @ v2.abs().t())
        w = c[t, place][:, None]
        out.index_add_(0, t, w * y)
        err.index_add_(0, t, w * (ey + y.abs() * (2.0 ** -21 + rel_c[t])))
    return out, err, c, ids
