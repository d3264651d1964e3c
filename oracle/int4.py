"""64-bit restatement of the 4-bit key/value cache and of attention over it (include/fp8attn.h): test
infrastructure only."""
from __future__ import annotations

import math

import torch

D = 128


def quantise(x: torch.Tensor):
    """bf16 rows [..., 128] -> (codes uint8 [..., 128], step bf16 [...], low bf16 [...])."""
    low, high = x.amin(-1), x.amax(-1)  # NaNs go through
    step = ((high.float() - low.float()) / 15).to(torch.bfloat16)
    bad = ~torch.isfinite(step)
    step = torch.where(bad, torch.full_like(step, math.nan), step)
    s, ok = step.double(), (~bad) & (step > 0)
    code = torch.round((x.double() - low.double()[..., None]) / torch.where(ok, s, 1.0)[..., None])
    code = torch.where(ok[..., None], code.clamp(0, 15), torch.zeros_like(code))
    return code.nan_to_num(0).to(torch.uint8), step, low


def pack(code: torch.Tensor) -> torch.Tensor:
    return code[..., 0::2] | (code[..., 1::2] << 4)


def unpack(cache: torch.Tensor) -> torch.Tensor:
    return torch.stack([cache & 15, cache >> 4], -1).flatten(-2)


def rows(cache: torch.Tensor, scale: torch.Tensor):
    """Packed rows [..., 64] and (step, low) [..., 2] -> (codes, step, low) in float64, [..., 128] and [..., 1]."""
    return unpack(cache).double(), scale[..., :1].double(), scale[..., 1:].double()


def store(key, value, k_cache, v_cache, kv_scale, slots):
    """Writes into the three tensors."""
    blocks, _, block, _ = k_cache.shape
    keep = (slots >= 0) & (slots < blocks * block)
    at = slots[keep].long()
    page, place = at // block, at % block
    for j, (x, cache) in enumerate(((key, k_cache), (value, v_cache))):
        code, step, low = quantise(x[keep])
        cache[page, :, place] = pack(code)
        kv_scale[page, :, place, 2 * j] = step
        kv_scale[page, :, place, 2 * j + 1] = low


def sequence(k_cache, v_cache, kv_scale, table, n):
    """Keys' and values' (codes, step, low) [n, KVH, ...] of a sequence's first n positions, and which of them
    lie in pages of the cache."""
    blocks, _, block, _ = k_cache.shape
    n = min(n, table.numel() * block)
    at = torch.arange(n, device=k_cache.device)
    page = table.long()[at // block]
    there = (page >= 0) & (page < blocks)
    page, place = page.clamp(0, blocks - 1), at % block
    scale = kv_scale[page, :, place]
    return (rows(k_cache[page, :, place], scale[..., :2]), rows(v_cache[page, :, place], scale[..., 2:]),
            there)


def attention(q, k_cache, v_cache, kv_scale, table, nk, softmax_scale, in_f16=False):
    """q [nq, heads, 128], the last nq of the sequence's nk positions.  (out, bound) in float64: what the
    kernels may be off by, before the rounding of the output.

    bound, from the kernels' arithmetic, with |k| = step c + |low| and the like for v:
      scores: products are exact; a sum of 128 terms is 8 matrix instructions of 17 terms, each of which may be
        cut at 2^-24 of the largest (under 2^-16.9 of the terms' magnitudes in all); the sum of q 2^-17 and the
        products with step and low 2^-23 of theirs: under 2^-16.  The argument of the exponential is a
        difference of scores, and the exponential itself is off by 2^-22.  An error e in every exponent moves
        an output by at most 2 e sum(p |v|) / sum(p);
      P step: one rounding to f16, 2^-11 of its term of sum(p step c), and 2^-25 of the largest step where
        it leaves f16's normal range (c up to 15, the largest p is 1 or more);
      sums over positions: at most 1024 additions in fp32 one after another (a thread's and the parts'), 2^-14
        of the magnitudes, in the numerator and in the denominator.

    in_f16: of the kernel for long chunks, which takes the values themselves as f16 operands.  Beside the above,
      each value of K and V is rounded to f16 (2^-11 of it, or 2^-25 where the tile's largest is 2^-7 or more: 2^-18
      of that), which for K is an error of the scores; so is P (2^-11 of its term, or 2^-25 where the largest is
      2^4 or more: 2^-29 for each position); and of the exponentials some are a polynomial's, off by 1e-4.
    """
    nq, heads, _ = q.shape
    kv = k_cache.shape[1]
    (kc, ks, kl), (vc, vs, vl), there = sequence(k_cache, v_cache, kv_scale, table, max(nk, 0))
    n = kc.shape[0]
    out = torch.zeros(nq, heads, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    if n == 0:
        return out, bound
    last = torch.arange(nq, device=q.device) + nk - nq
    seen = (torch.arange(n, device=q.device)[None] <= last[:, None]) & there[None]
    some = seen.any(-1)
    for h in range(heads):
        g = h // (heads // kv)
        x = q[:, h].double()
        kcg, ksg, klg, vcg, vsg, vlg = (t[:, g] for t in (kc, ks, kl, vc, vs, vl))
        hide = lambda t, v: t.masked_fill(~seen, v)  # noqa: E731
        used = seen.any(0)[:, None]  # rows that are never seen do not count, whatever they hold
        kcg, ksg, klg, vcg, vsg, vlg = (torch.where(used, t, torch.zeros_like(t))
                                        for t in (kcg, ksg, klg, vcg, vsg, vlg))
        s = hide((x @ (klg + ksg * kcg).T) * softmax_scale, -math.inf)
        size = hide((x.abs() @ (ksg * kcg + klg.abs()).T) * abs(softmax_scale), 0.0)
        p = torch.where(some[:, None], torch.softmax(s, -1), torch.zeros_like(s))
        out[:, h] = p @ (vlg + vsg * vcg)
        coded, whole = p @ (vsg * vcg), p @ (vsg * vcg + vlg.abs())
        e = 2.0 ** -16 * size.amax(-1, keepdim=True) + 2.0 ** -21
        if in_f16:
            k_top = (klg.abs() + ksg * 15).amax()
            e = e + 2.0 ** -11 * size.amax(-1, keepdim=True) + 2.0 ** -18 * abs(softmax_scale) * (
                x.abs().sum(-1, keepdim=True) * k_top) + 1e-4
            v_top = (vlg.abs() + vsg * 15).amax()
            bound[:, h] = 2.0 ** -10 * whole + (2.0 ** -18 + n * 2.0 ** -29) * v_top * some[:, None]
        bound[:, h] += (2 * e + 2.0 ** -13) * whole + 2.0 ** -11 * coded + 2.0 ** -21 * vsg.max() * p.sum(-1, keepdim=True)
        out[~some, h] = 0
    return out, bound


def attention_norm(q, k_cache, v_cache, kv_scale, table, nk, softmax_scale):
    """q [nq, heads, 128] as ``attention``'s: (out float64, room float64 [nq, heads]), what an output row of 128 may be off by
    in the 2-norm.  ``attention``'s bound holds for each value whatever the signs of the errors; this one counts them as
    independent, and so is narrow enough that a page left out or a scale 1 % off shows.

      rounding of the output to bf16: errors are spread evenly over half a step either way, at most 2^-8 / sqrt(3) of the
        value in the mean square; 2.5e-3 with what 128 values scatter; below 2^-126, where bf16's steps are 2^-133
        whatever the value, at most 2^-134 for each;
      P and values: rounded to f16 at each position for itself (2^-12 each), some exponentials 1e-4 off: errors of that size
        add up as their root mean square, 2^-10 sqrt(sum p^2 |v|^2) at the most of some four standard deviations;
      scores: 128 terms that carry 2^-12 of each (f16 operands), so off by e = 2^-12 (sum of squares of the terms)^1/2 and a
        weight by e of itself.  A weight is in the numerator and in the denominator of sum p v / sum p: it moves the output by
        e p (v - out).  Again for each position for itself, four times e;
      what is alike at all positions (sums cut in one direction): 2^-16 sum p |v|.
    """
    nq, heads, _ = q.shape
    kv = k_cache.shape[1]
    (kc, ks, kl), (vc, vs, vl), there = sequence(k_cache, v_cache, kv_scale, table, max(nk, 0))
    n = kc.shape[0]
    out = torch.zeros(nq, heads, D, dtype=torch.float64, device=q.device)
    room = torch.zeros(nq, heads, dtype=torch.float64, device=q.device)
    if n == 0:
        return out, room
    last = torch.arange(nq, device=q.device) + nk - nq
    seen = (torch.arange(n, device=q.device)[None] <= last[:, None]) & there[None]
    some = seen.any(-1)
    used = seen.any(0)[:, None]
    clean = lambda t: torch.where(used, t, torch.zeros_like(t))  # noqa: E731
    for h in range(heads):
        g = h // (heads // kv)
        x = q[:, h].double()
        k = clean(kl[:, g]) + clean(ks[:, g]) * kc[:, g]
        v = clean(vl[:, g]) + clean(vs[:, g]) * vc[:, g]
        s = (x @ k.T * softmax_scale).masked_fill(~seen, -math.inf)
        p = torch.where(some[:, None], torch.softmax(s, -1), torch.zeros_like(s))
        out[:, h] = p @ v
        root = torch.where(seen, (x.square() @ k.square().T).sqrt() * abs(softmax_scale), 0.0)
        size = v.norm(dim=-1)
        apart = (size.square() - 2 * out[:, h] @ v.T + out[:, h].square().sum(-1, keepdim=True)).clamp(min=0).sqrt()
        room[:, h] = (2.5e-3 * out[:, h].norm(dim=-1) + 2.0 ** -10 * ((p * size).square() + (root * p * apart).square())
                      .sum(-1).sqrt()
                      + 2.0 ** -16 * (p @ v.abs()).norm(dim=-1) + 2.0 ** -134 * D ** 0.5)
    return out, room
