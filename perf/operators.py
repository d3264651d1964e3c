"""The feed-forward operators of an FP8 layer, as cases that can be measured.

Three operators around the FP8 block-scaled linear layer (e4m3 values, one bf16 scale per row and
128 columns of an activation and per 128 x 128 block of a weight):

``norm``  residual addition + RMS norm, the result quantised for the next FP8 product;
``silu``  silu(gate) * up, the result quantised for the down projection;
``moe``   a whole mixture-of-experts layer for a few tokens: router, top-k, both products, on the
          norm's output and its quantised form.

``run`` computes a case with elementary torch operations, or, where ``own`` is set, with the
framework's kernels; ``exact`` computes it from the definitions in 64 bits.
"""
import math
import os
import sys

import torch

sys.path.append(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                             "my-nano-vllm_b200"))     # where the package lies

own = False

GROUP = 128   # columns that share an activation scale; weight blocks are GROUP x GROUP
E4M3_MAX = 448.0
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decoded token through the norm before a projection of a 4096-wide model
        dict(name="norm_decode_1", op="norm", tokens=1, hidden=4096, residual=True, norm=False,
             dtype="bf16"),
        # an ordinary decode batch, 5120-wide model
        dict(name="norm_batch_256", op="norm", tokens=256, hidden=5120, residual=True, norm=False,
             dtype="bf16"),
        # a whole prefill budget
        dict(name="norm_prefill_8192", op="norm", tokens=8192, hidden=4096, residual=True,
             norm=False, dtype="bf16"),
        # a ragged chunk of a first layer: no residual yet, the unquantised norm wanted too, fp16
        dict(name="norm_first_layer_fp16", op="norm", tokens=1237, hidden=1024, residual=False,
             norm=True, dtype="fp16"),
        # one decoded token between the two products of a dense feed-forward block
        dict(name="silu_decode_1", op="silu", tokens=1, inner=12288, dtype="bf16"),
        # a ragged mixed batch, the widest inner dimension, fp16
        dict(name="silu_mixed_fp16", op="silu", tokens=333, inner=25600, dtype="fp16"),
        # a whole prefill budget
        dict(name="silu_prefill_8192", op="silu", tokens=8192, inner=12288, dtype="bf16"),
        # one decoded token through 128 small experts
        dict(name="moe_decode_1", op="moe", tokens=1, hidden=2048, inner=768, experts=128, top_k=8,
             renormalize=True),
        # a small decode batch: most tokens have experts of their own
        dict(name="moe_batch_16", op="moe", tokens=16, hidden=2048, inner=768, experts=128,
             top_k=8, renormalize=True),
        # a decode batch that reaches nearly every expert
        dict(name="moe_batch_64", op="moe", tokens=64, hidden=2048, inner=768, experts=128,
             top_k=8, renormalize=True),
        # speculative verification (1 + 4 rows) through few large experts
        dict(name="moe_verify_5", op="moe", tokens=5, hidden=4096, inner=7168, experts=8, top_k=2,
             renormalize=True),
        # a ragged batch with many tokens to an expert, an odd number of blocks, raw probabilities
        dict(name="moe_ragged_250", op="moe", tokens=250, hidden=1152, inner=640, experts=60,
             top_k=6, renormalize=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["norm", "silu", "moe"])
    if op == "norm":
        hidden = GROUP * _log_int(rng, 2, 64)
        tokens = _log_int(rng, 1, min(16384, (8192 * 4096) // hidden))
        return dict(op=op, tokens=tokens, hidden=hidden, residual=rng.random() < 0.7,
                    norm=rng.random() < 0.3, dtype=rng.choice(["bf16", "fp16"]))
    if op == "silu":
        inner = GROUP * _log_int(rng, 2, 200)
        tokens = _log_int(rng, 1, min(16384, (8192 * 12288) // inner))
        return dict(op=op, tokens=tokens, inner=inner, dtype=rng.choice(["bf16", "fp16"]))
    experts = rng.choice([4, 8, 16, 40, 64, 128, 160, 256])
    hidden = GROUP * _log_int(rng, 2, 40)
    # all experts' weights at most 700 M values, and fewer tokens to the largest of them
    inner = GROUP * _log_int(rng, 1, min(64, 700_000_000 // (3 * experts * hidden * GROUP)))
    tokens = _log_int(rng, 1, min(256, 40_000_000_000 // (3 * experts * hidden * inner)))
    return dict(op=op, tokens=tokens, hidden=hidden, inner=inner, experts=experts,
                top_k=rng.randint(1, min(8, experts)), renormalize=rng.random() < 0.7)


# ------------------------------------------------------------------------------------ inputs
def _e4m3_weight(shape, gen):
    """Block-quantised weights as a checkpoint holds them: values that use the e4m3 range, and one
    bf16 scale per 128 x 128 block that brings a row's products back to about unit size."""
    *lead, n, k = shape
    w = torch.randn(shape, generator=gen, device="cuda").mul_(110).clamp_(-E4M3_MAX, E4M3_MAX).to(
        torch.float8_e4m3fn)
    scale = torch.rand(*lead, n // GROUP, k // GROUP, generator=gen, device="cuda") + 0.5
    return w, (scale / (110 * math.sqrt(k))).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    s = {"case": case}
    m = case["tokens"]
    if case["op"] == "norm":
        h, t = case["hidden"], DTYPES[case["dtype"]]
        s["x"] = randn(m, h).to(t)
        # a residual stream is wider than one block's output, and some of its channels stand out
        s["residual"] = (randn(m, h) * (1 + 8 * (torch.rand(h, generator=gen, device="cuda") > 0.99))
                         * 2).to(t) if case["residual"] else None
        s["weight"] = (1 + 0.2 * randn(h)).to(t)
    elif case["op"] == "silu":
        s["gate_up"] = (1.5 * randn(m, 2 * case["inner"])).to(DTYPES[case["dtype"]])
    else:
        e, h, i = case["experts"], case["hidden"], case["inner"]
        # what the norm before the layer leaves: its output, and the same quantised
        s["x"] = randn(m, h).to(torch.bfloat16)
        s["xq"], scale = _quantise(s["x"].float())
        s["x_scale"] = scale.to(torch.bfloat16)
        s["router"] = (1.5 * randn(e, h) / math.sqrt(h)).to(torch.bfloat16)
        s["w13"], s["w13_scale"] = _e4m3_weight((e, 2 * i, h), gen)
        s["w2"], s["w2_scale"] = _e4m3_weight((e, h, i), gen)
    return s


# ------------------------------------------------------------------- plain forms, 32 bits
def _quantise(y):
    """y fp32 [rows, columns] -> (e4m3 values, fp32 scales before their rounding to bf16)."""
    g = y.view(y.shape[0], -1, GROUP)
    d = g.abs().amax(-1) / E4M3_MAX
    d = torch.where(d > 0, d, torch.ones_like(d))
    q = (g / d[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.view(y.shape), d


def _dequantise(q, d):
    """The values that (q, bf16 scales) stand for, fp32."""
    return (q.float().view(q.shape[0], -1, GROUP) * d.to(torch.bfloat16).float()[..., None]).view(
        q.shape)


def _dequantise_weight(w, scale):
    e, n, k = w.shape
    blocks = w.float().view(e, n // GROUP, GROUP, k // GROUP, GROUP)
    return (blocks * scale.float()[:, :, None, :, None]).view(e, n, k)


def _silu_mul(g, u):
    return g / (1 + torch.exp(-g)) * u


def _norm_plain(s):
    x, t = s["x"].float(), s["x"].dtype
    res = None
    if s["residual"] is not None:
        x = x + s["residual"].float()
        res = x.to(t)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["weight"].float()
    q, d = _quantise(y)
    return q, d.to(torch.bfloat16), res, y.to(t) if s["case"]["norm"] else None


def _silu_plain(s):
    g, u = s["gate_up"].float().chunk(2, -1)
    q, d = _quantise(_silu_mul(g, u))
    return q, d.to(torch.bfloat16)


def _moe_plain(s):
    c = s["case"]
    k = c["top_k"]
    # the choice of experts is a comparison of sums: 64 bits
    logits = s["x"].double() @ s["router"].double().t()
    p = torch.softmax(logits, -1)
    p, ids = torch.sort(p, dim=-1, descending=True, stable=True)
    p, ids = p[:, :k], ids[:, :k]
    if c["renormalize"]:
        p = p / p.sum(-1, keepdim=True)
    p = p.float()
    xv = _dequantise(s["xq"], s["x_scale"])
    m = xv.shape[0]
    if m * k <= c["experts"]:  # few choices: only their experts' weights, one copy for each
        pick = ids.reshape(-1)
        rows = xv.repeat_interleave(k, 0)[:, :, None]
        y = torch.matmul(_dequantise_weight(s["w13"].view(torch.uint8)[pick].view(s["w13"].dtype),
                                            s["w13_scale"][pick]), rows)[:, :, 0]
        g, u = y.chunk(2, -1)
        hv = _dequantise(*_quantise(_silu_mul(g, u)))[:, :, None]
        y = torch.matmul(_dequantise_weight(s["w2"].view(torch.uint8)[pick].view(s["w2"].dtype),
                                            s["w2_scale"][pick]), hv)[:, :, 0]
        y = y.view(m, k, -1)
    else:  # every expert on every token, then the chosen ones
        g, u = torch.matmul(xv, _dequantise_weight(s["w13"], s["w13_scale"]).transpose(1, 2)).chunk(
            2, -1)
        h = _silu_mul(g, u)
        hv = _dequantise(*_quantise(h.reshape(-1, h.shape[-1]))).view(h.shape)
        y = torch.matmul(hv, _dequantise_weight(s["w2"], s["w2_scale"]).transpose(1, 2))
        y = y[ids, torch.arange(m, device=ids.device)[:, None]]
    return (p[:, :, None] * y).sum(1).to(torch.bfloat16), p, ids.to(torch.int32)


def run(state):
    op = state["case"]["op"]
    if own:
        from nanovllm_b200 import fp8_ffn
        if op == "norm":
            return fp8_ffn.add_rms_norm_fp8(state["x"], state["residual"], state["weight"], EPS,
                                            return_norm=state["case"]["norm"])
        if op == "silu":
            return fp8_ffn.silu_mul_fp8(state["gate_up"])
        return fp8_ffn.fp8_moe(state["x"], state["xq"], state["x_scale"], state["router"],
                               state["w13"], state["w13_scale"], state["w2"], state["w2_scale"],
                               state["case"]["top_k"], renormalize=state["case"]["renormalize"],
                               return_router=True)
    return {"norm": _norm_plain, "silu": _silu_plain, "moe": _moe_plain}[op](state)


# ------------------------------------------------------------------------------------- floors
def work(case):
    m = case["tokens"]
    if case["op"] == "norm":
        h = case["hidden"]
        per = 2 + 1 + 2 / GROUP + (4 if case["residual"] else 0) + (2 if case["norm"] else 0)
        return {"bytes": int(m * h * per) + 2 * h, "flops": 8 * m * h}
    if case["op"] == "silu":
        i = case["inner"]
        return {"bytes": int(m * i * (4 + 1 + 2 / GROUP)), "flops": 8 * m * i}
    e, h, i, k = case["experts"], case["hidden"], case["inner"], case["top_k"]
    # experts that are read: m tokens choose k of e each, evenly
    read = e * (1 - (1 - k / e) ** m)
    weights = read * 3 * i * h * (1 + 2 / GROUP ** 2)
    return {"bytes": int(weights) + 2 * e * h + 5 * m * h + 8 * m * k,
            "flops": 2 * m * e * h + 6 * m * k * i * h}


# --------------------------------------------------------------------- definitions, 64 bits
def _round_e4m3(v):
    """Nearest e4m3 value (ties to even), |v| <= 448, in float64: a step is 2^-3 of the value's
    power of two, and 2^-9 below 2^-6."""
    exponent = torch.frexp(v)[1] - 1
    step = torch.exp2(exponent.clamp(min=-6).double() - 3)
    return torch.round(v / step) * step


def _quantise_exact(y):
    part = y.reshape(y.shape[0], -1, GROUP)
    d = part.abs().max(dim=2).values / 448
    d[d == 0] = 1
    return _round_e4m3(part / d[:, :, None]).reshape(y.shape), d


def _bf16_values(d):
    return d.float().to(torch.bfloat16).double()


def _spread(scale, rows, columns):
    """One value per block -> one per element."""
    return scale.double().repeat_interleave(GROUP, 0)[:rows].repeat_interleave(GROUP, 1)[:, :columns]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x = s["x"].double()
        if s["residual"] is not None:
            x += s["residual"].double()
        y = x / torch.sqrt(x.square().sum(1, keepdim=True) / x.shape[1] + EPS)
        y *= s["weight"].double()
        q, d = _quantise_exact(y)
        return (q, d, x if s["residual"] is not None else None, y if case["norm"] else None)
    if case["op"] == "silu":
        inner = case["inner"]
        g, u = s["gate_up"][:, :inner].double(), s["gate_up"][:, inner:].double()
        return _quantise_exact(g * torch.sigmoid(g) * u)
    m, k, h, inner = case["tokens"], case["top_k"], case["hidden"], case["inner"]
    logits = s["x"].double() @ s["router"].double().T
    weight = torch.exp(logits - logits.max(1, keepdim=True).values)
    weight /= weight.sum(1, keepdim=True)
    left, ids, chosen = weight.clone(), [], []
    rows = torch.arange(m, device="cuda")
    for _ in range(k):
        best = (left == left.max(1, keepdim=True).values).double().argmax(1)  # the first of them
        ids.append(best)
        chosen.append(weight[rows, best])
        left[rows, best] = -1
    ids, chosen = torch.stack(ids, 1), torch.stack(chosen, 1)
    if case["renormalize"]:
        chosen /= chosen.sum(1, keepdim=True)
    xv = s["xq"].double() * s["x_scale"].double().repeat_interleave(GROUP, 1)
    out = torch.zeros(m, h, dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        token, place = (ids == e).nonzero(as_tuple=True)
        if not len(token):
            continue
        w13 = s["w13"][e].double() * _spread(s["w13_scale"][e], 2 * inner, h)
        both = xv[token] @ w13.T
        g, u = both[:, :inner], both[:, inner:]
        q, d = _quantise_exact(g * torch.sigmoid(g) * u)
        w2 = s["w2"][e].double() * _spread(s["w2_scale"][e], h, inner)
        y = (q * _bf16_values(d).repeat_interleave(GROUP, 1)) @ w2.T
        out.index_add_(0, token, y * chosen[token, place][:, None])
    return out, chosen, ids
