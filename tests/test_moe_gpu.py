"""fp8_moe against its definition in 64 bits (oracle/ffn.py).

The tolerance is the oracle's own bound on what fp32 sums may change (n 2^-24 of a dot product's
absolute terms, and what that may move across the midpoints of the 8-bit hidden values), then the
bf16 rounding of the result.  Router weights: within what the logits' sums allow; chosen experts are equal.
"""
import pytest
import torch

from oracle import ffn

pytestmark = pytest.mark.gpu


def _e4m3_weight(shape, gen):
    *lead, n, k = shape
    w = (torch.randn(shape, generator=gen, device="cuda") * 110).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = (torch.rand(*lead, n // 128, k // 128, generator=gen, device="cuda") + 0.5) / (110 * k ** 0.5)
    return w, s.to(torch.bfloat16)


def _inputs(T, H, I, E, seed, sd=1.0):
    from nanovllm_b200.fp8_linear import fp8_dyn_quant
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(T, H, generator=gen, device="cuda") * sd).to(torch.bfloat16)
    router = (torch.randn(E, H, generator=gen, device="cuda") * 1.5 / H ** 0.5).to(torch.bfloat16)
    w13, s13 = _e4m3_weight((E, 2 * I, H), gen)
    w2, s2 = _e4m3_weight((E, H, I), gen)
    xq, xs = fp8_dyn_quant(x)
    return dict(x=x, xq=xq, x_scale=xs, router=router, w13=w13, w13_scale=s13, w2=w2, w2_scale=s2)


def _run(a, top_k, renormalize=True, router=True):
    from nanovllm_b200.fp8_ffn import fp8_moe
    return fp8_moe(a["x"], a["xq"], a["x_scale"], a["router"], a["w13"], a["w13_scale"], a["w2"],
                   a["w2_scale"], top_k, renormalize=renormalize, return_router=router)


def _no_device_error():
    from nanovllm_b200 import fp8_attention
    torch.cuda.synchronize()
    assert fp8_attention.device_error(torch.device("cuda", 0)) == 0


def _check(a, top_k, renormalize=True):
    out, c, ids = _run(a, top_k, renormalize)
    T, H = a["x"].shape
    assert out.shape == (T, H) and out.dtype == torch.bfloat16
    assert c.shape == ids.shape == (T, top_k) and c.dtype == torch.float32 and ids.dtype == torch.int32
    ref, err, c64, ids64 = ffn.moe(a["x"], a["xq"], a["x_scale"], a["router"], a["w13"],
                                   a["w13_scale"], a["w2"], a["w2_scale"], top_k, renormalize)
    assert torch.equal(ids.long(), ids64)
    assert bool(((c.double() - c64).abs() <= c64 * ffn.route_rel(a["x"], a["router"])).all())
    ffn.assert_within(out, ref, err, ffn.bf16, "out")
    _no_device_error()
    return out, c, ids


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("T,H,I,E,k", [
    (1, 128, 128, 1, 1),            # the smallest of everything
    (1, 2048, 768, 128, 8),         # one token
    (2, 256, 384, 4, 4),            # every expert chosen
    (3, 384, 128, 7, 3),            # odd numbers of blocks and experts
    (5, 1024, 1664, 8, 2),          # an odd number of inner blocks
    (16, 2048, 768, 128, 8),
    (17, 1152, 640, 60, 6),         # one token past a 16-token tile
    (33, 512, 256, 33, 5),
    (64, 1024, 256, 64, 8),
    (64, 256, 128, 2, 1),           # many tokens to an expert
    (250, 1152, 640, 60, 6),
    (300, 256, 256, 3, 2),          # more than 128 tokens to an expert
    (1024, 256, 128, 512, 8),       # the most tokens, slots and experts
    (256, 128, 256, 40, 32),        # the largest top_k
    (7, 128, 2048, 16, 4),          # a wide inner dimension under a narrow hidden one
    (7, 4096, 128, 16, 4),
])
def test_moe(T, H, I, E, k, renormalize):
    _check(_inputs(T, H, I, E, T * 31 + H + E), k, renormalize)


@pytest.mark.parametrize("T", range(1, 41, 3))
def test_every_small_batch(T):
    _check(_inputs(T, 256, 256, 8, 1000 + T), 3)


@pytest.mark.parametrize("T", [15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200])
def test_all_tokens_to_one_expert(T):
    """The router sends every token to expert 2: token tiles of every fill."""
    a = _inputs(T, 256, 384, 4, 2000 + T)
    a["x"][:, 0] = 8
    a["router"][:] *= 0.01
    a["router"][2, 0] = 8
    from nanovllm_b200.fp8_linear import fp8_dyn_quant
    a["xq"], a["x_scale"] = fp8_dyn_quant(a["x"])
    _, _, ids = _check(a, 1)
    assert bool((ids == 2).all())


def test_ties_go_to_the_lower_expert():
    a = _inputs(6, 256, 128, 70, 3000)
    a["router"][:] = a["router"][0].clone()              # every logit of a token is the same
    _, c, ids = _check(a, 5)
    assert torch.equal(ids, torch.arange(5, device="cuda", dtype=torch.int32).expand(6, 5))
    assert bool((c - 0.2).abs().max() < 1e-6)
    a = _inputs(6, 256, 128, 70, 3001)
    a["router"][35:] = a["router"][:35].clone()          # pairs that tie
    _, _, ids = _check(a, 4)
    assert torch.equal(ids[:, 1] - ids[:, 0], torch.full((6,), 35, device="cuda", dtype=torch.int32))


def test_nan_and_infinite_tokens_stay_alone():
    a = _inputs(9, 512, 256, 16, 3100)
    clean = _run(a, 4)
    b = {n: t.clone() for n, t in a.items()}
    b["x"][2, 5] = float("nan")
    b["x"][7, 9] = float("inf")
    b["xq"].view(torch.uint8)[4, 100] = 0x7F             # a NaN in the quantised input alone
    out, c, ids = _run(b, 4)
    assert bool((ids >= 0).all()) and bool((ids < 16).all())
    assert bool((ids.sort(1).values.diff(dim=1) > 0).all())         # still top_k experts
    assert bool(torch.isnan(out[[2, 4]]).all())
    assert bool(torch.isnan(c[2]).all())
    keep = [0, 1, 3, 5, 6, 8]
    for p, q in zip((out, c, ids), clean):
        assert torch.equal(p[keep], q[keep])
    _no_device_error()


def test_nan_in_a_chosen_weight_reaches_its_tokens_only():
    a = _inputs(12, 256, 256, 8, 3200)
    clean, _, ids = _run(a, 2)
    a["w13"].view(torch.uint8)[3, 10, 20] = 0x7F         # one weight of expert 3
    out, _, _ = _run(a, 2)
    hit = (ids == 3).any(1)
    assert bool(hit.any()) and not bool(hit.all())
    assert torch.equal(out[~hit], clean[~hit])
    assert bool(torch.isnan(out[hit]).all())


def test_zero_tokens_and_zero_inputs():
    a = _inputs(4, 256, 128, 8, 3300)
    for n in ("x", "xq", "x_scale"):
        a[n] = a[n][:0]
    out, c, ids = _run(a, 2)
    assert out.shape == (0, 256) and c.shape == ids.shape == (0, 2)
    assert _run(a, 2, router=False).shape == (0, 256)
    a = _inputs(4, 256, 128, 8, 3301, sd=0.0)            # zeros: every logit ties, out is zero
    out, c, ids = _check(a, 3)
    assert bool((out == 0).all())


def test_strided_inputs_and_single_rows():
    a = _inputs(10, 384, 256, 8, 3400)
    want = _run(a, 2)
    b = dict(a)
    wide = torch.zeros(20, 512, dtype=torch.bfloat16, device="cuda")
    wide[::2, 64:448] = a["x"]
    b["x"] = wide[::2, 64:448]
    wq = torch.zeros(10, 640, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    wq.view(torch.uint8)[:, 16:400] = a["xq"].view(torch.uint8)
    b["xq"] = wq[:, 16:400]
    for p, q in zip(want, _run(b, 2)):
        assert torch.equal(p, q)
    one = dict(a, x=b["x"][3:4], xq=b["xq"][3:4], x_scale=a["x_scale"][3:4])
    for p, q in zip(want, _run(one, 2)):
        assert torch.equal(p[3:4], q)


def _bits(t):
    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("sd", [1.0, 0.0])
def test_repeated_calls_are_equal_bit_for_bit(sd):
    """Whichever CTA comes last: zeros and their signs included (zero inputs under weights of both
    signs)."""
    a = _inputs(48, 1024, 512, 32, 3500, sd=sd)
    if sd == 0.0:
        a["xq"].view(torch.uint8)[::2] = 0x80                # minus zero
    want = _run(a, 4)
    for _ in range(20):
        for p, q in zip(want, _run(a, 4)):
            assert torch.equal(_bits(p), _bits(q))


def test_a_token_s_result_does_not_depend_on_its_batch():
    """Which experts the other tokens take changes how the work is split, and fp32 sums with it: a
    row alone and in a batch agree within both bounds."""
    a = _inputs(40, 512, 384, 16, 3600)
    out, _, ids = _check(a, 3)
    for t in (0, 17, 39):
        one = dict(a, x=a["x"][t:t + 1], xq=a["xq"][t:t + 1], x_scale=a["x_scale"][t:t + 1])
        o, _, i = _check(one, 3)
        assert torch.equal(i[0], ids[t])


def _c_abi(a, top_k, workspace, out, err=0, weights=0, ids=0, stream=None):
    from nanovllm_b200 import _lib
    T, H = a["x"].shape
    E, I = a["router"].shape[0], a["w2"].shape[-1]
    s = torch.cuda.current_stream() if stream is None else stream
    _lib.check(_lib.lib.fp8attn_fp8_moe(
        a["x"].data_ptr(), H, a["xq"].data_ptr(), H, a["x_scale"].data_ptr(), a["router"].data_ptr(),
        a["w13"].data_ptr(), a["w13_scale"].data_ptr(), a["w2"].data_ptr(), a["w2_scale"].data_ptr(),
        out.data_ptr(), out.stride(0), weights, ids, T, H, I, E, top_k, 1, workspace.data_ptr(),
        workspace.numel(), err, s.cuda_stream))


@pytest.mark.parametrize("T", [1, 20, 100])
def test_uninitialised_workspace_and_rows_outside(T):
    from nanovllm_b200 import _lib
    a = _inputs(T, 512, 256, 16, 3700 + T)
    want = _run(a, 4)
    need = _lib.lib.fp8attn_fp8_moe_workspace_bytes(T, 512, 256, 16, 4)
    ws = torch.full((need + 512,), 0xFF, dtype=torch.uint8, device="cuda")
    out = torch.full((T + 2, 520), 7.0, dtype=torch.bfloat16, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    for _ in range(2):                                    # again, with what the first call left
        _c_abi(a, 4, ws[:need], out[1:T + 1], err=err.data_ptr())
        torch.cuda.synchronize()
        assert torch.equal(out[1:T + 1, :512], want[0])
        assert bool((out[0] == 7).all()) and bool((out[T + 1] == 7).all())
        assert bool((out[:, 512:] == 7).all()) and bool((ws[need:] == 0xFF).all())
    assert int(err) == 0


def test_two_streams_at_once():
    """Calls that overlap, each with its own scratch, over and over."""
    a, b = _inputs(24, 1024, 512, 32, 3800), _inputs(3, 2048, 256, 16, 3801)
    want_a, want_b = _run(a, 4)[0], _run(b, 2)[0]
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    got_a, got_b = [], []
    for _ in range(30):
        with torch.cuda.stream(s):
            got_a.append(_run(a, 4, router=False))
        with torch.cuda.stream(t):
            got_b.append(_run(b, 2, router=False))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want_a) for g in got_a)
    assert all(torch.equal(g, want_b) for g in got_b)
    _no_device_error()


def test_two_captured_graphs_replayed_at_once():
    a, b = _inputs(8, 1024, 512, 32, 3900), _inputs(8, 1024, 512, 32, 3901)
    _run(a, 4), _run(b, 4)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_run(i, 4))
        graphs.append(g)
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for seed in (1, 2, 3):
        for i, n in ((a, seed), (b, seed + 10)):
            new = _inputs(8, 1024, 512, 32, 4000 + n)
            for name in ("x", "xq", "x_scale"):
                i[name].view(torch.uint8).copy_(new[name].view(torch.uint8))
        torch.cuda.synchronize()
        for _ in range(5):
            with torch.cuda.stream(s):
                graphs[0].replay()
            with torch.cuda.stream(t):
                graphs[1].replay()
        torch.cuda.synchronize()
        got = [[t_.clone() for t_ in o] for o in outs]
        for i, o in zip((a, b), got):
            for p, q in zip(o, _run(i, 4)):
                assert torch.equal(p, q)
    _no_device_error()


def test_weights_past_32_bit_offsets():
    """Expert weights of more than 2^31 bytes: the last expert's rows."""
    E, H, I = 66, 4096, 4096                              # 66 x 32 MiB = 2.2e9 bytes of w13
    a = _inputs(2, H, I, 2, 4100)
    w13 = torch.zeros((E, 2 * I, H), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    s13 = torch.zeros((E, 2 * I // 128, H // 128), dtype=torch.bfloat16, device="cuda")
    w2 = torch.zeros((E, H, I), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    s2 = torch.zeros((E, H // 128, I // 128), dtype=torch.bfloat16, device="cuda")
    router = torch.zeros((E, H), dtype=torch.bfloat16, device="cuda")
    for e, src in ((0, 0), (E - 1, 1)):
        for big, small in ((w13, "w13"), (s13, "w13_scale"), (w2, "w2"), (s2, "w2_scale"),
                           (router, "router")):
            big[e].view(torch.uint8).copy_(a[small][src].view(torch.uint8))
    a["x"][:, 0] = 4
    router[:, 0] = 0
    router[0, 0] = router[E - 1, 0] = 8                   # both chosen by every token
    from nanovllm_b200.fp8_linear import fp8_dyn_quant
    a["xq"], a["x_scale"] = fp8_dyn_quant(a["x"])
    small = dict(a, router=torch.stack([router[0], router[E - 1]]))
    a.update(w13=w13, w13_scale=s13, w2=w2, w2_scale=s2, router=router)
    out, c, ids = _run(a, 2)
    ref, err, c64, ids64 = ffn.moe(**small, top_k=2, renormalize=True)
    assert torch.equal(ids.long(), ids64 * (E - 1))
    ffn.assert_within(out, ref, err, ffn.bf16, "out")
    _no_device_error()


def test_norm_then_experts():
    """As a layer runs them: the norm's two outputs are the experts' inputs."""
    from nanovllm_b200.fp8_ffn import add_rms_norm_fp8
    a = _inputs(21, 1024, 384, 24, 4200)
    gen = torch.Generator(device="cuda").manual_seed(5)
    h = torch.randn(21, 1024, generator=gen, device="cuda").to(torch.bfloat16)
    r = (3 * torch.randn(21, 1024, generator=gen, device="cuda")).to(torch.bfloat16)
    w = (1 + 0.1 * torch.randn(1024, generator=gen, device="cuda")).to(torch.bfloat16)
    a["xq"], a["x_scale"], res, a["x"] = add_rms_norm_fp8(h, r, w, 1e-6, return_norm=True)
    _check(a, 4)


def test_refusals():
    from nanovllm_b200._lib import Fp8AttnError
    a = _inputs(4, 256, 128, 8, 4300)
    with pytest.raises(Fp8AttnError):
        _run(a, 9)                                        # more than there are experts
    with pytest.raises((Fp8AttnError, RuntimeError)):
        _run(a, 0)
    for n, bad in [("x", a["x"].float()), ("x", a["x"].cpu()), ("xq", a["xq"][:3]),
                   ("xq", a["xq"].float()), ("x_scale", a["x_scale"].float()),
                   ("x_scale", a["x_scale"][:, :1]), ("router", a["router"].float()),
                   ("router", a["router"][:4]), ("w13", a["w13"][:, :128]), ("w13", a["w13"].float()),
                   ("w13_scale", a["w13_scale"][:, :1]), ("w2", a["w2"].cpu()),
                   ("w2_scale", a["w2_scale"].half())]:
        with pytest.raises(AssertionError):
            _run(dict(a, **{n: bad}), 2)
    big = dict(a, x=a["x"][:1].expand(1025, 256).contiguous(), xq=a["xq"][:1].view(torch.uint8).expand(
        1025, 256).contiguous().view(torch.float8_e4m3fn),
        x_scale=a["x_scale"][:1].expand(1025, 2).contiguous())
    with pytest.raises(Fp8AttnError):
        _run(big, 2)
