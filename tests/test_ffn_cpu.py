"""Refusals of the FP8 feed-forward entry points, before any device is touched, and the oracle's
roundings."""
import pytest
import torch

from nanovllm_b200 import _lib, fp8_ffn
from oracle import ffn

P = 4096                                          # an aligned address: never read


def _norm(**over):
    a = dict(x=P, xs=1024, r=P, rs=1024, w=P, eps=1e-6, q=P, d=P, ro=P, no=0, M=4, K=1024, dtype=0,
             stream=None)
    a.update(over)
    return _lib.lib.fp8attn_add_rms_norm_quant(*a.values())


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(w=None), dict(q=None), dict(d=None), dict(r=None), dict(ro=None),
    dict(x=P + 2), dict(r=P + 8), dict(w=P + 8), dict(q=P + 4), dict(d=P + 1), dict(ro=P + 8),
    dict(no=P + 8), dict(xs=1016), dict(xs=1028), dict(rs=1000), dict(rs=1030), dict(M=-1),
    dict(M=1 << 31), dict(K=0), dict(K=100), dict(K=16512, xs=16512, rs=16512), dict(dtype=2),
    dict(dtype=-1), dict(rs=2048)])                # in place with rows further apart
def test_norm_rejects(bad):
    assert _norm(**bad) == _lib.EINVAL
    assert _lib.lib.fp8attn_last_error()


def test_norm_empty_batch():
    assert _norm(M=0, x=None) == _lib.OK


def _silu(**over):
    a = dict(gu=P, rs=2048, q=P, d=P, M=4, I=1024, dtype=1, stream=None)
    a.update(over)
    return _lib.lib.fp8attn_silu_mul_quant(*a.values())


@pytest.mark.parametrize("bad", [
    dict(gu=None), dict(q=None), dict(d=None), dict(gu=P + 2), dict(q=P + 4), dict(d=P + 1),
    dict(rs=2040), dict(rs=2052), dict(M=-1), dict(M=1 << 40), dict(I=0), dict(I=64), dict(I=-128),
    dict(dtype=3)])
def test_silu_rejects(bad):
    assert _silu(**bad) == _lib.EINVAL


def test_silu_empty_batch():
    assert _silu(M=0, gu=None) == _lib.OK


def _moe(**over):
    a = dict(x=P, xs=1024, xq=P, xqs=1024, xscale=P, router=P, w13=P, w13s=P, w2=P, w2s=P, out=P,
             outs=1024, tw=0, ti=0, T=4, H=1024, I=512, E=16, k=4, renorm=1, ws=P, wsb=1 << 40, err=0,
             stream=None)
    a.update(over)
    return _lib.lib.fp8attn_fp8_moe(*a.values())


@pytest.mark.parametrize("bad", [
    *[{n: None} for n in ("x", "xq", "xscale", "router", "w13", "w13s", "w2", "w2s", "out")],
    *[{n: P + 8} for n in ("x", "xq", "router", "w13", "w2", "out")],
    *[{n: P + 1} for n in ("xscale", "w13s", "w2s", "tw", "ti", "err")],
    dict(xs=1020), dict(xs=512), dict(xqs=1032), dict(xqs=512), dict(outs=1028), dict(outs=1000),
    dict(T=-1), dict(T=1025), dict(H=0), dict(H=1000), dict(H=16512), dict(I=0), dict(I=500),
    dict(I=16512), dict(E=0), dict(E=513), dict(k=0), dict(k=17), dict(E=64, k=33),
    dict(T=1024, k=9), dict(ws=P + 16)])
def test_moe_rejects(bad):
    assert _moe(**bad) == _lib.EINVAL
    assert _lib.lib.fp8attn_last_error()


def test_moe_workspace():
    size = _lib.lib.fp8attn_fp8_moe_workspace_bytes
    assert size(4, 1000, 512, 16, 4) == -1 and size(-1, 1024, 512, 16, 4) == -1
    assert size(4, 1024, 512, 16, 17) == -1
    need = size(4, 1024, 512, 16, 4)
    assert need >= 4 * 4 * (4 + 4 + 512 + 1024 * 4)        # ids, weights, activations, results
    assert _moe(wsb=need - 1) == _lib.EWORKSPACE
    assert _moe(ws=None) == _lib.EWORKSPACE
    assert _moe(T=0, x=None) == _lib.OK


def test_python_refuses_cpu_tensors():
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    q = torch.zeros(4, 256, dtype=torch.float8_e4m3fn)
    s = torch.ones(4, 2, dtype=torch.bfloat16)
    with pytest.raises(AssertionError):
        fp8_ffn.add_rms_norm_fp8(x, None, x[0], 1e-6)
    with pytest.raises(AssertionError):
        fp8_ffn.silu_mul_fp8(x)
    with pytest.raises(AssertionError):
        fp8_ffn.fp8_moe(x, q, s, x, q, s, q, s, 1)


@pytest.mark.parametrize("dtype,rounding", [(torch.float8_e4m3fn, ffn.e4m3),
                                            (torch.bfloat16, ffn.bf16), (torch.float16, ffn.fp16)])
def test_oracle_roundings_are_torch_s(dtype, rounding):
    g = torch.Generator().manual_seed(0)
    v = torch.randn(20000, generator=g) * torch.exp2(torch.randint(-20, 9, (20000,), generator=g))
    v = v.clamp(-448, 448)
    assert torch.equal(rounding(v.double()), v.to(dtype).double())
