"""The largest and smallest arguments that the network operators' C entry points and Python functions take, and what lies
past them; before any device work (fake pointers, host only)."""

import ctypes

import pytest
import torch

import fermix_amd as fx
from fermix_amd import _lib

OK, INVALID, WORKSPACE, UNSUPPORTED = 0, 1, 2, 4
GOOD = 0x10000


def attention(**change):
    a = _lib.FxAttention(batch=2, nq=5, nk=7, heads=4, kv_heads=2, dim=8, dtype=_lib.FX_BF16, scale=0.3, q=GOOD, k=GOOD, v=GOOD, out=GOOD)
    for n, x in change.items():
        setattr(a, n, x)
    return ctypes.byref(a)


def test_attention_offset():
    """Positions offset + i stay within int32. (With no sample nothing is launched.)"""
    L = _lib.lib()
    last = 2**31 - 1 - 7
    assert L.fx_attention_forward(attention(offset=last, batch=0), None) == OK
    for bad in (last + 1, 2**31 - 1):
        assert L.fx_attention_forward(attention(offset=bad, batch=0), None) == INVALID
        assert L.fx_attention_grad(attention(offset=bad, batch=0), None, 0, None) == INVALID
    x, k = torch.zeros(2, 5, 4, 8), torch.zeros(2, 7, 2, 8)
    with pytest.raises(fx.FermixDeviceError):
        fx.attention(x, k, k, offset=last)
    with pytest.raises(ValueError):
        fx.attention(x, k, k, offset=last + 1)


def test_norm_gate_of_the_rows_alone():
    """The gradient of a gate that samples share and rows do not is a sum over samples: refused before any work."""
    L = _lib.lib()
    a = _lib.FxResidualNorm(samples=2, rows=3, columns=8, dtype=_lib.FX_BF16, wdtype=_lib.FX_F32, flags=6, eps=1e-6, alpha=1.0, x=GOOD, h=GOOD,
                            gate=GOOD, xs=24, xr=8, hs=24, hr=8, os=24, or_=8, gr=8, gc=1, stats=GOOD, grad_y=GOOD, grad_gate=GOOD)
    assert L.fx_residual_norm_grad(ctypes.byref(a), None, 0, None) == UNSUPPORTED
    a.gs = 24
    assert L.fx_residual_norm_grad(ctypes.byref(a), None, 0, None) == WORKSPACE
    a.gs, a.samples = 0, 1
    assert L.fx_residual_norm_grad(ctypes.byref(a), None, 0, None) == WORKSPACE


def test_bias_limits():
    """What the library cannot take is refused by name in Python, and by the C entry points."""
    L = _lib.lib()
    m, p = fx.distance_buckets(device="cpu"), torch.zeros(4, dtype=torch.int32)
    for heads in (0, 4097):
        with pytest.raises(ValueError, match="heads"):
            fx.relative_bias(torch.zeros(32, heads), m, p, p)
    with pytest.raises(fx.FermixDeviceError):
        fx.relative_bias(torch.zeros(256, 4096), m, p, p)
    with pytest.raises(ValueError, match="positions"):
        fx.relative_bias(torch.zeros(32, 1), m, torch.zeros(1, dtype=torch.int32).expand(2**30 + 1), p)
    for heads, nq, nk, want in ((4097, 0, 1, INVALID), (4096, 0, 1, OK), (1, 0, 2**30, OK), (1, 0, 2**30 + 1, INVALID), (1, 2**30 + 1, 0, INVALID)):
        assert L.fx_relative_bias(None, None, 8, 4, None, None, 1, heads, nq, nk, _lib.FX_F32, None, None) == want


def test_attention_lengths():
    L = _lib.lib()
    assert L.fx_attention_forward(attention(nq=2**30, nk=2**30, batch=0), None) == OK
    for bad in (dict(nq=2**30 + 1), dict(nk=2**30 + 1)):
        assert L.fx_attention_forward(attention(batch=0, **bad), None) == INVALID
    x = torch.zeros(1, 1, 1, 8)
    with pytest.raises(ValueError):
        fx.attention(x, x.expand(1, 2**32 + 5, 1, 8), x.expand(1, 2**32 + 5, 1, 8))


def test_step_pages():
    """A table of more tokens than int32 counts, and a page of 2^32 elements: refused by name."""
    q, n = torch.zeros(1, 1, 8), torch.zeros(1, dtype=torch.int32)
    cache = torch.zeros(1, 1, 1, 8)
    many = torch.zeros(1, 1, dtype=torch.int32).expand(1, 2**32 + 3)
    with pytest.raises(ValueError, match="pages"):
        fx.attention_step(q, cache, cache, many, n)
    meta = torch.empty(1, 2**29, 1, 8, device="meta")
    with pytest.raises(ValueError, match="pages"):
        fx.attention_step(q.to("meta"), meta, meta, many[:, :1].to("meta"), n.to("meta"))


def test_scales():
    L = _lib.lib()
    x, k = torch.zeros(1, 2, 1, 8), torch.zeros(1, 1, 1, 8)
    p, n = torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)

    def step(scale):
        return L.fx_attention_step_run(ctypes.byref(_lib.FxAttentionStep(batch=0, heads=1, kv_heads=1, dim=8, page_size=1, scale=scale)), None, 0, None)

    for scale in (1e-30, 1e30):
        assert L.fx_attention_forward(attention(scale=scale, batch=0), None) == OK and step(scale) == OK
        with pytest.raises(fx.FermixDeviceError):
            fx.attention(x, x, x, scale=scale)
    for bad in (0.0, -1.0, 1e-45, 9e-31, 1.1e30, 3e38, float("inf"), float("nan")):
        assert L.fx_attention_forward(attention(scale=bad, batch=0), None) == INVALID and step(bad) == INVALID
        with pytest.raises(ValueError, match="scale"):
            fx.attention(x, x, x, scale=bad)
        with pytest.raises(ValueError, match="scale"):
            fx.attention_step(x[0], k, k, p, n, scale=bad)
