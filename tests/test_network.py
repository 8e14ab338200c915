"""CPU checks of fermix_amd.network: the buckets' definition, what the Python functions refuse, and
what the C entry points refuse before any device work (fake pointers, host only)."""

import ctypes
import math
from fractions import Fraction

import pytest
import torch

import fermix_amd as fx
from fermix_amd import _lib
from tests import network64 as ref

OK, INVALID, WORKSPACE, UNSUPPORTED = 0, 1, 2, 4
GOOD, ODD = 0x10000, 0x10001


@pytest.mark.parametrize("nb,dist,two", [(32, 128, True), (32, 128, False), (4, 2, True), (2, 2, False), (20, 100, True), (64, 2048, True), (7, 9, True), (256, 2000, True)])
def test_distance_buckets(nb, dist, two):
    """Bucket b of a side holds distance b below the side's half, and above it the distances n with
    single (dist / single)^(t / grown) <= n, t = b - single, the largest such; compared as powers."""
    m = fx.distance_buckets(nb, dist, bidirectional=two, device="cpu")
    assert m.dtype == torch.uint8 and m.shape == (2 * dist + 1,)
    side = nb // 2 if two else nb
    single = side // 2
    grown = side - single

    def bucket(n):
        if n < single:
            return n
        t = max(t for t in range(grown) if Fraction(n, single) ** grown >= Fraction(dist, single) ** t)
        return single + t

    for d in list(range(-dist, -dist + 40)) + list(range(-45, 46)) + list(range(dist - 40, dist + 1)):
        if not -dist <= d <= dist:
            continue
        want = bucket(-d) if d <= 0 else side + bucket(d) if two else bucket(0)
        assert int(m[d + dist]) == want, d
    assert int(m.max()) < nb


def test_distance_buckets_refusals():
    for nb, dist, two in ((3, 10, True), (1, 10, False), (257, 300, False), (32, 8, True), (32, 2049, True)):
        with pytest.raises(ValueError):
            fx.distance_buckets(nb, dist, bidirectional=two, device="cpu")


def _attention(**change):
    a = dict(q=torch.zeros(2, 5, 4, 8), k=torch.zeros(2, 7, 2, 8), v=torch.zeros(2, 7, 2, 8), table=torch.zeros(32, 4), buckets=fx.distance_buckets(device="cpu"))
    a.update(change)
    return fx.attention(**a)


def test_attention_refusals():
    with pytest.raises(fx.FermixDeviceError):
        _attention()
    for bad in (
        dict(q=[1.0]), dict(q=torch.zeros(2, 5, 4, 8, dtype=torch.float64)), dict(k=torch.zeros(2, 7, 2, 8, dtype=torch.float16)),
        dict(table=torch.zeros(32, 4, dtype=torch.float16)), dict(buckets=torch.zeros(257, dtype=torch.int32)),
        dict(mask=torch.zeros(2, 7)), dict(lengths=torch.zeros(2)),
    ):
        with pytest.raises(TypeError):
            _attention(**bad)
    pos = lambda n: torch.zeros(2, n, dtype=torch.int32)
    for bad in (
        dict(q=torch.zeros(2, 4, 8)), dict(k=torch.zeros(3, 7, 2, 8), v=torch.zeros(3, 7, 2, 8)), dict(k=torch.zeros(2, 6, 2, 8)),
        dict(q=torch.zeros(2, 5, 4, 129), k=torch.zeros(2, 7, 2, 129), v=torch.zeros(2, 7, 2, 129)),
        dict(k=torch.zeros(2, 7, 3, 8), v=torch.zeros(2, 7, 3, 8)), dict(buckets=None), dict(table=None), dict(table=torch.zeros(32, 3)),
        dict(table=torch.zeros(65, 4)), dict(buckets=torch.zeros(256, dtype=torch.uint8)), dict(buckets=torch.zeros(4099, dtype=torch.uint8)),
        dict(q_pos=pos(5)), dict(q_pos=pos(5), k_pos=pos(6)), dict(lengths=torch.zeros(3, dtype=torch.int32)),
        dict(mask=torch.zeros(2, 8, dtype=torch.bool)), dict(offset=-1), dict(offset=2**31), dict(scale=0.0), dict(scale=math.nan),
    ):
        with pytest.raises(ValueError):
            _attention(**bad)


def _step(**change):
    a = dict(q=torch.zeros(2, 4, 8), k_cache=torch.zeros(6, 16, 2, 8), v_cache=torch.zeros(6, 16, 2, 8), pages=torch.zeros(2, 3, dtype=torch.int32),
             lengths=torch.zeros(2, dtype=torch.int32), k=torch.zeros(2, 2, 8), v=torch.zeros(2, 2, 8))
    a.update(change)
    return fx.attention_step(**a)


def test_step_refusals():
    with pytest.raises(fx.FermixDeviceError):
        _step()
    for bad in (dict(pages=torch.zeros(2, 3)), dict(k=torch.zeros(2, 2, 8, dtype=torch.float16)), dict(q=torch.zeros(2, 4, 8, dtype=torch.float64))):
        with pytest.raises(TypeError):
            _step(**bad)
    for bad in (
        dict(q=torch.zeros(3, 4, 8)), dict(v_cache=torch.zeros(6, 15, 2, 8)), dict(k=None), dict(k=torch.zeros(2, 2, 9)),
        dict(pages=torch.zeros(3, 3, dtype=torch.int32)), dict(lengths=torch.zeros(2, 1, dtype=torch.int32)),
        dict(k_cache=torch.zeros(6, 2, 16, 8).transpose(1, 2)), dict(table=torch.zeros(32, 4)),
    ):
        with pytest.raises(ValueError):
            _step(**bad)


def test_bias_refusals():
    m, t, p = fx.distance_buckets(device="cpu"), torch.zeros(32, 2), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(fx.FermixDeviceError):
        fx.relative_bias(t, m, p, p)
    for bad in ((t.int(), m, p, p), (t, m.int(), p, p), (t, m, p.float(), p), (t, m, p, [1])):
        with pytest.raises(TypeError):
            fx.relative_bias(*bad)
    for bad in ((t[0], m, p, p), (t, m[1:], p, p), (torch.zeros(257, 2), m, p, p), (t, m, p[0], p)):
        with pytest.raises(ValueError):
            fx.relative_bias(*bad)
    with pytest.raises(fx.FermixDeviceError):
        fx.relative_bias(t, m, p.expand(3, 4), p.expand(2, 4))


def test_norm_refusals():
    x, w = torch.zeros(3, 5, 8), torch.ones(8)
    with pytest.raises(fx.FermixDeviceError):
        fx.residual_norm(x, x)
    with pytest.raises(TypeError):
        fx.residual_norm(x, x.half())
    with pytest.raises(TypeError):
        fx.residual_norm(x.double(), x.double())
    with pytest.raises(TypeError):
        fx.residual_norm(x.half(), x.half(), post_weight=w, pre_weight=w.half())
    with pytest.raises(TypeError):
        fx.residual_norm(x, x, gate=w.half())
    for bad in (dict(h=x[:2]), dict(norm="batch"), dict(post_weight=w[:7]), dict(gate=torch.zeros(3, 5, 7)), dict(gate=torch.zeros(1, 3, 5, 8)), dict(eps=-1.0),
                dict(post_norm=False, post_weight=w), dict(pre_norm=False, pre_bias=w), dict(x=torch.zeros(2, 8193), h=torch.zeros(2, 8193)),
                dict(x=torch.zeros(2, 3, 4, 8), h=torch.zeros(2, 3, 4, 8), gate=torch.zeros(1, 3, 4, 8))):
        a = dict(x=x, h=x)
        a.update(bad)
        with pytest.raises(ValueError):
            fx.residual_norm(**a)


def _c_attention(**change):
    a = _lib.FxAttention(batch=2, nq=5, nk=7, heads=4, kv_heads=2, dim=8, dtype=_lib.FX_BF16, scale=0.3, q=GOOD, k=GOOD, v=GOOD, out=GOOD)
    for n, x in change.items():
        setattr(a, n, x)
    return ctypes.byref(a)


def test_c_attention():
    L = _lib.lib()
    assert L.fx_attention_forward(None, None) == INVALID
    assert L.fx_attention_forward(_c_attention(batch=0), None) == OK
    for bad in (dict(batch=-1), dict(dim=0), dict(dim=129), dict(heads=3), dict(kv_heads=0), dict(dtype=_lib.FX_F64), dict(dtype=9), dict(scale=0.0),
                dict(scale=math.inf), dict(offset=-1), dict(q=None), dict(v=None), dict(out=None), dict(q=ODD), dict(out=ODD), dict(buckets=32),
                dict(table=GOOD, buckets=32), dict(table=GOOD, map=GOOD, buckets=65), dict(table=GOOD, map=GOOD, buckets=32, radius=2049),
                dict(q_pos=GOOD), dict(stats=GOOD + 4), dict(lengths=GOOD + 2)):
        assert L.fx_attention_forward(_c_attention(**bad), None) == INVALID, bad
    grad = dict(stats=GOOD, grad_out=GOOD, grad_q=GOOD, grad_k=GOOD, grad_v=GOOD)
    need = L.fx_attention_grad_workspace(_c_attention(**grad))
    assert need >= 2 * 4 * 5 * 4
    assert L.fx_attention_grad(_c_attention(**grad), GOOD, need - 1, None) == WORKSPACE
    assert L.fx_attention_grad(_c_attention(**grad), GOOD + 8, need, None) == WORKSPACE
    assert L.fx_attention_grad(_c_attention(**grad), None, need, None) == WORKSPACE
    for bad in (dict(stats=None), dict(grad_out=None), dict(grad_k=None), dict(grad_q=ODD), dict(grad_table=GOOD)):
        assert L.fx_attention_grad(_c_attention(**{**grad, **bad}), GOOD, need, None) == INVALID, bad


def test_c_step():
    L = _lib.lib()

    def step(**change):
        a = _lib.FxAttentionStep(batch=2, heads=4, kv_heads=2, dim=8, dtype=_lib.FX_F32, pages=6, page_size=16, max_pages=300, scale=0.3,
                                 q=GOOD, k_cache=GOOD, v_cache=GOOD, page_table=GOOD, lengths=GOOD, out=GOOD)
        for n, x in change.items():
            setattr(a, n, x)
        return ctypes.byref(a)

    need = L.fx_attention_step_workspace(step())
    assert need > 0 and L.fx_attention_step_workspace(step(max_pages=4)) == 0
    assert L.fx_attention_step_run(step(), GOOD, need - 1, None) == WORKSPACE
    assert L.fx_attention_step_run(step(batch=0), None, 0, None) == OK
    assert L.fx_attention_step_run(step(max_pages=2**30, page_size=16), GOOD, 1 << 40, None) == UNSUPPORTED
    for bad in (dict(batch=-1), dict(page_size=0), dict(dim=129), dict(heads=3), dict(dtype=_lib.FX_F64), dict(scale=-1.0), dict(q=None), dict(lengths=None),
                dict(k_cache=None), dict(page_table=None), dict(k=GOOD), dict(q=ODD), dict(table=GOOD, buckets=4), dict(page_table=GOOD + 2)):
        assert L.fx_attention_step_run(step(**bad), GOOD, 1 << 40, None) == INVALID, bad


def test_c_bias():
    L = _lib.lib()

    def forward(table=GOOD, map_=GOOD, radius=8, buckets=4, q=GOOD, k=GOOD, batch=2, heads=2, nq=3, nk=5, dtype=_lib.FX_F32, out=GOOD):
        return L.fx_relative_bias(table, map_, radius, buckets, q, k, batch, heads, nq, nk, dtype, out, None)

    assert forward(batch=0, table=None) == OK and forward(nk=0, table=None) == OK
    for bad in (dict(table=None), dict(map_=None), dict(radius=-1), dict(radius=2049), dict(buckets=0), dict(buckets=257), dict(q=None), dict(batch=-1),
                dict(heads=0), dict(dtype=7), dict(out=None), dict(out=GOOD + 2), dict(dtype=_lib.FX_F64, out=GOOD + 4)):
        assert forward(**bad) == INVALID, bad
    need = L.fx_relative_bias_grad_workspace(4, 2, 2, 3, 5, _lib.FX_F32)
    args = lambda ws, n: (GOOD, GOOD, 8, 4, GOOD, GOOD, 2, 2, 3, 5, _lib.FX_F32, GOOD, ws, n, None)
    assert need > 0 and L.fx_relative_bias_grad(*args(GOOD, need - 1)) == WORKSPACE and L.fx_relative_bias_grad(*args(None, need)) == WORKSPACE
    assert L.fx_relative_bias_grad(None, *args(GOOD, need)[1:]) == INVALID


def test_c_norm():
    L = _lib.lib()

    def norm(**change):
        a = _lib.FxResidualNorm(samples=2, rows=3, columns=8, dtype=_lib.FX_BF16, wdtype=_lib.FX_F32, flags=6, eps=1e-6, alpha=1.0, x=GOOD, h=GOOD,
                                xs=24, xr=8, hs=24, hr=8, os=24, or_=8, y=GOOD, z=GOOD, stats=GOOD, grad_y=GOOD, grad_x=GOOD, grad_h=GOOD)
        for n, x in change.items():
            setattr(a, n, x)
        return ctypes.byref(a)

    assert L.fx_residual_norm_forward(norm(samples=0), None) == OK
    for bad in (dict(samples=-1), dict(columns=0), dict(columns=8193), dict(dtype=_lib.FX_F64), dict(wdtype=_lib.FX_F16), dict(flags=8), dict(gc=2), dict(x=None),
                dict(y=None), dict(z=None), dict(h=ODD), dict(post_weight=GOOD + 2), dict(stats=GOOD + 4)):
        assert L.fx_residual_norm_forward(norm(**bad), None) == INVALID, bad
    need = L.fx_residual_norm_grad_workspace(norm())
    assert need > 0 and L.fx_residual_norm_grad(norm(), GOOD, need - 1, None) == WORKSPACE
    assert L.fx_residual_norm_grad(norm(stats=None), GOOD, need, None) == INVALID
    assert L.fx_residual_norm_grad(norm(gate=GOOD), GOOD, 1 << 40, None) == INVALID


def test_reference_gradients():
    """The written-out gradients of tests/network64.py against torch's differentiation of its values."""
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)
    c = dict(q=r(2, 6, 4, 8), k=r(2, 9, 2, 8), v=r(2, 9, 2, 8), table=r(8, 4))
    kw = dict(buckets=fx.distance_buckets(8, 5, device="cpu"), causal=True, offset=1, lengths=torch.tensor([4, 9]), q_lengths=torch.tensor([6, 5]))
    g = r(2, 6, 4, 8)
    leaves = {n: x.clone().requires_grad_(True) for n, x in c.items()}
    want = torch.autograd.grad(ref.attention(**leaves, **kw), list(leaves.values()), g)
    for x, y in zip(ref.attention(**c, **kw, grad=g)[1:5], want):
        assert torch.allclose(x, y, atol=1e-12)
    for norm in ("rms", "layer"):
        c = dict(x=r(3, 4, 8), h=r(3, 4, 8), post_weight=r(8), post_bias=r(8), gate=r(3, 1, 8), scale=r(8), pre_weight=r(8), pre_bias=r(8))
        grads = (r(3, 4, 8), r(3, 4, 8))
        leaves = {n: x.clone().requires_grad_(True) for n, x in c.items()}
        want = torch.autograd.grad(ref.residual_norm(**leaves, norm=norm), list(leaves.values()), grads)
        got = ref.residual_norm(**c, norm=norm, grads=grads)[2]
        for n, y in zip(leaves, want):
            assert torch.allclose(got[n], y, atol=1e-12), n
