"""The operators of fermix_amd.network on the GPU where a size, a scale or an input goes to its end:
nothing to work on, the largest offsets, more work than one launch or one pass of a workgroup
holds, cotangents and weights that are small for float16. Oracle and tolerances: those of
test_gpu_network.py, unless a test derives its own."""

import ctypes
import math

import pytest
import torch

import fermix_amd as fx
from fermix_amd import _lib, network
from tests import network64 as ref
from tests.test_gpu_network import EPS, GATES, TYPES, U, attention_case, check_attention, check_norm, ids, near, near_sums, norm_case, rand, run_attention

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ nothing to work on


EMPTY = [(0, 5, 16), (5, 0, 16), (0, 1, 16), (0, 16), (3, 0, 2, 16), (0, 5, 300)]
WITH_ELEMENTS = [(s, g) for s in EMPTY for g in GATES if GATES[g](s) is not None and math.prod(GATES[g](s))]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("shape,gate", WITH_ELEMENTS, ids=lambda s: s if isinstance(s, str) else "x".join(map(str, s)))
def test_norm_gate_without_rows(dev, dtype, shape, gate):
    """Without rows every gradient is zero, a broadcast gate's too, which has elements all the same; the
    allocator's memory is filled with NaN beforehand, so that a result that nobody writes shows."""
    s = GATES[gate](shape)
    x, h = (torch.zeros(shape, dtype=dtype, device=dev, requires_grad=True) for _ in range(2))
    g = torch.ones(s, dtype=dtype, device=dev, requires_grad=True)
    w = torch.ones(shape[-1], device=dev, requires_grad=True)
    y, z = fx.residual_norm(x, h, gate=g, post_weight=w)
    fill = [torch.full((n,), math.nan, dtype=dtype, device=dev) for n in (1, 16, 80, 300, 1500) for _ in range(8)]
    del fill
    dg, dw = torch.autograd.grad((y, z), (g, w), (torch.zeros_like(y), torch.zeros_like(z)))
    assert dg.shape == g.shape and (dg == 0).all() and (dw == 0).all()


# ------------------------------------------------------------------ the largest offsets


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("N,K,D,causal", [(65, 65, 16, False), (300, 200, 64, False), (200, 330, 128, False), (130, 130, 40, True), (100, 90, 64, True)],
                         ids=lambda x: str(x))
def test_attention_largest_offset(dev, dtype, N, K, D, causal):
    """The last offset that is taken: every key is further below every query than the radius, also for tiles
    whose distances reach the lowest int32, and nothing is hidden by causal."""
    gen = torch.Generator().manual_seed(N + K)
    c = attention_case(gen, dtype, 2, N, K, 2, 1, D)
    c.update(causal=causal, offset=2**31 - 1 - max(N, K))
    check_attention(c, dev, dtype, gen, (N, K, D, causal))


# ------------------------------------------------------------------ float16's small numbers


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("size", [1e-2, 1e-3, 1e-4, "mixed"])
@pytest.mark.parametrize("N,K,H,Hkv,D,mode", [(64, 4096, 2, 1, 64, ""), (4096, 64, 1, 1, 64, ""), (70, 2100, 2, 2, 128, "p"), (1100, 1100, 2, 1, 128, "c"),
                                              (128, 128, 2, 2, 64, ""), (100, 128, 4, 2, 40, "lp"), (128, 90, 1, 1, 128, "m")], ids=lambda x: str(x))
def test_attention_small_cotangents(dev, dtype, size, N, K, H, Hkv, D, mode):
    """A loss that is a mean over many samples has small cotangents. P and dS then pass below float16's normal numbers
    (dS below its smallest) where the gradients do not: the error stays that of the roundings. k is large for dq, then
    q for dk, so that the results themselves are normal; "mixed": a cotangent of its own size for each query."""
    gen = torch.Generator().manual_seed(N + K + D)
    for big in "qk":
        c = attention_case(gen, dtype, 1, N, K, H, Hkv, D, mode=mode)
        small = "k" if big == "q" else "q"
        c[big], c[small] = c[big] * 64, c[small] / 64
        g = rand(gen, 1, N, H, D)
        g = (g * (2.0 ** -torch.randint(0, 14, (1, N, 1, 1), generator=gen) if size == "mixed" else size)).to(dtype)
        want = ref.attention(**c, grad=g)
        got = run_attention(c, dev, g)
        for name, x, y in zip(("out", "dq", "dk", "dv"), got, want):
            near(x, y, dtype, 2, (big, name))
        near_sums(got[4], want[4], want[5] + 1e-3 * want[5].mean(), dtype, what=(big, "dtable"), tol=EPS)


@pytest.mark.parametrize("N,K,D", [(100, 128, 64), (90, 700, 40), (200, 300, 128)])
def test_attention_large_cotangents(dev, N, K, D):
    """dS past float16's largest number, where the gradients are within it (small q and k)."""
    gen = torch.Generator().manual_seed(N)
    c = attention_case(gen, torch.float16, 2, N, K, 2, 2, D)
    c["q"], c["k"], c["v"] = c["q"] / 64, c["k"] / 64, c["v"] * 256
    g = rand(gen, 2, N, 2, D, dtype=torch.float16, scale=100.0)
    g[:, ::3] *= 100
    want = ref.attention(**c, grad=g)
    assert want[1].abs().max() < 6e4 and want[2].abs().max() < 6e4 and want[3].abs().max() < 6e4
    got = run_attention(c, dev, g)
    for name, x, y in zip(("out", "dq", "dk", "dv"), got, want):
        near(x, y, torch.float16, 2, name)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("gap", [14.0, 16.0, 18.0])
def test_attention_many_small_weights(dev, dtype, gap):
    """One key outweighs each of the others by exp(gap), but its value is 0: what is left is the others' sum, whose
    weights are below float16's normal numbers when the largest is 1. In a whole sequence and in one step."""
    K, H, D = 3000, 4, 32
    gen = torch.Generator().manual_seed(int(gap))
    q = torch.full((1, 1, H, D), 1.0, dtype=dtype)
    k, v = torch.zeros(1, K, 1, D, dtype=dtype), (1 + rand(gen, 1, K, 1, D, scale=0.25)).to(dtype)
    k[0, 1234], v[0, 1234] = gap / D, 0.0
    want = ref.attention(q, k, v, scale=1.0)
    near(fx.attention(q.to(dev), k.to(dev), v.to(dev), scale=1.0), want, dtype, 2, "attention")
    pages = torch.arange(K // 8, dtype=torch.int32, device=dev)[None]
    kc, vc = (t.reshape(K // 8, 8, 1, D).to(dev) for t in (k, v))
    got = fx.attention_step(q[:, 0].to(dev), kc, vc, pages, torch.tensor([K], dtype=torch.int32, device=dev), scale=1.0)
    near(got, want[:, 0], dtype, 2, "step")


# ------------------------------------------------------------------ more than one turn


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("shape,gate", [((700, 37, 512), "sample"), ((90, 130, 512), "none"), ((9, 130, 8192), "token"), ((10000, 7, 64), "full"), ((5, 21000, 40), "channel")],
                         ids=lambda x: "x".join(map(str, x)) if isinstance(x, tuple) else x)
def test_norm_many_rows(dev, dtype, shape, gate):
    """More rows than the workgroups of one launch hold at once, in samples that do not divide a turn."""
    gen = torch.Generator().manual_seed(sum(shape))
    c = norm_case(gen, dtype, shape, gate)
    check_norm(c, dev, dtype, gen, (shape, gate), norm="layer")


@pytest.mark.parametrize("dtype", TYPES + [torch.float64], ids=ids)
@pytest.mark.parametrize("B,H,Q,K,nb", [(6000, 3, 5, 9, 32), (5000, 1, 12, 12, 20), (3000, 2, 40, 24, 64), (9000, 1, 7, 130, 256)])
def test_relative_bias_many_samples(dev, dtype, B, H, Q, K, nb):
    """More samples than there are workgroups, each with positions of its own: a workgroup's sums go on over samples."""
    gen = torch.Generator().manual_seed(B + nb)
    table, m = rand(gen, nb, H, dtype=dtype), fx.distance_buckets(nb, 100, device="cpu")
    q, k = (torch.randint(-90, 90, (B, n), generator=gen).to(torch.int32) for n in (Q, K))
    t = table.to(dev).requires_grad_(True)
    out = fx.relative_bias(t, m.to(dev), q.to(dev), k.to(dev))
    assert torch.equal(out.detach().double().cpu(), ref.relative_bias(table, m, q, k))
    g = rand(gen, B, H, Q, K, dtype=dtype)
    (dt,) = torch.autograd.grad(out, t, g.to(dev))
    bucket = ref.bucket_of(m, nb, q, k)
    want, size = ref.bucket_sums(g.double(), bucket, nb), ref.bucket_sums(g.double().abs(), bucket, nb)
    if dtype == torch.float64:
        assert ((dt.cpu() - want).abs() <= 16 * U[dtype] * size).all()
    else:
        near_sums(dt, want, size, torch.float32, dtype)


def test_relative_bias_gradient_of_one_workgroup(dev):
    """Sums of one sign, which keep every rounding of a long chain: lanes add at most 64 values in float32 (a
    rounding error of some 0.3 u of the sum for 256 lanes), and the lanes' sums add nothing to that: 2 u, and u for the result."""
    gen = torch.Generator().manual_seed(1)
    for N, H in ((128, 8), (64, 16)):
        m, table = fx.distance_buckets(device="cpu"), torch.zeros(32, H)
        p = torch.arange(N, dtype=torch.int32)[None]
        t = table.to(dev).requires_grad_(True)
        g = 1 + torch.rand(1, H, N, N, generator=gen)
        (dt,) = torch.autograd.grad(fx.relative_bias(t, m.to(dev), p.to(dev), p.to(dev)), t, g.to(dev))
        want = ref.bucket_sums(g.double(), ref.bucket_of(m, 32, p, p), 32)
        near_sums(dt, want, want, torch.float32, tol=2 * U[torch.float32])


# ------------------------------------------------------------------ more than one launch


MANY = 2**32 // 256 + 12345  # workgroups of 256 lanes, which a launch counts in 32 bits


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("Hkv", [2, 1])
def test_attention_many_items(dev, dtype, Hkv):
    """One query, one key: out is v, dv the cotangent (summed over heads that share it), the other gradients vanish: the
    16-bit types form P = 1 from a score that has been rounded, to EPS, and so dS = P (dP - P dP) to EPS of dP."""
    gen = torch.Generator(device=dev).manual_seed(1)
    B = MANY // Hkv + 1
    r = lambda H: torch.randn(B, 1, H, 1, generator=gen, device=dev).to(dtype)
    q, k, v, g = r(2), r(Hkv), r(Hkv), r(2)
    table = torch.zeros(2, 2, device=dev)
    leaves = [x.requires_grad_(True) for x in (q, k, v, table)]
    out = fx.attention(q, k, v, table=table, buckets=torch.zeros(1, dtype=torch.uint8, device=dev))
    assert torch.equal(out, v.detach().expand(B, 1, 2, 1))
    dq, dk, dv, dt = torch.autograd.grad(out, leaves, g)
    dp = (g * v).detach().abs().double()
    tol = 0.0 if dtype == torch.float32 else EPS
    assert (dq.double().abs() <= tol * dp * k.detach().abs()).all() and dt.abs().max() <= tol * dp.sum()
    assert (dk.double().abs() <= tol * (dp * q.detach().abs()).reshape(B, 1, Hkv, -1).sum(-1, keepdim=True)).all()
    assert torch.equal(dv, g if Hkv == 2 else (g[:, :, :1].float() + g[:, :, 1:].float()).to(dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_norm_gate_of_many_samples(dev, dtype):
    gen = torch.Generator(device=dev).manual_seed(2)
    x, h, g, dy = (torch.randn(MANY, 1, 1, generator=gen, device=dev).to(dtype) for _ in range(4))
    for t in (h, g):
        t.requires_grad_(True)
    y = fx.residual_norm(x, h, gate=g, post_norm=False, pre_norm=False)
    dh, dg = torch.autograd.grad(y, (h, g), dy)
    assert torch.equal(dh, dy * g) and torch.equal(dg, dy * h)


# ------------------------------------------------------------------ tracing


def test_traces_replay_on_other_inputs(dev):
    """torch.jit.trace records a call, not only the memory that it returns: a replay gives the new input's values."""
    p = torch.arange(12, dtype=torch.int32, device=dev)[None]
    m, table = fx.distance_buckets(device=dev), torch.randn(32, 2, device=dev)
    calls = {
        (32, 2): lambda t: fx.relative_bias(t, m, p, p),
        (2, 12, 2, 16): lambda x: fx.attention(x, x, x, table=table, buckets=m, causal=True),
        (3, 5, 64): lambda x: fx.residual_norm(x, 2 * x, gate=x)[1],
    }
    for shape, f in calls.items():
        traced = torch.jit.trace(f, (torch.randn(shape, device=dev),), check_trace=False)
        for _ in range(3):
            x = torch.randn(shape, device=dev)
            fill = [torch.full((n,), math.nan, device=dev) for n in (256, 768, 960, 2048) for _ in range(8)]
            del fill
            assert torch.equal(traced(x), f(x)), shape
    cache = torch.zeros(3, 4, 2, 16, device=dev)
    z = torch.zeros(2, 1, dtype=torch.int32, device=dev)
    with pytest.raises(NotImplementedError, match="trace"):
        torch.jit.trace(lambda q: fx.attention_step(q, cache, cache.clone(), z, z[:, 0]), (torch.randn(2, 4, 16, device=dev),))


@pytest.mark.parametrize("transform", ["jvp", "vmap", "grad", "jacrev", "vmap of grad"])
@pytest.mark.parametrize("name", ["relative_bias", "attention", "residual_norm", "attention_step"])
def test_function_transforms_raise(dev, name, transform):
    """torch.func sees tensors that are not the caller's: every operator raises under each of them."""
    m, p = fx.distance_buckets(device=dev), torch.arange(4, dtype=torch.int32, device=dev)
    q, z = torch.randn(2, 4, 2, 8, device=dev), torch.zeros(2, 1, dtype=torch.int32, device=dev)
    cache = torch.zeros(2, 4, 2, 8, device=dev)
    f, x = {
        "relative_bias": (lambda t: fx.relative_bias(t, m, p, p), torch.randn(32, 2, device=dev)),
        "attention": (lambda t: fx.attention(t, q, q), q.clone()),
        "residual_norm": (lambda t: fx.residual_norm(t, 2 * q)[0], q.clone()),
        "attention_step": (lambda t: fx.attention_step(t, cache, cache, z, z[:, 0]), torch.randn(2, 2, 8, device=dev)),
    }[name]
    run = {
        "jvp": lambda: torch.func.jvp(f, (x,), (torch.ones_like(x),)),
        "vmap": lambda: torch.func.vmap(f)(torch.stack([x, x])),
        "grad": lambda: torch.func.grad(lambda t: f(t).sum())(x),
        "jacrev": lambda: torch.func.jacrev(f)(x),
        "vmap of grad": lambda: torch.func.vmap(torch.func.grad(lambda t: f(t).sum()))(torch.stack([x, x])),
    }[transform]
    f(x)
    with pytest.raises(RuntimeError):
        run()


# ------------------------------------------------------------------ the C entry points' own layouts


@pytest.mark.parametrize("gc", [1, 0])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_norm_gate_shared_by_samples(dev, dtype, gc):
    """A gate with no stride over samples and rows has one gradient, of the shape that its strides name, and nothing is
    written past it."""
    gen = torch.Generator().manual_seed(3)
    c = norm_case(gen, dtype, (7, 40, 96), "channel" if gc else "scalar", "")
    grads = rand(gen, 7, 40, 96, dtype=dtype), rand(gen, 7, 40, 96, dtype=dtype)
    want = ref.residual_norm(**c, grads=grads)[2]
    a = {n: x.to(dev) for n, x in c.items()}
    y, z, dx, dh = (torch.empty_like(a["x"]) for _ in range(4))
    stats = torch.empty(7, 40, 4, device=dev)
    s = network._norm_args(a["x"], a["h"], a["gate"], [None] * 5, 1.0, 1e-6, _lib.FX_NORM_POST | _lib.FX_NORM_PRE, y, z, stats)
    s.samples, s.rows, s.xs, s.hs, s.os = 7, 40, 40 * 96, 40 * 96, 40 * 96
    assert (s.gs, s.gr, s.gc) == (0, 0, gc)
    network._call("fx_residual_norm_forward", y, ctypes.byref(s))
    dy, dz = (g.to(dev) for g in grads)
    n = 96 if gc else 1
    dg = torch.full((8 * n,), 7.0, dtype=dtype, device=dev)
    s.grad_y, s.grad_z, s.grad_x, s.grad_h, s.grad_gate = (t.data_ptr() for t in (dy, dz, dx, dh, dg))
    size = _lib.lib().fx_residual_norm_grad_workspace(ctypes.byref(s))
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    network._call("fx_residual_norm_grad", y, ctypes.byref(s), ws.data_ptr(), size)
    near_sums(dg[:n].reshape(want["gate"].shape), want["gate"], want["size_gate"], dtype, dtype)
    assert (dg[n:] == 7.0).all()


# ------------------------------------------------------------------ many heads


@pytest.mark.parametrize("dtype", TYPES + [torch.float64], ids=ids)
@pytest.mark.parametrize("nb,H,Q,K", [(256, 65, 9, 24), (256, 300, 5, 7), (32, 4096, 3, 4)])
def test_relative_bias_many_heads(dev, dtype, nb, H, Q, K):
    """Tables that no workgroup holds as a whole."""
    gen = torch.Generator().manual_seed(H)
    table, m = rand(gen, nb, H, dtype=dtype), fx.distance_buckets(nb, 200, device="cpu")
    q, k = (torch.randint(-150, 150, (2, n), generator=gen).to(torch.int32) for n in (Q, K))
    t = table.to(dev).requires_grad_(True)
    out = fx.relative_bias(t, m.to(dev), q.to(dev), k.to(dev))
    assert torch.equal(out.detach().double().cpu(), ref.relative_bias(table, m, q, k))
    g = rand(gen, *out.shape, dtype=dtype)
    (dt,) = torch.autograd.grad(out, t, g.to(dev))
    bucket = ref.bucket_of(m, nb, q, k)
    want, size = ref.bucket_sums(g.double(), bucket, nb), ref.bucket_sums(g.double().abs(), bucket, nb)
    if dtype == torch.float64:
        assert ((dt.cpu() - want).abs() <= 16 * U[dtype] * size).all()
    else:
        near_sums(dt, want, size, torch.float32, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_attention_many_heads(dev, dtype):
    """More heads than a grid's second dimension holds."""
    gen = torch.Generator().manual_seed(70000)
    c = attention_case(gen, dtype, 1, 3, 4, 70000, 35000, 2, 4, 3)
    check_attention(c, dev, dtype, gen)


# ------------------------------------------------------------------ the smallest and the largest scale


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12, 1e30])
def test_attention_scales(dev, dtype, scale):
    """A scale at which the table alone decides (its entries of 0 among them), or the largest product does."""
    gen = torch.Generator().manual_seed(5)
    for mode in ("", "p"):
        c = attention_case(gen, dtype, 1, 70, 90, 2, 1, 32, mode=mode)
        c["table"][::3] = 0.0
        c["scale"] = scale
        near(run_attention(c, dev), ref.attention(**c), dtype, 2, (scale, mode))
    q, k, v = (c[n].to(dev) for n in "qkv")
    pages = torch.arange(9, dtype=torch.int32, device=dev)[None]
    out = fx.attention_step(q[:, 0], k.reshape(9, 10, 1, 32), v.reshape(9, 10, 1, 32), pages, torch.tensor([90], dtype=torch.int32, device=dev),
                            table=c["table"].to(dev), buckets=c["buckets"].to(dev), scale=scale)
    want = ref.attention(c["q"][:, :1], c["k"], c["v"], c["table"], c["buckets"], offset=89, scale=scale)
    near(out, want[:, 0], dtype, 2, (scale, "step"))
