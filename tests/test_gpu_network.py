"""The operators of fermix_amd.network on the GPU against their definitions in 64 bits
(tests/network64.py) on the same inputs.

Tolerances, with u the unit roundoff of a type (2^-24, 2^-11, 2^-8 for float32, float16, bfloat16):
* a value that is rounded once from float32 sums: 2-norm of the error at most u of the result's, for
  float32 EPS = 3e-6 (scores up to about 16 carry 16 roundings of u into the exponent, three times);
* attention's 16-bit results, which also round P or dS for a product: 2u (u for each rounding);
* sums over rows or buckets in float32: 16 u32 of the sum of the magnitudes that the terms are made
  of for float32 inputs (a term that is itself a difference has the error of what it is taken from), for
  16-bit inputs 32 u32, plus the result's own rounding; bucket sums of attention EPS of them, as
  each term has a weight whose error is that of a value.
"""

import math

import pytest
import torch

import fermix_amd as fx
from tests import network64 as ref

pytestmark = pytest.mark.gpu

U = {torch.float64: 2.0**-53, torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
EPS = 3e-6
TYPES = [torch.float32, torch.float16, torch.bfloat16]
ids = lambda x: str(x).replace("torch.", "") if isinstance(x, torch.dtype) else None


def near(got, want, dtype, rounds=1, what="", size=None):
    """2-norm of the error against that of the result (float32 results that are differences: of the magnitudes
    they are made of); non-finite places have to agree."""
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), what
    if not want.numel():
        return
    got, want = got.nan_to_num(0.0), want.nan_to_num(0.0)
    tol = EPS if dtype == torch.float32 else rounds * U[dtype]
    # a lone 16-bit value can be off by a whole roundoff, and tiny float16 values by half a subnormal step
    off, norm = (got - want).norm().item(), want.norm().item()
    floor = 2.0**-25 * math.sqrt(want.numel()) if dtype == torch.float16 else 1e-30
    floor += 0.0 if size is None else EPS * size.norm().item()
    assert off <= tol * norm + floor, (what, off / max(norm, 1e-300), tol)


def near_sums(got, want, size, dtype, out=torch.float32, what="", tol=None):
    got = got.detach().double().cpu()
    tol = tol or (16 if dtype == torch.float32 else 32) * U[torch.float32]
    floor = 2.0**-25 if out == torch.float16 else 1e-30  # half a subnormal step
    bad = (got - want).abs() > tol * size + U[out] * want.abs() + floor
    assert not bad.any(), (what, (got - want).abs()[bad].max().item(), size[bad].max().item())


def rand(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=gen, dtype=torch.float64) * scale).to(dtype)


def gpu(x, dev):
    return x.to(dev) if isinstance(x, torch.Tensor) else x


# ------------------------------------------------------------------ relative bias


@pytest.mark.parametrize("dtype", TYPES + [torch.float64], ids=ids)
@pytest.mark.parametrize("lead,H,Q,K,nb,dist", [
    ((), 1, 1, 1, 4, 3), ((), 3, 7, 13, 32, 128), ((2,), 2, 64, 96, 32, 20), ((2, 3), 1, 33, 40, 20, 17),
    ((5,), 5, 130, 264, 256, 2000), ((), 9, 300, 512, 64, 64),
])
def test_relative_bias(dev, dtype, lead, H, Q, K, nb, dist):
    gen = torch.Generator().manual_seed(Q * K + nb)
    table = rand(gen, nb, H, dtype=dtype)
    m = fx.distance_buckets(nb, dist, device="cpu")
    q = torch.randint(-300, 300, lead + (Q,), generator=gen).to(torch.int32)
    k = torch.randint(-300, 300, lead + (K,), generator=gen).to(torch.int32)
    t = table.to(dev).requires_grad_(True)
    out = fx.relative_bias(t, m.to(dev), q.to(dev), k.to(dev))
    want = ref.relative_bias(table, m, q, k)
    assert torch.equal(out.detach().double().cpu(), want)
    g = rand(gen, *out.shape, dtype=dtype)
    (dt,) = torch.autograd.grad(out, t, g.to(dev))
    (again,) = torch.autograd.grad(fx.relative_bias(t, m.to(dev), q.to(dev), k.to(dev)), t, g.to(dev))
    assert torch.equal(dt, again)
    flat = g.double().reshape(-1, H, Q, K)
    bucket = ref.bucket_of(m, nb, q, k).reshape(-1, Q, K)
    want, size = ref.bucket_sums(flat, bucket, nb), ref.bucket_sums(flat.abs(), bucket, nb)
    if dtype == torch.float64:
        assert ((dt.cpu() - want).abs() <= 16 * U[dtype] * size).all()
    else:
        near_sums(dt, want, size, torch.float32, dtype)


def test_relative_bias_extremes(dev):
    """Positions at the ends of int32 (the distance saturates), a map of one entry, one whose entries
    pass the table, int64 positions, broadcast leading dimensions, a misaligned cotangent."""
    table = torch.arange(12.0).reshape(6, 2)
    m = torch.tensor([0, 1, 2, 200, 4], dtype=torch.uint8)
    q = torch.tensor([[-(2**31), 0, 2**31 - 1, 5]])
    k = torch.tensor([[[2**31 - 1, 1, 6, -(2**31)]], [[4, 5, 6, 7]]])
    out = fx.relative_bias(table.to(dev), m.to(dev), q.to(dev), k.to(dev))
    assert out.shape == (2, 1, 2, 4, 4)
    assert torch.equal(out.double().cpu(), ref.relative_bias(table, m, q.expand(2, 1, 4), k))
    one = fx.relative_bias(table.to(dev), torch.tensor([3], dtype=torch.uint8, device=dev), q.to(dev), k.to(dev))
    assert torch.equal(one.cpu()[0, 0, 1], torch.full((4, 4), 7.0))
    t = table.to(dev).requires_grad_(True)
    out = fx.relative_bias(t, m.to(dev), q.to(dev), k.to(dev))
    g = torch.randn(out.numel() + 1, device=dev)[1:].view(out.shape)
    (dt,) = torch.autograd.grad(out, t, g)
    (want,) = torch.autograd.grad(fx.relative_bias(t, m.to(dev), q.to(dev), k.to(dev)), t, g.clone())
    # another order of the same few terms
    assert torch.allclose(dt, want, rtol=1e-6, atol=1e-6)
    for shape in ((0, 4), (4, 0)):
        t = table.to(dev).requires_grad_(True)
        z = [torch.zeros(n, dtype=torch.int32, device=dev) for n in shape]
        (dt,) = torch.autograd.grad(fx.relative_bias(t, m.to(dev), *z).sum(), t)
        assert torch.equal(dt.cpu(), torch.zeros(6, 2))


# ------------------------------------------------------------------ attention


def attention_case(gen, dtype, B, N, K, H, Hkv, D, nb=32, dist=128, mode=""):
    c = dict(q=rand(gen, B, N, H, D, dtype=dtype), k=rand(gen, B, K, Hkv, D, dtype=dtype), v=rand(gen, B, K, Hkv, D, dtype=dtype))
    if "n" not in mode:
        c["table"], c["buckets"] = rand(gen, nb, H), fx.distance_buckets(nb, dist, device="cpu")
    if "c" in mode:
        c.update(causal=True, offset=max(K - N, 0) if "o" in mode else 0)
    if "l" in mode:
        c["lengths"] = torch.randint(0, K + 2, (B,), generator=gen)
        c["lengths"][0] = 0
    if "L" in mode:
        c["q_lengths"] = torch.randint(0, N + 2, (B,), generator=gen)
    if "m" in mode:
        c["mask"] = torch.rand(B, K, generator=gen) < 0.6
        c["mask"][-1] = False
    if "p" in mode:
        c["q_pos"], c["k_pos"] = (torch.randint(-200, 200, (B, n), generator=gen) for n in (N, K))
    return c


def run_attention(c, dev, grad=None, leaves=("q", "k", "v", "table")):
    a = {n: gpu(x, dev) for n, x in c.items()}
    if grad is None:
        return fx.attention(**a)
    names = [n for n in leaves if n in a]
    for n in names:
        a[n].requires_grad_(True)
    out = fx.attention(**a)
    return (out.detach(), *torch.autograd.grad(out, [a[n] for n in names], grad.to(dev)))


def check_attention(c, dev, dtype, gen, what=""):
    B, N, H, D = c["q"].shape
    g = rand(gen, B, N, H, D, dtype=dtype)
    want = ref.attention(**c, grad=g)
    got = run_attention(c, dev, g)
    assert torch.equal(got[0], run_attention(c, dev))  # the value of a differentiated call
    again = run_attention(c, dev, g)
    for name, x, y, r in zip(("out", "dq", "dk", "dv"), got, want, (2, 2, 2, 2)):
        near(x, y, dtype, r, (what, name))
    assert all(torch.equal(x, y) for x, y in zip(got, again))
    if "table" in c:
        near_sums(got[4], want[4], want[5] + 1e-3 * want[5].mean(), dtype, what=(what, "dtable"), tol=EPS)


SHAPES = [
    # B, N, K, H, Hkv, D, mode
    (1, 1, 1, 1, 1, 1, ""), (2, 1, 5, 2, 1, 8, ""), (1, 12, 12, 4, 4, 16, ""), (2, 33, 33, 2, 2, 32, "c"), (1, 64, 64, 1, 1, 64, "n"),
    (2, 65, 63, 4, 2, 40, "l"), (1, 128, 128, 2, 2, 64, "c"), (2, 129, 200, 3, 1, 128, "co"), (2, 100, 130, 6, 2, 80, "lLp"),
    (2, 70, 300, 2, 2, 33, "mp"), (3, 130, 70, 4, 1, 7, "clm"), (1, 257, 257, 2, 1, 128, "cL"), (1, 300, 420, 2, 2, 96, "clmpo"),
    (2, 40, 600, 2, 1, 64, "n"), (1, 520, 520, 1, 1, 32, ""),
]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(str(x) for x in s))
def test_attention(dev, dtype, shape):
    gen = torch.Generator().manual_seed(sum(shape[:6]))
    check_attention(attention_case(gen, dtype, *shape[:6], mode=shape[6]), dev, dtype, gen, shape)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("shape", [(1, 1100, 1300, 2, 1, 64, "co"), (1, 1030, 1030, 1, 1, 128, "l"), (2, 90, 1500, 3, 3, 40, "mp"), (1, 1300, 70, 2, 1, 16, "")],
                         ids=lambda s: "-".join(str(x) for x in s))
def test_attention_long(dev, dtype, shape):
    """Many tiles, most of them past the radius as a whole; more queries than keys and the reverse."""
    gen = torch.Generator().manual_seed(sum(shape[:6]))
    check_attention(attention_case(gen, dtype, *shape[:6], mode=shape[6]), dev, dtype, gen, shape)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("nb,dist", [(4, 2), (64, 2048), (33, 17), (20, 100)])
def test_attention_buckets(dev, dtype, nb, dist):
    """The table's largest and smallest sizes, near and far tiles, with both kinds of positions."""
    gen = torch.Generator().manual_seed(nb)
    for mode in ("", "c", "p"):
        check_attention(attention_case(gen, dtype, 1, 200, 300, 2, 1, 128, nb, dist, mode), dev, dtype, gen, (nb, dist, mode))
    c = attention_case(gen, dtype, 1, 80, 90, 2, 2, 32, nb, dist)
    c["buckets"] = torch.randint(0, 256, (2 * dist + 1,), generator=gen).to(torch.uint8)  # any map, entries past the table
    check_attention(c, dev, dtype, gen, (nb, dist, "map"))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_attention_masked_places_hold_anything(dev, dtype):
    """Keys and values that lengths or mask hide, and queries past q_lengths, may be NaN or infinite: the
    results are those of zeros there, bit for bit, and finite."""
    gen = torch.Generator().manual_seed(7)
    for mode in ("lL", "mLp", "clmL"):
        c = attention_case(gen, dtype, 3, 70, 150, 4, 2, 64, mode=mode)
        g = rand(gen, 3, 70, 4, 64, dtype=dtype)
        hidden = torch.zeros(3, 150, dtype=torch.bool)
        if "lengths" in c:
            hidden |= torch.arange(150) >= c["lengths"][:, None]
        if "mask" in c:
            hidden |= ~c["mask"]
        past = torch.arange(70) >= c["q_lengths"][:, None]
        for n in "kv":
            c[n][hidden] = 0.0
        c["q"][past] = 0.0
        clean = run_attention(c, dev, g)
        bad = dict(c)
        for n, x in (("k", math.nan), ("v", math.inf)):
            bad[n] = c[n].clone()
            bad[n][hidden] = x
        bad["q"] = c["q"].clone()
        bad["q"][past] = -math.inf
        dirty = run_attention(bad, dev, g)
        assert all(torch.equal(x, y) and x.isfinite().all() for x, y in zip(clean, dirty))
        assert (clean[0][past.to(dev)] == 0).all() and (clean[1][past.to(dev)] == 0).all()
        assert (clean[2][hidden.to(dev)] == 0).all() and (clean[3][hidden.to(dev)] == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_attention_tables_that_forbid(dev, dtype):
    """-inf forbids a bucket (rows that it leaves empty give 0); the lowest float32 weighs like any
    other entry: alone in a row it cancels."""
    gen = torch.Generator().manual_seed(8)
    for low, mode in ((-math.inf, ""), (-math.inf, "p"), (torch.finfo(torch.float32).min, ""), (torch.finfo(torch.float32).min, "p")):
        c = attention_case(gen, dtype, 2, 90, 140, 2, 2, 64, 16, 20, mode)
        c["table"][:8] = low  # keys before the query, and itself
        if not mode:
            c.update(offset=100)  # the last queries see no key after them
        check_attention(c, dev, dtype, gen, (low, mode))


def test_attention_layouts(dev):
    """Strided, transposed and misaligned inputs, a fused projection's slices, a stream of its own: the
    packed call's results bit for bit."""
    gen = torch.Generator().manual_seed(9)
    B, N, H, D = 2, 100, 4, 64
    for dtype in TYPES:
        qkv = rand(gen, B, N, 3, H, D, dtype=dtype).to(dev)
        table, m = rand(gen, 32, H).to(dev), fx.distance_buckets(device=dev)
        g = rand(gen, B, N, H, D, dtype=dtype).to(dev)

        def run(q, k, v, g):
            q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
            out = fx.attention(q, k, v, table=table, buckets=m, causal=True)
            return (out.detach(), *torch.autograd.grad(out, (q, k, v), g))

        want = run(*(x.contiguous() for x in qkv.unbind(2)), g)
        heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in qkv.unbind(2)]
        odd = [torch.cat([x.new_zeros(1), x.flatten()])[1:].view(B, N, H, D) for x in qkv.unbind(2)]
        last = [x.transpose(2, 3).contiguous().transpose(2, 3) for x in qkv.unbind(2)]
        for inputs in (qkv.unbind(2), heads_first, odd, last):
            assert all(torch.equal(a, b) for a, b in zip(want, run(*inputs, g)))
        assert all(torch.equal(a, b) for a, b in zip(want, run(*qkv.unbind(2), g.transpose(1, 2).contiguous().transpose(1, 2))))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            other = run(*qkv.unbind(2), g)
        torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(a, b) for a, b in zip(want, other))


@pytest.mark.parametrize("N,K", [(0, 5), (5, 0), (0, 0)])
def test_attention_nothing(dev, N, K):
    gen = torch.Generator().manual_seed(1)
    c = attention_case(gen, torch.float32, 2, N, K, 2, 1, 16)
    got = run_attention(c, dev, torch.ones(2, N, 2, 16))
    for x in got:
        assert (x == 0).all()


def test_attention_differences(dev):
    """The gradient along directions against central differences of the 64-bit definition: the
    difference's own error is h^2, 1e-8 here, so float32's roundings decide."""
    gen = torch.Generator().manual_seed(11)
    c = attention_case(gen, torch.float32, 2, 40, 50, 4, 2, 24, 16, 30, "lmp")
    g = rand(gen, 2, 40, 4, 24)
    got = dict(zip(("q", "k", "v", "table"), run_attention(c, dev, g)[1:]))
    for n, d in got.items():
        step = torch.randn(d.shape, generator=gen, dtype=torch.float64)
        loss = lambda h: (ref.attention(**{**c, n: c[n].double() + h * step}) * g.double()).sum()
        want = (loss(1e-4) - loss(-1e-4)) / 2e-4
        have = (d.double().cpu() * step).sum()
        assert abs(have - want) <= 1e-5 * (d.double().cpu() * step).abs().sum(), (n, have, want)


def test_attention_some_gradients(dev):
    """Inputs that need no gradient, and a table that needs none, leave the others' as they are."""
    gen = torch.Generator().manual_seed(12)
    c = attention_case(gen, torch.bfloat16, 2, 80, 80, 2, 2, 64)
    g = rand(gen, 2, 80, 2, 64, dtype=torch.bfloat16)
    every = dict(zip(("out", "q", "k", "v", "table"), run_attention(c, dev, g)))
    for leaves in (("table",), ("q", "k"), ("v",)):
        got = run_attention({n: x.clone() for n, x in c.items()}, dev, g, leaves)
        assert all(torch.equal(every[n], x) for n, x in zip(("out",) + leaves, got))


# ------------------------------------------------------------------ one token


def step_case(gen, dtype, lengths, H, Hkv, D, page, M, nb=32, dist=128, extra=3):
    B = len(lengths)
    P = B * M + extra
    return dict(
        q=rand(gen, B, H, D, dtype=dtype), k_cache=rand(gen, P, page, Hkv, D, dtype=dtype), v_cache=rand(gen, P, page, Hkv, D, dtype=dtype),
        pages=torch.randperm(P, generator=gen)[: B * M].reshape(B, M).to(torch.int32), lengths=torch.tensor(lengths, dtype=torch.int32),
        k=rand(gen, B, Hkv, D, dtype=dtype), v=rand(gen, B, Hkv, D, dtype=dtype), table=rand(gen, nb, H), buckets=fx.distance_buckets(nb, dist, device="cpu"),
    )


def check_step(c, dev, dtype, what=""):
    a = {n: gpu(x, dev) if not n.endswith("cache") else x.to(dev).clone() for n, x in c.items()}
    got = fx.attention_step(**a)
    caches = c["k_cache"].clone(), c["v_cache"].clone()
    want = ref.attention_step(**{**c, "k_cache": caches[0], "v_cache": caches[1]})
    near(got, want, dtype, 2, what)
    for x, y in zip(caches, (a["k_cache"], a["v_cache"])):
        assert torch.equal(x.nan_to_num(7.0), y.cpu().nan_to_num(7.0)), what
    assert torch.equal(got.nan_to_num(7.0), fx.attention_step(**a).nan_to_num(7.0))
    return got


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("lengths,H,Hkv,D,page,M", [
    ([0], 1, 1, 1, 1, 1), ([0, 1, 2, 15, 16, 17, 30], 2, 2, 16, 16, 2), ([5, 0, 200, 99], 3, 1, 32, 7, 40), ([1000, 300, 64, 0], 8, 2, 64, 24, 42),
    ([700], 8, 1, 128, 64, 12), ([129, 511], 16, 1, 80, 100, 6), ([3, 77], 5, 5, 33, 8, 11), ([4000, 2500], 4, 2, 128, 16, 256), ([2047], 20, 1, 40, 1, 2100),
])
def test_step(dev, dtype, lengths, H, Hkv, D, page, M):
    gen = torch.Generator().manual_seed(H * D + page)
    c = step_case(gen, dtype, lengths, H, Hkv, D, page, M)
    check_step(c, dev, dtype, "append")
    check_step({**c, "k": None, "v": None}, dev, dtype, "read")
    check_step({**c, "table": None, "buckets": None, "scale": 0.3}, dev, dtype, "no bias")


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("B,H,Hkv,D", [(700, 6, 6, 32), (1100, 8, 4, 40), (2100, 6, 2, 64), (4200, 2, 1, 128)])
def test_step_many_units(dev, dtype, B, H, Hkv, D):
    """Enough samples and kv heads that each gets a wave of its own, in numbers that leave some waves spare."""
    gen = torch.Generator().manual_seed(B)
    lengths = torch.randint(-1, 60, (B,), generator=gen).tolist()
    c = step_case(gen, dtype, lengths, H, Hkv, D, 13, 5, 16, 12)
    c["pages"][7, 0] = -5
    check_step(c, dev, dtype)


def test_step_many_samples(dev):
    """More samples than a grid dimension holds, one token each of a small cache."""
    B = 66000
    gen = torch.Generator().manual_seed(2)
    q = rand(gen, B, 1, 16).to(dev)
    kc, vc = (torch.zeros(B, 1, 1, 16, device=dev) for _ in range(2))
    pages = torch.arange(B, dtype=torch.int32, device=dev)[:, None]
    k, v = rand(gen, B, 1, 16).to(dev), rand(gen, B, 1, 16).to(dev)
    out = fx.attention_step(q, kc, vc, pages, torch.zeros(B, dtype=torch.int32, device=dev), k=k, v=v)
    assert torch.equal(out, v) and torch.equal(kc[:, 0], k) and torch.equal(vc[:, 0], v)


def test_step_marks_the_caches_as_written(dev):
    """A graph that saved the caches before a token was appended refuses to go on with the new values."""
    k, v = (torch.randn(4, 8, 2, 32, device=dev) for _ in range(2))
    w = torch.ones((), device=dev, requires_grad=True)
    pages = torch.arange(2, dtype=torch.int32, device=dev)[:, None]
    lengths = torch.full((2,), 3, dtype=torch.int32, device=dev)
    q, new = torch.randn(2, 4, 32, device=dev), torch.randn(2, 2, 32, device=dev)
    for cache in (k, v):
        y = (cache * w).sum()
        with torch.no_grad():
            fx.attention_step(q, k, v, pages, lengths)  # only reads
        torch.autograd.grad(y, w)
        y = (cache * w).sum()
        with torch.no_grad():
            fx.attention_step(q, k, v, pages, lengths, k=new, v=new)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, w)


def test_step_refused_samples(dev):
    """Samples left out (0, nothing stored), past their pages and with a page outside the cache (NaN);
    the rest of the batch as ever. What lies past a sample's tokens may be NaN."""
    gen = torch.Generator().manual_seed(3)
    for dtype in TYPES:
        c = step_case(gen, dtype, [10, -1, 32, 5, 20, -(2**31), 2**31 - 1, 31], 4, 2, 64, 8, 4)
        c["pages"][3, 0] = -1
        c["pages"][4, 1] = c["k_cache"].shape[0]
        c["pages"][0, 2:] = 2**31 - 1  # not reached: 11 tokens
        for t in ("k_cache", "v_cache"):
            c[t][int(c["pages"][0, 1]), 3:] = math.nan
            c[t][int(c["pages"][7, 3]), 7:] = math.inf
        got = check_step(c, dev, dtype)
        assert (got[1] == 0).all() and (got[5] == 0).all()
        assert got[[2, 3, 4, 6]].isnan().all() and got[[0, 7]].isfinite().all()
        c = step_case(gen, dtype, [3], 2, 2, 64, 8, 1)
        c.update(k_cache=torch.zeros(0, 8, 2, 64, dtype=dtype), v_cache=torch.zeros(0, 8, 2, 64, dtype=dtype))
        assert check_step(c, dev, dtype).isnan().all()


def test_step_shared_pages(dev):
    """Two walkers that branched share their first pages."""
    gen = torch.Generator().manual_seed(4)
    c = step_case(gen, torch.float32, [40, 45], 4, 4, 32, 16, 3)
    c["pages"][1, :2] = c["pages"][0, :2]
    check_step(c, dev, torch.float32)


def test_step_forbidding_table(dev):
    gen = torch.Generator().manual_seed(5)
    for low in (-math.inf, torch.finfo(torch.float32).min):
        for dtype in TYPES:
            c = step_case(gen, dtype, [0, 3, 300], 4, 2, 64, 16, 19, 16, 20)
            c["table"][:] = low
            check_step(c, dev, dtype, low)
            c["table"][3] = 0.5
            check_step(c, dev, dtype, low)


def test_step_long_offsets(dev):
    """Pages past 2^31 elements of a cache, in both kernels: what the same pages give in a small one."""
    gen = torch.Generator().manual_seed(9)
    for H in (8, 16):
        c = step_case(gen, torch.bfloat16, [150, 190], H, 8, 128, 64, 3, extra=0)
        a = {n: gpu(x, dev) for n, x in c.items()}
        want = fx.attention_step(**a)
        pages = 2**31 // (64 * 8 * 128) + 10
        far = torch.arange(pages - 6, pages, device=dev)
        big = dict(a, pages=(a["pages"] + pages - 6).to(torch.int32))
        for n in ("k_cache", "v_cache"):
            big[n] = torch.empty(pages, 64, 8, 128, dtype=torch.bfloat16, device=dev)
            big[n][far] = c[n].to(dev)
        assert torch.equal(fx.attention_step(**big), want)
        for n in ("k_cache", "v_cache"):
            assert torch.equal(big[n][far], a[n])
        del big


def test_attention_long_offsets(dev):
    """A batch stride past 2^31 elements."""
    gen = torch.Generator().manual_seed(10)
    for dtype in (torch.bfloat16, torch.float32):
        c = attention_case(gen, dtype, 2, 70, 150, 2, 1, 64)
        a = {n: gpu(x, dev) for n, x in c.items()}
        want = fx.attention(**a)
        room = torch.empty(2**31 + 2**16, dtype=dtype, device=dev)
        for n in "kv":
            spread = room.as_strided((2, 150, 1, 64), (2**31 - 64, 64, 64, 1))
            spread.copy_(a[n])
            assert torch.equal(fx.attention(**{**a, n: spread}), want)
        del room, spread


def test_step_in_a_graph(dev):
    """A captured step, replayed while the sequence grows: every replay gives what an eager call gives."""
    gen = torch.Generator().manual_seed(11)
    for dtype, H in ((torch.bfloat16, 8), (torch.float32, 4)):
        c = step_case(gen, dtype, [700, 0, 64], H, 2, 64, 16, 64)
        a = {n: gpu(x, dev) for n, x in c.items()}
        eager = {n: x.clone() for n, x in a.items()}
        fx.attention_step(**{n: x.clone() for n, x in a.items()})
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fx.attention_step(**a)
        for turn in range(4):
            for n in ("q", "k", "v"):
                new = rand(gen, *a[n].shape, dtype=dtype).to(dev)
                a[n].copy_(new)
                eager[n].copy_(new)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, fx.attention_step(**eager)), turn
            assert torch.equal(a["k_cache"], eager["k_cache"]) and torch.equal(a["v_cache"], eager["v_cache"])
            a["lengths"] += 1
            eager["lengths"] += 1


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_step_follows_attention(dev, dtype):
    """A sequence token by token gives what attention gives it as a whole, to the roundings of both."""
    gen = torch.Generator().manual_seed(6)
    B, N, H, Hkv, D, page = 3, 37, 4, 2, 32, 8
    c = attention_case(gen, dtype, B, N, N, H, Hkv, D, 16, 12, "c")
    whole = ref.attention(**c)
    a = {n: gpu(x, dev) for n, x in c.items()}
    M = -(-N // page)
    kc, vc = (torch.full((B * M, page, Hkv, D), math.nan, dtype=dtype, device=dev) for _ in range(2))
    pages = torch.randperm(B * M, generator=gen).reshape(B, M).to(torch.int32).to(dev)
    outs = []
    for t in range(N):
        lengths = torch.full((B,), t, dtype=torch.int32, device=dev)
        outs.append(fx.attention_step(a["q"][:, t], kc, vc, pages, lengths, k=a["k"][:, t], v=a["v"][:, t], table=a["table"], buckets=a["buckets"]))
    near(torch.stack(outs, 1), whole, dtype, 2)


# ------------------------------------------------------------------ residual norm

GATES = {"none": lambda s: None, "scalar": lambda s: (1,) * len(s), "channel": lambda s: s[-1:], "token": lambda s: s[:-1] + (1,),
         "sample": lambda s: s[:-2] + (1, s[-1]), "sample_scalar": lambda s: s[:-2] + (1, 1), "full": lambda s: s,
         "position": lambda s: s[-2:], "position_scalar": lambda s: (s[-2], 1)}


def norm_case(gen, dtype, shape, gate="none", columns="wbspq", wide=True):
    C = shape[-1]
    wt = torch.float32 if wide else dtype
    c = dict(x=rand(gen, *shape, dtype=dtype), h=rand(gen, *shape, dtype=dtype, scale=2.0))
    for key, name in zip("wbspq", ("post_weight", "post_bias", "scale", "pre_weight", "pre_bias")):
        if key in columns:
            c[name] = (0.5 + rand(gen, C, dtype=torch.float64, scale=0.3)).to(wt)
    s = GATES[gate](tuple(shape))
    if s is not None:
        c["gate"] = rand(gen, *s, dtype=dtype)
    return c


def check_norm(c, dev, dtype, gen, what="", cotangents=(True, True), **kw):
    shape = c["x"].shape
    both = kw.get("pre_norm", True)
    grads = tuple(rand(gen, *shape, dtype=dtype) if on else None for on in cotangents)
    y, z, want = ref.residual_norm(**c, **kw, grads=grads)
    a = {n: gpu(x, dev) for n, x in c.items()}
    plain = fx.residual_norm(**a, **kw)
    leaves = [n for n in a if isinstance(a[n], torch.Tensor)]
    for n in leaves:
        a[n].requires_grad_(True)

    def run():
        out = fx.residual_norm(**a, **kw)
        out = out if both else (out,)
        used = [(o, g.to(dev)) for o, g in zip(out, grads) if g is not None]
        return out, torch.autograd.grad([o for o, _ in used], [a[n] for n in leaves], [g for _, g in used])

    out, got = run()
    for o, p, w in zip(out, plain if both else (plain,), (y, z)):
        near(o, w, dtype, 1, what)
        assert torch.equal(o, p)
    for n, g in zip(leaves, got):
        if n in ("x", "h") or (n == "gate" and c["gate"].shape == shape):
            near(g, want[n], dtype, 1, (what, n), want["size_" + n])
        else:
            near_sums(g, want[n], want["size_" + n], dtype, c[n].dtype, (what, n))
    assert all(torch.equal(x, y) for x, y in zip(got, run()[1]))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (2, 7, 64), (5, 3, 100), (2, 300, 256), (1, 9, 333), (4, 33, 512), (2, 2, 5, 1000), (3, 2048), (70, 4, 24), (2, 3, 5000), (2, 8192)],
                         ids=lambda s: "x".join(map(str, s)))
def test_norm(dev, dtype, norm, shape):
    gen = torch.Generator().manual_seed(sum(shape))
    check_norm(norm_case(gen, dtype, shape), dev, dtype, gen, norm=norm)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("shape", [(4, 40, 96), (3, 2, 7, 33), (2000, 2, 16), (1, 1, 40), (2, 600, 128)], ids=lambda s: "x".join(map(str, s)))
def test_norm_gates(dev, dtype, gate, shape):
    gen = torch.Generator().manual_seed(sum(shape))
    check_norm(norm_case(gen, dtype, shape, gate, wide=False), dev, dtype, gen, gate, norm="layer")
    check_norm(norm_case(gen, dtype, shape, gate, "sp"), dev, dtype, gen, gate)


def test_norm_options(dev):
    gen = torch.Generator().manual_seed(3)
    for dtype in TYPES:
        shape = (3, 20, 136)
        check_norm(norm_case(gen, dtype, shape, "full", ""), dev, dtype, gen, "bare")
        check_norm(norm_case(gen, dtype, shape, "sample", "spq"), dev, dtype, gen, "no post", post_norm=False)
        check_norm(norm_case(gen, dtype, shape, "sample", "wbs"), dev, dtype, gen, "no pre", cotangents=(True, False), pre_norm=False)
        check_norm(norm_case(gen, dtype, shape, "token"), dev, dtype, gen, "dy", cotangents=(True, False), norm="layer")
        check_norm(norm_case(gen, dtype, shape, "token"), dev, dtype, gen, "dz", cotangents=(False, True), norm="layer")
        c = norm_case(gen, dtype, shape, "full")
        a = {n: gpu(x, dev) for n, x in c.items()}
        y, z = fx.residual_norm(**{**a, "scale": 0.25}, eps=1e-3)
        wy, wz = ref.residual_norm(**{**c, "scale": 0.25}, eps=1e-3)
        near(y, wy, dtype)
        near(z, wz, dtype)


def test_norm_layouts_and_mean(dev):
    """Strided and misaligned inputs, another stream; a layer norm whose mean is a thousand deviations keeps
    its digits (the deviation is summed from the centred row)."""
    gen = torch.Generator().manual_seed(4)
    for dtype in TYPES:
        c = norm_case(gen, dtype, (4, 50, 72), "sample")
        a = {n: gpu(x, dev) for n, x in c.items()}
        want = fx.residual_norm(**a)
        b = dict(a)
        b["x"] = a["x"].transpose(0, 1).contiguous().transpose(0, 1)
        b["h"] = torch.cat([a["h"], a["h"]], -1)[..., :72]
        assert all(torch.equal(x, y) for x, y in zip(want, fx.residual_norm(**b)))
        odd = dict(a)
        odd["x"] = torch.cat([a["x"].new_zeros(1), a["x"].flatten()])[1:].view(4, 50, 72)
        for x, y in zip(want, fx.residual_norm(**odd)):
            near(x, y.cpu(), dtype)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            other = fx.residual_norm(**a)
        torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(x, y) for x, y in zip(want, other))
    x = torch.zeros(2, 3, 512)
    h = (1000 + rand(gen, 2, 3, 512, dtype=torch.float64)).float()
    y, z = fx.residual_norm(x.to(dev), h.to(dev), norm="layer")
    wy, wz = ref.residual_norm(x, h, norm="layer")
    # the mean itself is rounded to 2^-24 of a thousand, half of 1e-4 of a deviation
    assert (y.double().cpu() - wy).abs().max() < 1e-4 and (z.double().cpu() - wz).abs().max() < 1e-4


def test_norm_differences(dev):
    gen = torch.Generator().manual_seed(5)
    c = norm_case(gen, torch.float32, (3, 6, 40), "sample")
    dy, dz = rand(gen, 3, 6, 40), rand(gen, 3, 6, 40)
    for norm in ("rms", "layer"):
        a = {n: gpu(x, dev).requires_grad_(True) for n, x in c.items()}
        grads = torch.autograd.grad(fx.residual_norm(**a, norm=norm), list(a.values()), (dy.to(dev), dz.to(dev)))
        for n, d in zip(a, grads):
            step = torch.randn(d.shape, generator=gen, dtype=torch.float64)

            def loss(h):
                y, z = ref.residual_norm(**{**c, n: c[n].double() + h * step}, norm=norm)
                return (y * dy).sum() + (z * dz).sum()

            want = (loss(1e-4) - loss(-1e-4)) / 2e-4
            have = (d.double().cpu() * step).sum()
            assert abs(have - want) <= 1e-5 * (d.double().cpu() * step).abs().sum(), (norm, n)


def test_norm_nothing(dev):
    for shape in ((0, 5, 16), (5, 0, 16), (0, 16)):
        x, h = (torch.zeros(shape, device=dev, requires_grad=True) for _ in range(2))
        w = torch.ones(16, device=dev, requires_grad=True)
        y, z = fx.residual_norm(x, h, post_weight=w)
        grads = torch.autograd.grad((y, z), (x, h, w), (torch.zeros_like(y), torch.zeros_like(z)))
        assert y.shape == z.shape == shape and (grads[2] == 0).all()


# ------------------------------------------------------------------ all of them


def test_transforms_are_refused(dev):
    x = torch.randn(2, 3, 16, device=dev)
    with pytest.raises(RuntimeError):
        torch.func.vmap(torch.func.grad(lambda t: fx.residual_norm(t, t)[0].sum()))(x)
