"""The operators of fermix_amd.network on the GPU where a size, a scale or an input goes to its end:
nothing to work on, the largest offsets, more work than one launch or one pass of a workgroup
holds, cotangents and weights that are small for float16. Oracle and tolerances: those of
test_gpu_network.py, unless a test derives its own."""

import math

import pytest
import torch

import fermix_amd as fx
from tests import network64 as ref
from tests.test_gpu_network import GATES, TYPES, U, attention_case, check_attention, check_norm, ids, near_sums, norm_case, rand

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ nothing to work on


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("shape", [(0, 5, 16), (5, 0, 16), (0, 1, 16), (0, 16), (3, 0, 2, 16), (0, 5, 300)], ids=lambda s: "x".join(map(str, s)))
def test_norm_gate_without_rows(dev, dtype, gate, shape):
    """Without rows every gradient is zero, a broadcast gate's too, which has elements all the same; the
    allocator's memory is filled with NaN beforehand, so that a result that nobody writes shows."""
    s = GATES[gate](shape)
    if s is None or math.prod(torch.Size(s)) == 0:
        pytest.skip("no gate, or one without elements")
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
