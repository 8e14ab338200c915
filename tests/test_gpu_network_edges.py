"""The operators of fermix_amd.network on the GPU where a size, a scale or an input goes to its end:
nothing to work on, the largest offsets, more work than one launch or one pass of a workgroup
holds, cotangents and weights that are small for float16. Oracle and tolerances: those of
test_gpu_network.py, unless a test derives its own."""

import math

import pytest
import torch

import fermix_amd as fx
from tests.test_gpu_network import GATES, TYPES, attention_case, check_attention, ids

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
