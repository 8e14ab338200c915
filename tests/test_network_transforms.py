"""What fermix_amd.network's operators cannot do under a transform they refuse, each of them and for each of its
differentiable inputs, before anything is launched (so these run without a GPU)."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import fermix_amd as fx


def _calls():
    """name -> (function of its differentiable inputs, those inputs)"""
    m, p = fx.distance_buckets(device="cpu"), torch.arange(4, dtype=torch.int32)
    r = torch.randn
    heads, cache = lambda: r(2, 4, 2, 8), lambda: r(3, 4, 2, 8)
    pages, lengths = torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    return {
        "relative_bias": (lambda t: fx.relative_bias(t, m, p, p), [r(32, 2)]),
        "attention": (lambda q, k, v, t: fx.attention(q, k, v, table=t, buckets=m), [heads(), heads(), heads(), r(32, 2)]),
        "attention_step": (
            lambda q, kc, vc, k, v, t: fx.attention_step(q, kc, vc, pages, lengths, k=k, v=v, table=t, buckets=m),
            [r(2, 2, 8), cache(), cache(), r(2, 2, 8), r(2, 2, 8), r(32, 2)],
        ),
        "residual_norm": (
            lambda x, h, g, s, w1, b1, w2, b2: fx.residual_norm(
                x, h, gate=g, scale=s, post_weight=w1, post_bias=b1, pre_weight=w2, pre_bias=b2, norm="layer"),
            [r(3, 8), r(3, 8), r(3, 1)] + [r(8) for _ in range(5)],
        ),
    }


@pytest.mark.parametrize("name", _calls())
def test_forward_mode_is_refused(name):
    """A dual tensor raises, whichever input it is and whether autograd is on; the same call without one goes on
    to the next refusal (no GPU here)."""
    f, inputs = _calls()[name]
    with fwAD.dual_level():
        for i, x in enumerate(inputs):
            args = [fwAD.make_dual(y, torch.ones_like(y)) if j == i else y for j, y in enumerate(inputs)]
            with pytest.raises(NotImplementedError, match="forward mode"):
                f(*args)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward mode"):
                f(*args)
        with pytest.raises(fx.FermixDeviceError):
            f(*inputs)
