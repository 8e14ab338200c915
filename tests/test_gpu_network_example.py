"""examples/network.py: the operators together, in training and in sampling."""

import copy
import os
import sys
import types

import pytest
import torch

from tests import network64 as ref

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def test_network_example(dev):
    import network

    fit, nll, off = network.main(sites=24, electrons=10, batch=64, steps=25)
    assert fit[-1] < fit[0] and nll[-1] < nll[0]
    # 24 log probabilities of magnitude about 1, float32 throughout: some 1e-6 each
    assert off < 1e-3


def test_network_example_gradient(dev, monkeypatch):
    """log|psi| of the pairing function and its gradient through every operator against the same model in 64 bits
    with the operators' definitions. Only samples whose pairing matrix has a condition number below 100: it
    multiplies float32's roundings, some 1e-6 through the layers, to 1e-4 at most."""
    import network

    torch.manual_seed(1)
    where = torch.rand(64, 24).argsort(1)[:, :10].sort(1).values
    model = network.Pairing(24)
    double = copy.deepcopy(model).double()
    on_gpu = model.to(dev)
    double.buckets = double.buckets.cpu()
    matrices = []

    def slogpf(a):
        s = (a - a.transpose(1, 2)) / 2
        matrices.append(s)
        sign, logabs = torch.linalg.slogdet(s)
        return sign, logabs / 2

    names = dict(attention=ref.attention, relative_bias=ref.relative_bias, residual_norm=ref.residual_norm, slogpf=slogpf)
    with monkeypatch.context() as m:
        m.setattr(network, "fx", types.SimpleNamespace(**names))
        want = double(where)[1]
    good = torch.linalg.cond(matrices[0].detach()) < 100
    assert good.sum() >= 32
    weight = torch.where(good, torch.randn(64, dtype=torch.float64), 0.0)
    want_grads = torch.autograd.grad((want * weight).sum(), list(double.parameters()))
    got = on_gpu(where.to(dev))[1]
    assert ((got.double().cpu() - want)[good].abs() < 1e-4).all()
    grads = torch.autograd.grad((got * weight.float().to(dev)).sum(), list(on_gpu.parameters()))
    for (name, _), g, w in zip(on_gpu.named_parameters(), grads, want_grads):
        assert (g.double().cpu() - w).norm() <= 1e-3 * w.norm(), name
