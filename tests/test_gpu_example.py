"""examples/train_step.py runs all operators together: the loss falls well below a uniform guess, and V stays orthonormal"""
import importlib.util
import math
import os

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


def load():
    spec = importlib.util.spec_from_file_location("train_step", os.path.join(ROOT, "examples", "train_step.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_loss_falls(cuda):
    m = load()
    losses = m.train(steps=40, tokens=1024, vocab=500)
    assert all(math.isfinite(v) for v in losses)
    assert losses[-1] < 0.5 * math.log(500) < losses[0]


def test_layers_stay_orthonormal(cuda):
    m = load()
    model = m.Model(vocab=300, width=128, rank=32, layers=3)
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randint(0, 300, (257,), generator=g, device="cuda")
    for _ in range(3):
        loss, norm = m.step(model, x, (x * 7 + 1) % 300)
    assert math.isfinite(float(loss)) and float(norm) > 0.0
    for V, U, W in zip(model.V, model.U, model.W):
        # orth's own bound
        assert float((V.double().T @ V.double() - torch.eye(32, device=cuda, dtype=torch.float64)).abs().max()) <= 2e-7
        assert torch.equal(W, (U @ V.T).bfloat16())
