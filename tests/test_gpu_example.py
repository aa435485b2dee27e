"""The token model of examples/: its gradients against torch's automatic ones, and
that it learns."""
import math
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))


def test_gradients_of_a_step_are_torchs():
    import token_model
    import torch
    vocabulary, dimension, positions = 37, 48, 300
    model = token_model.TokenModel(vocabulary, dimension, positions, max_norm=0.05)
    g = torch.Generator(device="cuda").manual_seed(3)
    tokens = torch.randint(0, vocabulary, (positions,), generator=g, device="cuda")
    targets = torch.randint(0, vocabulary, (positions,), generator=g, device="cuda")
    p = {k: v.double().cpu().requires_grad_() for k, v in model.parameters.items()}
    x = p["table"][tokens.cpu()] * math.sqrt(dimension)
    v, m = torch.var_mean(x, 1, unbiased=False, keepdim=True)
    logits = ((x - m) / (v + 1e-5).sqrt() * p["weight"] + p["bias"]) @ p["head"]
    loss = torch.nn.functional.cross_entropy(logits, targets.cpu())
    loss.backward()
    norm = math.sqrt(sum(float((t.grad ** 2).sum()) for t in p.values()))
    assert norm > 0.05
    got = model.step(tokens, targets, rate=0.0)
    # float32 throughout: some hundred roundings of 6e-8 of the largest terms
    assert abs(float(got) - float(loss)) < 1e-4
    assert abs(float(model.norm) - norm) < 1e-4 * norm
    for name, t in p.items():
        exact = t.grad * (0.05 / norm)
        off = (model.gradients[name].double().cpu() - exact).abs().max()
        assert float(off) < 1e-4 * float(exact.abs().max()), name


@pytest.mark.parametrize("activations", ["float32", "bfloat16"])
def test_the_model_learns(activations):
    import token_model
    import torch
    losses = token_model.main(steps=41, vocabulary=128, dimension=128, positions=2048,
                              activations=getattr(torch, activations))
    assert losses[0] > 4.0 and losses[-1] < 0.7 * losses[0]


def test_a_step_over_fewer_positions_than_the_model_was_made_for():
    # The scratch was taken for 4096 positions; a last batch is a little shorter.
    import token_model
    import torch
    model = token_model.TokenModel(300, 2048, 4096)
    tokens = torch.arange(4097, device="cuda") * 7 % 300
    for n in (4096, 4064, 100, 1):
        loss = model.step(tokens[:n], tokens[1:n + 1], rate=0.01)
        assert math.isfinite(float(loss)) and math.isfinite(float(model.norm))
