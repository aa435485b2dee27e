"""The recurrent model of examples/: its gradients against torch's automatic ones, its steps
from token to token against the whole, and that it runs."""
import math
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))


def _reference(p, tokens, d, blocks, bounds):
    """The model in float64 with torch's automatic gradients."""
    import torch

    def norm(t, w):
        return t * torch.rsqrt((t * t).mean(1, keepdim=True) + 1e-5) * w

    total = p["table"][tokens] * math.sqrt(d)
    n = norm(total, p["weight0"])
    for i in range(blocks):
        gate, x, opened = (n @ p[f"mix{i}"]).split(d, 1)
        a = torch.sigmoid(gate)
        rows = []
        for begin, end in zip(bounds, bounds[1:]):
            h = torch.zeros(d, dtype=torch.float64)
            for t in range(begin, end):
                h = a[t] * h + (1 - a[t]) * x[t]
                rows.append(h)
        y = norm(torch.stack(rows), p[f"inner{i}"]) * torch.nn.functional.silu(opened)
        total = total + y
        n = norm(total, p[f"weight{i + 1}"])
    return n @ p["head"]


def _batch(torch, vocabulary, positions):
    g = torch.Generator(device="cuda").manual_seed(3)
    tokens = torch.randint(0, vocabulary, (positions,), generator=g, device="cuda")
    targets = torch.randint(0, vocabulary, (positions,), generator=g, device="cuda")
    return tokens, targets


def test_gradients_of_a_step_are_torchs():
    import recurrent_model
    import torch
    vocabulary, d, blocks, positions = 37, 48, 2, 150
    bounds = [0, 1, 60, 60, 149, 150]
    model = recurrent_model.RecurrentModel(vocabulary, d, blocks, positions, activations=torch.float32,
                                           max_norm=0.05)
    tokens, targets = _batch(torch, vocabulary, positions)
    p = {k: v.double().cpu().requires_grad_() for k, v in model.parameters.items()}
    logits = _reference(p, tokens.cpu(), d, blocks, bounds)
    loss = torch.nn.functional.cross_entropy(logits, targets.cpu())
    loss.backward()
    norm = math.sqrt(sum(float((t.grad ** 2).sum()) for t in p.values()))
    assert norm > 0.05
    offsets = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    before = {k: v.clone() for k, v in model.parameters.items()}
    got = model.step(tokens, targets, len(bounds) - 1, offsets)
    # float32 throughout: some hundred roundings of 6e-8 of the largest terms
    assert abs(float(got) - float(loss.detach())) < 1e-4
    assert abs(float(model.norm) - norm) < 1e-4 * norm
    for name, t in p.items():
        off = (model.gradients[name].double().cpu() - t.grad).abs().max()
        assert float(off) < 1e-4 * float(t.grad.abs().max()), name
    # The first step of AdamW moves every parameter by the rate, against the sign of its clipped
    # gradient, of those that are not next to nothing against epsilon.
    for name, t in p.items():
        g = t.grad * (0.05 / norm)
        far = g.abs() > 1e-5
        moved = (model.parameters[name] - before[name]).double().cpu()
        want = -model.rate * (g / (g.abs() + 1e-8) + 0.01 * before[name].double().cpu())
        assert float((moved - want)[far].abs().max()) < 1e-4 * model.rate + 4e-7, name
        assert torch.equal(model.copies[name], model.parameters[name])


def test_steps_from_token_to_token_are_the_whole():
    import recurrent_model
    import torch
    model = recurrent_model.RecurrentModel(50, 72, 2, 90, activations=torch.float32)
    tokens, _ = _batch(torch, 50, 90)
    whole = model.forward(tokens, sequences=3).clone()
    states = [torch.zeros(3, 72, device="cuda") for _ in range(2)]
    # twenty tokens of each sequence at once, then one by one
    parts = tokens.view(3, 30)
    first = model.forward(parts[:, :20].reshape(-1), sequences=3, states=states).view(3, 20, -1)
    logits = [first.clone()]
    for t in range(20, 30):
        logits.append(model.forward(parts[:, t].contiguous(), sequences=3, states=states)[:, None].clone())
    got = torch.cat(logits, 1).view(90, -1)
    # (float32; the products of torch may add up in another order for another number of rows)
    assert float((got - whole).abs().max()) < 1e-4 * float(whole.abs().max())


@pytest.mark.parametrize("eight_bits", [False, True])
def test_the_example_runs(eight_bits):
    import recurrent_model
    losses = recurrent_model.main(steps=3, vocabulary=50, dimension=72, blocks=2, positions=500,
                                  eight_bits=eight_bits)
    assert all(math.isfinite(x) for x in losses)


def test_a_step_is_captured_and_counts_on():
    # The step's number is on the device: replays are further steps, as eager ones are.
    import recurrent_model
    import torch
    tokens, targets = _batch(torch, 50, 400)
    offsets = torch.tensor([0, 100, 399, 400], dtype=torch.int32, device="cuda")
    models = [recurrent_model.RecurrentModel(50, 64, 1, 400, eight_bits=True) for _ in range(2)]
    for model in models:
        for _ in range(2):
            model.step(tokens, targets, 3, offsets)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        models[1].step(tokens, targets, 3, offsets)
    for _ in range(3):
        models[0].step(tokens, targets, 3, offsets)
        graph.replay()
        torch.cuda.synchronize()
        for name in models[0].parameters:
            a, b = (m.parameters[name] for m in models)
            # (torch's products may be others in a graph: a rounding of 16 bits in an activation)
            assert float((a - b).abs().max()) <= 0.1 * models[0].rate, name
    assert int(models[1].steps) == int(models[0].steps) == 5
