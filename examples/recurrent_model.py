"""A recurrent next-token model trained with the library's operators: embedding lookup,
blocks of a gated recurrence with the norms, the gate and the residual stream around it, their
gradients, the norm of all gradients and the AdamW step that clips by it.

    total, n = scale * table[token], norm(total)
    in every block:   gate, x, open = n @ mix
                      h = gated_recurrence(gate, x)
                      total = total + norm(h) * silu(open);  n = norm(total)
    logits = n @ head

The matrix products and the softmax are torch's; everything else is the library's, on torch's
current stream and without a synchronisation.  The AdamW step counts and clips on the device.
``python examples/recurrent_model.py`` trains on packed sequences of many lengths, with moments in
32 or (``--8bit``) in 8 bits, then continues sequences token by token from their states.
"""
from __future__ import annotations

import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from ilgpu_amd import capi  # noqa: E402

array, matrix = capi.DeviceArray.from_tensor, capi.DeviceMatrix.from_tensor


class RecurrentModel:
    """Parameters in float32; activations, their gradients and the parameters' copies that the
    products read in ``activations``."""

    def __init__(self, vocabulary: int, dimension: int, blocks: int, positions: int, *,
                 activations=torch.bfloat16, eight_bits: bool = False, rate: float = 1e-2,
                 max_norm: float = 1.0, seed: int = 1):
        g = torch.Generator(device="cuda").manual_seed(seed)
        d = dimension

        def normal(*shape, spread):
            return spread * torch.randn(*shape, generator=g, device="cuda")

        self.dimension, self.blocks, self.scale = d, blocks, math.sqrt(d)
        self.rate, self.max_norm = rate, max_norm
        p = {"table": normal(vocabulary, d, spread=d ** -0.5), "weight0": torch.ones(d, device="cuda"),
             "head": normal(d, vocabulary, spread=d ** -0.5)}
        for i in range(blocks):
            p[f"mix{i}"] = normal(d, 3 * d, spread=d ** -0.5)
            p[f"inner{i}"] = torch.ones(d, device="cuda")
            p[f"weight{i + 1}"] = torch.ones(d, device="cuda")
        self.parameters = p
        self.gradients = {k: torch.empty_like(v) for k, v in p.items()}
        self.copies = {k: v.to(activations) for k, v in p.items()}

        # The optimiser's state and the views of it, which every step uses again.
        def lists(tensors):
            return capi.TensorList([array(t) for t in tensors])

        sizes = [v.numel() for v in p.values()]
        kind = torch.uint8 if eight_bits else torch.float32
        moments = [[torch.zeros(n, dtype=kind, device="cuda") for n in sizes] for _ in range(2)]
        scales = [[torch.zeros(-(-n // capi.ADAMW_MOMENT_BLOCK), device="cuda") for n in sizes]
                  for _ in range(2)]
        self.moments = moments, scales
        self.lists = (lists(p.values()), lists(self.gradients.values()), lists(moments[0]),
                      lists(moments[1]))
        self.options = {"copies": lists(self.copies.values())}
        if eight_bits:
            self.options.update(first_scales=lists(scales[0]), second_scales=lists(scales[1]))
        self.norm = torch.empty(1, device="cuda")
        self.steps = torch.zeros(1, dtype=torch.int64, device="cuda")

        # Activations that the gradients need, and scratch.
        def empty(*shape, dtype=activations):
            return torch.empty(*shape, dtype=dtype, device="cuda")

        self.totals = [empty(positions, d) for _ in range(blocks + 1)]
        self.normed = [empty(positions, d) for _ in range(blocks + 1)]
        self.rstd = [empty(positions, dtype=torch.float32) for _ in range(blocks + 1)]
        self.inner_rstd = [empty(positions, dtype=torch.float32) for _ in range(blocks)]
        self.mixed = [empty(positions, 3 * d) for _ in range(blocks)]
        self.hidden = [empty(positions, d) for _ in range(blocks)]
        self.grads = [empty(positions, d) for _ in range(2)]
        self.grad_mixed = empty(positions, 3 * d)
        self.temps = [capi.temp_buffer(max(4, n)) for n in (
            capi.gated_recurrence_temp_bytes(positions, d),
            capi.residual_norm_gradient_temp_bytes(positions, d),
            capi.embedding_gradient_temp_bytes(positions, vocabulary, d),
            capi.gradient_norm_temp_bytes(len(p)))]

    def forward(self, tokens: torch.Tensor, sequences: int = 1, offsets=None,
                states=None) -> torch.Tensor:
        """Logits of the tokens that follow, of sequences packed behind one another (equal parts, or
        cut at offsets).  states: one float32 matrix (sequences x dimension) for each block, where
        the sequences begin and where they are left."""
        d, n, p, c = self.dimension, tokens.numel(), self.parameters, self.copies
        packed = {"sequences": sequences, "offsets": None if offsets is None else array(offsets)}
        total, normed = matrix(self.totals[0][:n]), matrix(self.normed[0][:n])
        capi.embedding(matrix(p["table"]), array(tokens), total, scale=self.scale)
        capi.residual_norm(total, None, None, normed, array(p["weight0"]), rstd=array(self.rstd[0]))
        for i in range(self.blocks):
            torch.matmul(self.normed[i][:n], c[f"mix{i}"], out=self.mixed[i][:n])
            gate, x, opened = (matrix(t) for t in self.mixed[i][:n].split(d, 1))
            hidden = matrix(self.hidden[i][:n])
            state = None if states is None else matrix(states[i])
            capi.gated_recurrence(gate, x, hidden, self.temps[0], initial=state, final=state,
                                  complement=True, **packed)
            after, normed = matrix(self.totals[i + 1][:n]), matrix(self.normed[i + 1][:n])
            capi.residual_norm(hidden, total, after, normed, array(p[f"weight{i + 1}"]), gate=opened,
                               gate_kind=capi.GATE_SILU, input_weight=array(p[f"inner{i}"]),
                               input_rstd=array(self.inner_rstd[i]), rstd=array(self.rstd[i + 1]))
            total = after
        return self.normed[self.blocks][:n] @ c["head"]

    def backward(self, tokens: torch.Tensor, grad_logits: torch.Tensor, sequences: int = 1,
                 offsets=None) -> None:
        """The gradients of all parameters from that of the logits, of sequences that began with
        states of zeros; the norm of them all goes to ``norm``."""
        d, n, p, c, g = self.dimension, tokens.numel(), self.parameters, self.copies, self.gradients
        packed = {"sequences": sequences, "offsets": None if offsets is None else array(offsets)}
        g["head"].copy_(self.normed[self.blocks][:n].t() @ grad_logits)
        grad_normed = grad_logits @ c["head"].t()
        grad_total, spare = None, [matrix(t[:n]) for t in self.grads]
        mixed = [matrix(t) for t in self.grad_mixed[:n].split(d, 1)]
        for i in reversed(range(self.blocks)):
            gate, x, opened = (matrix(t) for t in self.mixed[i][:n].split(d, 1))
            hidden, out = matrix(self.hidden[i][:n]), matrix(grad_normed)
            # (The gradient of the stream takes its own place, that of the state the output's.)
            capi.residual_norm_gradient(
                out, grad_total, hidden, matrix(self.totals[i + 1][:n]),
                array(p[f"weight{i + 1}"]), array(self.rstd[i + 1]), out, spare[0],
                array(g[f"weight{i + 1}"]), self.temps[1], gate=opened, gate_kind=capi.GATE_SILU,
                grad_gate=mixed[2], input_weight=array(p[f"inner{i}"]),
                input_rstd=array(self.inner_rstd[i]), grad_input_weight=array(g[f"inner{i}"]))
            grad_total = spare[0]
            capi.gated_recurrence_gradient(out, gate, x, hidden, mixed[0], mixed[1], self.temps[0],
                                           complement=True, **packed)
            g[f"mix{i}"].copy_(self.normed[i][:n].t() @ self.grad_mixed[:n])
            grad_normed = self.grad_mixed[:n] @ c[f"mix{i}"].t()
        total = matrix(self.totals[0][:n])
        capi.residual_norm_gradient(matrix(grad_normed), grad_total, total, total,
                                    array(p["weight0"]), array(self.rstd[0]), spare[1],
                                    grad_weight=array(g["weight0"]), temp=self.temps[1])
        capi.embedding_gradient(spare[1], array(tokens), matrix(g["table"]), self.temps[2],
                                scale=self.scale)
        capi.gradient_norm(self.lists[1], array(self.norm), self.temps[3])

    def step(self, tokens: torch.Tensor, targets: torch.Tensor, sequences: int = 1,
             offsets=None) -> torch.Tensor:
        """One step of AdamW; the mean loss, on the device."""
        logits = self.forward(tokens, sequences, offsets).float()
        log_p = logits - torch.logsumexp(logits, 1, keepdim=True)
        loss = -log_p.gather(1, targets[:, None]).mean()
        grad = log_p.exp()
        grad.scatter_add_(1, targets[:, None], torch.full_like(grad[:, :1], -1.0))
        self.backward(tokens, (grad / tokens.numel()).to(self.normed[0].dtype), sequences, offsets)
        self.steps += 1
        capi.adamw(*self.lists, array(self.steps), rate=self.rate, weight_decay=0.01,
                   norm=array(self.norm), max_norm=self.max_norm, seed=7, **self.options)
        return loss


def batch(g, positions: int, vocabulary: int):
    """Sequences of many lengths packed into `positions` tokens, each of which mostly follows from the
    two before it: tokens, those that follow them, and where the sequences begin and end."""
    cuts = torch.randint(1, positions, (positions // 64,), generator=g).unique()
    offsets = torch.cat((torch.tensor([0]), cuts, torch.tensor([positions]))).int()
    line, begins = [], set(offsets.tolist())
    for i in range(positions + 1):
        if i in begins or float(torch.rand(1, generator=g)) < 0.1:
            line.append(int(torch.randint(0, vocabulary, (1,), generator=g)))
        else:
            line.append((5 * line[-1] + 3 * line[-2 if i > 1 else -1] + 1) % vocabulary)
    line = torch.tensor(line)
    return line[:-1].cuda(), line[1:].cuda(), offsets.cuda()


def main(steps: int = 100, vocabulary: int = 128, dimension: int = 192, blocks: int = 2,
         positions: int = 2048, eight_bits: bool = False) -> list:
    g = torch.Generator().manual_seed(7)
    model = RecurrentModel(vocabulary, dimension, blocks, positions, eight_bits=eight_bits)
    losses = []
    for i in range(steps):
        tokens, targets, offsets = batch(g, positions, vocabulary)
        loss = model.step(tokens, targets, offsets.numel() - 1, offsets)
        if i % 10 == 0 or i == steps - 1:
            losses.append(float(loss))
            print(f"step {i:4d}  loss {losses[-1]:.4f}  norm of the gradients "
                  f"{float(model.norm):.3f}", flush=True)
    # Four sequences at once, token by token: all that is kept of them is a state a block.
    token = torch.arange(1, 5, device="cuda")
    states = [torch.zeros(4, dimension, device="cuda") for _ in range(blocks)]
    lines = [token]
    for _ in range(8):
        token = model.forward(token, sequences=4, states=states).argmax(1)
        lines.append(token)
    for line in torch.stack(lines, 1).tolist():
        print("continued:", *line, flush=True)
    return losses


if __name__ == "__main__":
    main(eight_bits="--8bit" in sys.argv)
