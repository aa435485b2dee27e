"""A next-token model trained with the library's operators: embedding lookup and its
gradient, layer norm and its gradients, the norm of all gradients and its clipping.

    logits = layer_norm(scale * table[token]) @ head

The two matrix products and the softmax are torch's; everything between the token
numbers and the products, and from the products' gradients to the clipped gradients
of the parameters, is the library's, on torch's current stream and without a
synchronisation.  ``python examples/token_model.py`` trains on a sequence whose next
token mostly follows from the last and prints the loss, then continues a sequence
token by token.
"""
from __future__ import annotations

import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from ilgpu_amd import capi  # noqa: E402

array, matrix = capi.DeviceArray.from_tensor, capi.DeviceMatrix.from_tensor


class TokenModel:
    """Parameters in float32, activations and their gradients in ``activations``."""

    def __init__(self, vocabulary: int, dimension: int, positions: int, *,
                 activations=torch.float32, max_norm: float = 1.0, seed: int = 1):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def normal(*shape, spread):
            return spread * torch.randn(*shape, generator=g, device="cuda")

        self.scale, self.max_norm = math.sqrt(dimension), max_norm
        self.parameters = {"table": normal(vocabulary, dimension, spread=dimension ** -0.5),
                           "weight": torch.ones(dimension, device="cuda"),
                           "bias": torch.zeros(dimension, device="cuda"),
                           "head": normal(dimension, vocabulary, spread=dimension ** -0.5)}
        self.gradients = {k: torch.empty_like(v) for k, v in self.parameters.items()}
        # What every step reuses: activations, statistics, scratch and the views of them.
        def empty(*shape, dtype=activations):
            return torch.empty(*shape, dtype=dtype, device="cuda")

        self.embedded, self.normed, self.grad_normed, self.grad_embedded = (
            empty(positions, dimension) for _ in range(4))
        self.mean, self.rstd = (empty(positions, dtype=torch.float32) for _ in range(2))
        self.norm = empty(1, dtype=torch.float32)
        self.clipped_list = capi.TensorList([array(t) for t in self.gradients.values()])
        self.temps = [capi.temp_buffer(n) for n in (
            capi.embedding_gradient_temp_bytes(positions, vocabulary, dimension),
            capi.layer_norm_gradient_temp_bytes(positions, dimension),
            capi.gradient_norm_temp_bytes(len(self.clipped_list)))]

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        """Logits of the tokens that follow; any number of tokens up to `positions`."""
        p, n = self.parameters, tokens.numel()
        capi.embedding(matrix(p["table"]), array(tokens), matrix(self.embedded[:n]),
                       scale=self.scale)
        capi.layer_norm(matrix(self.embedded[:n]), matrix(self.normed[:n]), array(p["weight"]),
                        array(p["bias"]), mean=array(self.mean), rstd=array(self.rstd))
        return self.normed[:n] @ p["head"].to(self.normed.dtype)

    def backward(self, tokens: torch.Tensor, grad_logits: torch.Tensor) -> None:
        """The gradients of all parameters from that of the logits, clipped together."""
        p, g, n = self.parameters, self.gradients, tokens.numel()
        head = p["head"].to(self.normed.dtype)
        g["head"].copy_(self.normed[:n].t() @ grad_logits)
        self.grad_normed[:n] = grad_logits @ head.t()
        capi.layer_norm_gradient(
            matrix(self.grad_normed[:n]), matrix(self.embedded[:n]), array(p["weight"]),
            array(self.mean), array(self.rstd), matrix(self.grad_embedded[:n]),
            array(g["weight"]), array(g["bias"]), self.temps[1])
        capi.embedding_gradient(matrix(self.grad_embedded[:n]), array(tokens), matrix(g["table"]),
                                self.temps[0], scale=self.scale)
        capi.gradient_norm(self.clipped_list, array(self.norm), self.temps[2])
        capi.clip_gradients(self.clipped_list, array(self.norm), self.max_norm)

    def step(self, tokens: torch.Tensor, targets: torch.Tensor, rate: float) -> torch.Tensor:
        """One step of gradient descent; the mean loss, on the device."""
        logits = self.forward(tokens).float()
        log_p = logits - torch.logsumexp(logits, 1, keepdim=True)
        loss = -log_p.gather(1, targets[:, None]).mean()
        grad = log_p.exp()
        grad.scatter_add_(1, targets[:, None], torch.full_like(grad[:, :1], -1.0))
        self.backward(tokens, (grad / tokens.numel()).to(self.normed.dtype))
        for name, value in self.parameters.items():
            value.sub_(self.gradients[name], alpha=rate)
        return loss


def sequence(g, length: int, vocabulary: int) -> torch.Tensor:
    """Tokens of which nine in ten follow from the one before."""
    jump = torch.rand(length, generator=g) < 0.1
    random = torch.randint(0, vocabulary, (length,), generator=g)
    tokens = [int(random[0])]
    for i in range(1, length):
        tokens.append(int(random[i]) if jump[i] else (5 * tokens[-1] + 3) % vocabulary)
    return torch.tensor(tokens)


def main(steps: int = 200, vocabulary: int = 512, dimension: int = 256, positions: int = 4096,
         activations=torch.bfloat16) -> list:
    g = torch.Generator().manual_seed(7)
    model = TokenModel(vocabulary, dimension, positions, activations=activations)
    losses = []
    for i in range(steps):
        tokens = sequence(g, positions + 1, vocabulary).to("cuda")
        loss = model.step(tokens[:-1], tokens[1:], rate=2.0)
        if i % 20 == 0 or i == steps - 1:
            losses.append(float(loss))
            print(f"step {i:4d}  loss {losses[-1]:.4f}  norm of the gradients "
                  f"{float(model.norm):.3f}", flush=True)
    token = torch.tensor([1], device="cuda")
    line = [1]
    for _ in range(10):
        token = model.forward(token).argmax(1)
        line.append(int(token))
    print("continued:", *line, flush=True)
    return losses


if __name__ == "__main__":
    main()
