"""The measured work of the operators around a language model's token table, its
normalisations and its optimiser step, through the public calls of
``ilgpu_amd.capi`` (``own``) or in plain torch operations.

    embedding             out[i] = scale * table[tokens[i]]; a token outside the
                          table (-1 fills up short sequences) gives a row of zeros
    embedding_gradient    grad_table[v] = scale * sum of grad_out[i] over the
                          positions i with tokens[i] = v, zeros where there is none
    layer_norm            out = (x - mean) / sqrt(variance + epsilon) * weight + bias
                          over each row, and the rows' mean and 1 / sqrt(...)
    layer_norm_gradient   the gradients of x, weight and bias
    clip                  the root of the sum of squares over a whole list of
                          gradients, and the gradients scaled to at most max_norm
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16,
         "int32": torch.int32, "int64": torch.int64}
SIZES = {"float32": 4, "float16": 2, "bfloat16": 2, "int32": 4, "int64": 8}
EPSILON = 1e-5
LARGEST = 1 << 28      # elements of the largest view a case makes


def listed():
    return [
        # Serving, one new token of one sequence: latency only.
        {"name": "embedding_one_token", "op": "embedding", "tokens": 1, "vocabulary": 32768,
         "dimension": 2048, "type": "bfloat16", "token_type": "int64", "ids": "zipf",
         "padding": 0.0, "scaled": False},
        # Training, a batch of long sequences, scaled by the root of the width.
        {"name": "embedding_64k_tokens", "op": "embedding", "tokens": 65536, "vocabulary": 131072,
         "dimension": 4096, "type": "bfloat16", "token_type": "int64", "ids": "zipf",
         "padding": 0.05, "scaled": True},
        # A small model's step: most of the table's rows get no gradient.
        {"name": "embedding_gradient_8k", "op": "embedding_gradient", "tokens": 8192,
         "vocabulary": 50021, "dimension": 1024, "type": "bfloat16", "table_type": "float32",
         "token_type": "int64", "ids": "zipf", "padding": 0.0, "scaled": True},
        # A large batch with padded sequences into a large table.
        {"name": "embedding_gradient_64k", "op": "embedding_gradient", "tokens": 65536,
         "vocabulary": 131072, "dimension": 2048, "type": "bfloat16", "table_type": "float32",
         "token_type": "int64", "ids": "zipf", "padding": 0.1, "scaled": False},
        # Characters or bytes: every row of a small table is met often; an odd width.
        {"name": "embedding_gradient_bytes", "op": "embedding_gradient", "tokens": 30011,
         "vocabulary": 1000, "dimension": 769, "type": "float32", "table_type": "float32",
         "token_type": "int32", "ids": "zipf", "padding": 0.0, "scaled": False},
        # Serving, one token: a single row.
        {"name": "layer_norm_one_row", "op": "layer_norm", "rows": 1, "columns": 4096,
         "type": "bfloat16", "weight_type": "bfloat16"},
        # An odd width and an odd number of rows: no row but the first is aligned.
        {"name": "layer_norm_ragged", "op": "layer_norm", "rows": 4099, "columns": 1537,
         "type": "float16", "weight_type": "float32"},
        # Training, a batch of long sequences of a wide model.
        {"name": "layer_norm_32k_rows", "op": "layer_norm", "rows": 32768, "columns": 4096,
         "type": "bfloat16", "weight_type": "float32"},
        # Training, a small model.
        {"name": "layer_norm_gradient_8k_rows", "op": "layer_norm_gradient", "rows": 8192,
         "columns": 1024, "type": "bfloat16", "weight_type": "float32"},
        # Training, a wide model.
        {"name": "layer_norm_gradient_32k_rows", "op": "layer_norm_gradient", "rows": 32768,
         "columns": 4096, "type": "bfloat16", "weight_type": "bfloat16"},
        # The gradients of a model of a few hundred thousand parameters: latency only.
        {"name": "clip_small_model", "op": "clip", "layers": 2, "width": 128, "vocabulary": 1000,
         "type": "float32", "norm": 8.0},
        # Matrices in 16 bits, vectors in 32: 285 million parameters.
        {"name": "clip_large_model", "op": "clip", "layers": 5, "width": 2048,
         "vocabulary": 16384, "type": "bfloat16", "norm": 5.0},
    ]


def _between(rng, smallest, largest):
    """Log-uniform over [smallest, largest], a multiple of 64 half of the time."""
    n = int(round(smallest * (largest / smallest) ** rng.random()))
    if n >= 64 and rng.random() < 0.5:
        n -= n % 64
    return max(smallest, min(largest, n))


def draw(rng):
    op = rng.choice(["embedding", "embedding_gradient", "layer_norm", "layer_norm_gradient", "clip"])
    kind = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    # The largest view in bytes is that of the listed cases: half as many elements of 32 bits.
    most = LARGEST // 2 if kind == "float32" else LARGEST
    if op == "embedding":
        dimension = _between(rng, 64, 4096)
        return {"op": op, "tokens": _between(rng, 1, min(65536, most // dimension)),
                "vocabulary": _between(rng, 1000, 131072), "dimension": dimension, "type": kind,
                "token_type": rng.choice(["int32", "int64"]), "ids": rng.choice(["zipf", "uniform"]),
                "padding": rng.choice([0.0, 0.05, 0.3]), "scaled": rng.random() < 0.5}
    if op == "embedding_gradient":
        dimension = _between(rng, 64, 2048)
        return {"op": op, "tokens": _between(rng, 1, 65536),
                "vocabulary": _between(rng, 1000, 131072), "dimension": dimension, "type": kind,
                "table_type": rng.choice(["float32", kind]),
                "token_type": rng.choice(["int32", "int64"]), "ids": rng.choice(["zipf", "uniform"]),
                "padding": rng.choice([0.0, 0.1, 0.5]), "scaled": rng.random() < 0.5}
    if op in ("layer_norm", "layer_norm_gradient"):
        columns = _between(rng, 64, 8192)
        return {"op": op, "rows": _between(rng, 1, min(65536, (most // 2) // columns)),
                "columns": columns, "type": kind, "weight_type": rng.choice(["float32", kind])}
    width = _between(rng, 64, 2048 if kind != "float32" else 1448)
    return {"op": op, "layers": rng.randint(1, 5), "width": width,
            "vocabulary": _between(rng, 1000, 16384), "type": kind,
            "norm": rng.choice([0.25, 3.0, 40.0])}


# ---- inputs ---------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(g, shape, kind):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32).to(TYPES[kind])


def _tokens(case, g):
    """Token numbers: by rank, the k-th of V about 1 / k as often (a tokenizer's table
    has its frequent entries first), or uniform; -1 at the ends of padded sequences of
    a 16th of the batch."""
    n, v = case["tokens"], case["vocabulary"]
    u = torch.rand(n, generator=g, device=DEVICE, dtype=torch.float64)
    if case["ids"] == "zipf":
        t = torch.exp(u * math.log(v + 1.0)) - 1.0
    else:
        t = u * v
    t = t.floor().clamp_(0, v - 1).to(TYPES[case["token_type"]])
    length = max(1, n // 16)
    t[torch.arange(n, device=DEVICE) % length >= length - int(length * case["padding"])] = -1
    return t


def _shapes(case):
    """A transformer's parameters: the token table, and per layer two norms of two
    vectors, four square matrices, two of four times the width and their biases."""
    w = case["width"]
    shapes = [((case["vocabulary"], w), case["type"])]
    for _ in range(case["layers"]):
        shapes += [((w,), "float32")] * 2 + [((w, w), case["type"])] * 4
        shapes += [((w,), "float32")] * 2 + [((4 * w, w), case["type"]), ((w, 4 * w), case["type"])]
    return shapes


def _inputs(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op == "embedding":
        return {"tokens": _tokens(case, g),
                "table": _normal(g, (case["vocabulary"], case["dimension"]), case["type"]),
                "scale": math.sqrt(case["dimension"]) if case["scaled"] else 1.0}
    if op == "embedding_gradient":
        return {"tokens": _tokens(case, g),
                "grad_out": _normal(g, (case["tokens"], case["dimension"]), case["type"]),
                "scale": math.sqrt(case["dimension"]) if case["scaled"] else 1.0}
    if op in ("layer_norm", "layer_norm_gradient"):
        rows, columns = case["rows"], case["columns"]
        # Activations: rows of different mean and spread, a few columns far larger.
        x = torch.randn((rows, columns), generator=g, device=DEVICE)
        x *= 0.5 + torch.rand((rows, 1), generator=g, device=DEVICE)
        x += 0.5 * torch.randn((rows, 1), generator=g, device=DEVICE)
        x[:, :: max(1, columns // 4)] *= 8.0
        inputs = {"x": x.to(TYPES[case["type"]]),
                  "weight": (1.0 + 0.2 * torch.randn(columns, generator=g, device=DEVICE)).to(
                      TYPES[case["weight_type"]]),
                  "bias": (0.2 * torch.randn(columns, generator=g, device=DEVICE)).to(
                      TYPES[case["weight_type"]])}
        if op == "layer_norm_gradient":
            inputs["grad_out"] = _normal(g, (rows, columns), case["type"])
            wide = inputs["x"].double()     # what the forward pass kept
            inputs["mean"] = wide.mean(1).float()
            inputs["rstd"] = (wide.var(1, unbiased=False) + EPSILON).rsqrt().float()
        return inputs
    shapes = _shapes(case)
    count = sum(math.prod(shape) for shape, _ in shapes)
    spread = case["norm"] / math.sqrt(count)
    return {"gradients": [(spread * torch.randn(shape, generator=g, device=DEVICE)).to(TYPES[kind])
                          for shape, kind in shapes], "max_norm": 1.0}


def prepare(case, seed):
    state = _inputs(case, seed)
    state["op"] = op = case["op"]
    if op == "embedding_gradient":
        state["table_type"] = TYPES[case["table_type"]]
        state["vocabulary"] = case["vocabulary"]
    if not own:
        return state
    from ilgpu_amd import capi
    array, matrix = capi.DeviceArray.from_tensor, capi.DeviceMatrix.from_tensor

    def empty(shape, like):
        return torch.empty(shape, dtype=like, device=DEVICE)

    state["capi"] = capi
    if op == "embedding":
        state["out"] = empty((case["tokens"], case["dimension"]), state["table"].dtype)
        state["views"] = (matrix(state["table"]), array(state["tokens"]), matrix(state["out"]))
    elif op == "embedding_gradient":
        state["out"] = empty((case["vocabulary"], case["dimension"]), state["table_type"])
        state["views"] = (matrix(state["grad_out"]), array(state["tokens"]), matrix(state["out"]))
        state["temp"] = capi.temp_buffer(capi.embedding_gradient_temp_bytes(
            case["tokens"], case["vocabulary"], case["dimension"]))
    elif op == "layer_norm":
        x = state["x"]
        state["out"] = (torch.empty_like(x), empty(x.shape[0], torch.float32),
                        empty(x.shape[0], torch.float32))
        state["views"] = (matrix(x), matrix(state["out"][0]), array(state["weight"]),
                          array(state["bias"]))
        state["statistics"] = {"mean": array(state["out"][1]), "rstd": array(state["out"][2])}
    elif op == "layer_norm_gradient":
        state["out"] = (torch.empty_like(state["x"]), torch.empty_like(state["weight"]),
                        torch.empty_like(state["weight"]))
        state["views"] = (matrix(state["grad_out"]), matrix(state["x"]), array(state["weight"]),
                          array(state["mean"]), array(state["rstd"]), matrix(state["out"][0]),
                          array(state["out"][1]), array(state["out"][2]))
        state["temp"] = capi.temp_buffer(capi.layer_norm_gradient_temp_bytes(
            case["rows"], case["columns"]))
    else:
        # The clipped gradients go into the optimiser's own copy.
        state["clipped"] = [torch.empty_like(t) for t in state["gradients"]]
        state["norm"] = empty(1, torch.float32)
        state["views"] = (capi.TensorList([array(t) for t in state["gradients"]]),
                          array(state["norm"]), capi.TensorList([array(t) for t in state["clipped"]]))
        state["temp"] = capi.temp_buffer(capi.gradient_norm_temp_bytes(len(state["gradients"])))
    return state


# ---- one pass -------------------------------------------------------------------
def run(state):
    op = state["op"]
    return _run_own(state, op) if own else _run_plain(state, op)


def _run_own(state, op):
    capi = state["capi"]
    if op == "embedding":
        capi.embedding(*state["views"], scale=state["scale"])
        return state["out"]
    if op == "embedding_gradient":
        capi.embedding_gradient(*state["views"], state["temp"], scale=state["scale"])
        return state["out"]
    if op == "layer_norm":
        x, out, weight, bias = state["views"]
        capi.layer_norm(x, out, weight, bias, epsilon=EPSILON, **state["statistics"])
        return state["out"]
    if op == "layer_norm_gradient":
        capi.layer_norm_gradient(*state["views"], state["temp"])
        return state["out"]
    gradients, norm, clipped = state["views"]
    capi.gradient_norm(gradients, norm, state["temp"])
    capi.clip_gradients(gradients, norm, state["max_norm"], clipped)
    return [state["norm"], *state["clipped"]]


def _run_plain(state, op):
    if op == "embedding":
        tokens = state["tokens"].long()
        there = (tokens >= 0) & (tokens < state["table"].shape[0])
        rows = state["table"][tokens * there].float() * state["scale"]
        return (rows * there[:, None]).to(state["table"].dtype)
    if op == "embedding_gradient":
        tokens, grad = state["tokens"].long(), state["grad_out"]
        there = (tokens >= 0) & (tokens < state["vocabulary"])
        out = torch.zeros((state["vocabulary"], grad.shape[1]), device=grad.device)
        out.index_add_(0, tokens * there, grad.float() * (state["scale"] * there[:, None]))
        return out.to(state["table_type"])
    if op == "layer_norm":
        x = state["x"].float()
        mean = x.mean(1, keepdim=True)
        away = x - mean
        rstd = torch.rsqrt((away * away).mean(1, keepdim=True) + EPSILON)
        out = away * rstd * state["weight"].float() + state["bias"].float()
        return out.to(state["x"].dtype), mean[:, 0], rstd[:, 0]
    if op == "layer_norm_gradient":
        grad, rstd = state["grad_out"].float(), state["rstd"][:, None]
        hat = (state["x"].float() - state["mean"][:, None]) * rstd
        weighted = grad * state["weight"].float()
        grad_x = rstd * (weighted - weighted.mean(1, keepdim=True)
                         - hat * (weighted * hat).mean(1, keepdim=True))
        kind = state["weight"].dtype
        return grad_x.to(state["x"].dtype), (grad * hat).sum(0).to(kind), grad.sum(0).to(kind)
    squares = [(t.float() * t.float()).sum() for t in state["gradients"]]
    norm = torch.sqrt(torch.stack(squares).sum())
    factor = torch.where(norm > state["max_norm"], state["max_norm"] / norm, 1.0)
    return [norm[None], *((t.float() * factor).to(t.dtype) for t in state["gradients"])]


# ---- what a pass cannot do without ----------------------------------------------
def _distinct(case):
    """Expected number of different tokens among those that are not padding."""
    n, v = case["tokens"] * (1.0 - case["padding"]), case["vocabulary"]
    if case["ids"] == "zipf":
        k = np.arange(v, dtype=np.float64)
        p = np.log1p(1.0 / (k + 1.0)) / math.log(v + 1.0)
    else:
        p = np.full(v, 1.0 / v)
    return float(np.sum(-np.expm1(n * np.log1p(-p))))


def work(case):
    op = case["op"]
    if op in ("embedding", "embedding_gradient"):
        n, d, size = case["tokens"], case["dimension"], SIZES[case["type"]]
        read = n * SIZES[case["token_type"]]
        if op == "embedding":
            return {"bytes": read + int(_distinct(case) * d * size) + n * d * size, "flops": n * d}
        met = n - 16 * int(max(1, n // 16) * case["padding"])
        return {"bytes": read + met * d * size
                + case["vocabulary"] * d * SIZES[case["table_type"]], "flops": 2 * met * d}
    if op in ("layer_norm", "layer_norm_gradient"):
        elements, size = case["rows"] * case["columns"], SIZES[case["type"]]
        small = case["columns"] * SIZES[case["weight_type"]]
        if op == "layer_norm":
            return {"bytes": 2 * elements * size + 2 * small + 8 * case["rows"], "flops": 8 * elements}
        return {"bytes": 3 * elements * size + 3 * small + 8 * case["rows"], "flops": 14 * elements}
    sizes = [(math.prod(shape), SIZES[kind]) for shape, kind in _shapes(case)]
    return {"bytes": 2 * sum(n * s for n, s in sizes), "flops": 3 * sum(n for n, _ in sizes)}


# ---- the definitions in 64 bits ---------------------------------------------------
def exact(case, seed):
    inputs = _inputs(case, seed)
    op = case["op"]
    if op == "embedding":
        out = torch.zeros((case["tokens"], case["dimension"]), dtype=torch.float64, device=DEVICE)
        at = torch.nonzero((inputs["tokens"] >= 0) & (inputs["tokens"] < case["vocabulary"]))[:, 0]
        out[at] = torch.index_select(inputs["table"], 0, inputs["tokens"][at]).double() * inputs["scale"]
        return out
    if op == "embedding_gradient":
        # Positions in the order of their tokens; a token's rows lie together and are
        # added up by halves: each round adds every second row to the one before it.
        tokens, order = torch.sort(inputs["tokens"].long(), stable=True)
        order = order[(tokens >= 0) & (tokens < case["vocabulary"])]
        tokens = tokens[(tokens >= 0) & (tokens < case["vocabulary"])]
        rows = inputs["grad_out"][order].double() * inputs["scale"]
        while tokens.numel() > 0:
            _, counts = torch.unique_consecutive(tokens, return_counts=True)
            if int(counts.max()) == 1:
                break
            first = torch.cumsum(counts, 0) - counts
            place = torch.arange(tokens.numel(), device=DEVICE) - torch.repeat_interleave(first, counts)
            left = torch.nonzero(place % 2 == 0)[:, 0]
            paired = torch.nonzero(place % 2 == 1)[:, 0]
            rows[paired - 1] += rows[paired]
            rows, tokens = rows[left], tokens[left]
        out = torch.zeros((case["vocabulary"], case["dimension"]), dtype=torch.float64, device=DEVICE)
        out[tokens] = rows
        return out
    if op == "layer_norm":
        x = inputs["x"].double()
        variance, mean = torch.var_mean(x, 1, unbiased=False)
        rstd = 1.0 / torch.sqrt(variance + EPSILON)
        out = x.sub_(mean[:, None]).mul_(rstd[:, None])
        return out.mul_(inputs["weight"].double()).add_(inputs["bias"].double()), mean, rstd
    if op == "layer_norm_gradient":
        # With g = weight * grad_out and h the normalised row: h and the constant row are
        # projected out of g, and what is left is divided by the deviation.
        grad, rstd = inputs["grad_out"].double(), inputs["rstd"].double()[:, None]
        hat = (inputs["x"].double() - inputs["mean"].double()[:, None]) * rstd
        n = case["columns"]
        grad_weight = torch.sum(grad * hat, 0)
        grad_bias = torch.sum(grad, 0)
        grad *= inputs["weight"].double()
        along_one, along_hat = grad.sum(1, keepdim=True) / n, (grad * hat).sum(1, keepdim=True) / n
        return rstd * (grad - along_one - hat * along_hat), grad_weight, grad_bias
    wide = [t.double() for t in inputs["gradients"]]
    norm = math.sqrt(math.fsum(float(torch.dot(t.flatten(), t.flatten())) for t in wide))
    factor = min(1.0, inputs["max_norm"] / norm)
    return [torch.tensor([norm], dtype=torch.float64, device=DEVICE), *(t * factor for t in wide)]
