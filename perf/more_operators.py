"""The measured work of the operators that a recurrent language model's training step
and its token-by-token form are made of, through the public calls of
``ilgpu_amd.capi`` (``own``) or in plain torch operations.

    recurrence           h[t] = a[t] h[t-1] + b[t] per channel over every sequence of a packed
                         batch; a = sigmoid(gate) or exp(gate), b = x or (1 - a) x; the first
                         h[t-1] is the sequence's initial state, the last h its final one
    recurrence_gradient  the gradients of gate, x and the initial states
    norm                 total = residual + scale * y, out = total * rstd * weight with
                         y = x [* input_rstd * input_weight] [* act(gate)] and
                         rstd = 1 / sqrt(mean of the row's squares + epsilon)
    norm_gradient        the gradients of x, gate, residual and both weights
    adamw                one step over a list of tensors from their gradients, scaled to
                         at most max_norm; moments in 32 bits, or in 8 with a scale for 256
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZES = {"float32": 4, "float16": 2, "bfloat16": 2}
EPSILON = 1e-5
LARGEST = 1 << 27      # elements of the largest matrix a case makes
BLOCK = 256            # moments in 8 bits that share a scale
RATE, BETAS, DAMPING, DECAY = 3e-4, (0.9, 0.95), 1e-8, 0.1
STEP, SEED = 1000, 0x1234567890


def listed():
    return [
        # Serving: one new token of each of 64 sequences, whose states are updated.
        {"name": "recurrence_one_token", "op": "recurrence", "sequences": 64, "rows": 64,
         "channels": 2048, "type": "bfloat16", "ragged": False, "initial": True,
         "decay": "sigmoid", "complement": True},
        # Prompts of many lengths packed behind one another, none of them too; an odd width.
        {"name": "recurrence_ragged", "op": "recurrence", "sequences": 37, "rows": 9001,
         "channels": 1537, "type": "float16", "ragged": True, "initial": True,
         "decay": "exponential", "complement": False},
        # One long document: few channels for the chip, many positions.
        {"name": "recurrence_64k", "op": "recurrence", "sequences": 1, "rows": 65536,
         "channels": 2048, "type": "bfloat16", "ragged": False, "initial": False,
         "decay": "sigmoid", "complement": True},
        # Training, a batch of sequences of a small model.
        {"name": "recurrence_gradient_8k", "op": "recurrence_gradient", "sequences": 8,
         "rows": 8192, "channels": 1024, "type": "bfloat16", "ragged": False, "initial": False,
         "decay": "sigmoid", "complement": True},
        # Training, packed documents of a wide model.
        {"name": "recurrence_gradient_packed", "op": "recurrence_gradient", "sequences": 41,
         "rows": 32768, "channels": 4096, "type": "bfloat16", "ragged": True, "initial": True,
         "decay": "exponential", "complement": True},
        # Serving, one token: a single row.
        {"name": "norm_one_row", "op": "norm", "rows": 1, "columns": 4096, "type": "bfloat16",
         "residual_type": "bfloat16", "weight_type": "bfloat16", "gate": "silu",
         "input_norm": True, "scale": 1.0},
        # Training: the residual stream in 32 bits, a gated block whose output is normalised.
        {"name": "norm_32k_rows", "op": "norm", "rows": 32768, "columns": 2048,
         "type": "bfloat16", "residual_type": "float32", "weight_type": "float32",
         "gate": "silu", "input_norm": True, "scale": 0.5},
        # An odd width, a block without a gate.
        {"name": "norm_gradient_ragged", "op": "norm_gradient", "rows": 4099, "columns": 1537,
         "type": "float16", "residual_type": "float16", "weight_type": "float32",
         "gate": "none", "input_norm": False, "scale": 1.0},
        # Training, a wide model.
        {"name": "norm_gradient_16k_rows", "op": "norm_gradient", "rows": 16384, "columns": 4096,
         "type": "bfloat16", "residual_type": "bfloat16", "weight_type": "float32",
         "gate": "sigmoid", "input_norm": True, "scale": 0.7},
        # A model of a few hundred thousand parameters: latency.
        {"name": "adamw_small_model", "op": "adamw", "layers": 2, "width": 128,
         "vocabulary": 1000, "type": "float32", "parameter_type": "float32", "copies": False,
         "states": 32, "norm": 3.0},
        # 285 million parameters in 32 bits, and a copy in 16 that the products read.
        {"name": "adamw_large_model", "op": "adamw", "layers": 5, "width": 2048,
         "vocabulary": 16384, "type": "bfloat16", "parameter_type": "float32", "copies": True,
         "states": 32, "norm": 5.0},
        # 8-bit moments, read back behind the step, as a checkpoint or a monitor does.
        {"name": "adamw_8bit", "op": "adamw", "layers": 3, "width": 1448, "vocabulary": 10007,
         "type": "bfloat16", "parameter_type": "float32", "copies": True, "states": 8,
         "norm": 5.0},
    ]


def _between(rng, smallest, largest):
    """Log-uniform over [smallest, largest], a multiple of 64 half of the time."""
    n = int(round(smallest * (largest / smallest) ** rng.random()))
    if n >= 64 and rng.random() < 0.5:
        n -= n % 64
    return max(smallest, min(largest, n))


def draw(rng):
    op = rng.choice(["recurrence", "recurrence", "recurrence_gradient", "norm", "norm_gradient",
                     "adamw"])
    kind = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    # Half as many elements of 32 bits.
    most = LARGEST // 2 if kind == "float32" else LARGEST
    if op in ("recurrence", "recurrence_gradient"):
        channels = _between(rng, 64, 4096)
        rows = _between(rng, 1, min(65536, most // channels))
        ragged = rng.random() < 0.5
        sequences = _between(rng, 1, rows if rng.random() < 0.3 else min(rows, 64))
        if not ragged:
            rows -= rows % sequences
        return {"op": op, "sequences": sequences, "rows": rows, "channels": channels,
                "type": kind, "ragged": ragged, "initial": rng.random() < 0.5,
                "decay": rng.choice(["sigmoid", "exponential"]),
                "complement": rng.random() < 0.5}
    if op in ("norm", "norm_gradient"):
        columns = _between(rng, 64, 8192)
        return {"op": op, "rows": _between(rng, 1, min(65536, (most // 2) // columns)),
                "columns": columns, "type": kind, "residual_type": rng.choice(["float32", kind]),
                "weight_type": rng.choice(["float32", kind]),
                "gate": rng.choice(["none", "sigmoid", "silu"]),
                "input_norm": rng.random() < 0.6, "scale": rng.choice([1.0, 0.5, 0.22])}
    width = _between(rng, 64, 1448)
    return {"op": op, "layers": rng.randint(1, 5), "width": width,
            "vocabulary": _between(rng, 1000, 16384), "type": kind,
            "parameter_type": rng.choice(["float32", "float32", kind]),
            "copies": rng.random() < 0.5, "states": rng.choice([32, 8]),
            "norm": rng.choice([0.25, 3.0, 40.0])}


# ---- inputs ---------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(g, shape, kind, spread=1.0):
    return (spread * torch.randn(shape, generator=g, device=DEVICE)).to(TYPES[kind])


def _used(case):
    """Rows of the sequences; of a ragged batch some rows are left behind the last."""
    return case["rows"] - (case["rows"] // 32 if case["ragged"] else 0)


def _offsets(case, g):
    """Where the sequences begin, and where the last ends: equal, or cut anywhere, with an
    empty one among them."""
    rows, sequences = _used(case), case["sequences"]
    if not case["ragged"]:
        return torch.arange(sequences + 1, device=DEVICE, dtype=torch.int32) * (rows // sequences)
    cuts = torch.randint(0, rows + 1, (sequences + 1,), generator=g, device=DEVICE)
    cuts[0], cuts[-1] = 0, rows
    cuts = cuts.sort().values
    if sequences > 2:
        cuts[2] = cuts[1]
    return cuts.to(torch.int32)


def _gates(case, g):
    """Channels of different memory, from a few positions to some hundreds."""
    rows, channels = case["rows"], case["channels"]
    gate = torch.randn((rows, channels), generator=g, device=DEVICE)
    gate += 6.0 * torch.rand(channels, generator=g, device=DEVICE)
    if case["decay"] == "exponential":
        gate = -torch.log1p(torch.exp(-gate))
    return gate.to(TYPES[case["type"]])


def _shapes(case):
    """A transformer's or recurrent model's parameters: the token table, and per layer two
    norms of two vectors, four square matrices, two of four times the width and their biases."""
    w = case["width"]
    shapes = [((case["vocabulary"], w), case["type"])]
    for _ in range(case["layers"]):
        shapes += [((w,), "float32")] * 2 + [((w, w), case["type"])] * 4
        shapes += [((w,), "float32")] * 2 + [((4 * w, w), case["type"]), ((w, 4 * w), case["type"])]
    return shapes


def _inputs(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op in ("recurrence", "recurrence_gradient"):
        shape, kind = (case["rows"], case["channels"]), case["type"]
        inputs = {"offsets": _offsets(case, g), "gate": _gates(case, g), "x": _normal(g, shape, kind)}
        if case["initial"]:
            inputs["initial"] = torch.randn((case["sequences"], case["channels"]), generator=g,
                                            device=DEVICE)
        if op == "recurrence_gradient":
            inputs["grad_out"] = _normal(g, shape, kind)
            if case["initial"]:
                inputs["grad_final"] = torch.randn((case["sequences"], case["channels"]),
                                                   generator=g, device=DEVICE)
            # What the forward pass left: the states, as it rounded them.
            inputs["out"] = _recurrence(case, inputs)[0].to(TYPES[kind])
        return inputs
    if op in ("norm", "norm_gradient"):
        shape, kind = (case["rows"], case["columns"]), case["type"]
        x = torch.randn(shape, generator=g, device=DEVICE)
        x *= 0.5 + torch.rand((shape[0], 1), generator=g, device=DEVICE)
        residual = torch.randn(shape, generator=g, device=DEVICE)
        residual[:, :: max(1, shape[1] // 4)] *= 8.0      # a few columns far larger
        inputs = {"x": x.to(TYPES[kind]), "residual": residual.to(TYPES[case["residual_type"]])}
        for name in ("weight",) + (("input_weight",) if case["input_norm"] else ()):
            inputs[name] = (1.0 + 0.2 * torch.randn(shape[1], generator=g, device=DEVICE)).to(
                TYPES[case["weight_type"]])
        if case["gate"] != "none":
            inputs["gate"] = _normal(g, shape, kind)
        if op == "norm_gradient":
            inputs["grad_out"] = _normal(g, shape, kind)
            inputs["grad_total"] = _normal(g, shape, case["residual_type"])
            # What the forward pass left.
            total, _, input_rstd, rstd = _norm(case, inputs)
            del inputs["residual"]
            inputs["total"] = total.to(TYPES[case["residual_type"]])
            inputs["rstd"] = rstd
            if case["input_norm"]:
                inputs["input_rstd"] = input_rstd
        return inputs
    shapes = _shapes(case)
    lengths = [math.prod(shape) for shape, _ in shapes]
    count = sum(lengths)
    spread = case["norm"] / math.sqrt(count)
    inputs = {"lengths": lengths,
              "gradients": [_normal(g, shape, kind, spread) for shape, kind in shapes],
              "norm": torch.full((1,), case["norm"], device=DEVICE), "max_norm": 1.0,
              "parameters": _normal(g, (count,), case["parameter_type"], 0.02)}
    # Moments of a run of some hundred steps: the second spread over some powers of two.
    first = 0.3 * spread * torch.randn(count, generator=g, device=DEVICE)
    second = spread * torch.exp(0.7 * torch.randn(count, generator=g, device=DEVICE))
    second.square_()
    if case["states"] == 32:
        inputs["first"], inputs["second"] = first, second
    else:
        codes, scales = ([], []), ([], [])
        for k, values in enumerate((first, second)):
            for part in values.split(lengths):
                blocks = _blocks(part)
                scale = blocks.abs().amax(1)
                root = (blocks.abs() / scale[:, None]).sqrt()
                code = (128 + torch.copysign(127 * root, blocks) if k == 0
                        else 255 * root.sqrt()).round().to(torch.uint8)
                codes[k].append(code.reshape(-1)[:part.numel()])
                scales[k].append(scale)
        inputs["first"], inputs["second"] = torch.cat(codes[0]), torch.cat(codes[1])
        inputs["first_scales"], inputs["second_scales"] = torch.cat(scales[0]), torch.cat(scales[1])
    if case["copies"]:
        inputs["copies"] = torch.zeros(count, dtype=TYPES[case["type"]], device=DEVICE)
    inputs["step"] = torch.full((1,), STEP, dtype=torch.int64, device=DEVICE)
    return inputs


def prepare(case, seed):
    state = _inputs(case, seed)
    state["op"], state["case"] = op, case = case["op"], case
    if op == "recurrence":
        state["result"] = [torch.zeros_like(state["x"]),
                           torch.empty((case["sequences"], case["channels"]), device=DEVICE)]
    elif op == "recurrence_gradient":
        state["result"] = [torch.zeros_like(state["x"]), torch.zeros_like(state["x"])]
        if case["initial"]:
            state["result"].append(torch.empty_like(state["initial"]))
    if not own:
        return state
    from ilgpu_amd import capi
    array, matrix = capi.DeviceArray.from_tensor, capi.DeviceMatrix.from_tensor

    def view(name):
        return matrix(state[name]) if name in state else None

    state["capi"] = capi
    if op in ("recurrence", "recurrence_gradient"):
        # Equal lengths need no offsets.
        state["options"] = {
            "sequences": case["sequences"], "initial": view("initial"),
            "offsets": array(state["offsets"]) if case["ragged"] else None,
            "decay": getattr(capi, "DECAY_" + case["decay"].upper()),
            "complement": case["complement"]}
        result = [matrix(t) for t in state["result"]]
        if op == "recurrence":
            state["options"]["final"] = result[1]
            state["views"] = (matrix(state["gate"]), matrix(state["x"]), result[0])
        else:
            state["options"]["grad_final"] = view("grad_final")
            state["options"]["grad_initial"] = result[2] if case["initial"] else None
            state["views"] = (matrix(state["grad_out"]), matrix(state["gate"]),
                              matrix(state["x"]), matrix(state["out"]), result[0], result[1])
        state["temp"] = capi.temp_buffer(capi.gated_recurrence_temp_bytes(
            case["rows"], case["channels"]))
    elif op in ("norm", "norm_gradient"):
        x = state["x"]
        state["options"] = options = {"scale": case["scale"]}
        if "gate" in state:
            options.update(gate=matrix(state["gate"]),
                           gate_kind=getattr(capi, "GATE_" + case["gate"].upper()))
        if case["input_norm"]:
            options["input_weight"] = array(state["input_weight"])
        if op == "norm":
            total = torch.empty_like(state["residual"])
            rstd = torch.empty(x.shape[0], device=DEVICE)
            input_rstd = torch.empty_like(rstd) if case["input_norm"] else None
            state["result"] = (total, torch.empty_like(x), input_rstd, rstd)
            options.update(epsilon=EPSILON, rstd=array(rstd),
                           input_rstd=array(input_rstd) if case["input_norm"] else None)
            state["views"] = (matrix(x), matrix(state["residual"]), matrix(total),
                              matrix(state["result"][1]), array(state["weight"]))
        else:
            result = {"x": torch.empty_like(x), "residual": torch.empty_like(state["total"]),
                      "weight": torch.empty_like(state["weight"]), "gate": None,
                      "input_weight": None}
            if "gate" in state:
                result["gate"] = torch.empty_like(x)
                options["grad_gate"] = matrix(result["gate"])
            if case["input_norm"]:
                result["input_weight"] = torch.empty_like(state["input_weight"])
                options.update(input_rstd=array(state["input_rstd"]),
                               grad_input_weight=array(result["input_weight"]))
            state["result"] = result
            state["views"] = (matrix(state["grad_out"]), matrix(state["grad_total"]), matrix(x),
                              matrix(state["total"]), array(state["weight"]), array(state["rstd"]),
                              matrix(result["x"]), matrix(result["residual"]),
                              array(result["weight"]))
            state["temp"] = capi.temp_buffer(capi.residual_norm_gradient_temp_bytes(
                case["rows"], case["columns"]))
    else:
        def parts(name, lengths):
            return capi.TensorList([array(t) for t in state[name].split(lengths)])

        lengths = state["lengths"]
        state["lists"] = (parts("parameters", lengths),
                          capi.TensorList([array(t) for t in state["gradients"]]),
                          parts("first", lengths), parts("second", lengths), array(state["step"]))
        state["options"] = {"rate": RATE, "betas": BETAS, "epsilon": DAMPING,
                            "weight_decay": DECAY, "norm": array(state["norm"]),
                            "max_norm": state["max_norm"]}
        if case["copies"]:
            state["options"]["copies"] = parts("copies", lengths)
        if case["states"] == 8:
            blocks = [-(-n // BLOCK) for n in lengths]
            state["options"].update(first_scales=parts("first_scales", blocks),
                                    second_scales=parts("second_scales", blocks), seed=SEED)
            state["values"] = [torch.empty(sum(lengths), dtype=torch.bfloat16, device=DEVICE)
                               for _ in range(2)]
            state["targets"] = [capi.TensorList([array(t) for t in v.split(lengths)])
                                for v in state["values"]]
    return state


# ---- one pass -------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state, state["op"], state["case"])


def _adamw_result(state, case, values):
    """Moments of 8 bits come back as the numbers they stand for, in 16."""
    result = {"parameters": state["parameters"], "copies": state.get("copies")}
    if case["states"] == 32:
        return {**result, "first": state["first"], "second": state["second"]}
    return {**result, "first": values[0], "second": values[1],
            "first_scales": state["first_scales"], "second_scales": state["second_scales"]}


def _run_own(state, op, case):
    capi = state["capi"]
    if op == "recurrence":
        capi.gated_recurrence(*state["views"], state["temp"], **state["options"])
        return state["result"]
    if op == "recurrence_gradient":
        capi.gated_recurrence_gradient(*state["views"], state["temp"], **state["options"])
        return state["result"]
    if op == "norm":
        capi.residual_norm(*state["views"], **state["options"])
        return state["result"]
    if op == "norm_gradient":
        capi.residual_norm_gradient(*state["views"], state["temp"], **state["options"])
        return state["result"]
    options, lists = state["options"], state["lists"]
    capi.adamw(*lists, **options)
    if case["states"] == 32:
        return _adamw_result(state, case, None)
    capi.adamw_moments(lists[2], options["first_scales"], state["targets"][0],
                       lists[3], options["second_scales"], state["targets"][1])
    return _adamw_result(state, case, state["values"])


def _decays(case, gate):
    """a and 1 - a, each with its own precision."""
    if case["decay"] == "sigmoid":
        return torch.sigmoid(gate), torch.sigmoid(-gate)
    return torch.exp(gate), -torch.expm1(gate)


def _ends(offsets):
    """The sequences that have positions, with their first and last ones."""
    there = torch.nonzero(offsets[1:] > offsets[:-1])[:, 0]
    return there, offsets[:-1][there].long(), offsets[1:][there].long() - 1


def _affine_scan(a, b):
    """h[t] = a[t] h[t-1] + b[t] from h = 0, by maps of 1, 2, 4, ... positions."""
    reach = 1
    while reach < a.shape[0]:
        more = a[reach:] * b[:-reach]
        b = torch.cat((b[:reach], b[reach:] + more))
        a = torch.cat((a[:reach], a[reach:] * a[:-reach]))
        reach *= 2
    return b


def _recurrence(case, state):
    """All states and the final ones in 32 bits; zeros behind the last sequence."""
    offsets, used = state["offsets"], _used(case)
    a, left = _decays(case, state["gate"][:used].float())
    b = state["x"][:used].float()
    if case["complement"]:
        b = b * left
    there, first, last = _ends(offsets)
    if case["initial"]:
        b[first] += a[first] * state["initial"][there]
    a[first] = 0.0
    h = _affine_scan(a, b)
    final = (state["initial"].clone() if case["initial"] else
             torch.zeros((case["sequences"], case["channels"]), device=DEVICE))
    final[there] = h[last]
    out = torch.zeros((case["rows"], case["channels"]), device=DEVICE)
    out[:used] = h
    return out, final


def _recurrence_gradient(case, state):
    used = _used(case)
    a, left = _decays(case, state["gate"][:used].float())
    there, first, last = _ends(state["offsets"])
    x, grad = state["x"][:used].float(), state["grad_out"][:used].float()
    if case["initial"]:
        grad[last] += state["grad_final"][there]
    # What reaches h[t]: grad[t] + a[t+1] * what reaches h[t+1], from the back.
    behind = torch.cat((a[1:], torch.zeros_like(a[:1])))
    behind[last] = 0.0
    reaches = _affine_scan(behind.flip(0), grad.flip(0)).flip(0)
    before = torch.cat((torch.zeros_like(x[:1]), state["out"][:used - 1].float()))
    before[first] = state["initial"][there] if case["initial"] else 0.0
    result = [torch.zeros_like(state["x"]), torch.zeros_like(state["x"])]
    slope = a * left if case["decay"] == "sigmoid" else a
    grad_gate = reaches * (before - x if case["complement"] else before) * slope
    result[0][:used] = grad_gate.to(result[0].dtype)
    result[1][:used] = (reaches * left if case["complement"] else reaches).to(result[1].dtype)
    if case["initial"]:
        grad_initial = state["grad_final"].clone()
        grad_initial[there] = a[first] * reaches[first]
        result.append(grad_initial)
    return result


def _activation(case, gate):
    """act(gate) and its slope."""
    s = torch.sigmoid(gate)
    if case["gate"] == "sigmoid":
        return s, s * (1.0 - s)
    return gate * s, s * (1.0 + gate * (1.0 - s))


def _rstd(rows):
    return torch.rsqrt((rows * rows).mean(1) + EPSILON)


def _norm(case, state):
    """Everything in 32 bits."""
    y, input_rstd = state["x"].float(), None
    if case["input_norm"]:
        input_rstd = _rstd(y)
        y = y * input_rstd[:, None] * state["input_weight"].float()
    if case["gate"] != "none":
        y = y * _activation(case, state["gate"].float())[0]
    total = state["residual"].float() + case["scale"] * y
    rstd = _rstd(total)
    return total, total * rstd[:, None] * state["weight"].float(), input_rstd, rstd


def _norm_gradient(case, state):
    grad = state["grad_out"].float()
    rstd = state["rstd"][:, None]
    hat = state["total"].float() * rstd
    grad_weight = (grad * hat).sum(0)
    grad = grad * state["weight"].float()
    grad_residual = state["grad_total"].float() + rstd * (
        grad - hat * (grad * hat).mean(1, keepdim=True))
    result = {"residual": grad_residual.to(state["total"].dtype), "gate": None,
              "weight": grad_weight.to(state["weight"].dtype), "input_weight": None}
    grad, kind = case["scale"] * grad_residual, state["x"].dtype
    x = state["x"].float()
    input_rstd = state["input_rstd"][:, None] if case["input_norm"] else None
    if case["gate"] != "none":
        act, slope = _activation(case, state["gate"].float())
        y = x * input_rstd * state["input_weight"].float() if case["input_norm"] else x
        result["gate"] = (grad * y * slope).to(kind)
        grad = grad * act
    if case["input_norm"]:
        hat = x * input_rstd
        result["input_weight"] = (grad * hat).sum(0).to(state["input_weight"].dtype)
        grad = grad * state["input_weight"].float()
        grad = input_rstd * (grad - hat * (grad * hat).mean(1, keepdim=True))
    result["x"] = grad.to(kind)
    return result


def _blocks(t):
    """Rows of 256, the last filled with zeros."""
    return torch.nn.functional.pad(t, (0, -t.numel() % BLOCK)).view(-1, BLOCK)


WORD = 0xFFFFFFFF


def _mixed(x):
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & WORD
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & WORD
    return x ^ (x >> 16)


def _chances(index, number):
    """Two numbers in [0, 1) for each of the elements `index` of tensor `number`."""
    key = _mixed(((SEED & WORD) + STEP * 0x3C6EF373) & WORD)
    key = _mixed((key + (SEED >> 32) + number * 0x9E3779B9) & WORD)
    word = _mixed((index * 0x9E3779B9 + key) & WORD)
    return (word & 0xFFFF).float() / 65536, (word >> 16).float() / 65536


def _first_value(code, scale):
    q = code.float() - 128
    return q * q.abs() * (scale / 127 ** 2)


def _second_value(code, scale):
    return code.float() ** 4 * (scale / 255 ** 4)


def _power_code(values, scale, levels, power, chance):
    """The last code whose power is not above the value, or the next one, with the chances
    that make the value right in the mean."""
    z = (values / torch.where(scale > 0, scale, 1.0)).double() * levels ** power
    low = z.pow(1.0 / power).floor().clamp(0, levels)
    up = z - low ** power > chance.double() * ((low + 1) ** power - low ** power)
    return (low + up).clamp(0, levels)


def _adamw(state, case):
    factor = min(1.0, state["max_norm"] / case["norm"])
    c1, c2 = 1.0 - BETAS[0] ** STEP, 1.0 - BETAS[1] ** STEP
    at, block, values = 0, 0, ([], [])
    for number, gradient in enumerate(state["gradients"]):
        n = gradient.numel()
        here, at = slice(at, at + n), at + n
        m, v = state["first"][here], state["second"][here]
        if case["states"] == 8:
            count = -(-n // BLOCK)
            scaled, block = slice(block, block + count), block + count
            scales = [state[k][scaled][:, None] for k in ("first_scales", "second_scales")]
            codes = m, v
            m = _first_value(_blocks(m), scales[0]).view(-1)[:n]
            v = _second_value(_blocks(v), scales[1]).view(-1)[:n]
        g = gradient.float().view(-1) * factor
        m = BETAS[0] * m + (1.0 - BETAS[0]) * g
        v = BETAS[1] * v + (1.0 - BETAS[1]) * (g * g)
        p = state["parameters"][here].float()
        p = p * (1.0 - RATE * DECAY) - RATE * ((m / c1) / ((v / c2).sqrt() + DAMPING))
        state["parameters"][here] = p.to(state["parameters"].dtype)
        if case["copies"]:
            state["copies"][here] = p.to(state["copies"].dtype)
        if case["states"] == 32:
            state["first"][here], state["second"][here] = m, v
            continue
        m, v = _blocks(m), _blocks(v)
        scales[0].copy_(m.abs().amax(1, keepdim=True))
        scales[1].copy_(v.amax(1, keepdim=True))
        index = torch.arange(m.numel(), device=m.device).view(-1, BLOCK)
        chances = _chances(index, number)
        m = 128 + torch.copysign(_power_code(m.abs(), scales[0], 127, 2, chances[0]), m.double())
        v = _power_code(v, scales[1], 255, 4, chances[1])
        codes[0].copy_(m.view(-1)[:n])
        codes[1].copy_(v.view(-1)[:n])
        values[0].append(_first_value(m, scales[0]).view(-1)[:n].to(torch.bfloat16))
        values[1].append(_second_value(v, scales[1]).view(-1)[:n].to(torch.bfloat16))
    if case["states"] == 8:
        values = [torch.cat(v) for v in values]
    return _adamw_result(state, case, values)


def _run_plain(state, op, case):
    if op == "recurrence":
        out, final = _recurrence(case, state)
        return [out.to(state["x"].dtype), final]
    if op == "recurrence_gradient":
        return _recurrence_gradient(case, state)
    if op == "norm":
        total, out, input_rstd, rstd = _norm(case, state)
        return total.to(state["residual"].dtype), out.to(state["x"].dtype), input_rstd, rstd
    if op == "norm_gradient":
        return _norm_gradient(case, state)
    return _adamw(state, case)


# ---- what a pass cannot do without ----------------------------------------------
def work(case):
    op = case["op"]
    if op in ("recurrence", "recurrence_gradient"):
        elements, size = _used(case) * case["channels"], SIZES[case["type"]]
        states = 4 * case["sequences"] * case["channels"]
        read = 4 * (case["sequences"] + 1) if case["ragged"] else 0
        if op == "recurrence":
            return {"bytes": read + 3 * elements * size + states * (2 if case["initial"] else 1),
                    "flops": 8 * elements}
        return {"bytes": read + 6 * elements * size + states * (3 if case["initial"] else 0),
                "flops": 14 * elements}
    if op in ("norm", "norm_gradient"):
        elements = case["rows"] * case["columns"]
        size, wide = SIZES[case["type"]], SIZES[case["residual_type"]]
        gated, normed = case["gate"] != "none", case["input_norm"]
        vectors = case["columns"] * SIZES[case["weight_type"]] * (1 + normed)
        statistics = 4 * case["rows"] * (1 + normed)
        if op == "norm":
            return {"bytes": elements * (size * (2 + gated) + 2 * wide) + vectors + statistics,
                    "flops": elements * (7 + 4 * normed + 5 * gated)}
        return {"bytes": elements * (size * (3 + 2 * gated) + 3 * wide) + 2 * vectors + statistics,
                "flops": elements * (11 + 9 * normed + 11 * gated)}
    elements = [(math.prod(shape), SIZES[kind]) for shape, kind in _shapes(case)]
    count = sum(n for n, _ in elements)
    each = 2 * SIZES[case["parameter_type"]] + (SIZES[case["type"]] if case["copies"] else 0)
    if case["states"] == 32:
        return {"bytes": sum(n * s for n, s in elements) + (each + 16) * count, "flops": 14 * count}
    # Both moments are read back: a byte each, written in two.
    blocks = sum(-(-n // BLOCK) for n, _ in elements)
    return {"bytes": sum(n * s for n, s in elements) + (each + 4 + 6) * count + 24 * blocks,
            "flops": 50 * count}


# ---- the definitions in 64 bits ---------------------------------------------------
def _lengths(offsets):
    """Starts and lengths on the host, and the sequences from the longest to the shortest, so
    that those with a position t are the first few."""
    ends = offsets.tolist()
    lengths = [e - b for b, e in zip(ends, ends[1:])]
    order = sorted(range(len(lengths)), key=lambda i: -lengths[i])
    return ends, lengths, order


def _gate_values(case, gate):
    if case["decay"] == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-gate)), 1.0 / (1.0 + torch.exp(gate))
    return torch.exp(gate), -torch.expm1(gate)


def _walk(case, inputs, backwards):
    """Position after position, all sequences that have one together: calls
    step(rows, which sequences' states)."""
    ends, lengths, order = _lengths(inputs["offsets"])
    starts = torch.tensor([ends[i] for i in order], device=DEVICE)
    order_t = torch.tensor(order, device=DEVICE)
    longest = lengths[order[0]] if order else 0
    alive, t_range = len(order), range(longest)
    counts = []
    for t in t_range:
        while alive and lengths[order[alive - 1]] <= t:
            alive -= 1
        counts.append(alive)
    for t in reversed(t_range) if backwards else t_range:
        yield starts[:counts[t]] + t, order_t[:counts[t]]


def exact(case, seed):
    op = case["op"]
    inputs = _inputs(case, seed)
    if op == "recurrence":
        state = (inputs["initial"].double() if case["initial"] else torch.zeros(
            (case["sequences"], case["channels"]), dtype=torch.float64, device=DEVICE))
        out = torch.zeros((case["rows"], case["channels"]), dtype=torch.float64, device=DEVICE)
        for rows, which in _walk(case, inputs, False):
            decay, left = _gate_values(case, inputs["gate"][rows].double())
            x = inputs["x"][rows].double()
            now = decay * state[which] + (left * x if case["complement"] else x)
            state[which] = now
            out[rows] = now
        return [out, state]
    if op == "recurrence_gradient":
        back = (inputs["grad_final"].double() if case["initial"] else torch.zeros(
            (case["sequences"], case["channels"]), dtype=torch.float64, device=DEVICE))
        grad_gate = torch.zeros((case["rows"], case["channels"]), dtype=torch.float64, device=DEVICE)
        grad_x = torch.zeros_like(grad_gate)
        starts = inputs["offsets"].long()
        for rows, which in _walk(case, inputs, True):
            decay, left = _gate_values(case, inputs["gate"][rows].double())
            x = inputs["x"][rows].double()
            at_start = (rows == starts[which])[:, None]
            first = inputs["initial"][which].double() if case["initial"] else torch.zeros_like(x)
            before = torch.where(at_start, first, inputs["out"][(rows - 1).clamp(min=0)].double())
            here = inputs["grad_out"][rows].double() + back[which]
            grad_x[rows] = here * left if case["complement"] else here
            by_decay = here * (before - x) if case["complement"] else here * before
            grad_gate[rows] = by_decay * decay * (left if case["decay"] == "sigmoid" else 1.0)
            back[which] = here * decay
        return [grad_gate, grad_x] + ([back] if case["initial"] else [])
    if op in ("norm", "norm_gradient"):
        n = case["columns"]
        x = inputs["x"].double()
        gate = inputs["gate"].double() if case["gate"] != "none" else None
        through = lambda t: torch.special.expit(t) * (t if case["gate"] == "silu" else 1.0)  # noqa: E731
        if op == "norm":
            input_rstd = None
            if case["input_norm"]:
                input_rstd = (torch.linalg.vector_norm(x, dim=1) ** 2 / n + EPSILON) ** -0.5
                x = x * input_rstd[:, None] * inputs["input_weight"].double()
            if gate is not None:
                x = x * through(gate)
            total = inputs["residual"].double() + x * case["scale"]
            rstd = (torch.linalg.vector_norm(total, dim=1) ** 2 / n + EPSILON) ** -0.5
            return total, total * rstd[:, None] * inputs["weight"].double(), input_rstd, rstd
        # A norm's gradient: what is along the normalised row is taken out of g * weight.
        def of_norm(g, hat, rstd):
            along = torch.linalg.vecdot(g, hat)[:, None] / n
            return rstd * torch.addcmul(g, along, hat, value=-1.0)

        rstd = inputs["rstd"].double()[:, None]
        hat = inputs["total"].double() * rstd
        grad = inputs["grad_out"].double()
        result = {"weight": torch.sum(hat * grad, 0), "gate": None, "input_weight": None}
        result["residual"] = inputs["grad_total"].double() + of_norm(
            grad * inputs["weight"].double(), hat, rstd)
        grad = result["residual"] * case["scale"]
        if case["input_norm"]:
            rstd = inputs["input_rstd"].double()[:, None]
            weight = inputs["input_weight"].double()
            hat = x * rstd
            x = hat * weight
        if gate is not None:
            s = torch.special.expit(gate)
            slope = s - s * s if case["gate"] == "sigmoid" else s + gate * (s - s * s)
            result["gate"] = grad * x * slope
            grad = grad * through(gate)
        if case["input_norm"]:
            result["input_weight"] = torch.sum(grad * hat, 0)
            grad = of_norm(grad * weight, hat, rstd)
        return {**result, "x": grad}
    # AdamW, tensor for tensor.
    beta1, beta2 = BETAS
    found = {"parameters": [], "first": [], "second": [], "first_scales": [], "second_scales": []}
    at = block = 0
    key = _mixed(((SEED & WORD) + STEP * 0x3C6EF373) & WORD)
    for number, gradient in enumerate(inputs["gradients"]):
        n = gradient.numel()
        g = gradient.double().flatten() / max(1.0, case["norm"] / inputs["max_norm"])
        m, v = inputs["first"][at:at + n].double(), inputs["second"][at:at + n].double()
        index = torch.arange(n, device=DEVICE)
        if case["states"] == 8:
            of_block = block + index // BLOCK
            m = torch.sign(m - 128) * ((m - 128) / 127) ** 2 * inputs["first_scales"][of_block]
            v = (v / 255) ** 4 * inputs["second_scales"][of_block]
        m = torch.lerp(g, m, beta1)
        v = torch.lerp(g ** 2, v, beta2)
        p = inputs["parameters"][at:at + n].double()
        slope = m / (1 - beta1 ** STEP) / (torch.sqrt(v / (1 - beta2 ** STEP)) + DAMPING)
        found["parameters"].append(p - RATE * (slope + DECAY * p))
        if case["states"] == 8:
            of_tensor = index // BLOCK
            word = _mixed((index * 0x9E3779B9 + _mixed(
                (key + (SEED >> 32) + number * 0x9E3779B9) & WORD)) & WORD)
            for name, values, chance, levels, power in (("first", m, word & 0xFFFF, 127, 2),
                                                        ("second", v, word >> 16, 255, 4)):
                size = values.abs()
                scale = torch.zeros(-(-n // BLOCK), dtype=torch.float64, device=DEVICE)
                scale.scatter_reduce_(0, of_tensor, size, "amax")
                steps = (size / scale[of_tensor]) ** (1.0 / power) * levels
                below = (steps * (1 + 1e-12)).floor()
                share = (steps ** power - below ** power) / ((below + 1) ** power - below ** power)
                code = below + (share > chance.double() / 65536)
                found[name].append(values.sign() * (code / levels) ** power * scale[of_tensor])
                found[name + "_scales"].append(scale)
            block += -(-n // BLOCK)
        else:
            found["first"].append(m)
            found["second"].append(v)
        at += n
    found = {k: torch.cat(v) for k, v in found.items() if v}
    return {**found, "copies": found["parameters"] if case["copies"] else None}
