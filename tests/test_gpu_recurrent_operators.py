"""The gated recurrence, the residual norm and the AdamW step through the C ABI against
their formulas in float64.

Tolerances follow from the arithmetic, not from measured differences.  With u = 2^-24
(float32):

  - a result is rounded to its type once;
  - a decay, what is left of it to 1 and their products are off by at most some units: the
    exponential by 4 u, a sum, a reciprocal and a product behind it by 8 u more, and a term of
    the state passes through one product a row and at most 13 joins a tile of at least 16
    rows.  STEP = 24 roundings a row cover it, each relative to the magnitudes of
    what is added up, which go through the same recurrence;
  - a sum of C elements by at least 64 lanes, or a block, takes L = C / 64 + 32 additions.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
STEP = 24
TYPES = ["float32", "float16", "bfloat16"]
KINDS = ["sigmoid", "exponential"]


def _t(name):
    import torch
    return getattr(torch, name)


def _u(dtype):
    import torch
    return {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]


def _tiny(dtype):
    import torch
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126


def _rng(*key):
    import torch
    return torch.Generator(device="cuda").manual_seed(
        sum(k * 1009 ** i for i, k in enumerate(key)) % (1 << 31))


def _normal(g, *shape, dtype):
    import torch
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _close(got, exact, slack):
    """|got - exact| <= slack + rounding to got's type, everywhere."""
    bound = slack + _u(got.dtype) * (exact.abs() + slack) + _tiny(got.dtype)
    off = (got.double() - exact).abs()
    worst = (off - bound).max() if off.numel() else None
    assert off.numel() == 0 or bool((off <= bound).all()), float(worst)


def _strided(t, stride, offset=0):
    """t's values as rows `stride` apart from `offset` elements into other memory, with NaN
    between them: (matrix tensor, the memory, its guard positions)."""
    import torch
    rows, columns = t.shape
    memory = torch.full((offset + rows * stride + 7,), float("nan"), dtype=t.dtype, device="cuda")
    view = torch.as_strided(memory, (rows, columns), (stride, 1), offset)
    view.copy_(t)
    guard = torch.ones(memory.numel(), dtype=torch.bool, device="cuda")
    torch.as_strided(guard, (rows, columns), (stride, 1), offset).fill_(False)
    return view, memory, guard


def _matrix(t):
    from ilgpu_amd import capi
    return None if t is None else capi.DeviceMatrix.from_tensor(t)


def _array(t):
    from ilgpu_amd import capi
    return None if t is None else capi.DeviceArray.from_tensor(t)


# ---- gated recurrence --------------------------------------------------------------
def _gates(g, rows, channels, kind, dtype):
    import torch
    gate = torch.randn(rows, channels, generator=g, device="cuda")
    gate += 5.0 * torch.rand(channels, generator=g, device="cuda")
    if kind == "exponential":
        gate = -torch.log1p(torch.exp(-gate))
    return gate.to(dtype)


def _decay(gate, kind):
    import torch
    gate = gate.double()
    if kind == "sigmoid":
        return torch.sigmoid(gate), torch.sigmoid(-gate)
    return torch.exp(gate), -torch.expm1(gate)


def _run(capi, gate, x, out, kind, complement, sequences=1, offsets=None, initial=None,
         final=None, **more):
    capi.gated_recurrence(_matrix(gate), _matrix(x), _matrix(out), sequences=sequences,
                          offsets=_array(offsets), initial=_matrix(initial),
                          final=_matrix(final), complement=complement,
                          decay=getattr(capi, "DECAY_" + kind.upper()), **more)


def _bounds(rows, sequences, offsets):
    return ([i * (rows // sequences) for i in range(sequences + 1)] if offsets is None
            else [int(o) for o in offsets.tolist()])


def _exact(gate, x, kind, complement, bounds, initial):
    """States and their error bounds, row after row, in float64 on the CPU; NaN in rows of no
    sequence.  Also the final states with theirs."""
    import torch
    a, left = (t.cpu() for t in _decay(gate, kind))
    b = x.double().cpu()
    if complement:
        b = b * left
    h = torch.full_like(b, float("nan"))
    slack = torch.zeros_like(b)
    final = torch.zeros(len(bounds) - 1, b.shape[1], dtype=torch.float64)
    final_slack = torch.zeros_like(final)
    for i, (begin, end) in enumerate(zip(bounds, bounds[1:])):
        now = (torch.zeros_like(b[0]) if initial is None else initial[i].double().cpu())
        size, off = now.abs(), torch.zeros_like(now)
        for t in range(begin, end):
            off = a[t] * off + STEP * U * (a[t] * size + b[t].abs())
            size = a[t] * size + b[t].abs()
            now = a[t] * now + b[t]
            h[t], slack[t] = now, off
        final[i], final_slack[i] = now, off
    return tuple(t.cuda() for t in (h, slack, final, final_slack))


def _check_recurrence(gate, x, kind, complement, sequences=1, offsets=None, initial=None, temp=None):
    import torch
    from ilgpu_amd import capi
    out = torch.full_like(x, 77.0)
    final = torch.full((sequences, x.shape[1]), float("nan"), device="cuda")
    _run(capi, gate, x, out, kind, complement, sequences, offsets, initial, final, temp=temp)
    bounds = _bounds(x.shape[0], sequences, offsets)
    h, slack, last, last_slack = _exact(gate, x, kind, complement, bounds, initial)
    rows = slice(bounds[0], bounds[-1])
    _close(out[rows], h[rows], slack[rows])
    _close(final, last, last_slack)
    left = torch.cat((out[:bounds[0]], out[bounds[-1]:]))
    assert bool((left == 77.0).all())      # rows of no sequence are left as they were
    return out, final


@pytest.mark.parametrize("complement", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels", [(1, 1), (1, 300), (2, 64), (31, 3), (33, 7), (64, 65),
                                           (127, 8), (129, 130), (257, 72), (1025, 100),
                                           (2100, 9)])
def test_recurrence(rows, channels, dtype, kind, complement):
    g = _rng(rows, channels)
    gate, x = _gates(g, rows, channels, kind, _t(dtype)), _normal(g, rows, channels, dtype=_t(dtype))
    _check_recurrence(gate, x, kind, complement)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("sequences,length", [(1, 1), (7, 1), (300, 1), (50, 2), (9, 33), (4, 256),
                                              (3, 700)])
def test_recurrence_of_equal_sequences_with_states(sequences, length, kind):
    import torch
    for dtype, channels in (("float32", 70), ("bfloat16", 136), ("float16", 5)):
        g = _rng(sequences, length, channels)
        rows = sequences * length
        gate, x = _gates(g, rows, channels, kind, _t(dtype)), _normal(g, rows, channels, dtype=_t(dtype))
        initial = torch.randn(sequences, channels, generator=g, device="cuda")
        _check_recurrence(gate, x, kind, True, sequences, None, initial)


RAGGED = {
    "one": [0, 900],
    "none": [0, 0],
    "empty ones": [0, 0, 0, 17, 17, 300, 300, 300, 901, 901, 901],
    "outside": [5, 6, 200, 200, 455, 456],
    "single rows": list(range(0, 701)),
    "tile borders": [0, 64, 128, 256, 257, 512, 767, 768, 1000],
    "many empty ones": [0] * 400 + [3] * 300 + [700] * 500,
}


@pytest.mark.parametrize("offset_type", ["int32", "int64"])
@pytest.mark.parametrize("way", sorted(RAGGED))
@pytest.mark.parametrize("dtype,channels", [("float32", 68), ("bfloat16", 129), ("float16", 6)])
def test_recurrence_of_ragged_sequences(dtype, channels, way, offset_type):
    import torch
    offsets = torch.tensor(RAGGED[way], dtype=_t(offset_type), device="cuda")
    g = _rng(channels, len(RAGGED[way]))
    rows, sequences = RAGGED[way][-1] + 40, len(RAGGED[way]) - 1
    gate = _gates(g, rows, channels, "sigmoid", _t(dtype))
    x = _normal(g, rows, channels, dtype=_t(dtype))
    initial = torch.randn(sequences, channels, generator=g, device="cuda")
    _check_recurrence(gate, x, "sigmoid", True, sequences, offsets, initial)
    _check_recurrence(gate, x, "sigmoid", False, sequences, offsets, None)


def test_recurrence_of_more_sequences_than_a_block_reads_at_a_time():
    import torch
    g = _rng(4)
    cuts = torch.randint(0, 3001, (70_001,), generator=g, device="cuda").sort().values
    gate, x = _gates(g, 3010, 24, "sigmoid", torch.bfloat16), _normal(g, 3010, 24, dtype=torch.bfloat16)
    initial = torch.randn(70_000, 24, generator=g, device="cuda")
    _check_recurrence(gate, x, "sigmoid", True, 70_000, cuts.int(), initial)


def test_recurrence_step_after_step_is_the_whole():
    import torch
    from ilgpu_amd import capi
    g = _rng(8)
    sequences, length, channels = 5, 40, 77
    gate = _gates(g, sequences * length, channels, "sigmoid", torch.float32)
    x = _normal(g, sequences * length, channels, dtype=torch.float32)
    out, final = _check_recurrence(gate, x, "sigmoid", True, sequences)
    state = torch.zeros(sequences, channels, device="cuda")
    gates, xs = (t.view(sequences, length, channels) for t in (gate, x))
    steps = torch.empty_like(xs)
    for t in range(length):       # the state is its own successor
        one = torch.empty(sequences, channels, device="cuda")
        _run(capi, gates[:, t].contiguous(), xs[:, t].contiguous(), one, "sigmoid", True, sequences,
             None, state, state)
        steps[:, t] = one
    _, slack, _, last = _exact(gate, x, "sigmoid", True, _bounds(sequences * length, sequences, None), None)
    _close(steps.view(-1, channels), out.double(), 2 * slack)
    _close(state, final.double(), 2 * last)


@pytest.mark.parametrize("dtype,channels", [("float32", 67), ("bfloat16", 70), ("bfloat16", 3)])
def test_recurrence_in_place_and_strided(dtype, channels):
    import torch
    from ilgpu_amd import capi
    g, rows, sequences = _rng(6, channels), 610, 10
    gate, x = _gates(g, rows, channels, "sigmoid", _t(dtype)), _normal(g, rows, channels, dtype=_t(dtype))
    initial = torch.randn(sequences, channels, generator=g, device="cuda")
    want = torch.empty_like(x)
    want_final = torch.empty_like(initial)
    _run(capi, gate, x, want, "sigmoid", True, sequences, None, initial, want_final)
    views = [_strided(t, channels + more, more) for more, t in
             ((1, gate), (3, x), (5, initial), (2, torch.zeros_like(x)), (7, torch.zeros_like(initial)))]
    out, final = views[3], views[4]
    _run(capi, views[0][0], views[1][0], out[0], "sigmoid", True, sequences, None, views[2][0], final[0])
    assert torch.equal(out[0], want) and torch.equal(final[0], want_final)
    for _, memory, guard in (out, final):
        assert bool(memory[guard].isnan().all())
    for over in (0, 1):           # over the gates, over the inputs, with the states in place
        both = [gate.clone(), x.clone()]
        state = initial.clone()
        _run(capi, both[0], both[1], both[over], "sigmoid", True, sequences, None, state, state)
        assert torch.equal(both[over], want) and torch.equal(state, want_final)
    # gates of one row for all, and initial states of one
    one = gate[:1].expand(rows, channels)
    _check_recurrence(one, x, "sigmoid", True, sequences, None, initial[:1].expand(sequences, channels))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", TYPES)
def test_recurrence_keeps_bad_values_to_their_sequences(dtype, bad):
    import torch
    from ilgpu_amd import capi
    g = _rng(9)
    bounds = [0, 10, 300, 300, 301, 640, 900]
    offsets = torch.tensor(bounds, device="cuda")
    gate, x = _gates(g, 930, 66, "sigmoid", _t(dtype)), _normal(g, 930, 66, dtype=_t(dtype))
    grad = _normal(g, 930, 66, dtype=_t(dtype))
    clean = torch.zeros_like(x)
    states = torch.zeros(6, 66, device="cuda")
    _run(capi, gate, x, clean, "sigmoid", False, 6, offsets, states)
    clean_grads = [torch.zeros_like(x), torch.zeros_like(x)]

    def gradients(gate, x, out, grad, states, to):
        capi.gated_recurrence_gradient(*(_matrix(t) for t in (grad, gate, x, out, *to)), sequences=6,
                                       offsets=_array(offsets), initial=_matrix(states))

    gradients(gate, x, clean, grad, states, clean_grads)
    for which in range(3):
        dirty = [gate.clone(), x.clone(), states.clone()]
        dirty_grad = grad.clone()
        if which == 2:
            dirty[2][1, 5] = dirty[2][4, 65] = bad
        else:
            for rows in (200, 299, 301, 639, 905):   # in sequences 1 and 4, and behind the last
                dirty[which][rows] = bad
            dirty_grad[10] = dirty_grad[639] = bad
        out = torch.zeros_like(x)
        final = torch.empty(6, 66, device="cuda")
        _run(capi, dirty[0], dirty[1], out, "sigmoid", False, 6, offsets, dirty[2], final)
        grads = [torch.zeros_like(x), torch.zeros_like(x)]
        gradients(dirty[0], dirty[1], clean, dirty_grad, dirty[2], grads)
        for i in (0, 3, 5):
            rows = slice(bounds[i], bounds[i + 1])
            assert torch.equal(out[rows], clean[rows])
            for got, want in zip(grads, clean_grads):
                assert torch.equal(got[rows], want[rows])
        assert bool(torch.isfinite(final[[0, 2, 3, 5]]).all())
        assert bool((out[900:] == 0).all()) and bool((grads[0][900:] == 0).all())


def test_recurrence_of_extreme_gates():
    # Open, shut and nearly so: the decay and what is left of it each keep their digits.
    import torch
    gate = torch.tensor([-float("inf"), -200.0, -100.0, -30.0, -1e-3, -1e-6, 0.0, 1e-6, 1e-3, 8.0,
                         16.6, 30.0, 90.0, 200.0, float("inf")], device="cuda")
    x = torch.linspace(0.5, 2.0, 15, device="cuda")
    initial = torch.linspace(-3.0, -1.0, 15, device="cuda")
    for complement in (False, True):
        _check_recurrence(gate[None], x[None], "sigmoid", complement, 1, None, initial[None])
        # (decays of more than 1 grow, up to infinity; that is the formula)
        shut = gate.clamp(max=1.0)
        _check_recurrence(shut[None], x[None], "exponential", complement, 1, None, initial[None])
        _check_recurrence(shut.expand(40, 15), x.expand(40, 15), "exponential", complement)
        # a step
        _check_recurrence(gate.expand(3, 15), x.expand(3, 15), "sigmoid", complement, 3, None,
                          initial.expand(3, 15))


def test_recurrence_forgets_nothing_it_should_keep():
    # A decay of 1 adds up: 20000 ones, exactly; and in a channel beside it everything is forgotten.
    import torch
    from ilgpu_amd import capi
    gate = torch.zeros(20_000, 2, device="cuda")
    gate[:, 1] = -float("inf")
    x = torch.ones(20_000, 2, device="cuda")
    out = torch.empty_like(x)
    _run(capi, gate, x, out, "exponential", False)
    assert torch.equal(out[:, 0], torch.arange(1.0, 20_001.0, device="cuda"))
    assert bool((out[:, 1] == 1.0).all())


def test_recurrence_gives_the_same_bits_again():
    import torch
    from ilgpu_amd import capi
    g = _rng(10)
    gate, x = _gates(g, 20_011, 136, "sigmoid", torch.bfloat16), _normal(g, 20_011, 136, dtype=torch.bfloat16)
    grad = _normal(g, 20_011, 136, dtype=torch.bfloat16)
    runs = []
    for _ in range(4):
        out, of_gate, of_x = (torch.empty_like(x) for _ in range(3))
        final, back = (torch.empty(1, 136, device="cuda") for _ in range(2))
        _run(capi, gate, x, out, "sigmoid", True, final=final)
        capi.gated_recurrence_gradient(*(_matrix(t) for t in (grad, gate, x, out, of_gate, of_x)),
                                       complement=True, grad_initial=_matrix(back))
        runs.append([t.view(torch.uint8).clone() for t in (out, final, of_gate, of_x, back)])
    for run in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(run, runs[0]))


def test_recurrence_of_no_rows_and_no_sequences():
    import torch
    from ilgpu_amd import capi
    none = torch.empty(0, 9, device="cuda")
    initial = torch.randn(4, 9, device="cuda")
    final = torch.full_like(initial, float("nan"))
    _run(capi, none, none, none, "sigmoid", True, 4, None, initial, final)
    assert torch.equal(final, initial)
    back = torch.full_like(initial, float("nan"))
    capi.gated_recurrence_gradient(*[_matrix(none)] * 6, sequences=4, grad_final=_matrix(initial),
                                   grad_initial=_matrix(back))
    assert torch.equal(back, initial)
    _run(capi, none, none, none, "sigmoid", True, 4, None, None, final)
    assert bool((final == 0).all())
    _run(capi, none, none, none, "sigmoid", True, 0)
    x = torch.ones(30, 9, device="cuda")
    out = torch.full_like(x, 5.0)
    _run(capi, x, x, out, "sigmoid", True, 0, torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert bool((out == 5.0).all())


def test_recurrence_of_rows_beyond_32_bit_offsets():
    import torch
    from ilgpu_amd import capi
    rows, stride = 70_001, 40_000          # 2.8 * 10^9 elements
    memory = torch.zeros(rows * stride + 64, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(memory, (rows, 16), (stride, 1), 0)
    out = torch.as_strided(memory, (rows, 16), (stride, 1), 16)
    x.fill_(1.0)
    gate = torch.full((1, 16), 1.0, device="cuda").bfloat16().expand(rows, 16)
    _run(capi, gate, x, out, "sigmoid", True)
    # h tends to 1
    assert bool((out[-1000:] == 1.0).all()) and float(out[0, 0]) < 0.5
    grads = torch.as_strided(memory, (rows, 16), (stride, 1), 32)
    capi.gated_recurrence_gradient(*(_matrix(t) for t in (x, gate, x, out, None, grads)), complement=True)
    assert bool((grads[0] - 1.0).abs().max() < 0.01)   # 1 - a of it, a of what comes behind, ...


def _gradient(capi, grad, gate, x, out, kind, complement, sequences, offsets, initial, grad_final,
              want=(True, True, True)):
    import torch
    to = [torch.full_like(x, 77.0) if w else None for w in want[:2]]
    back = torch.full((sequences, x.shape[1]), float("nan"), device="cuda") if want[2] else None
    capi.gated_recurrence_gradient(
        *(_matrix(t) for t in (grad, gate, x, out, *to)), sequences=sequences,
        offsets=_array(offsets), initial=_matrix(initial), grad_final=_matrix(grad_final),
        grad_initial=_matrix(back), decay=getattr(capi, "DECAY_" + kind.upper()),
        complement=complement)
    return (*to, back)


def _check_gradient(got, grad, gate, x, out, kind, complement, bounds, initial, grad_final):
    import torch
    a, left = (t.cpu() for t in _decay(gate, kind))
    slope = a * left if kind == "sigmoid" else a
    grad, xs, h = (t.double().cpu() for t in (grad, x, out))
    n = x.shape[1]
    reach, slack = torch.zeros_like(grad), torch.zeros_like(grad)
    before = torch.zeros_like(grad)
    back = torch.zeros(len(bounds) - 1, n, dtype=torch.float64)
    back_slack = torch.zeros_like(back)
    for i, (begin, end) in enumerate(zip(bounds, bounds[1:])):
        now = torch.zeros(n, dtype=torch.float64) if grad_final is None else grad_final[i].double().cpu()
        size, off = now.abs(), torch.zeros(n, dtype=torch.float64)
        for t in reversed(range(begin, end)):
            size, now = size + grad[t].abs(), now + grad[t]
            off = off + 2 * U * size
            reach[t], slack[t] = now, off
            off = a[t] * off + STEP * U * a[t] * size
            size, now = a[t] * size, a[t] * now
            before[t] = h[t - 1] if t > begin else 0.0 if initial is None else initial[i].double().cpu()
        back[i], back_slack[i] = now, off
    rows = slice(bounds[0], bounds[-1])
    distance = before - xs if complement else before
    sizes = before.abs() + (xs.abs() if complement else 0.0)
    exact_gate = reach * distance * slope
    slack_gate = (slack * distance.abs() + STEP * U * reach.abs() * sizes) * slope
    exact_x = reach * left if complement else reach
    slack_x = (slack + STEP * U * reach.abs()) * left.abs() if complement else slack
    for t, exact, off in ((got[0], exact_gate, slack_gate), (got[1], exact_x, slack_x)):
        if t is not None:
            _close(t[rows], exact[rows].cuda(), off[rows].cuda())
            assert bool((torch.cat((t[:rows.start], t[rows.stop:])) == 77.0).all())
    if got[2] is not None:
        _close(got[2], back.cuda(), back_slack.cuda())


@pytest.mark.parametrize("complement", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels", [(1, 1), (2, 64), (33, 7), (64, 65), (129, 130), (700, 72),
                                           (1300, 5)])
def test_recurrence_gradient(rows, channels, dtype, kind, complement):
    from ilgpu_amd import capi
    g = _rng(rows, channels, 2)
    gate, x, grad = (_gates(g, rows, channels, kind, _t(dtype)), _normal(g, rows, channels, dtype=_t(dtype)),
                     _normal(g, rows, channels, dtype=_t(dtype)))
    h, _, _, _ = _exact(gate, x, kind, complement, [0, rows], None)
    out = h.to(_t(dtype))
    got = _gradient(capi, grad, gate, x, out, kind, complement, 1, None, None, None)
    _check_gradient(got, grad, gate, x, out, kind, complement, [0, rows], None, None)


@pytest.mark.parametrize("way", ["equal"] + sorted(RAGGED))
@pytest.mark.parametrize("dtype,channels", [("float32", 68), ("bfloat16", 129), ("float16", 6)])
def test_recurrence_gradient_of_sequences(dtype, channels, way):
    import torch
    from ilgpu_amd import capi
    bounds = list(range(0, 1001, 100)) if way == "equal" else RAGGED[way]
    offsets = None if way == "equal" else torch.tensor(bounds, device="cuda")
    rows, sequences = bounds[-1] + (0 if way == "equal" else 33), len(bounds) - 1
    g = _rng(channels, sequences)
    gate, x, grad = (_gates(g, rows, channels, "sigmoid", _t(dtype)),
                     _normal(g, rows, channels, dtype=_t(dtype)), _normal(g, rows, channels, dtype=_t(dtype)))
    initial, grad_final = (torch.randn(sequences, channels, generator=g, device="cuda") for _ in range(2))
    for states in ((initial, grad_final), (None, None), (initial, None), (None, grad_final)):
        h, _, _, _ = _exact(gate, x, "sigmoid", True, bounds, states[0])
        out = h.nan_to_num(9.0).to(_t(dtype))
        got = _gradient(capi, grad, gate, x, out, "sigmoid", True, sequences, offsets, *states)
        _check_gradient(got, grad, gate, x, out, "sigmoid", True, bounds, *states)
    # parts of it, and over what is read
    for want in ((True, False, False), (False, True, False), (False, False, True)):
        some = _gradient(capi, grad, gate, x, out, "sigmoid", True, sequences, offsets, *states, want=want)
        for a, b in zip(some, got):
            assert a is None or torch.equal(a, b)
    used = slice(bounds[0], bounds[-1])
    for first, second in ((0, 1), (1, 2), (2, 0), (0, 2)):
        read = [grad.clone(), gate.clone(), x.clone()]
        state = grad_final.clone()
        capi.gated_recurrence_gradient(
            *(_matrix(t) for t in (*read, out, read[first], read[second])), sequences=sequences,
            offsets=_array(offsets), grad_final=_matrix(state), grad_initial=_matrix(state), complement=True)
        assert torch.equal(read[first][used], got[0][used]) and torch.equal(read[second][used], got[1][used])
        assert torch.equal(state, got[2])


# Many tiles of rows behind one another, and grids for which the gradients' tiles are longer.
@pytest.mark.parametrize("cuts", [None, [3, 3, 4000, 4001, 4001, 6400, 8170]])
@pytest.mark.parametrize("dtype,rows,channels", [("float32", 8321, 70), ("bfloat16", 16_700, 24),
                                                 ("float16", 16_500, 130), ("bfloat16", 8193, 799)])
def test_recurrence_and_gradient_of_many_tiles(dtype, rows, channels, cuts):
    import torch
    from ilgpu_amd import capi
    g = _rng(rows, channels)
    kind, complement = ("sigmoid", True) if cuts is None else ("exponential", False)
    bounds = [0, rows] if cuts is None else cuts
    sequences = len(bounds) - 1
    offsets = None if cuts is None else torch.tensor(cuts, device="cuda")
    gate, x, grad = (_gates(g, rows, channels, kind, _t(dtype)), _normal(g, rows, channels, dtype=_t(dtype)),
                     _normal(g, rows, channels, dtype=_t(dtype)))
    initial, grad_final = (torch.randn(sequences, channels, generator=g, device="cuda") for _ in range(2))
    out, _ = _check_recurrence(gate, x, kind, complement, sequences, offsets, initial)
    got = _gradient(capi, grad, gate, x, out, kind, complement, sequences, offsets, initial, grad_final)
    _check_gradient(got, grad, gate, x, out, kind, complement, bounds, initial, grad_final)
    again = _gradient(capi, grad, gate, x, out, kind, complement, sequences, offsets, initial, grad_final)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    # over what is read
    read, state = [grad.clone(), gate.clone()], grad_final.clone()
    capi.gated_recurrence_gradient(
        *(_matrix(t) for t in (read[0], read[1], x, out, read[0], read[1])), sequences=sequences,
        offsets=_array(offsets), initial=_matrix(initial), grad_final=_matrix(state),
        grad_initial=_matrix(state), decay=getattr(capi, "DECAY_" + kind.upper()), complement=complement)
    used = slice(bounds[0], bounds[-1])
    assert torch.equal(read[0][used], got[0][used]) and torch.equal(read[1][used], got[1][used])
    assert torch.equal(state, got[2])


def test_recurrence_gradient_against_differences():
    # In float32 with steps of 1/64: a difference is off by its curvature, of which a central one
    # keeps the third derivative, and by the roundings of the loss's terms over the step.
    import torch
    from ilgpu_amd import capi
    g = _rng(12)
    rows, channels, sequences = 45, 6, 3
    gate, x = _gates(g, rows, channels, "sigmoid", torch.float64), torch.randn(
        rows, channels, generator=g, device="cuda", dtype=torch.float64)
    initial = torch.randn(sequences, channels, generator=g, device="cuda", dtype=torch.float64)
    grad, grad_final = torch.randn_like(x), torch.randn_like(initial)
    bounds = [0, 15, 30, 45]

    def loss(gate, x, initial):
        h, _, final, _ = _exact(gate, x, "sigmoid", True, bounds, initial)
        return float((h * grad).sum() + (final * grad_final).sum())

    h, _, _, _ = _exact(gate, x, "sigmoid", True, bounds, initial)
    got = _gradient(capi, *(t.float() for t in (grad, gate, x, h)), "sigmoid", True, sequences, None,
                    initial.float(), grad_final.float())
    inputs = [gate, x, initial]
    for which in range(3):
        for row, channel in ((0, 0), (1, 3), (2, 5)):
            moved = []
            for sign in (1, -1):
                trial = [t.clone() for t in inputs]
                trial[which][row, channel] += sign * 1e-5
                moved.append(loss(*trial))
            # float64: the loss has some hundred terms of about 1, so a difference is good to 1e-9;
            # the gradient itself is in float32
            difference = (moved[0] - moved[1]) / 2e-5
            assert abs(float(got[which][row, channel]) - difference) < 1e-4 * max(1.0, abs(difference))


# ---- residual norm -------------------------------------------------------------------
def _rms(t, epsilon):
    return ((t * t).mean(1, keepdim=True) + epsilon).rsqrt()


def _act(gate, kind):
    import torch
    s = torch.sigmoid(gate)
    if kind == "sigmoid":
        return s, s * (1 - s), s * (1 - s)
    return gate * s, s * (1 + gate * (1 - s)), s + gate.abs() * s * (1 - s)


def _norm_inputs(g, rows, columns, dtype, residual_type, weight_type, gate, input_norm, residual=True):
    import torch
    s = {"x": _normal(g, rows, columns, dtype=dtype) * 1.5,
         "residual": _normal(g, rows, columns, dtype=residual_type) if residual else None,
         "gate": _normal(g, rows, columns, dtype=dtype) if gate else None, "kind": gate,
         "weight": (1 + 0.3 * torch.randn(columns, generator=g, device="cuda")).to(weight_type),
         "input_weight": (1 + 0.3 * torch.randn(columns, generator=g, device="cuda")).to(weight_type)
         if input_norm else None, "input_norm": input_norm, "scale": 0.7, "epsilon": 1e-5}
    return s


def _options(capi, s):
    return dict(scale=s["scale"], gate=_matrix(s["gate"]), input_norm=s["input_norm"],
                gate_kind=getattr(capi, "GATE_" + (s["kind"] or "silu").upper()),
                input_weight=_array(s["input_weight"]))


def _exact_norm(s):
    """total, out and both rstd in float64, with the slack of each."""
    import torch
    x = s["x"].double()
    lanes = (x.shape[1] / 64 + 40) * U
    y, input_rstd, off = x, None, 0.0
    if s["input_norm"]:
        input_rstd = _rms(x, s["epsilon"])
        y = x * input_rstd * (s["input_weight"].double() if s["input_weight"] is not None else 1.0)
        off = lanes
    if s["gate"] is not None:
        y = y * _act(s["gate"].double(), s["kind"])[0]
    scale = float(np.float32(s["scale"]))
    r = s["residual"].double() if s["residual"] is not None else torch.zeros_like(x)
    total = r + scale * y
    total_slack = (off + 32 * U) * (scale * y).abs() + 2 * U * total.abs()
    rstd = _rms(total, s["epsilon"])
    rstd_off = lanes + (total_slack * total_slack).mean(1, keepdim=True).sqrt() * rstd
    w = s["weight"].double() if s["weight"] is not None else 1.0
    out = total * rstd * w
    out_slack = (total_slack * rstd * (w.abs() if s["weight"] is not None else 1.0)
                 + (rstd_off + 8 * U) * out.abs())
    return total, total_slack, out, out_slack, input_rstd, lanes, rstd, rstd_off


def _norm(capi, s, total=True, out=True, statistics=True, over=None):
    import torch
    x = s["x"]
    rows = x.shape[0]
    kind = s["residual"].dtype if s["residual"] is not None else x.dtype
    got = {"total": torch.full(x.shape, 77.0, dtype=kind, device="cuda") if total else None,
           "out": torch.full_like(x, 77.0) if out else None,
           "rstd": torch.full((rows,), 77.0, device="cuda") if statistics else None,
           "input_rstd": torch.full((rows,), 77.0, device="cuda")
           if statistics and s["input_norm"] else None}
    got.update(over or {})
    capi.residual_norm(_matrix(x), _matrix(s["residual"]), _matrix(got["total"]), _matrix(got["out"]),
                       _array(s["weight"]), epsilon=s["epsilon"], rstd=_array(got["rstd"]),
                       input_rstd=_array(got["input_rstd"]), **_options(capi, s))
    return got


def _check_norm(got, s):
    total, total_slack, out, out_slack, input_rstd, input_off, rstd, rstd_off = _exact_norm(s)
    if got["total"] is not None:
        _close(got["total"], total, total_slack)
    if got["out"] is not None:
        _close(got["out"], out, out_slack)
    if got["rstd"] is not None:
        _close(got["rstd"], rstd[:, 0], (rstd * rstd_off)[:, 0])
    if got["input_rstd"] is not None:
        _close(got["input_rstd"], input_rstd[:, 0], (input_rstd * input_off)[:, 0])


COLUMNS = [1, 2, 3, 7, 8, 9, 64, 65, 127, 130, 256, 500, 512, 1000, 1024, 1025, 1537, 2048, 4096,
           4099, 8192, 8200, 16_384, 16_390, 33_000]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("columns", COLUMNS)
def test_residual_norm(columns, dtype):
    import torch
    from ilgpu_amd import capi
    for case, (gate, input_norm, residual_type, weight_type) in enumerate((
            (None, False, dtype, dtype), ("silu", True, "float32", "float32"),
            ("sigmoid", False, dtype, "float32"), (None, True, "float32", dtype))):
        rows = (1, 37, 300, 5)[case]
        s = _norm_inputs(_rng(columns, case), rows, columns, _t(dtype), _t(residual_type),
                         _t(weight_type), gate, input_norm)
        _check_norm(_norm(capi, s), s)


@pytest.mark.parametrize("columns", [9, 130, 1030, 5000, 40_000])
def test_residual_norm_parts_and_places(columns):
    import torch
    from ilgpu_amd import capi
    s = _norm_inputs(_rng(columns), 41, columns, torch.bfloat16, torch.bfloat16, torch.float32, "silu", True)
    whole = _norm(capi, s)
    _check_norm(whole, s)
    for parts in ((True, False, False), (False, True, False), (True, False, True), (False, True, True)):
        got = _norm(capi, s, *parts)
        for name in got:
            assert got[name] is None or torch.equal(got[name], whole[name]), name
    # over the residual, and over the input and the gate
    for a, b in (("residual", "x"), ("residual", "gate"), ("gate", "x"), ("x", "gate")):
        t = dict(s, x=s["x"].clone(), residual=s["residual"].clone(), gate=s["gate"].clone())
        got = _norm(capi, t, over={"total": t[a], "out": t[b]})
        assert torch.equal(got["total"], whole["total"]) and torch.equal(got["out"], whole["out"])
    t = dict(s, residual=s["residual"].clone())
    got = _norm(capi, t, out=False, statistics=False, over={"total": t["residual"]})
    assert torch.equal(got["total"], whole["total"])
    # strides, odd places, and a row that stands for all
    t = dict(s, x=_strided(s["x"], columns + 3, 1)[0], residual=_strided(s["residual"], columns + 5, 3)[0],
             gate=_strided(s["gate"], columns + 1, 5)[0])
    places = [_strided(torch.zeros_like(s["x"]), columns + 7, 3) for _ in range(2)]
    got = _norm(capi, t, over={"total": places[0][0], "out": places[1][0]})
    for (view, memory, guard), name in zip(places, ("total", "out")):
        assert torch.equal(view, whole[name]) and bool(memory[guard].isnan().all())
    t = dict(s, gate=s["gate"][:1].expand(41, columns), residual=s["residual"][3:4].expand(41, columns))
    _check_norm(_norm(capi, t), t)
    # without weights, without a residual: a plain norm
    t = dict(s, weight=None, input_weight=None, residual=None, gate=None, input_norm=False, scale=1.0)
    _check_norm(_norm(capi, t), t)
    t["input_norm"] = True
    _check_norm(_norm(capi, t), t)


def test_residual_norm_of_rows_of_zeros_infinities_and_shut_gates():
    import torch
    from ilgpu_amd import capi
    s = _norm_inputs(_rng(5), 6, 700, torch.bfloat16, torch.bfloat16, torch.float32, "silu", True)
    clean = _norm(capi, s)
    s["x"][1], s["residual"][1] = 0.0, 0.0
    s["x"][2, 5] = float("inf")
    s["residual"][3, 699] = float("nan")
    s["gate"][4] = -float("inf")          # nothing is added
    got = _norm(capi, s)
    assert bool((got["out"][1] == 0).all()) and bool(torch.isfinite(got["rstd"][1]))
    assert not bool(torch.isfinite(got["out"][2]).any()) or bool(got["out"][2].isnan().any())
    assert bool(got["out"][3].isnan().all())
    assert torch.equal(got["total"][4], s["residual"][4])
    for row in (0, 5):
        assert torch.equal(got["out"][row], clean["out"][row])
    s["gate"][4] = float("inf")
    assert bool(_norm(capi, s)["total"][4].isinf().any())


def _norm_gradient(capi, s, given, want=("x", "gate", "residual", "weight", "input_weight"), into=None,
                   accumulate=False, over=None):
    import torch
    x = s["x"]
    kind = given["total"].dtype
    like = {"x": x, "gate": s["gate"], "residual": given["total"],
            "weight": s["weight"] if given["grad_out"] is not None else None,
            "input_weight": s["input_weight"]}
    got = {k: torch.full(v.shape, 77.0, dtype=v.dtype, device="cuda") if v is not None and k in want else None
           for k, v in like.items()}
    for k, v in (into or {}).items():
        got[k] = v.clone()
    got.update(over or {})
    options = _options(capi, s)
    no_out = given["grad_out"] is None
    capi.residual_norm_gradient(
        _matrix(given["grad_out"]), _matrix(given["grad_total"]), _matrix(x),
        None if no_out else _matrix(given["total"]), _array(s["weight"]),
        None if no_out else _array(given["rstd"]), _matrix(got["x"]), _matrix(got["residual"]),
        _array(got["weight"]), grad_gate=_matrix(got["gate"]), input_rstd=_array(given["input_rstd"]),
        grad_input_weight=_array(got["input_weight"]), accumulate=accumulate, **options)
    return got


def _check_norm_gradient(got, s, given, into=None):
    import torch
    into = into or {}
    x = s["x"].double()
    rows, n = x.shape
    lanes = (n / 64 + 44) * U
    one = torch.ones(n, dtype=torch.float64, device="cuda")
    w = s["weight"].double() if s["weight"] is not None else one
    iw = s["input_weight"].double() if s["input_weight"] is not None else one
    d = torch.zeros_like(x)
    d_slack = torch.zeros_like(x)
    if given["grad_total"] is not None:
        d = d + given["grad_total"].double()
        d_slack = 2 * U * d.abs()
    if given["grad_out"] is not None:
        rstd = given["rstd"].double()[:, None]
        h = given["total"].double() * rstd
        grad = given["grad_out"].double()
        g = grad * w
        mean = (g * h).mean(1, keepdim=True)
        mean_off = lanes * (g * h).abs().mean(1, keepdim=True)
        d = d + rstd * (g - h * mean)
        d_slack = d_slack + rstd * (8 * U * (g.abs() + h.abs() * mean.abs()) + h.abs() * mean_off)
        if got["weight"] is not None:
            base = into["weight"].double() if "weight" in into else 0.0
            terms = (grad * h).abs().sum(0)
            _close(got["weight"], (grad * h).sum(0) + base, (rows + 8) * U * (terms + abs(base)))
    if got["residual"] is not None:
        _close(got["residual"], d, d_slack)
    scale = float(np.float32(s["scale"]))
    e, e_slack = d * scale, d_slack * scale + 2 * U * (d * scale).abs()
    k = x * given["input_rstd"].double()[:, None] if s["input_norm"] else x
    if s["gate"] is not None:
        act, slope, slope_size = _act(s["gate"].double(), s["kind"])
        y = k * iw if s["input_norm"] else k
        if got["gate"] is not None:
            _close(got["gate"], e * y * slope, e_slack * (y * slope).abs() + 24 * U * (e * y).abs() * slope_size)
        e, e_slack = e * act, e_slack * act.abs() + 16 * U * (e * act).abs()
    if s["input_norm"]:
        rstd = given["input_rstd"].double()[:, None]
        if got["input_weight"] is not None:
            base = into["input_weight"].double() if "input_weight" in into else 0.0
            terms = (e * k).abs().sum(0)
            _close(got["input_weight"], (e * k).sum(0) + base,
                   (rows + 8) * U * (terms + abs(base)) + (e_slack * k.abs()).sum(0))
        f, f_slack = e * iw, e_slack * iw.abs() + U * (e * iw).abs()
        mean = (f * k).mean(1, keepdim=True)
        mean_off = lanes * (f * k).abs().mean(1, keepdim=True) + (f_slack * k.abs()).mean(1, keepdim=True)
        e = rstd * (f - k * mean)
        e_slack = rstd * (f_slack + k.abs() * mean_off + 8 * U * (f.abs() + (k * mean).abs()))
    if got["x"] is not None:
        _close(got["x"], e, e_slack)


def _given(g, s, grad_out=True, grad_total=True):
    """What the forward call left, and the gradients that come in."""
    kind = s["residual"].dtype if s["residual"] is not None else s["x"].dtype
    total, _, _, _, input_rstd, _, rstd, _ = _exact_norm(s)
    shape = s["x"].shape
    return {"total": total.to(kind), "rstd": rstd[:, 0].float().contiguous(),
            "input_rstd": input_rstd[:, 0].float().contiguous() if s["input_norm"] else None,
            "grad_out": _normal(g, *shape, dtype=s["x"].dtype) if grad_out else None,
            "grad_total": _normal(g, *shape, dtype=kind) if grad_total else None}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("columns", COLUMNS)
def test_residual_norm_gradient(columns, dtype):
    from ilgpu_amd import capi
    for case, (gate, input_norm, residual_type, weight_type, outs) in enumerate((
            (None, False, dtype, dtype, (True, True)), ("silu", True, "float32", "float32", (True, True)),
            ("sigmoid", False, dtype, "float32", (True, False)), (None, True, "float32", dtype, (False, True)),
            ("silu", True, dtype, "float32", (True, False)))):
        rows = (1, 37, 300, 5, 1100)[case]
        g = _rng(columns, case, 3)
        s = _norm_inputs(g, rows, columns, _t(dtype), _t(residual_type), _t(weight_type), gate, input_norm)
        given = _given(g, s, *outs)
        _check_norm_gradient(_norm_gradient(capi, s, given), s, given)


@pytest.mark.parametrize("columns", [9, 130, 1030, 5000, 9000, 20_000])
def test_residual_norm_gradient_parts_accumulation_and_places(columns):
    import torch
    from ilgpu_amd import capi
    g = _rng(columns, 4)
    s = _norm_inputs(g, 333, columns, torch.bfloat16, torch.bfloat16, torch.float32, "silu", True)
    given = _given(g, s)
    whole = _norm_gradient(capi, s, given)
    _check_norm_gradient(whole, s, given)
    for name in whole:
        got = _norm_gradient(capi, s, given, want=(name,))
        assert torch.equal(got[name], whole[name]), name
    into = {k: torch.randn(columns, generator=g, device="cuda") for k in ("weight", "input_weight")}
    got = _norm_gradient(capi, s, given, into=into, accumulate=True)
    _check_norm_gradient(got, s, given, into)
    # each over another of what is read
    names = ["grad_out", "grad_total", "x", "gate", "total"]
    for shift in range(5):
        t = dict(s, x=s["x"].clone(), gate=s["gate"].clone())
        h = dict(given, **{k: given[k].clone() for k in ("grad_out", "grad_total", "total")})
        read = {**h, "x": t["x"], "gate": t["gate"]}
        over = {k: read[names[(i + shift) % 5]] for i, k in enumerate(("x", "gate", "residual"))}
        got = _norm_gradient(capi, t, h, over=over)
        for name in whole:
            assert torch.equal(got[name], whole[name]), (shift, name)
    # strides and odd places
    t = dict(s, x=_strided(s["x"], columns + 3, 1)[0], gate=_strided(s["gate"], columns + 1, 5)[0])
    h = dict(given, **{k: _strided(given[k], columns + 5, 3)[0] for k in ("grad_out", "grad_total", "total")})
    places = [_strided(torch.zeros_like(s["x"]), columns + 7, 3) for _ in range(3)]
    got = _norm_gradient(capi, t, h, over=dict(zip(("x", "gate", "residual"), (p[0] for p in places))))
    for name in whole:
        assert torch.equal(got[name], whole[name]), name
    for _, memory, guard in places:
        assert bool(memory[guard].isnan().all())


def test_residual_norm_gradient_of_no_rows():
    import torch
    from ilgpu_amd import capi
    s = _norm_inputs(_rng(3), 0, 70, torch.float32, torch.float32, torch.float32, "silu", True)
    given = {"total": s["x"], "rstd": torch.empty(0, device="cuda"), "input_rstd": torch.empty(0, device="cuda"),
             "grad_out": s["x"], "grad_total": s["x"]}
    got = _norm_gradient(capi, s, given)
    assert bool((got["weight"] == 0).all()) and bool((got["input_weight"] == 0).all())
    into = {k: torch.ones(70, device="cuda") for k in ("weight", "input_weight")}
    got = _norm_gradient(capi, s, given, into=into, accumulate=True)
    assert bool((got["weight"] == 1).all()) and bool((got["input_weight"] == 1).all())
    got = _norm(capi, s)
    assert got["out"].numel() == 0


def test_residual_norm_gradient_against_differences():
    import torch
    from ilgpu_amd import capi
    g = _rng(14)
    s = _norm_inputs(g, 7, 19, torch.float64, torch.float64, torch.float64, "silu", True)
    grad_out, grad_total = (_normal(g, 7, 19, dtype=torch.float64) for _ in range(2))

    def loss(s):
        total, _, out, *_ = _exact_norm(s)
        return float((total * grad_total).sum() + (out * grad_out).sum())

    f = {k: v.float() if hasattr(v, "float") else v for k, v in s.items()}
    given = _given(g, f)
    given.update(grad_out=grad_out.float(), grad_total=grad_total.float())
    got = _norm_gradient(capi, f, given)
    for name in ("x", "gate", "residual", "weight", "input_weight"):
        for at in (0, 11, s[name].numel() - 1):
            moved = []
            for sign in (1, -1):
                trial = dict(s, **{name: s[name].clone()})
                trial[name].view(-1)[at] += sign * 1e-5
                moved.append(loss(trial))
            # (float64, terms of about 1; the gradient itself is in float32)
            difference = (moved[0] - moved[1]) / 2e-5
            assert abs(float(got[name].view(-1)[at]) - difference) < 1e-4 * max(1.0, abs(difference)), name


def test_residual_norm_of_rows_beyond_32_bit_offsets():
    import torch
    from ilgpu_amd import capi
    rows, stride = 70_001, 40_000
    memory = torch.zeros(rows * stride + 512, dtype=torch.bfloat16, device="cuda")

    def part(at):
        return torch.as_strided(memory, (rows, 100), (stride, 1), at)

    x = part(0)
    x[-3:] = torch.randn(3, 100, device="cuda").bfloat16()
    w = torch.ones(100, device="cuda")
    rstd = torch.empty(rows, device="cuda")
    capi.residual_norm(_matrix(x), None, _matrix(part(100)), _matrix(part(200)), _array(w), rstd=_array(rstd))
    exact = x[-3:].double() * _rms(x[-3:].double(), 1e-5)
    _close(part(200)[-3:], exact, 60 * U * exact.abs())
    assert torch.equal(part(100), x) and bool((part(200)[:-3] == 0).all())
    capi.residual_norm_gradient(_matrix(x), None, _matrix(x), _matrix(part(100)), _array(w), _array(rstd),
                                _matrix(part(300)), _matrix(part(400)))
    # the gradient along the row itself is nearly nothing, that of rows of zeros is zero
    assert bool((part(300)[:-3] == 0).all()) and float(part(300)[-3:].abs().max()) < 0.02


# ---- AdamW ----------------------------------------------------------------------------
BLOCK = 256
WORD = 0xFFFFFFFF


def _mixed(x):
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & WORD
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & WORD
    return x ^ (x >> 16)


def _values(codes, scales, second):
    """What 8-bit moments stand for, in float64."""
    import torch
    at = torch.arange(codes.numel(), device="cuda") // BLOCK
    c = codes.double()
    return ((c / 255) ** 4 if second else (c - 128) * (c - 128).abs() / 127 ** 2) * scales.double()[at]


def _adam_state(g, sizes, types, eight, copies=None, fresh=False):
    import torch
    s = {"p": [_normal(g, n, dtype=_t(types[0])) * 0.1 for n in sizes],
         "g": [_normal(g, n, dtype=_t(types[1])) * 0.01 for n in sizes],
         "copies": [torch.full((n,), 77.0, dtype=_t(copies), device="cuda") for n in sizes] if copies else None,
         "step": torch.tensor([1 if fresh else 7], device="cuda")}
    if not eight:
        s["m"] = [torch.randn(n, generator=g, device="cuda") * (0.0 if fresh else 0.01) for n in sizes]
        s["v"] = [(torch.randn(n, generator=g, device="cuda") * (0.0 if fresh else 0.01)) ** 2 for n in sizes]
        s["ms"] = s["vs"] = None
    else:
        def codes(low, n):
            return torch.randint(low, 256, (n,), generator=g, device="cuda", dtype=torch.uint8)

        def scales(n, size):
            return size * (0.0 if fresh else 1.0) * (0.5 + torch.rand(-(-n // BLOCK), generator=g, device="cuda"))

        s["m"], s["v"] = [codes(1, n) for n in sizes], [codes(0, n) for n in sizes]
        s["ms"], s["vs"] = [scales(n, 0.03) for n in sizes], [scales(n, 1e-3) for n in sizes]
    return s


def _list(tensors):
    from ilgpu_amd import capi
    return None if tensors is None else capi.TensorList([_array(t) for t in tensors])


OPTIONS = dict(rate=1e-2, betas=(0.9, 0.99), epsilon=1e-8, weight_decay=0.1)


def _adamw(capi, s, stream=None, **more):
    capi.adamw(_list(s["p"]), _list(s["g"]), _list(s["m"]), _list(s["v"]), _array(s["step"]),
               first_scales=_list(s["ms"]), second_scales=_list(s["vs"]), copies=_list(s["copies"]),
               stream=stream, **{**OPTIONS, **more})


def _clone(s):
    return {k: [t.clone() for t in v] if isinstance(v, list) else v.clone() if v is not None else None
            for k, v in s.items()}


def _check_adamw(after, before, factor=1.0, rate=1.0, seed=0, only=None, **more):
    import torch
    o = {**OPTIONS, **more}
    b1, b2 = o["betas"]
    t = int(before["step"][0])
    c1, c2 = 1 - b1 ** t, 1 - b2 ** t
    r = o["rate"] * rate
    eight = before["ms"] is not None
    for k in range(len(before["p"])) if only is None else only:
        p, g = before["p"][k].double(), before["g"][k].double() * factor
        if p.numel() == 0:
            continue
        if eight:
            m, v = _values(before["m"][k], before["ms"][k], False), _values(before["v"][k], before["vs"][k], True)
        else:
            m, v = before["m"][k].double(), before["v"][k].double()
        m_size = b1 * m.abs() + (1 - b1) * g.abs()
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        root = (v / c2).sqrt() + o["epsilon"]
        exact = p - r * (m / c1 / root + o["weight_decay"] * p)
        slack = 4 * U * p.abs() * (1 + r * o["weight_decay"]) + r * 40 * U * m_size / c1 / root
        _close(after["p"][k], exact, slack)
        if after["copies"] is not None:
            _close(after["copies"][k], exact, slack)
        if not eight:
            _close(after["m"][k], m, 8 * U * m_size)
            _close(after["v"][k], v, 8 * U * v)
            continue
        # The scales are the largest of each block, the codes those that the hash chooses; values so
        # near to the border that roundings (some 40 u of the value) decide may go either way.
        n = p.numel()
        index = torch.arange(n, device="cuda")
        key = _mixed(((seed & WORD) + t * 0x3C6EF373) & WORD)
        key = _mixed((key + (seed >> 32 & WORD) + k * 0x9E3779B9) & WORD)
        word = _mixed((index * 0x9E3779B9 + key) & WORD)
        for codes, scales, values, size, power, levels, chance in (
                (after["m"][k].long() - 128, after["ms"][k], m, m_size, 2, 127, word & 0xFFFF),
                (after["v"][k].long(), after["vs"][k], v, v, 4, 255, word >> 16)):
            largest = torch.zeros(-(-n // BLOCK), dtype=torch.float64, device="cuda")
            largest.scatter_reduce_(0, index // BLOCK, values.abs(), "amax")
            sizes = torch.zeros_like(largest).scatter_reduce_(0, index // BLOCK, size, "amax")
            _close(scales, largest, 40 * U * sizes)
            scale = largest[index // BLOCK]
            there = scale > 2.0 ** -125
            share = torch.where(there, values.abs() / scale.clamp(min=1e-300), 0.0)
            z = share * levels ** power
            low = z.pow(1.0 / power).floor().clamp(0, levels)
            way = (z - low ** power) / ((low + 1) ** power - low ** power)
            u = chance.double() / 65536
            want = (low + (way > u)).clamp(max=levels)
            off = 80 * U * (z + size / scale.clamp(min=1e-300) * levels ** power) / (
                (low + 1) ** power - low ** power)
            # A value on a code, give or take `off`, is that code, or the one below with all the way to
            # it: only a chance of nearly 1, or of nearly 0 where it is the one above, tells them apart.
            unsure = ((way - u).abs() <= 2 * off) | ((way <= off) & (u >= 1 - 4 * off)) | (
                (way >= 1 - off) & (u <= 4 * off)) | ~there
            got = codes.abs().double()
            assert bool(((got == want) | unsure).all())
            assert bool(((got - want).abs() <= 1)[there].all())
            assert float(unsure[there].double().mean()) < 0.02 + 64 / n
            assert bool((codes[there & (got > 0)].sign() == values[there & (got > 0)].sign()).all())


SIZES = {"few": [5, 1, 300], "blocks": [256, 255, 257, 1024, 4096, 4097, 0, 1000],
         "many": [(37 * i) % 1500 for i in range(120)], "long": [300_007, 3, 65_536]}


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("types", [("float32", "float32", None), ("float32", "bfloat16", "bfloat16"),
                                   ("bfloat16", "bfloat16", None), ("float16", "float16", "float32"),
                                   ("float32", "float16", "float16")])
@pytest.mark.parametrize("sizes", sorted(SIZES))
def test_adamw(sizes, types, eight):
    from ilgpu_amd import capi
    for fresh in (False, True):
        s = _adam_state(_rng(len(sizes), fresh), SIZES[sizes], types, eight, types[2], fresh)
        before = _clone(s)
        _adamw(capi, s, seed=12345678901)
        _check_adamw(s, before, seed=12345678901)


@pytest.mark.parametrize("eight", [False, True])
def test_adamw_clips_schedules_and_counts_on_the_device(eight):
    import torch
    from ilgpu_amd import capi
    s = _adam_state(_rng(3), [700, 5000], ("float32", "float32", None), eight)
    norm, schedule = torch.tensor([4.0], device="cuda"), torch.tensor([0.25], device="cuda")
    for t in (1, 2, 1000, 1_000_000, 3_000_000_000):
        s["step"][0] = t
        before = _clone(s)
        _adamw(capi, s, norm=_array(norm), max_norm=1.0, schedule=_array(schedule))
        _check_adamw(s, before, factor=0.25, rate=0.25)
    before = _clone(s)
    _adamw(capi, s, norm=_array(norm), max_norm=5.0)        # within the limit
    _check_adamw(s, before)
    norm[0] = 3e38          # a factor below the normal numbers
    for t in s["g"]:
        t.mul_(3e38)
    before = _clone(s)
    _adamw(capi, s, norm=_array(norm), max_norm=1.0)
    _check_adamw(s, before, factor=1.0 / float(norm[0]))
    for bad in (float("inf"), float("nan"), -float("inf")):
        norm[0] = bad
        before = _clone(s)
        _adamw(capi, s, norm=_array(norm), max_norm=1.0)
        for k in ("p", "m", "v", "ms", "vs"):
            assert before[k] is None or all(torch.equal(a, b) for a, b in zip(s[k], before[k]))


def test_adamw_without_decay_momentum_or_rate():
    from ilgpu_amd import capi
    for more in (dict(weight_decay=0.0), dict(betas=(0.0, 0.0)), dict(rate=0.0), dict(epsilon=1.0),
                 dict(betas=(0.999, 0.9999), epsilon=1e-15)):
        for eight in (False, True):
            s = _adam_state(_rng(5), [900], ("float32", "float32", None), eight)
            before = _clone(s)
            _adamw(capi, s, **more)
            _check_adamw(s, before, **more)


def test_adamw_of_unaligned_tensors_and_what_lies_beside_them():
    import torch
    from ilgpu_amd import capi
    for eight in (False, True):
        s = _adam_state(_rng(6), [1003, 258, 7], ("float32", "bfloat16", None), eight, "float16")
        want = _clone(s)
        _adamw(capi, want)
        memory = {}
        for k in ("p", "g", "m", "v", "ms", "vs", "copies"):
            if s[k] is None:
                continue
            flat = torch.full((sum(t.numel() + 3 for t in s[k]) + 8,), 99, dtype=s[k][0].dtype, device="cuda")
            at, guard = 1, torch.ones(flat.numel(), dtype=torch.bool, device="cuda")
            for i, t in enumerate(s[k]):
                flat[at:at + t.numel()] = t
                guard[at:at + t.numel()] = False
                s[k][i] = flat[at:at + t.numel()]
                at += t.numel() + 3
            memory[k] = flat, guard
        _adamw(capi, s)
        for k, (flat, guard) in memory.items():
            assert bool((flat[guard] == 99).all()), k
            assert all(torch.equal(a, b) for a, b in zip(s[k], want[k])), k


def test_adamw_moments_of_very_small_and_of_bad_gradients():
    import torch
    from ilgpu_amd import capi
    s = _adam_state(_rng(7), [1024], ("float32", "float32", None), True, fresh=True)
    s["g"][0][:256] = torch.randn(256, device="cuda") * 1e-13    # v of 1e-28
    s["g"][0][256:512] = 1e-30                                   # v below the normal numbers
    s["g"][0][512:768] = 0.0
    s["g"][0][800] = float("nan")
    before = _clone(s)
    _adamw(capi, s)
    first, second = torch.empty(1024, device="cuda"), torch.empty(1024, device="cuda")
    capi.adamw_moments(_list(s["m"]), _list(s["ms"]), _list([first]), _list(s["v"]), _list(s["vs"]), _list([second]))
    assert bool((second[256:768] == 0).all()) and bool((first[512:768] == 0).all())
    assert bool(first[768:].isnan().all()) and bool(second[768:].isnan().all())
    assert bool(torch.isfinite(s["p"][0][:768]).all()) and bool(torch.isfinite(first[:768]).all())
    assert float(second[:256].max()) > 1e-28
    for t in (s, before):
        for k in ("p", "g", "m", "v"):
            t[k][0] = t[k][0][:256]
        for k in ("ms", "vs"):
            t[k][0] = t[k][0][:1]
    _check_adamw(s, before)


def test_adamw_moments_in_8_bits_are_right_in_the_mean():
    # Gradients of nothing: the second moment falls by a hundredth a step, less than a code's
    # distance, and the first by a tenth.  A rounding is right in the mean and at most one code's
    # distance away; of n elements and k steps the mean is off by distance * sqrt(k / n) times the
    # chance's deviation (1/2 at most): four of those.
    import torch
    from ilgpu_amd import capi
    n, steps = 1 << 17, 50
    s = _adam_state(_rng(8), [n], ("float32", "float32", None), True)
    s["m"][0][::BLOCK], s["v"][0][::BLOCK] = 255, 255    # (the scale falls with the largest)
    s["g"][0].zero_()
    start = [_values(s["m"][0], s["ms"][0], False), _values(s["v"][0], s["vs"][0], True)]
    for _ in range(steps):
        _adamw(capi, s, betas=(0.99, 0.99), rate=0.0)
        s["step"] += 1
    end = [_values(s["m"][0], s["ms"][0], False), _values(s["v"][0], s["vs"][0], True)]
    for a, b, distance, largest in ((start[0], end[0], 2 / 127, s["ms"][0]), (start[1], end[1], 4 / 255, s["vs"][0])):
        b = b / 0.99 ** steps
        off = abs(float((a - b).mean()))
        unit = distance * float(largest.max()) / 0.99 ** steps
        assert off < 4 * 0.5 * unit * math.sqrt(steps / n)
        assert float((a - b).abs().max()) > 0.1 * unit       # single ones do move


@pytest.mark.parametrize("target", TYPES)
def test_adamw_moments(target):
    import torch
    from ilgpu_amd import capi
    sizes = [3, 256, 0, 700, 5001] * 30
    s = _adam_state(_rng(9), sizes, ("float32", "float32", None), True)
    first, second = ([torch.full((n,), 77.0, dtype=_t(target), device="cuda") for n in sizes] for _ in range(2))
    capi.adamw_moments(_list(s["m"]), _list(s["ms"]), _list(first))
    capi.adamw_moments(second=_list(s["v"]), second_scales=_list(s["vs"]), second_targets=_list(second))
    for k in range(len(sizes)):
        for got, codes, scales, which in ((first, s["m"], s["ms"], False), (second, s["v"], s["vs"], True)):
            exact = _values(codes[k], scales[k], which) if sizes[k] else torch.empty(0, device="cuda").double()
            _close(got[k], exact, 8 * U * exact.abs())


def test_adamw_of_a_tensor_beyond_32_bits():
    import torch
    from ilgpu_amd import capi
    n = (1 << 31) + 4099
    for eight in (False, True):
        blocks = -(-n // BLOCK)
        kind = torch.uint8 if eight else torch.float32
        s = {"p": [torch.ones(n, dtype=torch.bfloat16, device="cuda")],
             "g": [torch.zeros(n, dtype=torch.bfloat16, device="cuda")],
             "m": [torch.zeros(n, dtype=kind, device="cuda")], "v": [torch.zeros(n, dtype=kind, device="cuda")],
             "ms": [torch.zeros(blocks, device="cuda")] if eight else None,
             "vs": [torch.zeros(blocks, device="cuda")] if eight else None, "copies": None,
             "step": torch.tensor([1], device="cuda")}
        s["g"][0][-1] = 1.0
        _adamw(capi, s, weight_decay=0.0, rate=0.5)
        assert float(s["p"][0][-1]) == 0.5 and bool((s["p"][0][-5000:-1] == 1.0).all())
        assert float(s["p"][0][0]) == 1.0 and float(s["p"][0][1 << 31]) == 1.0
        if eight:
            assert int(s["m"][0][-1]) == 255 and int(s["v"][0][-1]) == 255 and float(s["ms"][0][-1]) > 0.09
        else:
            assert abs(float(s["m"][0][-1]) - 0.1) < 1e-6


# ---- together, on other streams, in graphs ----------------------------------------------
def _together(torch, capi, rows=700, channels=264, sequences=7):
    """A recurrent block forwards and backwards, and the step of its weights: state and views."""
    g = _rng(rows, channels)
    bf, f = torch.bfloat16, torch.float32
    t = {"gate": _gates(g, rows, channels, "sigmoid", bf), "x": _normal(g, rows, channels, dtype=bf),
         "act": _normal(g, rows, channels, dtype=bf), "residual": _normal(g, rows, channels, dtype=bf),
         "grad_out": _normal(g, rows, channels, dtype=bf), "grad_total": _normal(g, rows, channels, dtype=bf),
         "weights": 1 + 0.1 * torch.randn(2 * channels, generator=g, device="cuda"),
         "m": torch.zeros(2 * channels, device="cuda"), "v": torch.zeros(2 * channels, device="cuda"),
         "m8": torch.zeros(2 * channels, dtype=torch.uint8, device="cuda"),
         "v8": torch.zeros(2 * channels, dtype=torch.uint8, device="cuda"),
         "ms": torch.zeros(2 * -(-channels // BLOCK), device="cuda"),
         "vs": torch.zeros(2 * -(-channels // BLOCK), device="cuda"),
         "weights8": torch.ones(2 * channels, device="cuda"),
         "step": torch.zeros(1, dtype=torch.int64, device="cuda"),
         "offsets": torch.tensor([0, 5, 5, 300, 301, 500, 600, 650], dtype=torch.int32, device="cuda"),
         "initial": torch.randn(sequences, channels, generator=g, device="cuda")}
    for k in ("h", "total", "out", "grad_h", "grad_act", "grad_residual", "grad_gate", "grad_x"):
        t[k] = torch.zeros(rows, channels, dtype=bf, device="cuda")
    for k in ("rstd", "input_rstd"):
        t[k] = torch.empty(rows, device="cuda")
    for k in ("final", "grad_initial"):
        t[k] = torch.empty(sequences, channels, device="cuda")
    t["grads"] = torch.empty(2 * channels, dtype=f, device="cuda")
    t["norm"] = torch.empty(1, device="cuda")
    t["_views"] = v = {k: _matrix(a) if a.dim() == 2 else _array(a) for k, a in t.items()}
    for k in ("weights", "m", "v", "m8", "v8", "weights8", "grads"):
        v[k + "_list"] = _list([t[k][:channels], t[k][channels:]])
    for k in ("ms", "vs"):
        v[k + "_list"] = _list(t[k].chunk(2))
    v["w"], v["iw"] = _array(t["weights"][:channels]), _array(t["weights"][channels:])
    v["gw"], v["giw"] = _array(t["grads"][:channels]), _array(t["grads"][channels:])
    t["_temps"] = [capi.temp_buffer(n) for n in (capi.gated_recurrence_temp_bytes(rows, channels),
                                                 capi.residual_norm_gradient_temp_bytes(rows, channels),
                                                 capi.gradient_norm_temp_bytes(2))]
    return t


def _train(torch, capi, t, stream=None):
    v = t["_views"]
    sequences = dict(sequences=7, offsets=v["offsets"], initial=v["initial"], complement=True, stream=stream)
    gate = dict(gate=v["act"], gate_kind=capi.GATE_SILU, input_weight=v["iw"], scale=0.5, stream=stream)
    capi.gated_recurrence(v["gate"], v["x"], v["h"], t["_temps"][0], final=v["final"], **sequences)
    capi.residual_norm(v["h"], v["residual"], v["total"], v["out"], v["w"], input_rstd=v["input_rstd"],
                       rstd=v["rstd"], **gate)
    capi.residual_norm_gradient(
        v["grad_out"], v["grad_total"], v["h"], v["total"], v["w"], v["rstd"], v["grad_h"],
        v["grad_residual"], v["gw"], t["_temps"][1], grad_gate=v["grad_act"], input_rstd=v["input_rstd"],
        grad_input_weight=v["giw"], **gate)
    capi.gated_recurrence_gradient(v["grad_h"], v["gate"], v["x"], v["h"], v["grad_gate"], v["grad_x"],
                                   t["_temps"][0], grad_initial=v["grad_initial"], **sequences)
    capi.gradient_norm(v["grads_list"], v["norm"], t["_temps"][2], stream=stream)
    capi.adamw(v["weights_list"], v["grads_list"], v["m_list"], v["v_list"], v["step"], rate=0.01,
               norm=v["norm"], max_norm=1.0, stream=stream)
    capi.adamw(v["weights8_list"], v["grads_list"], v["m8_list"], v["v8_list"], v["step"], rate=0.01,
               first_scales=v["ms_list"], second_scales=v["vs_list"], norm=v["norm"], max_norm=1.0,
               stream=stream)


def _results(t):
    return {k: a.clone() for k, a in t.items() if not k.startswith("_")}


def test_operators_together_in_a_graph():
    import torch
    from ilgpu_amd import capi
    eager, graphed = _together(torch, capi), _together(torch, capi)
    capi.lib()
    for t in (eager, graphed):
        t["step"] += 1
        _train(torch, capi, t)
        t["step"] += 1
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _train(torch, capi, graphed)
        graphed["step"] += 1
    for turn in range(4):
        _train(torch, capi, eager)
        eager["step"] += 1
        graph.replay()
        torch.cuda.synchronize()
        a, b = _results(eager), _results(graphed)
        for k in a:
            assert torch.equal(a[k].view(torch.uint8), b[k].view(torch.uint8)), (turn, k)
        for t in (eager, graphed):       # new inputs, and other work in between
            t["x"].copy_(torch.randn(t["x"].shape, generator=_rng(turn), device="cuda"))
            t["gate"].copy_(torch.randn(t["x"].shape, generator=_rng(turn, 1), device="cuda"))
            t["grad_out"].mul_(1.5)


def test_operators_together_on_another_stream():
    import torch
    from ilgpu_amd import capi
    want, got = _together(torch, capi), _together(torch, capi)
    for t in (want, got):
        t["step"] += 1
    _train(torch, capi, want)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    _train(torch, capi, got, stream)
    stream.synchronize()
    a, b = _results(want), _results(got)
    for k in a:
        assert torch.equal(a[k].view(torch.uint8), b[k].view(torch.uint8)), k


def test_scans_on_two_streams_at_once():
    import torch
    from ilgpu_amd import capi
    g = _rng(40)
    gate, x = _gates(g, 30_000, 200, "sigmoid", torch.bfloat16), _normal(g, 30_000, 200, dtype=torch.bfloat16)
    want = torch.empty_like(x)
    _run(capi, gate, x, want, "sigmoid", True)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [torch.empty_like(x) for _ in streams]
    temps = [capi.temp_buffer(capi.gated_recurrence_temp_bytes(30_000, 200)) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(3):
        for stream, out, temp in zip(streams, outs, temps):
            _run(capi, gate, x, out, "sigmoid", True, temp=temp, stream=stream)
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for out in outs)


def test_a_temp_serves_fewer_rows():
    import torch
    from ilgpu_amd import capi
    g = _rng(41)
    gate, x = _gates(g, 5000, 72, "sigmoid", torch.float32), _normal(g, 5000, 72, dtype=torch.float32)
    temp = capi.temp_buffer(capi.gated_recurrence_temp_bytes(5000, 72))
    for rows in (5000, 4001, 300, 64, 1):
        _check_recurrence(gate[:rows], x[:rows], "sigmoid", True, temp=temp)
