"""The gated recurrence, the residual norm and the AdamW step at the ends of their ranges, against
their formulas in float64.

Inputs and tolerances are those of test_gpu_recurrent_operators, which says where they come from;
u = 2^-24 here too.
"""
import pytest

from tests.test_gpu_recurrent_operators import (
    BLOCK, KINDS, TYPES, U, WORD, _adam_state, _adamw, _array, _check_adamw, _check_gradient,
    _check_recurrence, _clone, _close, _gradient, _matrix, _mixed, _normal, _rng, _run, _t)

pytestmark = pytest.mark.gpu


# ---- decays whose product over some rows leaves float32 ------------------------------------
# Rows whose gates add up to more than 88.7 grow beyond float32 together, whatever comes in.
@pytest.mark.parametrize("backwards", [False, True])
@pytest.mark.parametrize("dtype,rows,channels", [("float32", 700, 70), ("float16", 900, 136),
                                                 ("bfloat16", 900, 136), ("bfloat16", 300, 3),
                                                 ("bfloat16", 17_000, 24)])
def test_growing_decays_leave_nothing_where_nothing_comes_in(dtype, rows, channels, backwards):
    import torch
    from ilgpu_amd import capi
    g = _rng(rows, channels, backwards)
    gate = (0.3 + 2.0 * torch.rand(rows, channels, generator=g, device="cuda")).to(_t(dtype))
    given = torch.zeros(rows, channels, dtype=_t(dtype), device="cuda")
    # (every third channel has a number at the end of the scan, which does not pass any rows)
    given[0 if backwards else rows - 1, ::3] = 1.5
    zeros, out, grads = torch.zeros_like(given), torch.empty_like(given), torch.empty_like(given)
    last = torch.empty(1, channels, device="cuda")
    if backwards:
        capi.gated_recurrence_gradient(
            *(_matrix(t) for t in (given, gate, zeros, zeros, out, grads)),
            grad_initial=_matrix(last), decay=capi.DECAY_EXPONENTIAL)
        assert torch.equal(grads, given) and bool((out == 0).all())
        want = given[0].double() * gate[0].double().exp()
        _close(last[0], want, 24 * U * want)
    else:
        _run(capi, gate, given, out, "exponential", False, final=last)
        assert torch.equal(out, given) and torch.equal(last[0], given[-1].float())


def _growth(rows, dtype):
    """Gates of 512 rows that leave a state as it is and of `rows` through which it grows by e^0 to
    e^150, a channel each, and what grows to 1e30."""
    import torch
    total = torch.linspace(0.0, 150.0, 76, dtype=torch.float64, device="cuda")
    gate = (total / rows).to(dtype)
    gates = torch.cat((torch.zeros(512, 76, dtype=dtype, device="cuda"), gate.expand(rows, 76)))
    return gates, (1e30 * torch.exp(-rows * gate.double())).float()[None]


# A tile has 256 rows at most, which is all of the growth, or more of it than float32 holds.
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [100, 256, 1200])
def test_states_that_grow_or_fall_through_all_of_float32(rows, dtype):
    import torch
    from ilgpu_amd import capi
    gates, start = _growth(rows, _t(dtype))
    large, none = torch.full_like(start, 1e30), torch.zeros_like(gates)
    _check_recurrence(gates, none, "exponential", False, 1, None, start)
    _, final = _check_recurrence(-gates, none, "exponential", False, 1, None, large)
    assert bool((final > 0).all())
    # up and down again, with something added in all rows
    _check_recurrence(torch.cat((gates, -gates)), torch.cat((none, none + 1.0)), "exponential", False, 1, None,
                      start)
    # and backwards; states of zero, so that the gates' gradients are
    for way, grad_final in ((gates.flip(0), start), (-gates.flip(0), large)):
        got = _gradient(capi, none, way, none, none, "exponential", False, 1, None, None, grad_final)
        _check_gradient(got, none, way, none, none, "exponential", False, [0, len(gates)], None, grad_final)


# (Of gates of -20 the decays of eight rows, a thread's, are below float32 together.)
@pytest.mark.parametrize("gate", [-3.0, -20.0])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES)
def test_an_infinite_state_stays_infinite_however_long(dtype, kind, gate):
    import torch
    from ilgpu_amd import capi
    rows, channels = 2500, 72
    gates = torch.full((rows, channels), gate, dtype=_t(dtype), device="cuda")
    x = _normal(_rng(rows, 11), rows, channels, dtype=_t(dtype))
    x[0, ::2] = float("inf")
    x[0, 1::4] = -float("inf")
    back = x.flip(0).contiguous()
    out, grads = torch.empty_like(x), torch.empty_like(x)
    _run(capi, gates, x, out, kind, False)
    capi.gated_recurrence_gradient(*(_matrix(t) for t in (back, gates, x, x, None, grads)),
                                   decay=getattr(capi, "DECAY_" + kind.upper()))
    for got in (out, grads):
        assert bool((got[:, ::2] == float("inf")).all()) and bool((got[:, 1::4] == -float("inf")).all())
        assert bool(torch.isfinite(got[:, 3::4]).all())


def test_growing_decays_give_the_same_bits_again():
    import torch
    from ilgpu_amd import capi
    g = _rng(12)
    gate, x = (0.05 * torch.randn(20_011, 136, generator=g, device="cuda")).bfloat16(), \
        _normal(g, 20_011, 136, dtype=torch.bfloat16)
    runs = []
    for _ in range(4):
        out, of_gate, of_x = (torch.empty_like(x) for _ in range(3))
        _run(capi, gate, x, out, "exponential", False)
        capi.gated_recurrence_gradient(*(_matrix(t) for t in (x, gate, x, x, of_gate, of_x)),
                                       decay=capi.DECAY_EXPONENTIAL)
        runs.append([t.view(torch.uint8).clone() for t in (out, of_gate, of_x)])
    for run in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(run, runs[0]))


# ---- AdamW's codes ---------------------------------------------------------------------
def test_moments_in_8_bits_near_the_largest_float32():
    # Squares of 1.3e19 to 1.8e19 are floats, and the half of them is above 2^126, whose
    # reciprocal is below the normal numbers; beside them a block with smaller ones.
    import torch
    from ilgpu_amd import capi
    s = _adam_state(_rng(21), [1024], ("float32", "float32", None), True, fresh=True)
    s["g"][0] = s["g"][0].sign() * torch.linspace(1e17, 1.8e19, 1024, device="cuda")
    s["g"][0][512:768] = torch.linspace(1.0, 1.8e19, 256, device="cuda")
    before = _clone(s)
    _adamw(capi, s, betas=(0.9, 0.5))
    _check_adamw(s, before, betas=(0.9, 0.5))
    assert bool((s["v"][0].view(4, 256).max(1).values == 255).all())
    assert bool(((s["m"][0].long() - 128).abs().view(4, 256).max(1).values == 127).all())


def _codes(shares, power, levels, chance):
    """The codes of shares of a scale, exactly: float64 holds a float32 times levels^power to a unit of 2^-53."""
    import torch
    z = shares.double() * float(levels) ** power
    low = z.pow(1.0 / power).floor()
    low = torch.where(low ** power > z, low - 1, low)
    low = torch.where((low + 1) ** power <= z, low + 1, low)
    way, span = z - low ** power, (low + 1) ** power - low ** power
    return (low + (way * 65536 > chance * span)).clamp(max=levels)


@pytest.mark.parametrize("second", [False, True])
def test_codes_beside_what_a_code_stands_for(second):
    # Values some units from a code's, at the first and last chances: the code above is raised from the one
    # or the other side.  Without what was before (beta 0) the moments are the gradient and its square.
    import torch
    from ilgpu_amd import capi
    power, levels = (4, 255) if second else (2, 127)
    n, t = 1 << 25, 1
    index = torch.arange(n, device="cuda")
    g = _rng(22, second)
    s = _adam_state(g, [n], ("float32", "float32", None), True, fresh=True)
    s["step"][0] = t
    compared = 0
    for seed in range(77, 87):
        key = _mixed(((seed & WORD) + t * 0x3C6EF373) & WORD)
        key = _mixed((key + (seed >> 32 & WORD)) & WORD)
        word = _mixed((index * 0x9E3779B9 + key) & WORD)
        chance = word >> 16 if second else word & 0xFFFF
        at = (((chance > 0) & (chance < 6)) | (chance > 65530)).nonzero()[:, 0]
        at = at[(at % BLOCK) != 0]
        largest = 1.0 + torch.rand(n // BLOCK, generator=g, device="cuda")
        scale = (largest * largest if second else largest)[at // BLOCK]
        code = torch.randint(levels // 2, levels, (at.numel(),), generator=g, device="cuda").double()
        value = ((code / levels) ** power * scale.double()).float()
        near = value.view(torch.int32) + torch.randint(-9, 10, (at.numel(),), generator=g, device="cuda").int()
        s["g"][0].zero_()
        s["g"][0][::BLOCK] = largest
        s["g"][0][at] = near.view(torch.float32).sqrt() if second else near.view(torch.float32)
        for k in ("m", "v", "ms", "vs"):
            s[k][0].zero_()
        _adamw(capi, s, betas=(0.0, 0.0), seed=seed)
        assert torch.equal(s["vs" if second else "ms"][0][at // BLOCK], scale)
        got = (s["v"][0][at].long() if second else s["m"][0][at].long() - 128).double()
        values = s["g"][0][at] * s["g"][0][at] if second else s["g"][0][at]
        shares = (values.cpu() / scale.cpu()).cuda()      # (rounded to float32 to the nearest)
        want = _codes(shares, power, levels, chance[at].double())
        assert torch.equal(got, want), (seed, int((got != want).sum()))
        compared += at.numel()
    assert compared > 30_000


# ---- the exponential of float32 gates ------------------------------------------------------
def _decays(gates, kind):
    """Decays and what is left of them to 1, each alone: a state of 1 a row on, and an input of 1."""
    import torch
    from ilgpu_amd import capi
    x = gates.reshape(-1, 64)
    zero, one = torch.zeros_like(x), torch.ones_like(x)
    a, left = torch.empty_like(x), torch.empty_like(x)
    _run(capi, x, zero, a, kind, False, len(x), None, one)
    _run(capi, x, one, left, kind, True, len(x))
    return a.flatten(), left.flatten()


def test_decays_of_large_float32_gates_keep_their_digits():
    # The exponential is off by 4 u: the instruction's unit in the last place (2 u), the two roundings of what
    # the product's rest makes of it; the rest itself is off by a thousandth of u.  The logistic function
    # adds a sum, a reciprocal (2 u) and a product; 1 - exp is -1 and more of the exponential.
    import torch
    gates = torch.linspace(0.5, 87.0, 64 * 4096, device="cuda")
    for sign in (1, -1):
        x = sign * gates
        e = torch.exp(x.double())
        a, left = _decays(x, "exponential")
        _close(a, e, 4 * U * e)
        if sign > 0:
            _close(left, 1 - e, 5 * U * e)
        a, left = _decays(x, "sigmoid")
        for got, exact in ((a, torch.sigmoid(x.double())), (left, torch.sigmoid(-x.double()))):
            _close(got, exact, 12 * U * exact)


# ---- more rows than a grid of the largest blocks has ------------------------------------------
def test_norm_gradient_of_very_many_long_rows():
    # One row in the place of all.  Sums of ones are exact; with a weight of 1 of both norms the
    # input's statistics take part too: the gradient of total is grad_out - mean(grad_out * h) * h = 0.
    import torch
    from ilgpu_amd import capi
    rows, columns = (1 << 22) + 3, 8200
    one = torch.ones(1, columns, dtype=torch.bfloat16, device="cuda").expand(rows, columns)
    rstd = torch.ones(rows, device="cuda")
    rstd[-3:] = 0.0
    of_weight, of_input = (torch.full((columns,), 77.0, device="cuda") for _ in range(2))
    capi.residual_norm_gradient(_matrix(one), None, _matrix(one), _matrix(one), None, _array(rstd),
                                grad_weight=_array(of_weight), input_rstd=_array(rstd),
                                grad_input_weight=_array(of_input))
    assert bool((of_weight == 1 << 22).all()) and bool((of_input == 0).all())


# ---- more tiles than a launch has blocks ---------------------------------------------------
# 2^22 blocks a launch; of one channel a tile has 32 rows, backwards 16.  A state of 1 has to come through
# all of them unchanged.
@pytest.mark.parametrize("backwards", [False, True])
def test_a_state_passes_through_more_tiles_than_a_launch_has(backwards):
    import torch
    from ilgpu_amd import capi
    rows = (1 << 27) // (2 if backwards else 1) + 77
    gate = torch.zeros(1, 1, dtype=torch.bfloat16, device="cuda").expand(rows, 1)
    given = torch.zeros(rows, 1, dtype=torch.bfloat16, device="cuda")
    given[-1 if backwards else 0] = 1.0
    out, last = torch.zeros_like(given), torch.empty(1, 1, device="cuda")
    if backwards:
        capi.gated_recurrence_gradient(*(_matrix(t) for t in (given, gate, gate, gate, None, out)),
                                       grad_initial=_matrix(last), decay=capi.DECAY_EXPONENTIAL)
    else:
        _run(capi, gate, given, out, "exponential", False, final=last)
    assert bool((out == 1.0).all()) and float(last) == 1.0
