"""The operators of language models (embedding, layer norm, gradient norm and
clipping) through the C ABI against their formulas in float64.

Tolerances follow from the arithmetic, not from measured differences.  With
u = 2^-24 (float32) and u_out the unit roundoff of the result's type:

  - a result is rounded to its type once: u_out * |exact|, and half the spacing
    of float16's subnormal numbers;
  - a sum whose elements pass through at most L additions is off by at most
    L * u times the sum of their magnitudes, whatever the order.  A row of C
    columns is shared by at least 64 lanes: L = C / 64 + 32.  Sums over
    positions or rows take L = their number.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = ["float32", "float16", "bfloat16"]


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
    """t's values as rows `stride` apart from `offset` elements into other memory,
    with NaN between them: (matrix tensor, the memory, its guard positions)."""
    import torch
    rows, columns = t.shape
    memory = torch.full((offset + rows * stride + 7,), float("nan"), dtype=t.dtype, device="cuda")
    view = torch.as_strided(memory, (rows, columns), (stride, 1), offset)
    view.copy_(t)
    guard = torch.ones(memory.numel(), dtype=torch.bool, device="cuda")
    torch.as_strided(guard, (rows, columns), (stride, 1), offset).fill_(False)
    return view, memory, guard


def _tokens(g, n, vocabulary, dtype, outside=True):
    import torch
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    t = (vocabulary * u * u * u).floor().clamp(0, max(vocabulary - 1, 0)).to(dtype)
    if outside and n > 3:
        t[n // 2] = -1
        t[n // 3] = vocabulary
        t[n - 1] = torch.iinfo(dtype).min
        if dtype == torch.int64:
            t[1] = (1 << 32) + 1      # its lower half is a token of the table
    return t


# ---- embedding ------------------------------------------------------------------
@pytest.mark.parametrize("token_type", ["int32", "int64"])
@pytest.mark.parametrize("table_type", TYPES)
@pytest.mark.parametrize("out_type", TYPES)
@pytest.mark.parametrize("n,vocabulary,dimension", [
    (1, 1, 1), (1, 50, 4096), (5, 17, 3), (63, 1000, 64), (1030, 301, 129), (257, 40, 1000),
    (66, 70, 2051)])
def test_embedding(n, vocabulary, dimension, out_type, table_type, token_type):
    import torch
    from ilgpu_amd import capi
    g = _rng(n, vocabulary, dimension)
    table = _normal(g, vocabulary, dimension, dtype=_t(table_type))
    tokens = _tokens(g, n, vocabulary, _t(token_type))
    out = torch.full((n, dimension), float("nan"), dtype=_t(out_type), device="cuda")
    scale = 1.7
    capi.embedding(capi.DeviceMatrix.from_tensor(table), capi.DeviceArray.from_tensor(tokens),
                   capi.DeviceMatrix.from_tensor(out), scale=scale)
    wide = tokens.long()
    there = (wide >= 0) & (wide < vocabulary)
    exact = table.double()[wide * there] * float(np.float32(scale)) * there[:, None]
    _close(out, exact, U * exact.abs())
    assert bool((out[~there] == 0).all())


@pytest.mark.parametrize("kind", TYPES)
def test_embedding_without_scale_copies_bits(kind):
    import torch
    from ilgpu_amd import capi
    table = _normal(_rng(3), 100, 77, dtype=_t(kind))
    table[7, 0], table[7, 1], table[7, 2] = float("inf"), -0.0, float("-inf")
    tokens = torch.arange(99, -1, -1, device="cuda")
    out = torch.empty_like(table)
    capi.embedding(capi.DeviceMatrix.from_tensor(table), capi.DeviceArray.from_tensor(tokens),
                   capi.DeviceMatrix.from_tensor(out))
    assert torch.equal(out.view(torch.uint8), table.flip(0).contiguous().view(torch.uint8))


def test_embedding_strides_and_unaligned_rows():
    import torch
    from ilgpu_amd import capi
    for kind in TYPES:
        table = _normal(_rng(5), 40, 85, dtype=_t(kind))
        tokens = _tokens(_rng(6), 70, 40, torch.int32)
        t_view, _, _ = _strided(table, 91, 3)
        o_view, o_memory, guard = _strided(torch.zeros(70, 85, dtype=_t(kind), device="cuda"), 87, 1)
        capi.embedding(capi.DeviceMatrix.from_tensor(t_view), capi.DeviceArray.from_tensor(tokens),
                       capi.DeviceMatrix.from_tensor(o_view))
        there = (tokens >= 0) & (tokens < 40)
        assert torch.equal(o_view, table[(tokens * there).long()] * there[:, None])
        assert bool(o_memory[guard].isnan().all())      # nothing between the rows was written


def test_embedding_ignores_what_no_token_names():
    import torch
    from ilgpu_amd import capi
    table = torch.full((9, 33), float("nan"), device="cuda")
    table[4] = 2.0
    tokens = torch.tensor([4, -1, 9, 4], device="cuda")
    out = torch.empty(4, 33, device="cuda")
    capi.embedding(capi.DeviceMatrix.from_tensor(table), capi.DeviceArray.from_tensor(tokens),
                   capi.DeviceMatrix.from_tensor(out), scale=0.5)
    assert out[[0, 3]].eq(1).all() and out[[1, 2]].eq(0).all()


# ---- embedding gradient -----------------------------------------------------------
def _embedding_gradient(grad, tokens, vocabulary, table_type, scale=1.0, padding=-1, into=None):
    import torch
    from ilgpu_amd import capi
    out = torch.full((vocabulary, grad.shape[1]), float("nan"), dtype=table_type,
                     device="cuda") if into is None else into.clone()
    capi.embedding_gradient(capi.DeviceMatrix.from_tensor(grad), capi.DeviceArray.from_tensor(tokens),
                            capi.DeviceMatrix.from_tensor(out), scale=scale, padding_token=padding,
                            accumulate=into is not None)
    return out


def _check_embedding_gradient(out, grad, tokens, vocabulary, scale, padding=-1, into=None):
    import torch
    wide = tokens.long()
    there = (wide >= 0) & (wide < vocabulary) & (wide != padding)
    s = float(np.float32(scale))
    rows = grad.double()[there] * s
    shape = (vocabulary, grad.shape[1])
    exact = torch.zeros(shape, dtype=torch.float64, device="cuda")
    size = torch.zeros(shape, dtype=torch.float64, device="cuda")
    met = torch.zeros(vocabulary, dtype=torch.float64, device="cuda")
    exact.index_put_((wide[there],), rows, accumulate=True)
    size.index_put_((wide[there],), rows.abs(), accumulate=True)
    met.index_put_((wide[there],), torch.ones_like(wide[there], dtype=torch.float64), accumulate=True)
    slack = (met[:, None] + 2) * U * size
    if into is not None:
        exact = exact + into.double()
        slack = slack + U * (size + into.double().abs()) * (met[:, None] > 0)
        assert torch.equal(out[met == 0], into[met == 0])
    else:
        assert bool((out[met == 0] == 0).all())
    _close(out, exact, slack)


@pytest.mark.parametrize("table_type", TYPES)
@pytest.mark.parametrize("grad_type", TYPES)
@pytest.mark.parametrize("n,vocabulary,dimension", [
    (1, 1, 1), (1, 300, 2048), (2, 3, 5), (64, 2, 64), (65, 1, 130), (1000, 4099, 96),
    (4097, 50, 33), (5000, 20011, 257), (300, 100, 1537)])
def test_embedding_gradient(n, vocabulary, dimension, grad_type, table_type):
    import torch
    g = _rng(n, vocabulary, dimension, 1)
    grad = _normal(g, n, dimension, dtype=_t(grad_type))
    for token_type in (torch.int32, torch.int64):
        tokens = _tokens(g, n, vocabulary, token_type)
        out = _embedding_gradient(grad, tokens, vocabulary, _t(table_type), 0.3)
        _check_embedding_gradient(out, grad, tokens, vocabulary, 0.3)


@pytest.mark.parametrize("n,vocabulary", [(20_000, 32_003), (70_001, 1000), (150_000, 250_007),
                                          (300_000, 70_000), (40_000, 1_500_000),
                                          (20_000, 500_009), (30_000, 1_048_576),
                                          (131_072, 50_000), (131_073, 50_000), (65_537, 300_000)])
def test_embedding_gradient_of_many_tokens(n, vocabulary):
    import torch
    g = _rng(n, vocabulary)
    grad = _normal(g, n, 24, dtype=torch.bfloat16)
    tokens = _tokens(g, n, vocabulary, torch.int64)
    out = _embedding_gradient(grad, tokens, vocabulary, torch.float32)
    _check_embedding_gradient(out, grad, tokens, vocabulary, 1.0)
    again = _embedding_gradient(grad, tokens, vocabulary, torch.float32)
    assert torch.equal(out, again)


@pytest.mark.parametrize("distribution", ["one", "two", "alternating", "runs", "all_outside",
                                          "ascending", "mostly_one"])
@pytest.mark.parametrize("n", [31, 64, 1000, 1024, 30_000, 120_001])
def test_embedding_gradient_of_skewed_tokens(n, distribution):
    import torch
    vocabulary = 513
    at = torch.arange(n, device="cuda")
    tokens = {"one": at * 0 + 512, "two": (at * 7 // max(n, 1)) % 2 * 511, "alternating": at % 2,
              "runs": at // 40 % vocabulary, "all_outside": at + vocabulary,
              "ascending": at % vocabulary,
              "mostly_one": torch.where(at % 11 == 0, at % vocabulary, 7)}[distribution]
    grad = _normal(_rng(n, 9), n, 100, dtype=torch.bfloat16)
    out = _embedding_gradient(grad, tokens, vocabulary, torch.float32, 2.0)
    _check_embedding_gradient(out, grad, tokens, vocabulary, 2.0)
    assert torch.equal(out, _embedding_gradient(grad, tokens, vocabulary, torch.float32, 2.0))


@pytest.mark.parametrize("dimension", [1, 5, 36, 64, 130, 300])
@pytest.mark.parametrize("unit", [8, 32])
def test_embedding_gradient_of_runs_of_many_lengths(unit, dimension):
    # whole numbers, whose sums are exact in float32 in any order, in runs of up to 5000 chunks
    import torch
    lengths = [unit * c + more for c in (1, 2, 63, 64, 65, 128, 255, 256, 257, 320, 321, 700, 5000)
               for more in (-1, 0, 1)]
    tokens = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths)).cuda()
    g = _rng(unit, dimension)
    grad = torch.randint(-3, 4, (len(tokens), dimension), generator=g, device="cuda").float()
    out = _embedding_gradient(grad, tokens, len(lengths), torch.float32)
    exact = torch.zeros(len(lengths), dimension, dtype=torch.float64, device="cuda")
    exact.index_add_(0, tokens, grad.double())
    assert torch.equal(out.double(), exact)


@pytest.mark.parametrize("table_type", TYPES)
@pytest.mark.parametrize("n", [40, 3000])
@pytest.mark.parametrize("dimension", [3, 64, 65, 257])
def test_embedding_gradient_gives_zeros_one_sign(dimension, n, table_type):
    # 0 * -1 is -0 in every column, the last ones of a row that is no whole number of vectors too
    import torch
    tokens = torch.zeros(n, dtype=torch.int32, device="cuda")
    out = _embedding_gradient(torch.zeros(n, dimension, device="cuda"), tokens, 2, _t(table_type), -1.0)
    assert bool((out == 0).all())
    assert bool(torch.signbit(out[0]).all()) and not bool(torch.signbit(out[1]).any())


@pytest.mark.parametrize("table_type", TYPES)
@pytest.mark.parametrize("n", [40, 3000])
def test_embedding_gradient_accumulates_and_skips_padding(n, table_type):
    import torch
    vocabulary = 700
    g = _rng(11)
    grad = _normal(g, n, 65, dtype=torch.float16)
    tokens = _tokens(g, n, vocabulary, torch.int32)
    # what padding contributes must not be read into anything
    grad[tokens == 0] = float("nan")
    grad[(tokens < 0) | (tokens >= vocabulary)] = float("inf")
    clean = torch.where((tokens == 0)[:, None] | ~torch.isfinite(grad), torch.zeros_like(grad), grad)
    out = _embedding_gradient(grad, tokens, vocabulary, _t(table_type), 0.7, padding=0)
    _check_embedding_gradient(out, clean, tokens, vocabulary, 0.7, padding=0)
    old = _normal(g, vocabulary, 65, dtype=_t(table_type))
    out = _embedding_gradient(grad, tokens, vocabulary, _t(table_type), 0.7, padding=0, into=old)
    _check_embedding_gradient(out, clean, tokens, vocabulary, 0.7, padding=0, into=old)


def test_embedding_gradient_of_no_tokens_and_of_broadcast_rows():
    import torch
    from ilgpu_amd import capi
    none = torch.empty(0, 12, device="cuda")
    tokens = torch.empty(0, dtype=torch.int64, device="cuda")
    assert bool((_embedding_gradient(none, tokens, 5, torch.float32) == 0).all())
    old = torch.ones(5, 12, device="cuda")
    assert torch.equal(_embedding_gradient(none, tokens, 5, torch.float32, into=old), old)
    # the gradient of a sum: one row for all positions, at a stride of 0
    tokens = torch.arange(100, device="cuda") % 3
    grad = torch.full((1, 12), 0.5, device="cuda").expand(100, 12)
    matrix = capi.DeviceMatrix.from_tensor(grad)
    assert matrix.row_stride == 0
    out = _embedding_gradient(grad, tokens, 4, torch.float32)
    assert out[:, 0].tolist() == [17.0, 16.5, 16.5, 0.0]


@pytest.mark.parametrize("n", [50, 900])
def test_embedding_gradient_strides(n):
    import torch
    grad = _normal(_rng(21), n, 35, dtype=torch.bfloat16)
    tokens = _tokens(_rng(22), n, 60, torch.int64)
    g_view, _, _ = _strided(grad, 41, 1)
    o_view, o_memory, guard = _strided(torch.zeros(60, 35, device="cuda"), 37, 1)
    from ilgpu_amd import capi
    capi.embedding_gradient(capi.DeviceMatrix.from_tensor(g_view),
                            capi.DeviceArray.from_tensor(tokens),
                            capi.DeviceMatrix.from_tensor(o_view))
    _check_embedding_gradient(o_view, grad, tokens, 60, 1.0)
    assert bool(o_memory[guard].isnan().all())


def test_embedding_gradient_against_differences():
    # The lookup is linear in the table: a step of any size gives the exact difference.
    import torch
    from ilgpu_amd import capi
    vocabulary, n, dimension = 11, 40, 6
    g = _rng(31)
    table = torch.randint(-8, 9, (vocabulary, dimension), generator=g, device="cuda").float()
    grad = torch.randint(-8, 9, (n, dimension), generator=g, device="cuda").float()
    tokens = _tokens(g, n, vocabulary, torch.int64)

    def loss(t):
        out = torch.empty(n, dimension, device="cuda")
        capi.embedding(capi.DeviceMatrix.from_tensor(t), capi.DeviceArray.from_tensor(tokens),
                       capi.DeviceMatrix.from_tensor(out), scale=0.5)
        return float((out * grad).double().sum())

    got = _embedding_gradient(grad, tokens, vocabulary, torch.float32, 0.5)
    base = loss(table)
    for v in range(vocabulary):
        for c in range(0, dimension, 2):
            step = table.clone()
            step[v, c] += 4.0
            assert (loss(step) - base) / 4.0 == float(got[v, c]), (v, c)


def test_offsets_beyond_32_bits():
    # 2^31 elements and more in the table: rows in front of and behind that.
    import torch
    from ilgpu_amd import capi
    vocabulary, dimension = 1_060_000, 2048
    table = torch.zeros(vocabulary, dimension, dtype=torch.bfloat16, device="cuda")
    tokens = torch.tensor([0, 1_048_575, 1_048_576, 1_059_999, 1_048_576], device="cuda")
    grad = _normal(_rng(41), 5, dimension, dtype=torch.bfloat16)
    capi.embedding_gradient(capi.DeviceMatrix.from_tensor(grad), capi.DeviceArray.from_tensor(tokens),
                            capi.DeviceMatrix.from_tensor(table), accumulate=True)
    out = torch.empty(5, dimension, dtype=torch.float32, device="cuda")
    capi.embedding(capi.DeviceMatrix.from_tensor(table), capi.DeviceArray.from_tensor(tokens),
                   capi.DeviceMatrix.from_tensor(out))
    exact = grad.double()
    exact[2] += exact[4]
    exact[4] = exact[2]
    _close(out.to(torch.bfloat16), exact, U * grad.double().abs().sum(0))


@pytest.mark.parametrize("n", [60, 300, 5000])
def test_embedding_gradient_keeps_bad_rows_to_their_tokens(n):
    import torch
    vocabulary = 97
    g = _rng(n, 51)
    grad = _normal(g, n, 300, dtype=torch.bfloat16)
    tokens = torch.randint(0, vocabulary, (n,), generator=g, device="cuda")
    good = _embedding_gradient(grad, tokens, vocabulary, torch.float32)
    bad = [int(tokens[k]) for k in (3, n // 2, n - 1)]
    grad[3], grad[n // 2, 7], grad[n - 1, 299] = float("nan"), float("inf"), float("nan")
    out = _embedding_gradient(grad, tokens, vocabulary, torch.float32)
    kept = torch.ones(vocabulary, dtype=torch.bool, device="cuda")
    kept[bad] = False
    assert torch.equal(out[kept], good[kept])
    assert bool(out[bad[0]].isnan().all()) and not bool(torch.isfinite(out[bad[1], 7]))
    others = torch.arange(300, device="cuda") != 7
    if bad[1] not in (bad[0], bad[2]):
        assert torch.equal(out[bad[1], others], good[bad[1], others])


def _whole_numbers(g, *shape, dtype=None):
    """Small whole numbers: sums of up to 2^22 of them are exact in float32 in any order."""
    import torch
    return torch.randint(-3, 4, shape, generator=g, device="cuda").to(dtype or torch.float32)


def _equal_sums(out, grad, tokens, vocabulary):
    """out is the sum of each token's rows, to the bit."""
    import torch
    wide = tokens.long()
    at = torch.nonzero((wide >= 0) & (wide < vocabulary))[:, 0]
    at = at[wide[at].argsort()]
    # sums up to each token's last row less those up to the one before it, all whole numbers
    sums = torch.zeros(len(at) + 1, grad.shape[1], dtype=torch.float64, device="cuda")
    sums[1:] = grad.double()[at].cumsum(0)
    counts = torch.bincount(wide[at], minlength=vocabulary)
    ends = counts.cumsum(0)
    assert torch.equal(out.double(), sums[ends] - sums[ends - counts])


@pytest.mark.parametrize("token_type", ["int32", "int64"])
@pytest.mark.parametrize("n,places", [(65_536, 512), (131_072, 1024)])
@pytest.mark.parametrize("more", [-1, 0, 1, 64, None])
def test_embedding_gradient_of_position_lists_about_full(more, n, places, token_type):
    # Sixteen waves of a block list the positions of its tokens in a sixteenth of the input each;
    # a list has `places` of them. Tokens 7, 263 and 519 belong to the same block.
    import torch
    vocabulary, stretch = 600, n // 16
    g = _rng(n, places, 0 if more is None else more + 2)
    listed = stretch if more is None else places + more
    tokens = torch.randint(0, 7, (16, stretch), generator=g, device="cuda")
    tokens[:, :listed] = 7 + 256 * torch.randint(0, 3, (16, listed), generator=g, device="cuda")
    order = torch.rand(16, stretch, generator=g, device="cuda").argsort(1)
    tokens = tokens.gather(1, order).reshape(-1).to(_t(token_type))
    grad = _whole_numbers(g, n, 24)
    out = _embedding_gradient(grad, tokens, vocabulary, torch.float32)
    _equal_sums(out, grad, tokens, vocabulary)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dimension", [1, 3, 4, 20, 64, 130, 1030])
@pytest.mark.parametrize("vocabulary", [1, 2, 17, 63, 65, 257, 1021])
def test_embedding_gradient_of_few_tokens_and_rows_that_end_inside_a_wave(vocabulary, dimension,
                                                                         accumulate):
    # Rows of the table share waves and the table ends inside one; tokens lie in all 64 lanes.
    import torch
    g = _rng(vocabulary, dimension, 61)
    for n in (33, 64):
        tokens = torch.randint(max(0, vocabulary - 9), vocabulary, (n,), generator=g, device="cuda")
        grad = _whole_numbers(g, n, dimension)
        old = _whole_numbers(g, vocabulary, dimension) if accumulate else None
        out = _embedding_gradient(grad, tokens, vocabulary, torch.float32, into=old)
        _equal_sums(out if old is None else out - old, grad, tokens, vocabulary)


@pytest.mark.parametrize("most,vocabulary,dimension", [(4096, 900, 2048), (40_000, 3000, 256),
                                                       (131_073, 1000, 64), (140_000, 300_000, 24)])
def test_embedding_gradient_of_fewer_tokens_in_the_same_temp(most, vocabulary, dimension):
    import torch
    from ilgpu_amd import capi
    g = _rng(most, vocabulary, 71)
    temp = capi.temp_buffer(capi.embedding_gradient_temp_bytes(most, vocabulary, dimension))
    for n in (most, most - 1, most - 32, most // 2, most // 5, 100, 3):
        tokens = _tokens(g, n, vocabulary, torch.int64)
        grad = _whole_numbers(g, n, dimension)
        out = torch.full((vocabulary, dimension), float("nan"), device="cuda")
        capi.embedding_gradient(capi.DeviceMatrix.from_tensor(grad),
                                capi.DeviceArray.from_tensor(tokens),
                                capi.DeviceMatrix.from_tensor(out), temp)
        _equal_sums(out, grad, tokens, vocabulary)


@pytest.mark.parametrize("n", [1, 33, 64])
@pytest.mark.parametrize("vocabulary,dimension,in_one", [
    (49_152, 1024, True), (65_536, 1024, False), (300_000, 200, True), (300_000, 300, False),
    (1_100_000, 60, True), (1_100_000, 100, False)])
def test_embedding_gradient_of_few_tokens_accumulated_into_large_tables(vocabulary, dimension,
                                                                        in_one, n):
    # One launch has blocks for every row of the table, which is more than the tokens' rows take.
    import torch
    from ilgpu_amd import capi
    g = _rng(vocabulary, dimension, n)
    tokens = _tokens(g, n, vocabulary, torch.int64)
    tokens[: n // 2] = tokens[n // 2:n // 2 * 2].clone()
    grad = _whole_numbers(g, n, dimension)
    old = _whole_numbers(g, vocabulary, dimension)
    capi.profile_enable(True)
    try:
        out = _embedding_gradient(grad, tokens, vocabulary, torch.float32, into=old)
        torch.cuda.synchronize()
        launches = capi.profile_query("embedding_gradient_of_few")[0]
    finally:
        capi.profile_enable(False)
    assert launches == (1 if in_one else 0)
    _equal_sums(out - old, grad, tokens, vocabulary)


@pytest.mark.parametrize("grad_type", ["float32", "bfloat16"])
@pytest.mark.parametrize("dimension", [1, 36, 100, 513])
@pytest.mark.parametrize("distribution", ["one", "two", "alternating", "runs", "ascending",
                                          "mostly_one"])
@pytest.mark.parametrize("n", [31, 65, 1000, 1024, 30_000, 120_001, 131_073])
def test_embedding_gradient_sums_skewed_tokens_to_the_bit(n, distribution, dimension, grad_type):
    # A sum that misses a row, or has one twice, is another number, however long its run.
    import torch
    vocabulary = 513
    at = torch.arange(n, device="cuda")
    tokens = {"one": at * 0 + 512, "two": (at * 7 // n) % 2 * 511, "alternating": at % 2,
              "runs": at // 40 % vocabulary, "ascending": at % vocabulary,
              "mostly_one": torch.where(at % 11 == 0, at % vocabulary, 7)}[distribution]
    grad = _whole_numbers(_rng(n, dimension, 93), n, dimension, dtype=_t(grad_type))
    _equal_sums(_embedding_gradient(grad, tokens, vocabulary, torch.float32), grad, tokens, vocabulary)


# Runs of lengths around whole chunks, in the four ways that positions are grouped and cut: chunks of
# 8 up to 32736 tokens of at most 256 columns, of 32 beyond; grouped in one launch up to 131072
# tokens of at most 2^20 rows, sorted beyond.
RUNS = {"grouped_8": (8, (1, 2, 3, 63, 64, 65, 257, 700), 1),
        "sorted_8": (8, (1, 2, 3, 63, 64, 65, 257, 700), 50_000),
        "grouped_32": (32, (1, 2, 3, 63, 64, 65, 128, 257, 320), 1),
        "sorted_32": (32, (1, 2, 3, 63, 64, 65, 257, 1500), 1)}


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("shuffled", [False, True])
@pytest.mark.parametrize("dimension", [1, 5, 64, 130, 256])
@pytest.mark.parametrize("way", sorted(RUNS))
def test_embedding_gradient_of_runs_about_whole_chunks(way, dimension, shuffled, accumulate):
    import torch
    unit, chunks, apart = RUNS[way]
    lengths = [unit * c + more for c in chunks for more in (-1, 0, 1)]
    n, vocabulary = sum(lengths), (len(lengths) - 1) * apart + 1
    assert (n <= 32 * 1023) == (unit == 8)
    assert (n <= 1 << 17 and vocabulary <= 1 << 20) == way.startswith("grouped")
    g = _rng(n, dimension, vocabulary)
    tokens = torch.repeat_interleave(torch.arange(len(lengths)) * apart, torch.tensor(lengths)).cuda()
    if shuffled:
        tokens = tokens[torch.randperm(n, generator=g, device="cuda")]
    grad = _whole_numbers(g, n, dimension)
    old = _whole_numbers(g, vocabulary, dimension) if accumulate else None
    out = _embedding_gradient(grad, tokens, vocabulary, torch.float32, into=old)
    _equal_sums(out if old is None else out - old, grad, tokens, vocabulary)


# ---- layer norm -------------------------------------------------------------------
def _layer_norm(x, weight, bias, epsilon=1e-5, out=None):
    import torch
    from ilgpu_amd import capi
    array, matrix = capi.DeviceArray.from_tensor, capi.DeviceMatrix.from_tensor
    rows = x.shape[0]
    out = torch.full_like(x, float("nan"), memory_format=torch.contiguous_format) if out is None else out
    mean, rstd = (torch.full((rows,), float("nan"), device="cuda") for _ in range(2))
    capi.layer_norm(matrix(x), matrix(out), None if weight is None else array(weight),
                    None if bias is None else array(bias), epsilon=epsilon, mean=array(mean),
                    rstd=array(rstd))
    return out, mean, rstd


def _check_layer_norm(out, mean, rstd, x, weight, bias, epsilon=1e-5):
    import torch
    wide = x.double()
    columns = x.shape[1]
    level = columns / 64 + 32
    m = wide.mean(1, keepdim=True)
    away = wide - m
    v = (away * away).mean(1, keepdim=True) + float(np.float32(epsilon))
    r = 1.0 / v.sqrt()
    w = 1.0 if weight is None else weight.double()
    b = torch.zeros((), dtype=torch.float64, device="cuda") if bias is None else bias.double()
    m_off = (level + 1) * U * wide.abs().mean(1, keepdim=True)
    r_off = (level + 4) * U / 2 + m_off * m_off / (2 * v) + 4 * U   # relative
    y = away * r * w
    slack = m_off * r * abs(w) + y.abs() * (r_off + 4 * U) + U * (y.abs() + b.abs())
    _close(mean, m[:, 0], m_off[:, 0])
    _close(rstd, r[:, 0], (r * r_off)[:, 0])
    _close(out, y + b, slack)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("columns", [1, 2, 3, 7, 64, 65, 127, 256, 500, 768, 1000, 1024, 1025, 1537,
                                     2048, 4096, 4099, 8192, 10_000, 16_384, 16_391, 40_000])
def test_layer_norm(columns, kind):
    import torch
    for rows in (1, 3, 33, 300):
        g = _rng(rows, columns)
        for weight_type in sorted({kind, "float32"}):
            x = (2 * _normal(g, rows, columns, dtype=torch.float32)
                 + 3 * _normal(g, rows, 1, dtype=torch.float32)).to(_t(kind))
            weight = _normal(g, columns, dtype=_t(weight_type))
            bias = _normal(g, columns, dtype=_t(weight_type))
            out, mean, rstd = _layer_norm(x, weight, bias)
            _check_layer_norm(out, mean, rstd, x, weight, bias)


@pytest.mark.parametrize("kind", TYPES)
def test_layer_norm_without_weight_bias_or_statistics(kind):
    import torch
    from ilgpu_amd import capi
    x = _normal(_rng(51), 70, 333, dtype=_t(kind))
    weight, bias = _normal(_rng(52), 333, dtype=_t(kind)), _normal(_rng(53), 333, dtype=_t(kind))
    for w, b in ((None, None), (weight, None), (None, bias)):
        out, mean, rstd = _layer_norm(x, w, b, 0.5)
        _check_layer_norm(out, mean, rstd, x, w, b, 0.5)
        matrix, array = capi.DeviceMatrix.from_tensor, capi.DeviceArray.from_tensor
        alone = torch.empty_like(x)
        capi.layer_norm(matrix(x), matrix(alone), None if w is None else array(w),
                        None if b is None else array(b), epsilon=0.5)
        assert torch.equal(out, alone)


@pytest.mark.parametrize("columns", [100, 1537, 4096, 9000, 20_000])
def test_layer_norm_in_place_and_strided(columns):
    import torch
    for kind in TYPES:
        x = _normal(_rng(61, columns), 50, columns, dtype=_t(kind))
        weight = _normal(_rng(62), columns, dtype=torch.float32)
        bias = _normal(_rng(63), columns, dtype=torch.float32)
        out, mean, rstd = _layer_norm(x, weight, bias)
        view, memory, guard = _strided(x, columns + 3, 1)
        got, mean2, rstd2 = _layer_norm(view, weight, bias, out=view)
        _check_layer_norm(got, mean2, rstd2, x, weight, bias)
        assert bool(memory[guard].isnan().all())
        same = x.clone()
        _layer_norm(same, weight, bias, out=same)
        assert torch.equal(same, out)


def test_layer_norm_of_large_means_and_constant_rows():
    import torch
    g = _rng(71)
    x = torch.randn(20, 1000, generator=g, device="cuda") + 4096.0
    x[3] = 7.25          # no variance: epsilon alone
    x[4] = 0.0
    weight = _normal(g, 1000, dtype=torch.float32)
    bias = _normal(g, 1000, dtype=torch.float32)
    out, mean, rstd = _layer_norm(x, weight, bias)
    _check_layer_norm(out, mean, rstd, x, weight, bias)
    assert torch.equal(out[3], bias) and torch.equal(out[4], bias)


def test_layer_norm_keeps_bad_rows_to_themselves():
    import torch
    x = _normal(_rng(81), 64, 700, dtype=torch.float32)
    good, _, _ = _layer_norm(x, None, None)
    x[5, 3], x[17, 699], x[40, 0] = float("nan"), float("inf"), float("-inf")
    out, mean, rstd = _layer_norm(x, None, None)
    bad = torch.zeros(64, dtype=torch.bool, device="cuda")
    bad[[5, 17, 40]] = True
    assert torch.equal(out[~bad], good[~bad]) and bool(out[bad].isnan().all())


def test_layer_norm_of_rows_beyond_32_bit_offsets():
    import torch
    # three rows 2^30 elements apart: the last one begins at element 2^31
    rows, columns, stride = 3, 100, 1 << 30
    memory = torch.zeros(2 * stride + columns, dtype=torch.bfloat16, device="cuda")
    view = torch.as_strided(memory, (rows, columns), (stride, 1))
    x = _normal(_rng(95), rows, columns, dtype=torch.bfloat16)
    view.copy_(x)
    weight = _normal(_rng(96), columns, dtype=torch.float32)
    grad = _normal(_rng(97), rows, columns, dtype=torch.bfloat16)
    mean, rstd = _statistics(x)
    result = _layer_norm_gradient(grad, view, weight, mean, rstd, torch.float32)
    _check_layer_norm_gradient(result, grad, x, weight, mean, rstd)
    out, mean, rstd = _layer_norm(view, weight, None, out=view)
    _check_layer_norm(out, mean, rstd, x, weight, None)


def test_layer_norm_of_no_rows():
    import torch
    x = torch.empty(0, 9, device="cuda")
    out, mean, rstd = _layer_norm(x, None, None)
    assert out.shape == (0, 9)


@pytest.mark.parametrize("kind,middle,spread", [
    ("float32", 0.0, 1.0), ("float32", 1e4, 1.0), ("float32", -1e6, 1.0), ("float32", 3e7, 40.0),
    ("float16", 1000.0, 3.0), ("bfloat16", -300.0, 8.0)])
@pytest.mark.parametrize("columns", [5, 64, 100, 769, 1024, 4096, 4099, 16_384, 16_391, 100_000])
def test_layer_norm_of_rows_far_from_zero(columns, kind, middle, spread):
    # A sum passes through at most L additions: a thread adds up to 16 elements of a row in the
    # registers (V vectors of W) and of a longer one its 1024th part, W at a time; then come at most
    # six steps over lanes and four over waves.  With A the mean of |x - mean|:
    #   the first mean is off by D = (L + 1) u mean|x|,
    #   the mean of the deviations from it by d = (L + 2) u (A + D), and so is the second mean
    #   (rows whose mean is at most two deviations from zero keep the first: D + d),
    #   a deviation from that by 2 u (|x - mean| + D) + d,
    #   the variance v by (L + 6) u (v + D D) + 2 D d + d d.
    import torch
    rows = 40
    g = _rng(columns, int(abs(middle)), 91)
    x = (middle + spread * torch.randn(rows, columns, generator=g, device="cuda",
                                       dtype=torch.float64)).to(_t(kind))
    weight, bias = (_normal(g, columns, dtype=torch.float32) for _ in range(2))
    out, mean, rstd = _layer_norm(x, weight, bias)
    L = 30 + columns / 4096
    wide = x.double()
    m = wide.mean(1, keepdim=True)
    away = wide - m
    v = (away * away).mean(1, keepdim=True)
    r = 1.0 / (v + float(np.float32(1e-5))).sqrt()
    D = (L + 1) * U * wide.abs().mean(1, keepdim=True)
    d = (L + 2) * U * (away.abs().mean(1, keepdim=True) + D) + D * (m * m <= 4.01 * v)
    r_off = ((L + 6) * U * (v + D * D) + 2 * D * d + d * d) * r * r / 2 + 4 * U     # relative
    y = away * r * weight.double()
    slack = (2 * U * (away.abs() + D) + d) * r * weight.abs() + y.abs() * (1.1 * r_off + 4 * U) \
        + U * (y.abs() + bias.abs())
    _close(mean, m[:, 0], d[:, 0])
    _close(rstd, r[:, 0], (1.1 * r * r_off)[:, 0])
    _close(out, y + bias.double(), slack)


@pytest.mark.parametrize("columns", [64, 700, 20_000])
def test_layer_norm_of_rows_with_infinities_keeps_their_mean(columns):
    import torch
    x = _normal(_rng(columns, 92), 6, columns, dtype=torch.float32)
    x[1, 3], x[2, columns - 1], x[3, 0], x[3, 1] = float("inf"), float("-inf"), float("inf"), float("-inf")
    out, mean, rstd = _layer_norm(x, None, None)
    assert float(mean[1]) == float("inf") and float(mean[2]) == float("-inf")
    assert bool(mean[3].isnan()) and bool(rstd[1:4].isnan().all()) and bool(out[1:4].isnan().all())
    assert bool(torch.isfinite(out[[0, 4, 5]]).all())


# ---- layer norm's gradient ----------------------------------------------------------
def _layer_norm_gradient(grad, x, weight, mean, rstd, weight_type, want=("x", "w", "b"), into=None,
                         grad_x=None):
    import torch
    from ilgpu_amd import capi
    array, matrix = capi.DeviceArray.from_tensor, capi.DeviceMatrix.from_tensor
    columns = x.shape[1]

    def vector(k):
        return (torch.full((columns,), float("nan"), dtype=weight_type, device="cuda")
                if into is None else into[k].clone())

    if grad_x is None:
        grad_x = torch.full(x.shape, float("nan"), dtype=x.dtype, device="cuda")
    grad_w, grad_b = vector(0), vector(1)
    capi.layer_norm_gradient(
        matrix(grad), matrix(x), None if weight is None else array(weight), array(mean),
        array(rstd), matrix(grad_x) if "x" in want else None,
        array(grad_w) if "w" in want else None, array(grad_b) if "b" in want else None,
        accumulate=into is not None)
    return grad_x, grad_w, grad_b


def _check_layer_norm_gradient(result, grad, x, weight, mean, rstd, into=None):
    import torch
    grad_x, grad_w, grad_b = result
    rows, columns = x.shape
    level = columns / 64 + 32
    dy, r = grad.double(), rstd.double()[:, None]
    hat = (x.double() - mean.double()[:, None]) * r
    g = dy if weight is None else dy * weight.double()
    mean_g, mean_gh = g.mean(1, keepdim=True), (g * hat).mean(1, keepdim=True)
    exact = r * (g - mean_g - hat * mean_gh)
    slack = (level + 8) * U * r * (g.abs() + g.abs().mean(1, keepdim=True)
                                   + hat.abs() * (g * hat).abs().mean(1, keepdim=True))
    _close(grad_x, exact, slack)
    exact_w, exact_b = (dy * hat).sum(0), dy.sum(0)
    slack_w, slack_b = (rows + 4) * U * (dy * hat).abs().sum(0), rows * U * dy.abs().sum(0)
    if into is not None:
        exact_w, exact_b = exact_w + into[0].double(), exact_b + into[1].double()
        slack_w, slack_b = slack_w + U * exact_w.abs(), slack_b + U * exact_b.abs()
    _close(grad_w, exact_w, slack_w)
    _close(grad_b, exact_b, slack_b)


def _statistics(x):
    import torch
    v, m = torch.var_mean(x.double(), 1, unbiased=False)
    return m.float(), (v + 1e-5).rsqrt().float()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,columns", [
    (1, 1), (1, 4096), (2, 3), (7, 65), (64, 64), (300, 127), (1000, 256), (33, 500), (5, 768),
    (515, 1024), (2100, 1025), (70, 1537), (129, 2048), (130, 4096), (66, 4099), (300, 8192),
    (40, 10_000), (300, 16_384), (20, 16_391), (9, 40_000), (5000, 96)])
def test_layer_norm_gradient(rows, columns, kind):
    import torch
    g = _rng(rows, columns, 2)
    for weight_type in sorted({kind, "float32"}):
        x = _normal(g, rows, columns, dtype=_t(kind))
        grad = _normal(g, rows, columns, dtype=_t(kind))
        weight = _normal(g, columns, dtype=_t(weight_type))
        mean, rstd = _statistics(x)
        result = _layer_norm_gradient(grad, x, weight, mean, rstd, _t(weight_type))
        _check_layer_norm_gradient(result, grad, x, weight, mean, rstd)
        again = _layer_norm_gradient(grad, x, weight, mean, rstd, _t(weight_type))
        assert all(torch.equal(a, b) for a, b in zip(result, again))


@pytest.mark.parametrize("rows,columns", [(37, 200), (400, 1024), (90, 5000), (12, 30_000)])
def test_layer_norm_gradient_parts_accumulation_and_places(rows, columns):
    import torch
    for kind in TYPES:
        g = _rng(rows, columns, 3)
        x, grad = (_normal(g, rows, columns, dtype=_t(kind)) for _ in range(2))
        mean, rstd = _statistics(x)
        whole = _layer_norm_gradient(grad, x, None, mean, rstd, torch.float32)
        _check_layer_norm_gradient(whole, grad, x, None, mean, rstd)
        for k, part in enumerate("xwb"):
            alone = _layer_norm_gradient(grad, x, None, mean, rstd, torch.float32, want=part)
            assert torch.equal(alone[k], whole[k])
            assert all(bool(alone[j].isnan().all()) for j in range(3) if j != k)
        old = [_normal(g, columns, dtype=_t(kind)) for _ in range(2)]
        weight = _normal(g, columns, dtype=_t(kind))
        result = _layer_norm_gradient(grad, x, weight, mean, rstd, _t(kind), into=old)
        _check_layer_norm_gradient(result, grad, x, weight, mean, rstd, into=old)
        # grad_in over grad_out, over in, and between rows that are not touched
        for place in range(2):
            sources = [grad.clone(), x.clone()]
            over = _layer_norm_gradient(sources[0], sources[1], weight, mean, rstd, _t(kind),
                                        into=old, grad_x=sources[place])
            assert all(torch.equal(a, b) for a, b in zip(over, result))
        g_view, _, _ = _strided(grad, columns + 5, 3)
        x_view, _, _ = _strided(x, columns + 1, 1)
        o_view, memory, guard = _strided(torch.zeros_like(x), columns + 9, 2)
        apart = _layer_norm_gradient(g_view, x_view, weight, mean, rstd, _t(kind), into=old,
                                     grad_x=o_view)
        _check_layer_norm_gradient(apart, grad, x, weight, mean, rstd, into=old)
        assert bool(memory[guard].isnan().all())
        # one gradient row for all rows
        row = grad[:1].expand(rows, columns)
        _check_layer_norm_gradient(
            _layer_norm_gradient(row, x, weight, mean, rstd, _t(kind)), row, x, weight, mean, rstd)


def test_layer_norm_gradient_of_no_rows():
    import torch
    none = torch.empty(0, 9, device="cuda")
    stat = torch.empty(0, device="cuda")
    _, w, b = _layer_norm_gradient(none, none, None, stat, stat, torch.float32)
    assert w.eq(0).all() and b.eq(0).all()
    old = [torch.ones(9, device="cuda"), torch.full((9,), 2.0, device="cuda")]
    _, w, b = _layer_norm_gradient(none, none, None, stat, stat, torch.float32, into=old)
    assert torch.equal(w, old[0]) and torch.equal(b, old[1])


def test_layer_norm_gradient_against_differences():
    import torch
    rows, columns, epsilon, step = 4, 19, 1e-5, 1e-5
    g = _rng(91)
    x, grad = (_normal(g, rows, columns, dtype=torch.float32) for _ in range(2))
    weight, bias = (_normal(g, columns, dtype=torch.float32) for _ in range(2))
    _, mean, rstd = _layer_norm(x, weight, bias, epsilon)
    grad_x, grad_w, grad_b = _layer_norm_gradient(grad, x, weight, mean, rstd, torch.float32)

    def loss(x, w, b):
        v, m = torch.var_mean(x, 1, unbiased=False, keepdim=True)
        return float((((x - m) / torch.sqrt(v + float(np.float32(epsilon))) * w + b)
                      * grad.double()).sum())

    inputs = [x.double(), weight.double(), bias.double()]
    # central differences in float64 are off by step^2 times a third derivative of
    # size 10 and 1e-16 / step times a loss of size 10; the kernel by its sums'
    # roundings of about 40 u per unit of |grad| rstd |weight|, all at most 10 here
    tolerance = 400 * U + 1e-8
    for k, got in enumerate((grad_x, grad_w, grad_b)):
        for i in range(got.numel()):
            around = []
            for sign in (1.0, -1.0):
                moved = [t.clone() for t in inputs]
                moved[k].view(-1)[i] += sign * step
                around.append(loss(*moved))
            slope = (around[0] - around[1]) / (2 * step)
            assert abs(slope - float(got.view(-1)[i])) <= tolerance * 10, (k, i)


def test_layer_norm_gradient_of_rows_longer_than_a_grid_of_threads():
    # 2^28 columns at 16 threads each are 2^32. With a mean of 0 and a deviation of 1, whole numbers
    # stay whole.
    import torch
    rows, columns = 2, (1 << 28) + 70
    g = _rng(28, 81)
    x = _whole_numbers(g, rows, columns, dtype=torch.float16)
    grad = _whole_numbers(g, rows, columns, dtype=torch.float16)
    mean, rstd = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    _, grad_w, grad_b = _layer_norm_gradient(grad, x, None, mean, rstd, torch.float16, want="wb",
                                             grad_x=x)
    assert torch.equal(grad_b, grad[0] + grad[1])
    assert torch.equal(grad_w, grad[0] * x[0] + grad[1] * x[1])


# ---- gradient norm and clipping --------------------------------------------------------
def _lists(g, sizes, spread=1.0):
    import torch
    kinds = [torch.bfloat16, torch.float32, torch.float16]
    return [(spread * torch.randn(n, generator=g, device="cuda")).to(kinds[k % 3])
            for k, n in enumerate(sizes)]


def _norm(tensors):
    import torch
    from ilgpu_amd import capi
    norm = torch.full((1,), float("nan"), device="cuda")
    capi.gradient_norm([capi.DeviceArray.from_tensor(t) for t in tensors],
                       capi.DeviceArray.from_tensor(norm))
    return norm


def _exact_norm(tensors):
    import torch
    return float(sum((t.double() ** 2).sum() for t in tensors) ** 0.5) if tensors else 0.0


SIZES = {
    "none": [], "empty": [0, 0], "one": [1], "few": [5, 0, 3, 1000, 7],
    "chunks": [16384, 16383, 16385, 65536, 1], "large": [3_000_017, 12],
    "many": [1 + 37 * k % 4001 for k in range(300)],
    "full_table": [3] * 120, "beyond_a_table": [40_000] * 121, "tables": [9_000] * 240, "large_many": [70_001] * 260,
}


@pytest.mark.parametrize("sizes", sorted(SIZES))
def test_gradient_norm_and_clipping(sizes):
    import torch
    from ilgpu_amd import capi
    array = capi.DeviceArray.from_tensor
    tensors = _lists(_rng(len(sizes), sum(SIZES[sizes])), SIZES[sizes])
    exact = _exact_norm(tensors)
    norm = _norm(tensors)
    assert abs(float(norm) - exact) <= 1.01 * U * exact
    assert torch.equal(norm, _norm(tensors))
    listed = capi.TensorList([array(t) for t in tensors])
    for max_norm in (0.37 * exact, 2 * exact + 1, 0.0):
        n = float(norm)
        limit = float(np.float32(max_norm))
        factor = limit / n if n > limit else 1.0
        targets = [torch.full_like(t, float("nan")) for t in tensors]
        capi.clip_gradients(listed, array(norm), max_norm, [array(t) for t in targets])
        for source, target in zip(tensors, targets):
            wide = source.double() * factor
            if factor == 1.0:
                assert torch.equal(source, target)
            else:
                _close(target, wide, 2 * U * wide.abs())
        places = [t.clone() for t in tensors]
        capi.clip_gradients([array(t) for t in places], array(norm), max_norm)
        assert all(torch.equal(a, b) for a, b in zip(places, targets))


def test_gradient_norm_beyond_float32_squares():
    import torch
    big = torch.full((1000,), 1e25, device="cuda")
    small = torch.full((1000,), 1e-30, device="cuda")
    for t in (big, small):
        exact = _exact_norm([t])
        assert abs(float(_norm([t])) - exact) <= 1.01 * U * exact


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("max_norm", [2.0, 1.0, 1e-3, 1e-10, 1e-30, 0.0])
def test_clipping_by_factors_below_the_normal_numbers(max_norm, kind):
    # 1 / 3e38 is a subnormal number; norm, factor and product are rounded once each.
    import torch
    from ilgpu_amd import capi
    array = capi.DeviceArray.from_tensor
    t = torch.randn(10_007, generator=_rng(113), device="cuda", dtype=torch.float64)
    t = (t * (3e38 / float(t.norm()))).to(_t(kind))
    norm = _norm([t])
    assert 2.9e38 < float(norm) < 3.1e38
    out = torch.empty_like(t)
    capi.clip_gradients([array(t)], array(norm), max_norm, [array(out)])
    exact = t.double() * (float(np.float32(max_norm)) / _exact_norm([t]))
    _close(out, exact, 3 * U * exact.abs())


@pytest.mark.parametrize("bad", ["inf", "-inf", "nan"])
def test_clipping_leaves_gradients_of_no_finite_norm(bad):
    import torch
    from ilgpu_amd import capi
    array = capi.DeviceArray.from_tensor
    tensors = _lists(_rng(101), [1000, 20, 4000])
    tensors[1][7] = float(bad)
    norm = _norm(tensors)
    assert bool(norm.isnan().all()) if bad == "nan" else float(norm) == float("inf")
    before = [t.clone() for t in tensors]
    targets = [torch.zeros_like(t) for t in tensors]
    capi.clip_gradients([array(t) for t in tensors], array(norm), 1.0, [array(t) for t in targets])
    capi.clip_gradients([array(t) for t in tensors], array(norm), 1.0)
    for t, b, o in zip(tensors, before, targets):
        assert torch.equal(t.view(torch.uint8), b.view(torch.uint8))
        assert torch.equal(o.view(torch.uint8), b.view(torch.uint8))


def test_gradient_norm_of_unaligned_tensors():
    import torch
    from ilgpu_amd import capi
    array = capi.DeviceArray.from_tensor
    for kind in TYPES:
        memory = _normal(_rng(111), 50_000, dtype=_t(kind))
        kept = memory.clone()
        parts = [memory[1:20_000], memory[20_003:20_010], memory[30_001:49_999]]
        exact = _exact_norm(parts)
        norm = _norm(parts)
        assert abs(float(norm) - exact) <= 1.01 * U * exact
        capi.clip_gradients([array(t) for t in parts], array(norm), 0.5 * float(norm))
        for a, b in ((0, 1), (20_000, 20_003), (20_010, 30_001), (49_999, 50_000)):
            assert torch.equal(memory[a:b], kept[a:b])
        wide = kept[30_001:49_999].double() * 0.5
        _close(parts[2], wide, 3 * U * wide.abs())


def test_gradient_norm_of_a_tensor_beyond_32_bits():
    import torch
    from ilgpu_amd import capi
    array = capi.DeviceArray.from_tensor
    n = (1 << 31) + 5
    t = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    t[0], t[n // 2], t[n - 1] = 3.0, 4.0, 12.0
    norm = _norm([t])
    assert float(norm) == 13.0
    capi.clip_gradients([array(t)], array(norm), 6.5)
    assert [float(t[k]) for k in (0, 1, n // 2, n - 2, n - 1)] == [1.5, 0.0, 2.0, 0.0, 6.0]


# ---- streams and graphs -------------------------------------------------------------
def _step(capi, torch, s, stream=None):
    """Lookup, norm, both gradients, norm of the gradients and clipping, as one program."""
    array, matrix = capi.DeviceArray.from_tensor, capi.DeviceMatrix.from_tensor
    capi.embedding(matrix(s["table"]), array(s["tokens"]), matrix(s["x"]), scale=2.0, stream=stream)
    capi.layer_norm(matrix(s["x"]), matrix(s["y"]), array(s["w"]), array(s["b"]),
                    mean=array(s["mean"]), rstd=array(s["rstd"]), stream=stream)
    capi.layer_norm_gradient(matrix(s["y"]), matrix(s["x"]), array(s["w"]), array(s["mean"]),
                             array(s["rstd"]), matrix(s["dx"]), array(s["dw"]), array(s["db"]),
                             s.get("temp_norm"), stream=stream)
    capi.embedding_gradient(matrix(s["dx"]), array(s["tokens"]), matrix(s["dt"]),
                            s.get("temp_embedding"), scale=2.0, stream=stream)
    grads = [array(s[k]) for k in ("dt", "dw", "db")]
    capi.gradient_norm(grads, array(s["norm"]), s.get("temp_list"), stream=stream)
    capi.clip_gradients(grads, array(s["norm"]), 0.01, stream=stream)


def _step_state(torch, capi, n=5000, vocabulary=3001, dimension=520):
    g = _rng(n, vocabulary, dimension, 7)

    def empty(*shape):
        return torch.full(shape, float("nan"), device="cuda")

    return {"table": _normal(g, vocabulary, dimension, dtype=torch.float32),
            "tokens": _tokens(g, n, vocabulary, torch.int64),
            "w": _normal(g, dimension, dtype=torch.float32),
            "b": _normal(g, dimension, dtype=torch.float32), "x": empty(n, dimension),
            "y": empty(n, dimension), "dx": empty(n, dimension), "mean": empty(n),
            "rstd": empty(n), "dw": empty(dimension), "db": empty(dimension),
            "dt": empty(vocabulary, dimension), "norm": empty(1)}


RESULTS = ("x", "y", "mean", "rstd", "dx", "dw", "db", "dt", "norm")


def test_operators_on_another_stream():
    import torch
    from ilgpu_amd import capi
    s = _step_state(torch, capi)
    _step(capi, torch, s)
    torch.cuda.synchronize()
    first = {k: s[k].clone() for k in RESULTS}
    side = torch.cuda.Stream()
    for handle in (side, side.cuda_stream):
        for k in RESULTS:
            s[k].fill_(float("nan"))
        side.wait_stream(torch.cuda.current_stream())
        _step(capi, torch, s, stream=handle)
        # memory that the call's own temps would share with work on this stream
        for _ in range(4):
            torch.full((1 << 20,), -1, dtype=torch.int32, device="cuda")
        side.synchronize()
        for k in RESULTS:
            assert torch.equal(s[k], first[k]), k


def test_operators_in_a_graph():
    import torch
    from ilgpu_amd import capi
    s = _step_state(torch, capi, 9000, 2000, 130)
    s["temp_norm"] = capi.temp_buffer(capi.layer_norm_gradient_temp_bytes(9000, 130))
    s["temp_embedding"] = capi.temp_buffer(capi.embedding_gradient_temp_bytes(9000, 2000, 130))
    s["temp_list"] = capi.temp_buffer(capi.gradient_norm_temp_bytes(3))
    capi.sort_check_device()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(capi, torch, s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _step(capi, torch, s)
    for round_ in range(4):
        s["table"].copy_(_normal(_rng(round_, 5), 2000, 130, dtype=torch.float32))
        s["tokens"].copy_(_tokens(_rng(round_, 6), 9000, 2000, torch.int64))
        _step(capi, torch, s)
        torch.cuda.synchronize()
        eager = {k: s[k].clone() for k in RESULTS}
        for k in RESULTS:
            s[k].fill_(float("nan"))
        for name in ("temp_norm", "temp_embedding", "temp_list"):
            s[name].bytes.fill_(0xA5)
        graph.replay()
        torch.cuda.synchronize()
        for k in RESULTS:
            assert torch.equal(s[k], eager[k]), (round_, k)
