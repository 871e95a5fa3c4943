"""Attention at the ends of the number ranges: scores near and beyond f32's ends, one key far above all others, infinities among
the values that a row sees, large values behind it. Against the definitions in 64 bits, or against the same call without them.

Tolerances. `_HALF` is half a step of a 16-bit type. Results in 32 bits: 4.1e-6 of the norm for scores of a standard deviation
below 2.5 (every factor keeps 21 bits, 16 partial sums rounded towards zero), and a score of g adds its own 22 bits, g * 2^-22.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
_HALF = {F16: 2.0 ** -11, BF16: 2.0 ** -8}
_PAIRS = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]


@pytest.fixture(autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from fuel_b200 import ops
    ops.device_error(clear=True)
    yield
    assert ops.device_error(clear=True) == 0


def _randn(shape, seed, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _sink(n, h, d, act, cache, gap, seed):
    """q [1, h, d], k and v [n, 1, d]: the first key scores `gap` in every head and holds values of zero, the others' scores have a
    standard deviation of 0.3."""
    q, k, v = _randn((1, h, d), seed, act, 0.3), _randn((n, 1, d), seed + 1, cache), _randn((n, 1, d), seed + 2, cache)
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    k[0] = 0.0
    k[0, 0, 0] = gap / (8.0 * d ** -0.5)
    v[0] = 0.0
    return q, k, v


def _attend(q, k, v, scale):
    """q [h, d], k and v [n, d] in 64 bits -> (out, sum of p |v|)"""
    p = torch.softmax(q @ k.T * scale, -1)
    return p @ v, p @ v.abs()


def _near_the_end(shape, seed, dtype):
    """Values up to 0.95 of the type's largest"""
    return (torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").clamp(-1.9, 1.9) / 2.0
            * torch.finfo(dtype).max).to(dtype)


def _pages(k, v, page):
    """k and v [n, 1, d] as a paged cache of one sequence, its pages in reverse"""
    n, _, d = k.shape
    pages = -(-n // page)
    kc, vc = (torch.zeros(pages * page, 1, d, dtype=k.dtype, device="cuda") for _ in range(2))
    kc[:n], vc[:n] = k, v
    kc, vc = (c.view(pages, page, 1, d).transpose(1, 2).flip(0).contiguous() for c in (kc, vc))
    return kc, vc, _ints([list(range(pages - 1, -1, -1))])


# ---- one key far above all others

@pytest.mark.parametrize("gap", [8.0, 12.0, 16.0, 20.0])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("act,cache", _PAIRS)
def test_decode_keeps_small_weights_beside_one_large(act, cache, d, gap):
    """The result is the sum of two thousand weights of e^-gap: each has to keep its type's bits."""
    from fuel_b200 import ops
    n, h = 2049, 4
    q, k, v = _sink(n, h, d, act, cache, gap, 3)
    kc, vc, table = _pages(k, v, 16)
    out = ops.paged_attn_decode(q, kc, vc, table, _ints([n]))
    want, mag = _attend(q[0].double(), k[:, 0].double(), v[:, 0].double(), d ** -0.5)
    err = (out[0].double() - want).abs()
    if act == F32:
        assert (err.norm() / want.norm()).item() <= 4.1e-6 + gap * 2.0 ** -22
    else:
        # beside the roundings of the weights and of the result: scores of `gap` in f32 sums of 128 terms. Results below 2^-14 are
        # whole multiples of 2^-24 in f16, whatever they come from: half of one is off
        least = 2.0 ** -25 if act == F16 else 0.0
        assert (err <= _HALF[act] * (want.abs() + mag) + (2.0 ** -15 + gap * 2.0 ** -17) * mag + least).all()


@pytest.mark.parametrize("act,gap", [(F16, 12.0), (F16, 16.0), (BF16, 16.0), (F32, 16.0)])
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_keeps_small_weights_beside_one_large(act, d, gap):
    from fuel_b200 import ops
    n, h = 1500, 2
    q1, k, v = _sink(n, h, d, act, act, gap, 3)
    q = q1.expand(n, h, d).contiguous()
    out = ops.prompt_attn(q, k, v, _ints([0, n]))
    for row in (500, 1023, 1499):
        want, mag = _attend(q[row].double(), k[:row + 1, 0].double(), v[:row + 1, 0].double(), d ** -0.5)
        err = (out[row].double() - want).abs()
        if act == F32:
            assert (err.norm() / want.norm()).item() <= 4.1e-6 + gap * 2.0 ** -22
        else:
            least = 2.0 ** -25 if act == F16 else 0.0       # as above
            assert (err <= _HALF[act] * (want.abs() + mag) + (2.0 ** -15 + gap * 2.0 ** -17) * mag + least).all(), row


# ---- values that are not finite, seen by the row

@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("act,cache", _PAIRS)
def test_decode_of_infinite_values(act, cache, d, bad):
    """A value of infinity has a weight above zero: its column is that infinity, the others are as they were. Infinities of both
    signs make NaN."""
    from fuel_b200 import ops
    h, n = 6, 700
    q, k, v = _randn((2, h, d), 3, act), _randn((n, 1, d), 4, cache), _randn((n, 1, d), 5, cache)
    for at in (0, 77, 699):
        b = v.clone()
        b[at, 0, 9] = bad
        b[at, 0, 40] = -bad
        b[at // 2, 0, 50], b[at // 2 + 300 if at < 699 else 3, 0, 50] = math.inf, -math.inf
        kc, vc, table = _pages(k, v, 16)
        _, bc, _ = _pages(k, b, 16)
        table, lens = table.repeat(2, 1), _ints([n, n])
        good, out = ops.paged_attn_decode(q, kc, vc, table, lens), ops.paged_attn_decode(q, kc, bc, table, lens)
        for c, want in ((9, bad), (40, -bad), (50, math.nan)):
            col = out[..., c].float()
            assert (col.isnan() if want != want else col == want).all(), (at, c, col)
        cols = [c for c in range(d) if c not in (9, 40, 50)]
        assert torch.equal(out[..., cols], good[..., cols])


@pytest.mark.parametrize("act", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_of_infinite_values_of_hardly_any_weight(act, d):
    """Beside a key of e^100 times their weight: the weights round to zero, the infinities are there all the same, and nowhere else."""
    from fuel_b200 import ops
    n, h = 700, 3
    q, k, v = _randn((n, h, d), 1, act, 0.3), _randn((n, 1, d), 2, act), _randn((n, 1, d), 3, act)
    q[..., 0], k[..., 0], k[0] = 16.0, 0.0, 0.0
    k[0, 0, 0] = 100.0 / (16.0 * d ** -0.5)
    good = ops.prompt_attn(q, k, v, _ints([0, n]))
    b = v.clone()
    b[50, 0, 7], b[50, 0, 9], b[300, 0, 9], b[140, 0, 11], b[699, 0, 13] = math.inf, -math.inf, math.inf, math.nan, math.inf
    out = ops.prompt_attn(q, k, b, _ints([0, n]))
    want = good.clone()
    want[50:, :, 7], want[50:, :, 9], want[300:, :, 9], want[140:, :, 11], want[699:, :, 13] = math.inf, -math.inf, math.nan, math.nan, math.inf
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(nan=7.0), want.nan_to_num(nan=7.0))


@pytest.mark.parametrize("act", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_of_infinite_values_in_every_short_prompt(act, d):
    """Each thread block takes many items one after the other, nearly all of them with an infinity in their last key tile: what is
    noted of one is not lost to the next."""
    from fuel_b200 import ops
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(1, 129, (2500,), generator=g)
    lens[::9] += 128
    start = torch.cat((torch.zeros(1, dtype=torch.long), lens.cumsum(0)))
    rows, h = int(start[-1]), 2
    q, k, v = _randn((rows, h, d), 1, act), _randn((rows, 1, d), 2, act), _randn((rows, 1, d), 3, act)
    where, col = start[:-1] + (torch.rand(2500, generator=g) * lens).long(), torch.randint(0, d, (2500,), generator=g)
    sign = torch.where(torch.rand(2500, generator=g) < 0.5, -1.0, 1.0)
    v[where.cuda(), 0, col.cuda()] = (sign * math.inf).to(act).cuda()
    want = torch.zeros(rows, d)
    for a, b, c, x in zip(where.tolist(), start[1:].tolist(), col.tolist(), sign.tolist()):
        want[a:b, c] = x
    want = want.cuda()[:, None].expand(rows, h, d)
    for _ in range(10):
        out = ops.prompt_attn(q, k, v, start.int().cuda()).float()
        assert torch.equal(torch.where(out.isinf(), out.sign(), 0.0 * out), want)


@pytest.mark.parametrize("act,cache", _PAIRS)
def test_decode_of_nothing_but_infinite_values(act, cache):
    """Every column of every key, in items of one block and of several; then a page of NaN."""
    from fuel_b200 import ops
    h, kv, d, page, lens = 8, 2, 128, 16, [5000, 1, 130, 0, 64]
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(1)).tolist()
    table, at = torch.full((len(lens), max(need)), -1, dtype=torch.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    q, kc = _randn((len(lens), h, d), 1, act), _randn((at, kv, page, d), 2, cache)
    vc = torch.full((at, kv, page, d), -math.inf, dtype=cache, device="cuda")
    out = ops.paged_attn_decode(q, kc, vc, table.cuda(), _ints(lens))
    live = [0, 1, 2, 4]
    assert (out[live] == -math.inf).all() and not out[3].any()
    vc[table[0, 7]] = math.nan
    out = ops.paged_attn_decode(q, kc, vc, table.cuda(), _ints(lens))
    assert out[0].isnan().all() and (out[live[1:]] == -math.inf).all()


# ---- scores at the ends of their range

@pytest.mark.parametrize("act", [F32, BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("scale", [1.0, 5.0])
def test_prompt_of_scores_at_the_ends_of_their_type(act, d, scale):
    """Scores whose product with log2(e) passes f32's range: the softmax is that of the scores. Among keys of the type's lowest value
    another takes all; if there are no others they share alike; a key at the highest value takes all."""
    from fuel_b200 import ops
    n, h = 300, 2
    low = torch.finfo(act).min
    if act == F16:
        scale *= 2.0 ** 110         # f16's ends are not f32's: the scale takes the scores there
    v = _randn((n, 1, d), 2, act)
    q = torch.zeros(n, h, d, dtype=act, device="cuda")
    q[..., 0] = 1.0
    half = _HALF.get(act, 0.0)
    cu = _ints([0, n])

    def close(got, want, mag):      # means of 300 values in f32 sums: 300 * 2^-24 at most
        assert ((got.double() - want).abs() <= half * (want.abs() + mag) + 2.0 ** -15 * mag).all()

    def same(got, want):            # 32 bits: two f16 parts of each value, the lower one a whole multiple of 2^-24 beside 2^14
        off = (got.double() - want.double()).abs()
        assert (off <= (2.0 ** -21 * want.abs() + 2.0 ** -37 * want.abs().max() if act == F32 else 0.0)).all()

    k = torch.zeros(n, 1, d, dtype=act, device="cuda")
    k[..., 0] = low
    k[130, 0, 0] = 2.0
    out = ops.prompt_attn(q, k, v, cu, scale=scale)
    for row in (0, 1, 127, 129):
        close(out[row, 0], v[:row + 1, 0].double().mean(0), v[:row + 1, 0].double().abs().mean(0))
    for row in (130, 131, 255, 299):
        same(out[row, 0], v[130, 0])
    k.zero_()
    for high in (140, 290):
        k[high, 0, 0] = -low
    out = ops.prompt_attn(q, k, v, cu, scale=scale)
    close(out[139, 1], v[:140, 0].double().mean(0), v[:140, 0].double().abs().mean(0))
    for row in (140, 200, 256, 289):
        same(out[row, 1], v[140, 0])
    two = v[[140, 290], 0].double()
    close(out[295, 0], two.mean(0), two.abs().mean(0))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 17, 2.0 ** 20, 2.0 ** 24, 2.0 ** 60])
def test_prompt_of_large_scores_alike(d, size):
    """Equal keys of large scores, in two key tiles and more, values of different magnitudes: every row is the mean of the values, in
    place of the queries too."""
    from fuel_b200 import ops
    n, h = 1000, 2
    q, k, v = _randn((n, h, d), 1, F32), _randn((1, 1, d), 2, F32, size).expand(n, 1, d).contiguous(), _randn((n, 1, d), 3, F32)
    v[::7] *= 2.0 ** -12
    out = ops.prompt_attn(q, k, v, _ints([0, n]))
    want = v.double().cumsum(0) / torch.arange(1, n + 1, device="cuda")[:, None, None]
    assert ((out.double() - want).norm() / (want.norm() * h ** 0.5)).item() <= 4.1e-6
    assert torch.equal(ops.prompt_attn(q, k, v, _ints([0, n]), out=q), out) and torch.equal(q, out)


@pytest.mark.parametrize("act,size", [(F16, 300.0), (F16, 5000.0), (F16, 30000.0), (BF16, 1e6), (BF16, 1e15)])
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_of_large_queries_and_keys(act, size, d):
    """Scores far above what an exponent holds: the key with the largest takes all, wherever it is clear of the next. Rows beside such
    rows keep their bits."""
    from fuel_b200 import ops
    n = 600
    q, k, v = _randn((n, 2, d), 1, act), _randn((n, 1, d), 2, act), _randn((n, 1, d), 3, act)
    size = min(size, torch.finfo(act).max / 5.0)       # five deviations
    large_q, large_k = (q.float() * size).to(act), (k.float() * size).to(act)
    out = ops.prompt_attn(large_q, large_k, v, _ints([0, n]))
    s = torch.einsum("ihd,jhd->hij", large_q.double(), large_k.double().expand(n, 2, d)) * d ** -0.5
    s = s.masked_fill(torch.arange(n, device="cuda")[None, :] > torch.arange(n, device="cuda")[:, None], -math.inf)
    two = s.topk(2, -1)
    clear = two.values[..., 0] - two.values[..., 1] > 40.0 + 2.0 ** -16 * s.abs().nan_to_num(posinf=0.0).amax(-1)
    clear[:, 0] = True
    assert clear.sum() > 0.8 * clear.numel()
    want = v[two.indices[..., 0], 0].transpose(0, 1)
    # one weight rounded to the type beside its sum that is not, and the result: two half steps; f16 steps are 2^-24 at least
    tol = 2.02 * _HALF[act] * want.double().abs() + (2.0 ** -25 if act == F16 else 0.0)
    assert ((out.double() - want.double()).abs() <= tol)[clear.T].all()
    good, mixed = ops.prompt_attn(q, k, v, _ints([0, n])), q.clone()
    mixed[::3] = large_q[::3]
    out = ops.prompt_attn(mixed, k, v, _ints([0, n]))
    keep = [i for i in range(n) if i % 3]
    assert torch.equal(out[keep], good[keep])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("act", [F16, BF16])
@pytest.mark.parametrize("large", [2.0 ** 8, 2.0 ** 11, 2.0 ** 13, 2.0 ** 14, 2.0 ** 15])
def test_prompt_of_close_scores_far_from_zero(act, large, d):
    """Scores of up to 2^30, exact in f32, that lie a few units apart and rise from key tile to key tile: their weights are those of the
    distances, at either sign."""
    from fuel_b200 import ops
    n, scale = 500, 0.125
    step = max(1.0, large * large * 2.0 ** -23)         # the least that f32 tells apart there
    q, k = (torch.zeros(n, 1, d, dtype=act, device="cuda") for _ in range(2))
    v = _randn((n, 1, d), 3, act)
    rise = torch.randint(0, 6, (n,), generator=torch.Generator().manual_seed(1)) + 3 * (torch.arange(n) // 100)
    q[..., 0], q[..., 1], k[..., 0], k[:, 0, 1] = large, step, large, rise.cuda().to(act)
    for sign in (1.0, -1.0):
        k[..., 0] = sign * large
        out = ops.prompt_attn(q, k, v, _ints([0, n]), scale=scale)
        for row in (0, 1, 99, 127, 128, 200, 301, 499):
            want, mag = _attend(q[row].double(), k[:row + 1, 0].double(), v[:row + 1, 0].double(), scale)
            off = (out[row].double() - want).abs()
            # differences of up to 20 steps, exact but for the factor's 24 bits: the weights' rounding and the result's
            assert (off <= _HALF[act] * (want.abs() + mag) + 2.0 ** -15 * mag).all(), (sign, row)


def test_prompt_of_factors_whose_powers_pass_f32():
    """Large columns of q meet columns of zero in k and the other way round: the scores are of a few units."""
    from fuel_b200 import ops
    n, d = 200, 64
    q, k, v = (_randn((n, 1, d), s, F32) for s in (1, 2, 3))
    q[..., 0], k[..., 0] = 2.0 ** 100, 0.0
    q[..., 1], k[..., 1] = 0.0, 2.0 ** 100
    q[..., 2:], k[..., 2:] = 0.0, 0.0         # what is left of them beside 2^100 is zero in any 22 bits
    out = ops.prompt_attn(q, k, v, _ints([0, n]))
    want = v.double().cumsum(0) / torch.arange(1, n + 1, device="cuda")[:, None, None]
    assert ((out.double() - want).norm() / want.norm()).item() <= 4.1e-6


@pytest.mark.parametrize("act,cache", _PAIRS)
def test_the_largest_scale(act, cache):
    """Large queries at a scale of 2^127: the key of the largest product takes all, equal ones share, zeros are zeros."""
    from fuel_b200 import ops
    n, d, scale = 300, 64, 2.0 ** 127
    q = torch.zeros(n, 1, d, dtype=act, device="cuda")
    q[..., 0] = 2.0 ** 15
    k, v = torch.zeros(n, 1, d, dtype=cache, device="cuda"), _randn((n, 1, d), 2, cache)
    k[7::100, 0, 0] = 0.5
    for last, seen in ((299, [7, 107, 207]), (6, range(7))):
        want = v[list(seen), 0].double().mean(0)
        tol = 2 * _HALF.get(act, 2.0 ** -17) * v.double().abs().max()
        kc, vc, table = _pages(k, v, 16)
        got = ops.paged_attn_decode(q[last:last + 1], kc, vc, table, _ints([last + 1]), scale=scale)
        assert ((got[0, 0].double() - want).abs() <= tol).all(), last
        if act == cache:
            assert ((ops.prompt_attn(q, k, v, _ints([0, n]), scale=scale)[last, 0].double() - want).abs() <= tol).all(), last


@pytest.mark.parametrize("act", [F32, BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_rows_with_a_score_of_infinity_are_nan(act, d):
    """inf - inf is in the softmax of such a row, wherever the key lies; the rows before it do not see it."""
    from fuel_b200 import ops
    n = 400
    q, k, v = _randn((n, 2, d), 1, act), _randn((n, 1, d), 2, act), _randn((n, 1, d), 3, act)
    q[..., 0] = 1.0
    want = ops.prompt_attn(q, k, v, _ints([0, n]))
    for at in list(range(0, 34)) + [129, 138, 139, 143, 255, 256, 300, 399]:
        b = k.clone()
        b[at, 0, 0] = math.inf
        out = ops.prompt_attn(q, b, v, _ints([0, n]))
        assert out[at:].isnan().all(), at
        assert torch.equal(out[:at], want[:at])


@pytest.mark.parametrize("act,cache", [(F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("d", [64, 128])
def test_decode_of_scores_of_infinity(act, cache, d):
    """+inf makes the row NaN, -inf is a weight of zero, and a row with no other scores has no weights: zeros."""
    from fuel_b200 import ops
    n, h = 300, 3
    q, k, v = _randn((1, h, d), 1, act), _randn((n, 1, d), 2, cache), _randn((n, 1, d), 3, cache)
    q[..., 0] = 1.0
    for at in (0, 5, 150, 299):
        b = k.clone()
        b[at, 0, 0] = math.inf
        kc, vc, table = _pages(b, v, 32)
        assert ops.paged_attn_decode(q, kc, vc, table, _ints([n])).isnan().all(), at
    b = k.clone()
    b[:290, 0, 0] = -math.inf
    kc, vc, table = _pages(b, v, 32)
    out = ops.paged_attn_decode(q, kc, vc, table, _ints([n]))
    want, mag = _attend(q[0].double(), k[290:, 0].double(), v[290:, 0].double(), d ** -0.5)
    assert ((out[0].double() - want).abs() <= _HALF[act] * (want.abs() + mag) + 2.0 ** -15 * mag).all()
    assert not ops.paged_attn_decode(q, kc, vc, table, _ints([290])).any()


@pytest.mark.parametrize("act", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_rows_whose_first_keys_score_minus_infinity(act, d):
    """Two key tiles and more of weights of zero, then others."""
    from fuel_b200 import ops
    n, first = 500, 300
    q, k, v = _randn((n, 2, d), 1, act), _randn((n, 1, d), 2, act), _randn((n, 1, d), 3, act)
    q[..., 0] = 1.0
    k[:first, 0, 0] = -math.inf
    out = ops.prompt_attn(q, k, v, _ints([0, n]))
    assert not out[:first].any()
    for row in (300, 301, 383, 384, 499):
        want, mag = _attend(q[row].double(), k[first:row + 1, 0].double(), v[first:row + 1, 0].double(), d ** -0.5)
        assert ((out[row].double() - want).abs() <= _HALF[act] * (want.abs() + mag) + 2.0 ** -15 * mag).all(), row


# ---- large values

@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("act", [F32, F16, BF16])
def test_prompt_of_values_at_the_ends_of_their_type(act, d):
    """Their means are finite, whatever their sums are."""
    from fuel_b200 import ops
    n = 700
    q, k, v = _randn((n, 2, d), 1, act), _randn((n, 1, d), 2, act), _near_the_end((n, 1, d), 3, act)
    v[::5] = torch.finfo(act).max * 0.9
    out = ops.prompt_attn(q, k, v, _ints([0, n]))
    for row in (0, 1, 127, 128, 300, 699):
        want, mag = _attend(q[row].double(), k[:row + 1, 0].double(), v[:row + 1, 0].double(), d ** -0.5)
        off = (out[row].double() - want).abs()
        if act == F32:
            assert (off.norm() / want.norm()).item() <= 4.1e-6, row
        else:
            assert (off <= _HALF[act] * (want.abs() + mag) + 2.0 ** -15 * mag).all(), row


@pytest.mark.parametrize("act,cache", _PAIRS)
def test_decode_of_values_at_the_ends_of_their_type(act, cache):
    """One row in one block's run and one that is joined from several."""
    from fuel_b200 import ops
    n, h, d = 3000, 3, 128
    q, k, v = _randn((2, h, d), 1, act), _randn((n, 1, d), 2, cache), _near_the_end((n, 1, d), 3, cache)
    v[::5] = torch.finfo(cache).max * 0.9
    kc, vc, table = _pages(k, v, 16)
    out = ops.paged_attn_decode(q, kc, vc, table.repeat(2, 1), _ints([n, 5]))
    for s, m in ((0, n), (1, 5)):
        want, mag = _attend(q[s].double(), k[:m, 0].double(), v[:m, 0].double(), d ** -0.5)
        off = (out[s].double() - want).abs()
        if act == F32:
            assert (off.norm() / want.norm()).item() <= 4.1e-6, s
        else:
            assert (off <= _HALF[act] * (want.abs() + mag) + 2.0 ** -15 * mag).all(), s


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("gap", [-30.0, 0.0, 10.0, 14.0])
def test_prompt_of_values_as_far_apart_as_f32_goes(d, gap):
    """A value of 2^125 among values of one, in the same key tile and in others: what the others weigh is in the softmax's sum."""
    from fuel_b200 import ops
    n = 400
    q, k, v = _randn((n, 1, d), 1, F32, 0.3), _randn((n, 1, d), 2, F32), _randn((n, 1, d), 3, F32)
    q[..., 0], k[..., 0] = 8.0, 0.0
    for at in (50, 300):
        k[at], v[at] = 0.0, v[at] * 2.0 ** 125
        k[at, 0, 0] = gap / (8.0 * d ** -0.5)
    out = ops.prompt_attn(q, k, v, _ints([0, n]))
    for row in (0, 49, 50, 51, 127, 128, 255, 299, 300, 399):
        want, _ = _attend(q[row].double(), k[:row + 1, 0].double(), v[:row + 1, 0].double(), d ** -0.5)
        off = out[row].double() - want
        assert (off.norm() / want.norm()).item() <= 4.1e-6 + abs(gap) * 2.0 ** -22, row


def test_long_prompt_of_infinite_values():
    """Two columns infinite in every row of 40000: told apart from the others without a pass over them for each row."""
    from fuel_b200 import ops
    n, d = 40000, 128
    q, k, v = _randn((n, 1, d), 1, F32), _randn((n, 1, d), 2, F32), _randn((n, 1, d), 3, F32)
    v[:, 0, 3], v[:, 0, 77] = math.inf, -math.inf
    v[20000, 0, 3] = -math.inf
    out = ops.prompt_attn(q, k, v, _ints([0, n]))
    assert (out[:20000, 0, 3] == math.inf).all() and out[20000:, 0, 3].isnan().all() and (out[:, 0, 77] == -math.inf).all()
    cols = [c for c in range(d) if c not in (3, 77)]
    for row in (0, 5000, 20000, n - 1):
        want, _ = _attend(q[row].double(), k[:row + 1, 0].double(), v[:row + 1, 0][:, cols].double(), d ** -0.5)
        assert ((out[row][:, cols].double() - want).norm() / want.norm()).item() <= 4.1e-6


# ---- large values behind a row

@pytest.mark.parametrize("act", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_rows_do_not_see_large_values_behind_them(act, d):
    """The type's largest values in later rows of the sequence, in the next one and behind the last: weights of zero, not nearly."""
    from fuel_b200 import ops
    rows, cu = 360, _ints([0, 300, 350])
    q, k, v = _randn((rows, 2, d), 1, act), _randn((rows, 1, d), 2, act), _randn((rows, 1, d), 3, act)
    want = ops.prompt_attn(q, k, v, cu)
    for bad in (torch.finfo(act).max, torch.finfo(act).min):
        for at in list(range(1, 19)) + [137, 138, 256, 299]:
            b = v.clone()
            b[at:300] = bad
            b[300:] = bad
            out = ops.prompt_attn(q, k, b, cu)
            assert torch.equal(out[:at], want[:at]), (bad, at)


# ---- nothing in the cache yet

@pytest.mark.parametrize("act,cache", [(F32, F16), (BF16, BF16)])
def test_a_batch_of_free_slots_without_pages(act, cache):
    """No page and no column of the table: padding is skipped, free slots are zeros, anything else is told."""
    from fuel_b200 import _lib, ops
    n, h, kv, d = 3, 4, 2, 64
    q, k, v = _randn((n, h, d), 1, act), _randn((n, kv, d), 2, act), _randn((n, kv, d), 3, act)
    kc, vc = (torch.empty(0, kv, 16, d, dtype=cache, device="cuda") for _ in range(2))
    table, cos = torch.empty(n, 0, dtype=torch.int32, device="cuda"), torch.empty(0, d, device="cuda")
    ops.paged_append(k, v, kc, vc, table, _ints([-1, -1, -1]), cos, cos, q=q)
    assert not ops.paged_attn_decode(q, kc, vc, table, _ints([0, -3, 0])).any()
    assert ops.device_error() == 0
    ops.paged_append(k, v, kc, vc, table, _ints([-1, 0, -1]), cos, cos, q=q)
    assert ops.device_error() == _lib.DEVICE_ERROR_INDEX
    assert not ops.paged_attn_decode(q, kc, vc, table, _ints([0, 2, 0])).any()
    assert ops.device_error() == _lib.DEVICE_ERROR_INDEX
