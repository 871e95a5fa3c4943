"""Paged-cache append, attention of single tokens over the pages, and attention inside packed prompts, against their
definitions in 64 bits.

Tolerances. A result in 16 bits is off by half a step (`_HALF` of its value), and the weights of the softmax are rounded once to
the same type before they meet the values: half a step of sum(p |v|) at worst. What f32 adds is below 2^-15 of that sum: scores
here are below 16, f32 sums of 128 terms err by at most 128 * 2^-24 of them. With 32-bit activations every factor keeps 21 bits
or more: scores of a standard deviation s err by about s * 2^-21 from the factors and, in 16 partial sums each rounded
towards zero, by up to s * 16 * 2^-24 from the sums, with s < 2.5 here: 3.6e-6 of each weight, and the weighted sum adds its
own 2^-21: 4.1e-6 of the norm in all. Were a low-order factor lost, it would be some 1e-4.
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


def _randn(shape, seed, dtype, scale=1.25):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _reference(q, k, v, scale, causal_from=None):
    """q [n, h, d], k and v [m, kv, d] in f64 -> (out, sum of p |v|); causal_from: position of q's first row."""
    n, h, d = q.shape
    m, kv = k.shape[:2]
    if m == 0 or n == 0:
        return torch.zeros(n, h, d, dtype=torch.float64, device="cuda"), torch.zeros(n, h, d, dtype=torch.float64, device="cuda")
    out, mag = [], []
    for j in range(h):
        s = q[:, j] @ k[:, j // (h // kv)].T * scale
        vj = v[:, j // (h // kv)]
        if causal_from is not None:
            s = s.masked_fill(torch.arange(m, device="cuda")[None, :] > torch.arange(n, device="cuda")[:, None] + causal_from, float("-inf"))
        p = torch.softmax(s, dim=-1)
        out.append(p @ vj)
        mag.append(p @ vj.abs())
    return torch.stack(out, 1), torch.stack(mag, 1)


def _check(got, want, mag, what):
    assert torch.isfinite(got.float()).all(), what
    err = (got.double() - want).abs()
    if got.dtype == F32:
        rel = (err.norm() / want.norm().clamp(min=1e-30)).item()
        assert rel <= 4.1e-6, (what, rel)
    else:
        tol = _HALF[got.dtype] * (want.abs() + mag) + 2.0 ** -15 * mag
        assert (err <= tol).all(), (what, (err / tol.clamp(min=1e-30)).max().item())


def _table(lens, page, seed, extra=2, width=None):
    """Pages of the sequences in no order, -1 behind the last one; and the number of pages."""
    need = [-(-max(n, 0) // page) for n in lens]
    total = sum(need) + extra
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    width = width or max(1, max(need))
    rows, at = [], 0
    for n in need:
        rows.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return _ints(rows), total


def _gather(cache, table, s, n):
    page = cache.shape[2]
    ids = table[s, :-(-n // page)].long()
    return cache[ids].transpose(1, 2).reshape(-1, cache.shape[1], cache.shape[3])[:n].double()


def _tables(n, d):
    inv = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    ang = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * inv
    ang = torch.cat((ang, ang), 1)
    return ang.cos().float(), ang.sin().float()


def _stacked(rows, h, kv, d, seed, dtype):
    qkv = _randn((rows, (h + 2 * kv) * d), seed, dtype)
    return qkv[:, :h * d].view(rows, h, d), qkv[:, h * d:(h + kv) * d].view(rows, kv, d), qkv[:, (h + kv) * d:].view(rows, kv, d)


def _turn(x, pos, cos, sin):
    """The rotation in f32, every product and difference rounded by itself as the kernel does it."""
    half = x.shape[-1] // 2
    c, s = cos[pos.long()][:, None, :half], sin[pos.long()][:, None, :half]
    lo, hi = x[..., :half].float(), x[..., half:].float()
    return torch.cat((lo * c - hi * s, hi * c + lo * s), -1)


# ---- append

@pytest.mark.parametrize("act,cache", _PAIRS)
@pytest.mark.parametrize("h,kv,d,page,lens", [(8, 2, 128, 16, [17, 1, 300]), (5, 5, 64, 1, [3, 40]), (32, 1, 128, 64, [65]),
                                              (32, 8, 64, 1024, [1] * 70), (1, 1, 128, 8, [9, 8, 7])])
def test_append(act, cache, h, kv, d, page, lens):
    from fuel_b200 import ops
    table, pages = _table(lens, page, 3)
    rows = sum(lens)
    q, k, v = _stacked(rows, h, kv, d, 5, act)
    kc, vc = (torch.full((pages, kv, page, d), float("nan"), dtype=cache, device="cuda") for _ in range(2))
    seq = _ints([s for s, n in enumerate(lens) for _ in range(n)])
    pos = _ints([p for n in lens for p in range(n)])
    cos, sin = _tables(max(lens), d)
    k_out = torch.empty(k.shape, dtype=act, device="cuda")
    got = ops.paged_append(k, v, kc, vc, table, pos, cos, sin, seq_ids=seq, q=q, k_out=k_out)
    rot_q, rot_k = _turn(q, pos, cos, sin), _turn(k, pos, cos, sin)
    assert torch.equal(got, rot_q.to(act)) and torch.equal(k_out, rot_k.to(act))
    at = table.long()[seq.long(), (pos // page).long()] * page + (pos % page).long()
    written = torch.zeros(pages * page, dtype=torch.bool, device="cuda")
    written[at] = True
    for c, want in ((kc, rot_k.to(cache)), (vc, v.to(cache))):
        flat = c.transpose(1, 2).reshape(-1, kv, d)
        assert torch.equal(flat[at], want)
        assert flat[~written].isnan().all()            # every other place as it was
    # without queries and without the second copy of the keys: the same caches; one row per sequence without seq_ids
    kc2, vc2 = torch.full_like(kc, float("nan")), torch.full_like(vc, float("nan"))
    assert ops.paged_append(k, v, kc2, vc2, table, pos, cos, sin, seq_ids=seq) is None
    assert torch.equal(kc2.nan_to_num(7), kc.nan_to_num(7)) and torch.equal(vc2.nan_to_num(7), vc.nan_to_num(7))
    first = _ints([0] * len(lens))
    kc2.fill_(float("nan")), vc2.fill_(float("nan"))
    n = len(lens)
    ops.paged_append(k[:n], v[:n], kc2, vc2, table, first, cos, sin)
    flat = kc2.transpose(1, 2).reshape(-1, kv, d)
    assert torch.equal(flat[table[:, 0].long() * page], k[:n].to(cache))   # position 0 turns by nothing


def test_append_rotates_as_the_single_sequence_step_does():
    """The same bits as fuelq_rope_store with a cache that has one page per sequence."""
    from fuel_b200 import _lib, ops
    h, kv, d, room, at = 4, 2, 128, 64, 37
    q, k, v = (_randn((1, n, d), s, F32) for n, s in ((h, 1), (kv, 2), (kv, 3)))
    cos, sin = _tables(room, d)
    kc, vc = torch.zeros(1, kv, room, d, device="cuda"), torch.zeros(1, kv, room, d, device="cuda")
    kc2, vc2, q2, pos = kc.clone(), vc.clone(), q.clone(), _ints([at])
    got = ops.paged_append(k, v, kc, vc, _ints([[0]]), pos, cos, sin, q=q)
    _lib.check(_lib.lib.fuelq_rope_store(q2.data_ptr(), k.data_ptr(), v.data_ptr(), kc2.data_ptr(), vc2.data_ptr(), cos.data_ptr(),
                                         sin.data_ptr(), pos.data_ptr(), h, kv, d, room, torch.cuda.current_stream().cuda_stream), "rope")
    assert torch.equal(got, q2) and torch.equal(kc, kc2) and torch.equal(vc, vc2)


def test_append_padding_in_place_and_bad_indices():
    from fuel_b200 import _lib, ops
    h, kv, d, page = 4, 2, 64, 16
    q, k, v = (_randn((6, n, d), s, F16) for n, s in ((h, 1), (kv, 2), (kv, 3)))
    cos, sin = _tables(64, d)
    kc, vc = torch.zeros(4, kv, page, d, dtype=F16, device="cuda"), torch.zeros(4, kv, page, d, dtype=F16, device="cuda")
    q0, k0 = q.clone(), k.clone()
    # rows 1 and 3 are padding; in place
    seq, pos = _ints([0, 0, 1, -1, 1, 0]), _ints([20, -1, 5, 7, 6, 21])
    assert ops.paged_append(k, v, kc, vc, _ints([[2, 0], [3, -1]]), pos, cos, sin, seq_ids=seq, q=q, q_out=q, k_out=k) is q
    real = torch.tensor([0, 2, 4, 5], device="cuda")
    assert torch.equal(q[[1, 3]], q0[[1, 3]]) and torch.equal(k[[1, 3]], k0[[1, 3]])
    assert torch.equal(q[real], _turn(q0, pos.clamp(min=0), cos, sin).half()[real])
    assert torch.equal(kc[3, :, 5], k[2]) and torch.equal(kc[0, :, 4], k[0]) and torch.equal(vc[0, :, 5], v[5])
    assert int((kc != 0).any(-1).any(1).sum()) == 4
    assert ops.device_error() == 0
    # a position behind the angles, behind the table, a page that is none, a sequence that is none: left out, and told
    for s, p, row in ((0, 64, [1, 1, 1, 1, 1]), (0, 32, [1, 1]), (1, 0, [1, 1]), (1, 16, [1, 1]), (2, 0, [1, 1]), (0, 40, [1, 1, 4])):
        table = _ints([row, [-1, 9] + [0] * (len(row) - 2)])
        kc.zero_(), vc.zero_()
        ops.paged_append(k0[:2], v[:2], kc, vc, table, _ints([p, 1]), cos, sin, seq_ids=_ints([s, 0]))
        assert ops.device_error() == _lib.DEVICE_ERROR_INDEX
        assert int((kc != 0).any(-1).any(1).sum()) == 1 and torch.equal(vc[1, :, 1], v[1])


# ---- one token over the pages

_LENS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 200, 0, 1000]


@pytest.mark.parametrize("act,cache", _PAIRS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("h,kv,page", [(4, 4, 16), (8, 2, 64), (3, 1, 1), (14, 2, 8), (16, 2, 32), (16, 1, 1024), (40, 1, 4)])
def test_decode(act, cache, d, h, kv, page):
    from fuel_b200 import ops
    table, pages = _table(_LENS, page, 11)
    kc, vc = _randn((pages, kv, page, d), 1, cache), _randn((pages, kv, page, d), 2, cache)
    q, _, _ = _stacked(len(_LENS), h, kv, d, 3, act)
    ws = ops.paged_attn_workspace(len(_LENS), h, kv, d, "cuda").fill_(255)
    out = ops.paged_attn_decode(q, kc, vc, table, _ints(_LENS), workspace=ws)
    want, mag = zip(*(_reference(q[s:s + 1].double(), _gather(kc, table, s, n), _gather(vc, table, s, n), d ** -0.5)
                      for s, n in enumerate(_LENS)))
    _check(out, torch.cat(want), torch.cat(mag), (act, cache))
    assert not out[0].any() and not out[11].any()
    again = ops.paged_attn_decode(q, kc, vc, table, _ints(_LENS))
    assert torch.equal(out, again)


@pytest.mark.parametrize("act,cache,h,kv,n", [(F32, F32, 8, 8, 3001), (F32, F16, 32, 8, 70001), (BF16, BF16, 4, 1, 33333), (F16, F16, 64, 2, 9000)])
def test_decode_of_one_long_sequence(act, cache, h, kv, n):
    """Few rows: the length is split over the device and joined."""
    from fuel_b200 import ops
    d, page = 128, 32
    table, pages = _table([n], page, 5)
    kc, vc = _randn((pages, kv, page, d), 1, cache), _randn((pages, kv, page, d), 2, cache)
    q = _randn((1, h, d), 3, act, 2.0)     # wider scores: the softmax has to find its maximum again and again
    out = ops.paged_attn_decode(q, kc, vc, table, _ints([n]), scale=0.06)
    want, mag = _reference(q.double(), _gather(kc, table, 0, n), _gather(vc, table, 0, n), 0.06)
    _check(out, want, mag, n)


@pytest.mark.parametrize("act,cache", _PAIRS)
def test_decode_reads_nothing_behind_a_sequence(act, cache):
    """NaN and infinities in the rest of the last page and in pages of nobody, -1 and stale numbers behind the last page."""
    from fuel_b200 import ops
    lens, page, h, kv, d = [5, 16, 0, 33], 16, 4, 2, 128
    table, pages = _table(lens, page, 7, width=5)
    kc = torch.full((pages, kv, page, d), float("nan"), dtype=cache, device="cuda")
    vc = torch.full((pages, kv, page, d), float("inf"), dtype=cache, device="cuda")
    good_k, good_v = _randn((pages, kv, page, d), 1, cache), _randn((pages, kv, page, d), 2, cache)
    for s, n in enumerate(lens):
        for p in range(n):
            kc[table[s, p // page], :, p % page] = good_k[table[s, p // page], :, p % page]
            vc[table[s, p // page], :, p % page] = good_v[table[s, p // page], :, p % page]
    table[0, 2], table[1, 3] = 10 ** 6, 0
    q = _randn((4, h, d), 3, act)
    out = ops.paged_attn_decode(q, kc, vc, table, _ints(lens))
    want, mag = zip(*(_reference(q[s:s + 1].double(), _gather(kc, table, s, n), _gather(vc, table, s, n), d ** -0.5) for s, n in enumerate(lens)))
    _check(out, torch.cat(want), torch.cat(mag), (act, cache))


def test_decode_bad_pages_and_lengths_are_told():
    from fuel_b200 import _lib, ops
    page, h, kv, d = 16, 4, 2, 64
    kc, vc = _randn((6, kv, page, d), 1, F16), _randn((6, kv, page, d), 2, F16)
    q = _randn((3, h, d), 3, F16)
    good = ops.paged_attn_decode(q, kc, vc, _ints([[1, 2], [3, 4], [5, 0]]), _ints([20, 30, 32]))
    out = ops.paged_attn_decode(q, kc, vc, _ints([[1, 2], [-1, 4], [5, 0]]), _ints([20, 30, 32]))
    assert ops.device_error() == _lib.DEVICE_ERROR_INDEX
    assert torch.equal(out[[0, 2]], good[[0, 2]])
    only = ops.paged_attn_decode(q[1:2], kc, vc, _ints([[4]]), _ints([14]))    # the keys of the page that is there
    assert (out[1].float() - only[0].float()).abs().max() <= 2 ** -9
    out = ops.paged_attn_decode(q, kc, vc, _ints([[1, 2], [3, 4], [5, 0]]), _ints([20, 30, 33]))   # longer than its row of the table
    assert ops.device_error() == _lib.DEVICE_ERROR_INDEX
    assert torch.equal(out, good)
    out = ops.paged_attn_decode(q, kc, vc, _ints([[6, 2], [3, 4], [5, 0]]), _ints([16, -5, 32]))   # no such page; a length below zero
    assert ops.device_error() == _lib.DEVICE_ERROR_INDEX
    assert not out[0].any() and not out[1].any() and torch.equal(out[2], good[2])


def test_decode_of_scores_at_the_ends_of_their_type():
    """One key far above others of the type's lowest value takes all; all of them at the lowest value share alike."""
    from fuel_b200 import ops
    page, h, kv, d = 16, 2, 1, 64
    low = torch.finfo(F32).min
    kc, vc = torch.zeros(3, kv, page, d, device="cuda"), _randn((3, kv, page, d), 2, F32)
    q = torch.zeros(3, h, d, device="cuda")
    q[:, :, 0] = 1.0
    kc[0, 0, :, 0] = low
    kc[0, 0, 3, 0] = 2.0
    kc[1, 0, :, 0] = low
    kc[2, 0, 5, 0] = -low
    out = ops.paged_attn_decode(q, kc, vc, _ints([[0], [1], [2]]), _ints([16, 16, 16]), scale=1.0)
    assert (out[0, 0] - vc[0, 0, 3]).abs().max() <= 1e-6
    assert (out[1, 0] - vc[1, 0].mean(0)).abs().max() <= 1e-6
    assert (out[2, 0] - vc[2, 0, 5]).abs().max() <= 1e-6


def test_decode_of_pages_behind_four_gigabytes():
    """Element offsets beyond 2^31, byte offsets beyond 2^32."""
    from fuel_b200 import ops
    page, h, kv, d = 64, 8, 8, 128
    pages = (1 << 32) // (2 * kv * page * d) + 40
    if torch.cuda.mem_get_info()[0] < 3 * pages * kv * page * d * 2:
        pytest.skip("not enough memory")
    kc, vc = (torch.empty(pages, kv, page, d, dtype=F16, device="cuda") for _ in range(2))
    table = _ints([[pages - 1, 0, pages - 2], [pages - 3, pages - 4, 1]])
    used = table.flatten().long()
    kc[used], vc[used] = _randn((6, kv, page, d), 1, F16), _randn((6, kv, page, d), 2, F16)
    q, k, v = _stacked(2, h, kv, d, 3, F16)
    lens = _ints([130, 192])
    cos, sin = _tables(256, d)
    qr = ops.paged_append(k, v, kc, vc, table, lens - 1, cos, sin, q=q)
    out = ops.paged_attn_decode(qr, kc, vc, table, lens)
    small, at = _ints([[0, 1, 2], [3, 4, 5]]), used
    out2 = ops.paged_attn_decode(qr, kc[at].contiguous(), vc[at].contiguous(), small, lens)
    assert torch.equal(out, out2)
    assert torch.equal(kc[pages - 2, :, 1], _turn(k, lens - 1, cos, sin).half()[0])


# ---- prompts

_PACKS = [[1], [2, 0, 1], [0, 5, 0, 130, 128, 129, 1, 0], [255, 256, 257], [700, 64, 1025]]


@pytest.mark.parametrize("act", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("h,kv", [(2, 2), (8, 2), (3, 1)])
@pytest.mark.parametrize("lens", _PACKS, ids=lambda x: "_".join(map(str, x)))
def test_prompt(act, d, h, kv, lens):
    """Rows apart in a stacked projection; rows behind the last sequence hold NaN and stay as they were in the result."""
    from fuel_b200 import ops
    rows, pad = sum(lens), 7
    q, k, v = _stacked(rows + pad, h, kv, d, 3, act)
    for t in (q, k, v):
        t[rows:] = float("nan")
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    out = torch.full((rows + pad, h, d), 5.0, dtype=act, device="cuda")
    ws = ops.prompt_attn_workspace(q, k).fill_(255)
    ops.prompt_attn(q, k, v, _ints(starts), out=out, workspace=ws)
    assert (out[rows:] == 5.0).all()
    for s, n in enumerate(lens):
        a, b = starts[s], starts[s] + n
        if n:
            want, mag = _reference(q[a:b].double(), k[a:b].double(), v[a:b].double(), d ** -0.5, 0)
            _check(out[a:b], want, mag, (act, d, h, kv, s))
    again = ops.prompt_attn(q, k, v, _ints(starts))
    assert torch.equal(out[:rows], again[:rows])


@pytest.mark.parametrize("act", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_rows_do_not_see_what_stands_behind_them(act, d):
    """NaN and infinities in later rows of the sequence and in the next one."""
    from fuel_b200 import ops
    lens, h, kv = [300, 50], 2, 1
    q, k, v = _stacked(350, h, kv, d, 3, act)
    want = ops.prompt_attn(q, k, v, _ints([0, 300, 350]))
    for at in (0, 1, 17, 130, 256, 299):
        for bad in (float("nan"), float("inf"), float("-inf")):
            for which in (k, v):
                t = which.clone()
                t[at, 0, 5] = bad
                t[300:] = bad
                out = ops.prompt_attn(q, t if which is k else k, t if which is v else v, _ints([0, 300, 350]))
                assert torch.equal(out[:at], want[:at]), (at, bad, which is k)
                if which is v:     # from there on that column holds it, and no other column does
                    col = out[at:300, :, 5].float()
                    assert (col.isnan().all() if bad != bad else (col == bad).all()), (at, bad)
                    cols = [c for c in range(d) if c != 5]
                    assert torch.equal(out[:300][:, :, cols], want[:300][:, :, cols]), (at, bad)


@pytest.mark.parametrize("act", [F32, BF16])
def test_prompt_of_very_uneven_magnitudes(act):
    """A later row a thousand million times larger: the rows before it keep their accuracy."""
    from fuel_b200 import ops
    q, k, v = _stacked(200, 2, 2, 128, 3, act)
    v[100:] *= 2.0 ** 30
    out = ops.prompt_attn(q, k, v, _ints([0, 200]))
    want, mag = _reference(q.double(), k.double(), v.double(), 128 ** -0.5, 0)
    _check(out[:100], want[:100], mag[:100], "before")
    _check(out[100:], want[100:], mag[100:], "behind")


def test_prompt_of_a_long_sequence_samples():
    from fuel_b200 import ops
    n, h, kv, d = 9001, 4, 2, 128
    for act in (F16, BF16, F32):
        q, k, v = _stacked(n, h, kv, d, 3, act)
        q.mul_(2.0)
        out = ops.prompt_attn(q, k, v, _ints([0, n]), scale=0.06)
        for a in (0, 127, 4000, 8190, n - 40):
            want, mag = _reference(q[a:a + 40].double(), k[:a + 40].double(), v[:a + 40].double(), 0.06, a)
            _check(out[a:a + 40], want, mag, (act, a))


def test_prompt_boundaries_that_are_none():
    """Sequences that end before they begin or behind the rows: left out, and told; the others are right."""
    from fuel_b200 import _lib, ops
    q, k, v = _stacked(64, 2, 2, 64, 3, F16)
    good = ops.prompt_attn(q, k, v, _ints([0, 20, 40]))
    for cu in ([0, 20, 40, 90], [0, 20, 40, 30], [0, 20, 40, -3]):
        out = torch.full_like(good, 9.0)
        ops.prompt_attn(q, k, v, _ints(cu), out=out)
        assert ops.device_error() == _lib.DEVICE_ERROR_INDEX, cu
        assert torch.equal(out[:40], good[:40]), cu
        assert (out[40:] == 9.0).all(), cu


@pytest.mark.parametrize("act", [F32, F16])
def test_thousands_of_short_prompts(act):
    """More sequences than rows of most of them: the search for a block's sequence takes several rounds, many slots are empty."""
    from fuel_b200 import ops
    lens = [(i * 7) % 5 for i in range(1500)] + [0] * 700 + [130]
    h, kv, d, rows = 2, 1, 64, sum(lens)
    q, k, v = _stacked(rows, h, kv, d, 3, act)
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    out = ops.prompt_attn(q, k, v, _ints(starts))
    # all at once: rows of one sequence see each other and nothing else
    seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), _ints(lens).long())
    idx = torch.arange(rows, device="cuda")
    hidden = (seq[:, None] != seq[None, :]) | (idx[None, :] > idx[:, None])
    want, mag = [], []
    for j in range(h):
        p = torch.softmax((q[:, j].double() @ k[:, 0].double().T * d ** -0.5).masked_fill(hidden, float("-inf")), -1)
        want.append(p @ v[:, 0].double()), mag.append(p @ v[:, 0].double().abs())
    _check(out, torch.stack(want, 1), torch.stack(mag, 1), act)


def test_decode_of_thousands_of_sequences():
    from fuel_b200 import ops
    lens = [(i * 13) % 40 for i in range(3000)]
    h, kv, d, page = 2, 1, 64, 8
    table, pages = _table(lens, page, 1)
    kc, vc = _randn((pages, kv, page, d), 1, F16), _randn((pages, kv, page, d), 2, F16)
    q = _randn((len(lens), h, d), 3, F16)
    out = ops.paged_attn_decode(q, kc, vc, table, _ints(lens))
    ids = table.clamp(min=0).long()
    kk, vv = (c[ids].transpose(1, 2).reshape(len(lens), -1, d).double() for c in (kc, vc))     # [sequences, keys, d]
    s = q.double() @ kk.transpose(1, 2) * d ** -0.5
    seen = torch.arange(kk.shape[1], device="cuda") < _ints(lens)[:, None]
    p = torch.softmax(s.masked_fill(~seen[:, None], float("-inf")), -1).nan_to_num(0.0)
    _check(out, p @ vv, p @ vv.abs(), "many")


# ---- together

@pytest.mark.parametrize("act,cache", _PAIRS)
def test_prompts_then_tokens(act, cache):
    """Two prompts packed with padding behind them, their keys into the pages, then single tokens as decoding adds them, one
    sequence leaving on the way: every row against the definition over all of its sequence's rows."""
    from fuel_b200 import ops
    h, kv, d, page, room = 8, 2, 128, 16, 4
    lens, steps = [37, 18, 0], 20
    cos, sin = _tables(64, d)
    table = _ints([[7, 1, 9, 3], [2, 0, 8, 4], [5, -1, -1, -1]])
    kc, vc = (torch.full((10, kv, page, d), float("nan"), dtype=cache, device="cuda") for _ in range(2))
    rows = sum(lens)
    q, k, v = _stacked(rows + 3, h, kv, d, 1, act)
    seq, pos = _ints([0] * 37 + [1] * 18 + [-1] * 3), _ints(list(range(37)) + list(range(18)) + [0] * 3)
    k_rot = torch.empty(k.shape, dtype=act, device="cuda")
    q_rot = ops.paged_append(k, v, kc, vc, table, pos, cos, sin, seq_ids=seq, q=q, k_out=k_rot)
    out = ops.prompt_attn(q_rot, k_rot, v, _ints([0, 37, 55]))
    keys, vals = [k_rot[:37].double(), k_rot[37:55].double()], [v[:37].double(), v[37:55].double()]
    for s, a in ((0, 0), (1, 37)):
        want, mag = _reference(q_rot[a:a + lens[s]].double(), keys[s], vals[s], d ** -0.5, 0)
        _check(out[a:a + lens[s]], want, mag, ("prompt", s))
    for step in range(steps):
        live = step < 12
        q, k, v = _stacked(3, h, kv, d, 100 + step, act)
        pos = _ints([37 + step, 18 + step if live else -1, -1])
        q_rot = torch.zeros(3, h, d, dtype=act, device="cuda")
        ops.paged_append(k, v, kc, vc, table, pos, cos, sin, q=q, q_out=q_rot)
        out = ops.paged_attn_decode(q_rot, kc, vc, table, (pos + 1).clamp(min=0))
        for s in range(2 if live else 1):
            n = int(pos[s]) + 1
            kk, vv = _gather(kc, table, s, n), _gather(vc, table, s, n)
            assert torch.equal(kk[-1], _turn(k, pos.clamp(min=0), cos, sin).to(cache).double()[s])
            want, mag = _reference(q_rot[s:s + 1].double(), kk, vv, d ** -0.5)
            _check(out[s:s + 1], want, mag, ("step", step, s))
        assert not out[2].any()


def test_decode_agrees_with_the_single_sequence_step():
    """fuelq_attn_decode over a contiguous f32 cache, and the same keys in pages: two f32 orders of the same sums."""
    from fuel_b200 import _lib, ops
    h, kv, d, room, n, page = 32, 8, 128, 640, 513, 16
    kc, vc = _randn((kv, room, d), 1, F32), _randn((kv, room, d), 2, F32)
    q, pos = _randn((1, h, d), 3, F32), _ints([n - 1])
    one = torch.empty(1, h, d, device="cuda")
    ws = torch.empty(_lib.lib.fuelq_attn_decode_workspace_bytes(h), dtype=torch.uint8, device="cuda")
    _lib.check(_lib.lib.fuelq_attn_decode(q.data_ptr(), kc.data_ptr(), vc.data_ptr(), one.data_ptr(), pos.data_ptr(), h, kv, d, room,
                                          d ** -0.5, ws.data_ptr(), ws.numel(), None, torch.cuda.current_stream().cuda_stream), "attn")
    table = _ints([torch.randperm(room // page).tolist()])
    pk, pv = torch.empty(room // page, kv, page, d, device="cuda"), torch.empty(room // page, kv, page, d, device="cuda")
    pk[table[0].long()] = kc.view(kv, -1, page, d).transpose(0, 1)
    pv[table[0].long()] = vc.view(kv, -1, page, d).transpose(0, 1)
    got = ops.paged_attn_decode(q, pk, pv, table, _ints([n]))
    assert ((got - one).norm() / one.norm()).item() <= 8.2e-6     # twice the bound of one


def test_captured_step_with_other_lengths():
    """Append and decode captured once, replayed with other positions, pages and lengths; two graphs on one workspace in turn."""
    from fuel_b200 import ops
    h, kv, d, page, n = 8, 2, 128, 16, 5
    cos, sin = _tables(512, d)
    kc, vc = _randn((200, kv, page, d), 1, F16), _randn((200, kv, page, d), 2, F16)
    ws = ops.paged_attn_workspace(n, h, kv, d, "cuda")
    q, k, v = _stacked(n, h, kv, d, 3, F32)
    table, pos = torch.zeros(n, 32, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    lens = torch.ones(n, dtype=torch.int32, device="cuda")

    def step():
        qr = ops.paged_append(k, v, kc, vc, table, pos, cos, sin, q=q)
        return ops.paged_attn_decode(qr, kc, vc, table, lens, workspace=ws)

    graphs, outs = [], []
    stream = torch.cuda.Stream()
    for _ in range(2):
        with torch.cuda.stream(stream):
            step()
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(step())
        graphs.append(g)
    kc0, vc0 = kc.clone(), vc.clone()
    for i, now in enumerate(([1, 500, 17, 64, 3], [100, 1, 1, 300, 511], [16, 16, 16, 16, 16])):
        kc.copy_(kc0), vc.copy_(vc0)
        new, _ = _table(now, page, i, width=32)
        table.copy_(new)
        lens.copy_(_ints(now))
        pos.copy_(lens - 1)
        torch.cuda.synchronize()
        graphs[i % 2].replay()
        graphs[1 - i % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1])
        want, mag = [], []
        qr = _turn(q, pos, cos, sin).double()
        for s, m in enumerate(now):
            w, g = _reference(qr[s:s + 1], _gather(kc, table, s, m), _gather(vc, table, s, m), d ** -0.5)
            want.append(w), mag.append(g)
        _check(outs[0], torch.cat(want), torch.cat(mag), now)


@pytest.mark.parametrize("act", [F32, F16])
def test_captured_prompts_with_other_boundaries(act):
    """Captured once, replayed with other sequences in the same rows; the result in place of the queries."""
    from fuel_b200 import ops
    rows, h, kv, d = 700, 4, 2, 128
    q, k, v = (_randn((rows, n, d), s, act) for n, s in ((h, 1), (kv, 2), (kv, 3)))
    q0, cu, ws = q.clone(), _ints([0, 1, 2, 3]), ops.prompt_attn_workspace(q, k)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ops.prompt_attn(q, k, v, cu, out=q, workspace=ws)
    stream.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        ops.prompt_attn(q, k, v, cu, out=q, workspace=ws)
    for starts in ([0, 300, 300, 700], [0, 1, 129, 400], [0, 0, 0, 700]):
        cu.copy_(_ints(starts))
        q.copy_(q0)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(starts, starts[1:]):
            want, mag = _reference(q0[a:b].double(), k[a:b].double(), v[a:b].double(), d ** -0.5, 0)
            if b > a:
                _check(q[a:b], want, mag, (act, starts))
        assert torch.equal(q[starts[-1]:], q0[starts[-1]:])


def test_two_streams_with_a_workspace_each():
    from fuel_b200 import ops
    h, kv, d, page = 16, 4, 128, 16
    lens = [3000, 1, 700, 64]
    table, pages = _table(lens, page, 1)
    kc, vc = _randn((pages, kv, page, d), 1, BF16), _randn((pages, kv, page, d), 2, BF16)
    q, k, v = _stacked(900, h, kv, d, 3, BF16)
    cu, ln = _ints([0, 400, 900]), _ints(lens)
    want_d, want_p = ops.paged_attn_decode(q[:4], kc, vc, table, ln), ops.prompt_attn(q, k, v, cu)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((ops.paged_attn_decode(q[:4], kc, vc, table, ln), ops.prompt_attn(q, k, v, cu)))
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a, want_d) and torch.equal(b, want_p)


def test_refusals_of_the_python_entries():
    from fuel_b200 import _lib, ops
    q, k, v = _stacked(4, 4, 2, 64, 3, F16)
    kc, vc = _randn((3, 2, 16, 64), 1, F16), _randn((3, 2, 16, 64), 2, F16)
    table, ints, cu = _ints([[0], [1], [2], [0]]), _ints([1, 2, 3, 4]), _ints([0, 4])
    cos, sin = _tables(8, 64)
    for bad in (dict(kc=kc.float()), dict(table=table[:3]), dict(table=table.long()), dict(lens=ints[:3]), dict(q=q.float().bfloat16()),
                dict(q=q.transpose(1, 2)), dict(kc=kc[:, :1]), dict(out=torch.empty(4, 4, 64, device="cuda"))):
        a = dict(q=q, kc=kc, table=table, lens=ints, out=None) | bad
        with pytest.raises((ValueError, _lib.FuelqError)):
            ops.paged_attn_decode(a["q"], a["kc"], vc, a["table"], a["lens"], out=a["out"])
    for bad in (dict(k=k[:3]), dict(k=k.float()), dict(v=v[:, :1]), dict(cu=cu.long()), dict(cu=cu[:0]), dict(q=q[:, :3])):
        a = dict(q=q, k=k, v=v, cu=cu) | bad
        with pytest.raises((ValueError, _lib.FuelqError)):
            ops.prompt_attn(a["q"], a["k"], a["v"], a["cu"])
    for bad in (dict(k=k[:3]), dict(pos=ints[:2]), dict(cos=cos.half()), dict(cos=cos[:, :32]), dict(q=q[:3]), dict(q_out=q.float()),
                dict(k_out=k), dict(seq=ints[:2]), dict(table=table[:2], seq=None)):
        a = dict(k=k, pos=ints, cos=cos, q=q, q_out=None, k_out=None, seq=ints, table=table) | bad
        with pytest.raises((ValueError, _lib.FuelqError)):
            ops.paged_append(a["k"], v, kc, vc, a["table"], a["pos"], a["cos"], sin, seq_ids=a["seq"], q=a["q"], q_out=a["q_out"], k_out=a["k_out"])
    small = torch.empty(16, dtype=torch.uint8, device="cuda")
    if _lib.lib.fuelq_paged_attn_workspace_bytes(4, 4, 2, 64) > 16:
        with pytest.raises(_lib.FuelqError):
            ops.paged_attn_decode(q, kc, vc, table, ints, workspace=small)
