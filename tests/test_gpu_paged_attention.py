"""The paged cache's operators on the GPU against plain 64-bit arithmetic: every type, the lengths and page
sizes at which a tile, a chunk or a page ends, ragged and padded batches, any order of the pools in memory,
far pages, bad pages, and the append -> attend -> verify -> roll back cycle of a serving loop."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import nanocamelid_amd as nc  # noqa: E402

from tests.paged_util import Pages, attend, close, ints, starts, weights_rounded  # noqa: E402

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]
ids = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731


@pytest.fixture(scope="module")
def ctx():
    assert torch.cuda.is_available(), "GPU tests need the MI355X"
    return nc.Context(0)


def _randn(shape, seed, gain=1.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * gain).to(dtype).cuda()


def _sequences(lens, page, kv, hd, dtype, seed, **more):
    """A filled cache; each sequence's last key and first key attract queries like 'strong' below."""
    cache = Pages(lens, page, kv, hd, dtype, seed, **more)
    for s, n in enumerate(lens):
        if n > 0:
            cache.fill(s, _randn((n, kv, hd), seed + 31 * s), _randn((n, kv, hd), seed + 31 * s + 1))
    return cache


def _check(ctx, cache, lens, rows, heads, kv, hd, qt, seed, row_start=True, scale=None, **batch):
    starts_ = starts(rows)
    q = _randn((int(starts_[-1]), heads, hd), seed, 1.5, qt)
    b = nc.PagedBatch(cache.table, ints(lens), ints(starts_) if row_start else None, **batch)
    out = nc.paged_attention(ctx, nc.PagedKV(cache.k, cache.v), b, q, scale)
    for s, (n, m) in enumerate(zip(rows, lens)):
        k, v = cache.read(s, max(m, 0))
        a = int(starts_[s])
        want, tol = attend(q[a:a + n], k, v, scale if scale is not None else hd**-0.5)
        if m > 0:
            tol = weights_rounded(tol, v, qt)
        close(out[a:a + n], want, tol, ("sequence", s, n, m))
    return q, b, out


# lengths on both sides of 16, 32, 64, 128, 256 and 512 positions, from one on
LENS = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 255, 256, 257, 511, 512, 513, 600, 1030]


@pytest.mark.parametrize("qt,ct", TYPES, ids=ids)
@pytest.mark.parametrize("heads,kv,hd,page", [(8, 2, 128, 16), (8, 8, 64, 24), (12, 4, 128, 5), (20, 2, 64, 64), (17, 1, 128, 100)])
def test_one_row_a_sequence(ctx, qt, ct, heads, kv, hd, page):
    cache = _sequences(LENS, page, kv, hd, ct, 5)
    _check(ctx, cache, LENS, [1] * len(LENS), heads, kv, hd, qt, 6, row_start=False)


@pytest.mark.parametrize("qt,ct", TYPES, ids=ids)
@pytest.mark.parametrize("heads,kv,hd,page", [(8, 2, 128, 16), (32, 8, 64, 7), (64, 8, 128, 256), (3, 3, 64, 1)])
def test_verify_rows(ctx, qt, ct, heads, kv, hd, page):
    """Ragged rows, none among them, more than a tile of them, and all of a sequence's."""
    lens = [9, 40, 5, 300, 64, 258, 129, 700]
    rows = [9, 5, 0, 3, 64, 4, 70, 1]
    cache = _sequences(lens, page, kv, hd, ct, 11)
    _check(ctx, cache, lens, rows, heads, kv, hd, qt, 12)


@pytest.mark.parametrize("rows", [1, 2, 4, 5, 8, 9, 16, 17, 33])
def test_every_row_count(ctx, rows):
    lens = [rows, rows + 250, 513]
    cache = _sequences(lens, 16, 2, 128, F16, 21)
    _check(ctx, cache, lens, [rows] * 3, 8, 2, 128, F32, 22)


def test_padded_batch_and_rows_without_positions(ctx):
    """Sequences of no positions, and rows that stand before the first one: zeros, whatever the cache holds."""
    lens, rows = [0, 3, -5, 2, 20], [1, 5, 2, 2, 0]
    cache = _sequences([max(n, 0) for n in lens], 16, 2, 64, F32, 31)
    q, _, out = _check(ctx, cache, lens, rows, 4, 2, 64, F32, 32)
    assert (out[:3] == 0).all() and (out[3:6] != 0).all() and (out[6:8] == 0).all()


def test_rows_outside_every_sequence_are_left(ctx):
    cache = _sequences([30, 40], 16, 2, 64, F32, 41)
    q = _randn((12, 4, 64), 42)
    out = torch.full_like(q, 7.0)
    b = nc.PagedBatch(cache.table, ints([30, 40]), ints([2, 5, 9]))
    nc.paged_attention(ctx, nc.PagedKV(cache.k, cache.v), b, q, out=out)
    assert (out[:2] == 7).all() and (out[9:] == 7).all() and (out[2:9] != 7).all()


@pytest.mark.parametrize("order", [(0, 1, 2), (0, 2, 1), (2, 0, 1), (1, 0, 2)])
@pytest.mark.parametrize("ct", [F32, BF16], ids=ids)
def test_any_order_of_the_pools(ctx, order, ct):
    lens = [70, 300]
    cache = _sequences(lens, 16, 4, 128, ct, 51, order=order)
    _check(ctx, cache, lens, [2, 3], 8, 4, 128, F32, 52)


def test_interleaved_pools_and_strided_rows(ctx):
    """k and v pages side by side in one tensor, layers apart; queries inside a fused buffer."""
    both = torch.full((2, 9, 2, 16, 2, 64), float("nan"), dtype=F16, device="cuda")
    cache = Pages([100], 16, 2, 64, F16, 61)
    cache.k, cache.v = both[1, :, 0], both[1, :, 1]
    cache.fill(0, _randn((100, 2, 64), 62), _randn((100, 2, 64), 63))
    fused = _randn((3, 8 * 64), 64)
    q = fused[:, :256].view(3, 4, 64)
    b = nc.PagedBatch(cache.table, ints([100]), ints([0, 3]))
    out = nc.paged_attention(ctx, nc.PagedKV(cache.k, cache.v), b, q)
    k, v = cache.read(0, 100)
    want, tol = attend(q, k, v, 0.125)
    close(out, want, tol)
    assert torch.isnan(both[0]).all()


def test_scale_and_bounds_of_lengths(ctx):
    """A scale of its own, zero, negative; max_len as tight as it may be; a table with rows apart."""
    lens = [5, 600, 257]
    cache = _sequences(lens, 16, 2, 64, F32, 71, width=40)
    for scale in (1.0, 0.0, -0.3):
        _check(ctx, cache, lens, [1, 1, 1], 4, 2, 64, F32, 72, scale=scale, max_len=600)
    wide = torch.full((3, 200), -1, dtype=torch.int32, device="cuda")
    wide[:, :cache.table.shape[1]] = cache.table
    cache.table = wide[:, :cache.table.shape[1] + 2]
    _check(ctx, cache, lens, [2, 2, 2], 4, 2, 64, F32, 73)


def test_large_and_infinite_scores(ctx):
    """Scores far from zero, one key far above all, and keys of infinite size: as the formula says."""
    cache = _sequences([400], 16, 1, 64, F32, 81)
    k, v = cache.read(0, 400)
    k[7] *= 60
    k[300] *= 80
    cache.fill(0, k, v)
    _check(ctx, cache, [400], [1], 2, 1, 64, F32, 82)
    q = torch.ones((1, 2, 64), device="cuda")
    k[:] = 0
    k[5, 0, 0] = -math.inf
    cache.fill(0, k, v)
    b = nc.PagedBatch(cache.table, ints([400]))
    out = nc.paged_attention(ctx, nc.PagedKV(cache.k, cache.v), b, q)
    keep = torch.arange(400) != 5
    want = v.cpu().double()[keep, 0].mean(0)
    # 399 equal weights: sums of 399 terms
    assert ((out.cpu().double()[0] - want).abs() <= 2 * 500 * 2.0**-24 * v.abs().max().item()).all()
    k[:, 0, 0] = -math.inf
    cache.fill(0, k, v)
    assert (nc.paged_attention(ctx, nc.PagedKV(cache.k, cache.v), b, q) == 0).all()
    k[:, 0, 0] = 0
    k[9, 0, 3] = math.nan
    cache.fill(0, k, v)
    assert torch.isnan(nc.paged_attention(ctx, nc.PagedKV(cache.k, cache.v), b, q)).all()


@pytest.mark.parametrize("qt,ct", TYPES, ids=ids)
@pytest.mark.parametrize("what", ["inf", "nan", "largest", "lowest"])
def test_later_rows_reach_no_earlier_one(ctx, qt, ct, what):
    """What the later of a sequence's new rows hold, and the places behind its end, is not seen before them."""
    lens, rows = [300, 37, 257], [5, 3, 2]
    cache = _sequences(lens, 16, 2, 128, ct, 85)
    q = _randn((10, 8, 128), 86, 1.5, qt)
    info = torch.finfo(ct)
    x = {"inf": math.inf, "nan": math.nan, "largest": info.max, "lowest": info.min}[what]
    for s, n in enumerate(lens):
        pg, at = cache.place(s, n - 1)
        cache.k[pg, at], cache.v[pg, at] = x, x
    out = nc.paged_attention(ctx, nc.PagedKV(cache.k, cache.v), nc.PagedBatch(cache.table, ints(lens), ints(starts(rows))), q)
    a = starts(rows)
    for s, (n, m) in enumerate(zip(rows, lens)):
        k, v = cache.read(s, m - 1)
        r = slice(int(a[s]), int(a[s + 1]) - 1)
        want, tol = attend(q[r], k, v, 128**-0.5)
        close(out[r], want, weights_rounded(tol, v, qt), (what, s))


@pytest.mark.parametrize("ct", [F32, F16], ids=ids)
def test_bad_pages_and_lengths_answer_nan(ctx, ct):
    lens = [40, 300, 64]
    cache = _sequences(lens, 16, 2, 64, ct, 91)
    for bad in (-1, cache.k.shape[0], 2**31 - 1, -2**31):
        table = cache.table.clone()
        table[1, 3] = bad
        b = nc.PagedBatch(table, ints(lens), ints([0, 2, 4, 6]))
        q = _randn((6, 4, 64), 92)
        out = nc.paged_attention(ctx, nc.PagedKV(cache.k, cache.v), b, q)
        assert torch.isnan(out[2:4]).all() and torch.isfinite(out[:2]).all() and torch.isfinite(out[4:]).all(), bad
    # a length past the table, past max_len: only the rows that would see past it
    width = cache.table.shape[1] * 16
    table = cache.table[1:2].clone()
    table[table < 0] = 0
    # the places behind the sequence's 300 positions hold NaN, which these longer rows would rightly answer
    cache.k.nan_to_num_(0.0)
    cache.v.nan_to_num_(0.0)
    b = nc.PagedBatch(table, ints([width + 1]), ints([0, 2]))
    out = nc.paged_attention(ctx, nc.PagedKV(cache.k, cache.v), b, q[:2])
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1]).all()
    b = nc.PagedBatch(cache.table, ints(lens), ints([0, 1, 2, 3]), max_len=299)
    out = nc.paged_attention(ctx, nc.PagedKV(cache.k, cache.v), b, q[:3])
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1]).all() and torch.isfinite(out[2]).all()


@pytest.mark.parametrize("seqs", [1, 40])
@pytest.mark.parametrize("ct", [F16, F32], ids=ids)
def test_bad_pages_and_lengths_of_joined_rows(ctx, ct, seqs):
    lens = [2500] + [2450 - 60 * s for s in range(1, seqs)]
    cache = _sequences(lens, 16, 2, 64, ct, 95)
    q = _randn((3 * seqs, 4, 64), 96)
    pool, at = nc.PagedKV(cache.k, cache.v), ints([3 * s for s in range(seqs + 1)])
    good = nc.paged_attention(ctx, pool, nc.PagedBatch(cache.table, ints(lens), at), q)
    assert torch.isfinite(good).all()
    short = nc.paged_attention(ctx, pool, nc.PagedBatch(cache.table, ints(lens), at, max_len=2498), q)
    assert torch.equal(short[:1], good[:1]) and torch.isnan(short[1:3]).all() and torch.equal(short[3:], good[3:])
    table = cache.table.clone()
    table[0, 2496 // 16] = cache.k.shape[0]  # the page of positions 2496 on: rows at 2497, 2498 and 2499 see it
    table[0, 2500 // 16 + 1:] = -1           # pages that none sees
    bad = nc.paged_attention(ctx, pool, nc.PagedBatch(table, ints(lens), at), q)
    assert torch.isnan(bad[:3]).all() and torch.equal(bad[3:], good[3:])


def test_row_starts_of_any_value_stay_inside(ctx):
    cache = _sequences([40, 50, 60], 16, 2, 64, F32, 101)
    q = _randn((8, 4, 64), 102)
    guard = torch.full((24, 4, 64), 3.0, device="cuda")
    for start in ([0, 100, 50, 8], [-7, 2, -3, 2**31 - 1], [5, 3, 1, 0], [8, 8, 8, 8], [-2**31, -1, 4, 2**31 - 1]):
        b = nc.PagedBatch(cache.table, ints([40, 50, 60]), ints(start))
        nc.paged_attention(ctx, nc.PagedKV(cache.k, cache.v), b, q, out=guard[8:16])
        nc.paged_kv_append(ctx, nc.PagedKV(cache.k, cache.v), b, q[:, :2].contiguous(), q[:, :2].contiguous(), q=q, q_out=guard[8:16])
        assert (guard[:8] == 3).all() and (guard[16:] == 3).all(), start


@pytest.mark.parametrize("qt,ct", [(F32, F32), (F32, F16), (BF16, BF16)], ids=ids)
def test_a_rows_result_depends_on_no_other_row(ctx, qt, ct):
    """Alone, in a verify step, in another batch, under another table width: the same bits."""
    cache = _sequences([700, 90, 1100], 16, 2, 128, ct, 111, width=60)
    q = _randn((6, 8, 128), 112, 1.0, qt)
    kv = nc.PagedKV(cache.k, cache.v)
    step = nc.paged_attention(ctx, kv, nc.PagedBatch(cache.table, ints([700, 90, 1100]), ints([0, 5, 5, 6])), q)
    for i in range(5):
        alone = nc.paged_attention(ctx, kv, nc.PagedBatch(cache.table[:1], ints([696 + i]), max_len=700), q[i:i + 1])
        assert torch.equal(alone[0], step[i]), i
    last = nc.paged_attention(ctx, kv, nc.PagedBatch(cache.table[2:], ints([1100])), q[5:])
    assert torch.equal(last[0], step[5])
    again = nc.paged_attention(ctx, kv, nc.PagedBatch(cache.table, ints([700, 90, 1100]), ints([0, 5, 5, 6])), q)
    assert torch.equal(again, step)


@pytest.mark.parametrize("qt,ct,heads,kv,hd,seqs,most,rows", [
    (F32, F32, 32, 8, 128, 12, 1400, 1), (F16, F16, 8, 2, 64, 40, 2600, 1), (F32, BF16, 4, 4, 128, 24, 2400, 1),
    (F32, F32, 8, 1, 128, 20, 1400, 5), (BF16, BF16, 16, 2, 64, 30, 2500, 3), (F32, F16, 12, 1, 128, 8, 9000, 4), (F32, F32, 2, 1, 128, 300, 1200, 1)], ids=ids)
def test_long_ragged_batches(ctx, qt, ct, heads, kv, hd, seqs, most, rows):
    """More chunks than workgroups: each takes a part of all of them, which begins and ends within sequences.  The
    answers are those of each sequence by itself."""
    lens = [most] + [max(rows, most * (s * 7 % 23) // (23 if s % 3 else 230)) for s in range(1, seqs)]
    cache = _sequences(lens, 16, kv, hd, ct, 121)
    q, _, out = _check(ctx, cache, lens, [rows] * seqs, heads, kv, hd, qt, 122)
    for s in {0, 1, seqs // 2, seqs - 1}:
        own = nc.PagedBatch(cache.table[s:s + 1], ints([lens[s]]), ints([0, rows]))
        alone = nc.paged_attention(ctx, nc.PagedKV(cache.k, cache.v), own, q[s * rows:(s + 1) * rows])
        assert torch.equal(alone, out[s * rows:(s + 1) * rows]), s


def test_one_long_sequence_among_many(ctx):
    lens = [1 + s * 13 % 60 for s in range(150)] + [17000] + [1 + s * 7 % 40 for s in range(59)]
    cache = _sequences(lens, 16, 4, 64, F16, 125)
    _check(ctx, cache, lens, [1] * len(lens), 8, 4, 64, F16, 126, row_start=False)


@pytest.mark.parametrize("ct", [F16, F32], ids=ids)
def test_offsets_past_32_bits(ctx, ct):
    """Pools of more than 2^31 elements, the sequence's pages at their end."""
    kv, hd, page = 2, 128, 64
    pages = (2**31 + 2**24) // (kv * hd * page)
    k = torch.empty((pages, page, kv, hd), dtype=ct, device="cuda")
    v = torch.empty_like(k)
    ids_ = [pages - 1, 0, pages - 3, 1, pages - 2]
    keys, values = _randn((300, kv, hd), 121, 1.0, ct), _randn((300, kv, hd), 122, 1.0, ct)
    batch = nc.PagedBatch(ints([ids_]), ints([300]), ints([0, 300]))
    nc.paged_kv_append(ctx, nc.PagedKV(k, v), batch, keys, values)
    at = torch.arange(300)
    pg = torch.tensor(ids_)[at // page].cuda()
    assert torch.equal(k[pg, (at % page).cuda()], keys) and torch.equal(v[pg, (at % page).cuda()], values)
    q = _randn((2, 4, hd), 123)
    out = nc.paged_attention(ctx, nc.PagedKV(k, v), nc.PagedBatch(ints([ids_]), ints([300]), ints([0, 2])), q)
    want, tol = attend(q, keys, values, hd**-0.5)
    close(out, want, tol)


@pytest.mark.parametrize("seqs", [70, 300])
def test_many_sequences(ctx, seqs):
    rng = np.random.default_rng(seqs)
    lens = rng.integers(1, 90, seqs).tolist()
    rows = [int(min(n, r)) for n, r in zip(lens, rng.integers(0, 4, seqs))]
    cache = _sequences(lens, 16, 1, 64, F32, 131)
    _check(ctx, cache, lens, rows, 2, 1, 64, F32, 132)


# ---------------------------------------------------------------- append
def _turned(x, pos, table):
    """Pairs (2j, 2j + 1) turned by their position's angle, in 64 bits; x [n][heads][hd]."""
    half = table.shape[1]
    out = x.detach().cpu().double().clone()
    a, b = out[..., 0:2 * half:2].clone(), out[..., 1:2 * half:2].clone()
    sin, cos = (torch.from_numpy(table[pos, :, j].astype(np.float64))[:, None] for j in (0, 1))
    out[..., 0:2 * half:2], out[..., 1:2 * half:2] = a * cos - b * sin, a * sin + b * cos
    return out


def _rotation_room(x):
    # two products and a sum, each rounded: 3 half steps of |a| + |b| (twice the largest value)
    return 3 * 2.0**-24 * 2 * x.detach().abs().max().cpu().double()


@pytest.mark.parametrize("ct", [F32, F16, BF16], ids=ids)
@pytest.mark.parametrize("qt", [F32, F16, BF16], ids=ids)
@pytest.mark.parametrize("heads,kv,hd,page,dim", [(8, 2, 128, 16, 128), (4, 4, 64, 5, 64), (6, 2, 128, 24, 74)])
def test_append(ctx, qt, ct, heads, kv, hd, page, dim):
    """Fresh prompts, verify rows, single rows, none: cache, rotated rows, and everything else untouched."""
    lens, rows = [37, 260, 1, 90, 64], [37, 5, 1, 0, 64]
    cache = Pages(lens, page, kv, hd, ct, 141)
    angles = nc.rope_table(300, dim, 10000.0)
    t = sum(rows)
    fused = _randn((t, (heads + 2 * kv) * hd), 142, 1.0, qt)
    q, k, v = (fused[:, a * hd:b * hd].view(t, -1, hd) for a, b in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv)))
    keep = fused.clone()
    batch = nc.PagedBatch(cache.table, ints(lens), ints(starts(rows)))
    q_out, k_out = nc.paged_kv_append(ctx, nc.PagedKV(cache.k, cache.v), batch, k, v, torch.from_numpy(angles).cuda(), q=q, want_k=True)
    assert torch.equal(fused, keep)
    at = starts(rows)
    written = torch.zeros(cache.k.shape[:2], dtype=torch.bool)
    for s, (n, m) in enumerate(zip(rows, lens)):
        pos, rows_ = np.arange(m - n, m), slice(int(at[s]), int(at[s + 1]))
        for got, x in ((q_out, q), (k_out, k)):
            close(got[rows_], _turned(x[rows_], pos, angles), _rotation_room(x), s)
        got_k, got_v = (c[m - n:] for c in cache.read(s, m))
        if n:
            close(got_k, _turned(k[rows_], pos, angles), _rotation_room(k), s)
            assert torch.equal(got_v, v[rows_].to(ct))
        for p in pos:
            written[cache.place(s, int(p))] = True
    assert torch.isnan(cache.k[~written.cuda()]).all() and torch.isnan(cache.v[~written.cuda()]).all()


def test_append_rotates_as_the_sessions_do(ctx):
    """Bit for bit: x0 cos - x1 sin and x0 sin + x1 cos with every operation rounded to f32."""
    x = _randn((50, 2, 64), 151)
    angles = nc.rope_table(50, 64)
    cache = Pages([50], 16, 2, 64, F32, 152)
    batch = nc.PagedBatch(cache.table, ints([50]), ints([0, 50]))
    nc.paged_kv_append(ctx, nc.PagedKV(cache.k, cache.v), batch, x, x, torch.from_numpy(angles).cuda())
    a = x.cpu().numpy()
    sn, cs = angles[:, None, :, 0], angles[:, None, :, 1]
    want = np.empty_like(a)
    want[..., 0::2] = a[..., 0::2] * cs - a[..., 1::2] * sn
    want[..., 1::2] = a[..., 0::2] * sn + a[..., 1::2] * cs
    got, values = cache.read(0, 50)
    assert np.array_equal(got.cpu().numpy().view(np.uint32), want.view(np.uint32))
    assert torch.equal(values, x)


def test_append_in_place_and_without_rotation(ctx):
    cache = Pages([20], 16, 2, 64, F16, 161)
    kv, batch = nc.PagedKV(cache.k, cache.v), nc.PagedBatch(cache.table, ints([20]), ints([0, 20]))
    q, k, v = _randn((20, 4, 64), 162), _randn((20, 2, 64), 163), _randn((20, 2, 64), 164)
    angles = torch.from_numpy(nc.rope_table(20, 64)).cuda()
    q_ref, k_ref = nc.paged_kv_append(ctx, kv, batch, k, v, angles, q=q, want_k=True)
    q2, k2 = q.clone(), k.clone()
    q_out, k_out = nc.paged_kv_append(ctx, kv, batch, k2, v, angles, q=q2, q_out=q2, k_out=k2)
    assert q_out is q2 and k_out is k2 and torch.equal(q2, q_ref) and torch.equal(k2, k_ref)
    q_out, k_out = nc.paged_kv_append(ctx, kv, batch, k, v, None, q=q, want_k=True)
    assert torch.equal(q_out, q) and torch.equal(k_out, k) and torch.equal(cache.read(0, 20)[0], k.half())
    assert nc.paged_kv_append(ctx, kv, batch, k, v) == (None, None)


def test_append_of_rows_that_have_no_place(ctx):
    """Padding rows, rows past the table, past the angles, of a bad page: nothing is written, the rest is."""
    cache = Pages([40, 40, 40, 40], 16, 2, 64, F32, 171, width=0)
    table = cache.table.clone()
    table[3, 2] = cache.k.shape[0]
    angles = torch.from_numpy(nc.rope_table(47, 64)).cuda()
    # a padded sequence; one whose rows end past the table (48 positions) and past the angles (47); a bad page
    lens, rows = [0, 1, 50, 34], [2, 2, 5, 4]
    batch = nc.PagedBatch(table, ints(lens), ints(starts(rows)))
    k, v = _randn((13, 2, 64), 172), _randn((13, 2, 64), 173)
    q = _randn((13, 2, 64), 174)
    q_out, k_out = nc.paged_kv_append(ctx, nc.PagedKV(cache.k, cache.v), batch, k, v, angles, q=q, want_k=True)
    assert torch.equal(q_out[:3], q[:3]) and torch.equal(k_out[:3], k[:3])
    assert torch.isfinite(q_out[4:6]).all() and torch.isnan(q_out[6:9]).all() and torch.isnan(k_out[6:9]).all()
    assert torch.isfinite(q_out[9:]).all()
    want = {(1, 0): 3, (2, 45): 4, (2, 46): 5, (3, 30): 9, (3, 31): 10}
    written = torch.zeros(cache.k.shape[:2], dtype=torch.bool)
    for (s, p), row in want.items():
        written[cache.place(s, p)] = True
        assert torch.equal(cache.v[cache.place(s, p)], v[row])
    assert torch.isnan(cache.v[~written.cuda()]).all() and torch.isnan(cache.k[~written.cuda()]).all()


# ---------------------------------------------------------------- together
def test_serving_cycle(ctx):
    """Prompts, decode steps, verify steps of which a part is rolled back, a sequence that ends and one that
    takes its pages: after every step each new row's attention is that of the whole kept sequence."""
    heads, kv, hd, page, ct = 8, 2, 128, 16, F16
    angles_h = nc.rope_table(400, hd)
    angles = torch.from_numpy(angles_h).cuda()
    cache = Pages([400, 400, 400], page, kv, hd, ct, 181)
    pool = nc.PagedKV(cache.k, cache.v)
    kept = [[], [], []]  # per sequence: (rotated key, value) in the cache's type, 64-bit copies
    lens = [0, 0, 0]
    plan = [([60, 17, 130], [60, 17, 130]), ([1, 1, 1], [1, 1, 1]), ([5, 3, 4], [2, 3, 1]), ([1, 0, 5], [1, 0, 5]),
            ([4, 9, 1], [4, 1, 1]), ([1, 1, 1], [1, 1, 1])]
    for step, (rows, keep) in enumerate(plan):
        t = sum(rows)
        q, k, v = _randn((t, heads, hd), 200 + step), _randn((t, kv, hd), 300 + step), _randn((t, kv, hd), 400 + step)
        total = [n + r for n, r in zip(lens, rows)]
        batch = nc.PagedBatch(cache.table, ints(total), ints(starts(rows)))
        q_rot, k_rot = nc.paged_kv_append(ctx, pool, batch, k, v, angles, q=q, want_k=True)
        out = nc.paged_attention(ctx, pool, batch, q_rot)
        if step == 0:
            packed = nc.packed_attention(ctx, q_rot, k_rot, v, ints(starts(rows)))
        at = starts(rows)
        for s in range(3):
            rows_ = slice(int(at[s]), int(at[s + 1]))
            keys = torch.cat([x[0] for x in kept[s]] + [k_rot[rows_].to(ct).cpu()])
            values = torch.cat([x[1] for x in kept[s]] + [v[rows_].to(ct).cpu()])
            want, tol = attend(q_rot[rows_], keys, values, hd**-0.5)
            close(out[rows_], want, tol, (step, s))
            if step == 0:
                want, tol = attend(q_rot[rows_], k_rot[rows_], v[rows_], hd**-0.5)
                close(packed[rows_], want, tol, ("packed", s))
            kept[s].append((keys[sum(len(x[0]) for x in kept[s]):][:keep[s]], values[sum(len(x[0]) for x in kept[s]):][:keep[s]]))
            lens[s] += keep[s]
        if step == 3:  # sequence 1 ends; the next one starts in its pages
            kept[1], lens[1] = [], 0


def test_captured_step_follows_its_inputs(ctx):
    """A decode step captured into a graph, replayed over changing lengths, rows and pages, between eager calls."""
    heads, kv, hd, seqs = 8, 2, 64, 3
    cache = _sequences([300, 520, 40], 16, kv, hd, F16, 211, width=4)
    pool = nc.PagedKV(cache.k, cache.v)
    lens = ints([300, 520, 40])
    batch = nc.PagedBatch(cache.table, lens)
    angles = torch.from_numpy(nc.rope_table(600, hd)).cuda()
    q, k, v = _randn((seqs, heads, hd), 212), _randn((seqs, kv, hd), 213), _randn((seqs, kv, hd), 214)

    def step():
        q_rot, _ = nc.paged_kv_append(ctx, pool, batch, k, v, angles, q=q)
        return nc.paged_attention(ctx, pool, batch, q_rot)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs of the same step, each with scratch of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for i in range(4):
        q.copy_(_randn((seqs, heads, hd), 220 + i))
        k.copy_(_randn((seqs, kv, hd), 230 + i))
        lens.copy_(ints([300 - 90 * i, 520 - 100 * i, 40 - 13 * i]))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        eager = step()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, eager), i


@pytest.mark.parametrize("seqs", [2, 40])
def test_captured_joins_have_scratch_of_their_own(ctx, seqs):
    """Attention that is split and joined, in two graphs, replayed over lengths that change the chunks in use."""
    heads, kv, hd, most = 8, 2, 64, 2600
    lens_ = [most] + [1 + most * (s * 11 % 17) // 40 for s in range(1, seqs)]
    cache = _sequences(lens_, 16, kv, hd, F16, 215)
    pool, lens, q = nc.PagedKV(cache.k, cache.v), ints(lens_), _randn((seqs, heads, hd), 216)
    batch = nc.PagedBatch(cache.table, lens)
    assert nc.lib().nc_paged_attention_work_bytes(pool.ref, batch.ref, seqs, heads) > 0
    qs = [q, _randn((seqs, heads, hd), 217)]
    nc.paged_attention(ctx, pool, batch, q)
    torch.cuda.synchronize()
    graphs = []
    for x in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = nc.paged_attention(ctx, pool, batch, x)
        graphs.append((graph, out))
    for i in range(4):
        lens.copy_(ints([max(1, n - 700 * i) for n in lens_]))
        q.copy_(_randn((seqs, heads, hd), 218 + i))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        eager = [nc.paged_attention(ctx, pool, batch, x) for x in qs]
        torch.cuda.synchronize()
        for (_, out), want in zip(graphs, eager):
            assert torch.equal(out, want), i


def test_two_streams_at_once(ctx):
    caches = [_sequences([900, 700], 16, 2, 128, F16, 241 + i) for i in range(2)]
    qs = [_randn((2, 8, 128), 251 + i) for i in range(2)]
    batches = [nc.PagedBatch(c.table, ints([900, 700])) for c in caches]
    want = [nc.paged_attention(ctx, nc.PagedKV(c.k, c.v), b, q) for c, b, q in zip(caches, batches, qs)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(nc.paged_attention(ctx, nc.PagedKV(caches[i].k, caches[i].v), batches[i], qs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_nothing_to_do(ctx):
    cache = _sequences([10], 16, 2, 64, F32, 261)
    pool = nc.PagedKV(cache.k, cache.v)
    none = torch.empty((0, 4, 64), device="cuda")
    b = nc.PagedBatch(cache.table, ints([10]), ints([0, 0]))
    assert nc.paged_attention(ctx, pool, b, none).shape == (0, 4, 64)
    nc.paged_kv_append(ctx, pool, b, none[:, :2], none[:, :2])
    empty = nc.PagedBatch(cache.table[:0], ints([]), ints([0]))
    out = torch.full((2, 4, 64), 5.0, device="cuda")
    nc.paged_attention(ctx, pool, empty, _randn((2, 4, 64), 262), out=out)
    assert (out == 5).all()


@pytest.mark.parametrize("what", ["type", "heads", "head_dim", "row_shape", "other_rows", "strided_heads", "unaligned", "rows_without_starts",
                                  "pools_differ", "pool_inner_stride", "pool_type", "table_type", "cpu_rows", "rope_type", "rope_wide", "out_is_q", "no_dimensions",
                                  "out_shape"])
def test_refusals(ctx, what):
    cache = _sequences([20, 20], 16, 2, 64, F16, 271)
    pool, batch = nc.PagedKV(cache.k, cache.v), nc.PagedBatch(cache.table, ints([20, 20]))
    q, k = _randn((2, 4, 64), 272), _randn((2, 2, 64), 273)
    angles = torch.from_numpy(nc.rope_table(20, 64)).cuda()
    calls = {
        "type": lambda: nc.paged_attention(ctx, pool, batch, q.bfloat16()),
        "heads": lambda: nc.paged_attention(ctx, pool, batch, q[:, :3].contiguous()),
        "head_dim": lambda: nc.paged_attention(ctx, nc.PagedKV(cache.k[..., :32].contiguous(), cache.v[..., :32].contiguous()), batch, q[..., :32].contiguous()),
        "row_shape": lambda: nc.paged_attention(ctx, pool, batch, q.view(2, 256)),
        "other_rows": lambda: nc.paged_kv_append(ctx, pool, batch, k, k[:1]),
        "strided_heads": lambda: nc.paged_attention(ctx, pool, batch, _randn((2, 8, 64), 1)[:, ::2]),
        "unaligned": lambda: nc.paged_attention(ctx, pool, batch, _randn((2, 257), 1)[:, 1:].view(2, 4, 64)),
        "rows_without_starts": lambda: nc.paged_attention(ctx, pool, batch, q[:1]),
        "pools_differ": lambda: nc.PagedKV(cache.k, cache.v.transpose(1, 2).contiguous().transpose(1, 2)),
        "pool_inner_stride": lambda: nc.PagedKV(cache.k[..., ::2], cache.v[..., ::2]),
        "pool_type": lambda: nc.PagedKV(cache.k.to(torch.int16), cache.v.to(torch.int16)),
        "table_type": lambda: nc.PagedBatch(cache.table.long(), ints([20, 20])),
        "cpu_rows": lambda: nc.paged_attention(ctx, pool, batch, q.cpu()),
        "rope_type": lambda: nc.paged_kv_append(ctx, pool, batch, k, k, angles.double()),
        "rope_wide": lambda: nc.paged_kv_append(ctx, pool, batch, k, k, torch.from_numpy(nc.rope_table(20, 128)).cuda()),
        "out_is_q": lambda: nc.paged_attention(ctx, pool, batch, q, out=q),
        "no_dimensions": lambda: nc.paged_kv_append(ctx, pool, batch, k[0, 0, 0], k),
        "out_shape": lambda: nc.paged_attention(ctx, pool, batch, q, out=torch.empty((2, 4, 128), device="cuda")),
    }
    with pytest.raises(nc.NcError) as e:
        calls[what]()
    assert e.value.code == -1
