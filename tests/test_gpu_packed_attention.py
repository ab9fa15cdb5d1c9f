"""Attention over packed prompts on the GPU against plain 64-bit arithmetic: every type, ragged lengths around
the tiles' edges, heads in groups, continued prompts, rows that see nothing, strides, streams and graphs."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import nanocamelid_amd as nc  # noqa: E402

from tests.paged_util import attend, close, ints, starts, weights_rounded  # noqa: E402

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ids = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731


@pytest.fixture(scope="module")
def ctx():
    assert torch.cuda.is_available(), "GPU tests need the MI355X"
    return nc.Context(0)


def _randn(shape, seed, gain=1.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * gain).to(dtype).cuda()


def _fused(rows, heads, kv, hd, seed, dtype):
    x = _randn((rows, (heads + 2 * kv) * hd), seed, 1.3, dtype)
    return (x[:, a * hd:b * hd].view(rows, b - a, hd) for a, b in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv)))


def _check(out, q, k, v, rows, keys, scale):
    a, b = starts(rows), starts(keys)
    for s in range(len(rows)):
        r, c = slice(int(a[s]), int(a[s + 1])), slice(int(b[s]), int(b[s + 1]))
        want, tol = attend(q[r], k[c], v[c], scale)
        if keys[s]:
            tol = weights_rounded(tol, v[c], q.dtype)
        close(out[r], want, tol, ("sequence", s, rows[s], keys[s]))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=ids)
@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 128), (3, 3, 64), (8, 1, 64), (5, 1, 128), (8, 2, 128), (12, 1, 64)])
def test_ragged_prompts(ctx, dtype, heads, kv, hd):
    rows = [1, 2, 31, 32, 33, 0, 63, 64, 65, 127, 128, 129, 16, 17, 200]
    q, k, v = _fused(sum(rows), heads, kv, hd, 1, dtype)
    out = nc.packed_attention(ctx, q, k, v, ints(starts(rows)))
    _check(out, q, k, v, rows, rows, hd**-0.5)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=ids)
@pytest.mark.parametrize("n,hd", [(1, 128), (255, 64), (256, 128), (257, 128), (513, 64), (770, 128)])
@pytest.mark.parametrize("heads", [2, 4])
def test_one_prompt(ctx, dtype, n, hd, heads):
    q, k, v = _fused(n, heads, 1, hd, 2 + n, dtype)
    out = nc.packed_attention(ctx, q, k, v, ints([0, n]))
    _check(out, q, k, v, [n], [n], hd**-0.5)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=ids)
@pytest.mark.parametrize("hd,heads", [(64, 4), (128, 4), (128, 8)])
def test_continued_prompts_and_rows_that_see_nothing(ctx, dtype, hd, heads):
    """More keys than rows (a prompt that goes on), fewer (the first rows see none), none at all."""
    rows, keys = [5, 130, 40, 10, 7, 64, 0], [300, 131, 33, 0, 7, 129, 20]
    a = starts(rows)
    q = _randn((sum(rows), heads, hd), 11, 1.3, dtype)
    k, v = _randn((sum(keys), 2, hd), 12, 1.0, dtype), _randn((sum(keys), 2, hd), 13, 1.0, dtype)
    out = nc.packed_attention(ctx, q, k, v, ints(a), ints(starts(keys)))
    _check(out, q, k, v, rows, keys, hd**-0.5)
    assert (out[a[2]:a[2] + 7] == 0).all() and (out[a[3]:a[4]] == 0).all()


@pytest.mark.parametrize("heads", [4, 8])
@pytest.mark.parametrize("dtype", [F32, F16], ids=ids)
def test_neighbours_do_not_leak(ctx, dtype, heads):
    """What other sequences and the rows between them hold, NaN and infinities too, reaches no row."""
    q, k, v = (x.contiguous() for x in _fused(200, heads, 2, 128, 21, dtype))
    alone = nc.packed_attention(ctx, q[70:130].contiguous(), k[70:130].contiguous(), v[70:130].contiguous(), ints([0, 60]))
    for x in (k, v):
        x[:70], x[130:] = math.nan, math.inf
    out = torch.full_like(q, 3.0)
    nc.packed_attention(ctx, q, k, v, ints([70, 130]), out=out)
    assert torch.equal(out[70:130], alone) and (out[:70] == 3).all() and (out[130:] == 3).all()


@pytest.mark.parametrize("dtype,heads,hd", [(F32, 2, 128), (F32, 4, 128), (F32, 4, 64), (F16, 2, 64), (BF16, 4, 128)], ids=ids)
def test_causal_mask_hides_infinities(ctx, dtype, heads, hd):
    """A row sees nothing of the later rows, whatever they hold."""
    q, k, v = (x.contiguous() for x in _fused(150, heads, 1, hd, 31, dtype))
    want = nc.packed_attention(ctx, q, k, v, ints([0, 150]))
    k2, v2 = k.clone(), v.clone()
    k2[100:], v2[100:] = math.inf, math.nan
    got = nc.packed_attention(ctx, q, k2, v2, ints([0, 150]))
    # f32: the 32 keys from 96 on, some of them not finite, take another product of the same accuracy, so the rows
    # that see some of the finite ones agree within the bound of f32 arithmetic, not in their bits
    same = 96 if dtype == F32 else 100
    assert torch.equal(got[:same], want[:same]) and torch.isnan(got[100:]).all()
    _check(got[:100], q[:100], k[:100], v[:100], [100], [100], hd**-0.5)


@pytest.mark.parametrize("heads,hd", [(2, 64), (4, 128)])
def test_extreme_scores(ctx, heads, hd):
    q, k, v = (x.contiguous() for x in _fused(140, heads, 1, hd, 41, F32))
    k[3] *= 50
    k[90] *= 70
    out = nc.packed_attention(ctx, q, k, v, ints([0, 140]))
    _check(out, q, k, v, [140], [140], hd**-0.5)
    q[:] = 1.0
    k[:] = -math.inf
    assert (nc.packed_attention(ctx, q, k, v, ints([0, 140])) == 0).all()


@pytest.mark.parametrize("heads,hd", [(2, 64), (4, 128)])
@pytest.mark.parametrize("size", [1e-30, 1e-6, 3e4, 1e15])
def test_f32_values_of_any_size(ctx, heads, hd, size):
    """Sizes far from one, and sizes that grow and shrink along the sequence: relative accuracy holds."""
    q, k, v = (x.contiguous() for x in _fused(200, heads, 1, hd, 45, F32))
    k, v, q = k * size, v * size, q / size
    _check(nc.packed_attention(ctx, q, k, v, ints([0, 200])), q, k, v, [200], [200], hd**-0.5)
    # values by row: tiny ones first, large ones later, which rows before them must not feel
    grow = (10.0 ** torch.linspace(-4, 4, 200)).cuda()[:, None, None]
    v = v * grow
    out = nc.packed_attention(ctx, q, k, v, ints([0, 200]))
    rows = [40, 80, 120, 160, 200]
    for n in rows:
        want, tol = attend(q[n - 1:n], k[:n], v[:n], hd**-0.5)
        close(out[n - 1:n], want, tol, n)


@pytest.mark.parametrize("dtype,heads,hd", [(F32, 2, 128), (F32, 4, 128), (F32, 4, 64), (F16, 2, 64), (BF16, 4, 128)], ids=ids)
def test_masked_values_of_the_largest_size(ctx, dtype, heads, hd):
    """Rows before a key of the type's largest or lowest values answer as if it were not there."""
    q, k, v = (x.contiguous() for x in _fused(150, heads, 1, hd, 47, dtype))
    for low in (True, False):
        k2, v2 = k.clone(), v.clone()
        info = torch.finfo(dtype)
        k2[100:], v2[100:] = (info.min, info.min) if low else (info.max, info.max)
        got = nc.packed_attention(ctx, q, k2, v2, ints([0, 150]))
        _check(got[:100], q[:100], k[:100], v[:100], [100], [100], hd**-0.5)


@pytest.mark.parametrize("heads,hd", [(2, 64), (2, 128), (4, 128)])
def test_f32_rows_of_unlike_size(ctx, heads, hd):
    """Keys and values whose rows differ in size by more than 16-bit parts hold together, in and across tiles."""
    q, k, v = (x.contiguous() for x in _fused(200, heads, 1, hd, 49, F32))
    wide = (10.0 ** torch.linspace(-18, 18, 200)).cuda()[:, None, None]
    for keys, values in ((k, v * wide), (k, v * wide.flip(0)), (k * 1e-9 * wide.clamp(1e-9, 1e9), v)):
        out = nc.packed_attention(ctx, q, keys, values, ints([0, 200]))
        for n in (1, 30, 33, 64, 95, 130, 200):
            want, tol = attend(q[n - 1:n], keys[:n], values[:n], hd**-0.5)
            close(out[n - 1:n], want, tol, n)
    # one in a tile
    for at in (5, 70, 199):
        keys, values = k.clone(), v.clone()
        keys[at] *= 3e6
        values[at] *= 1e12
        _check(nc.packed_attention(ctx, q, keys, values, ints([0, 200])), q, keys, values, [200], [200], hd**-0.5)
    # both tiny: scores of zero under masks
    tiny = nc.packed_attention(ctx, q * 1e-25, k * 1e-25, v, ints([0, 200]))
    _check(tiny, q * 1e-25, k * 1e-25, v, [200], [200], hd**-0.5)


@pytest.mark.parametrize("heads,hd", [(2, 64), (4, 128)])
@pytest.mark.parametrize("e", [-122, 122])
def test_f32_ordinary_scores_of_sizes_at_the_ends(ctx, heads, hd, e):
    q, k, v = (x.contiguous() for x in _fused(70, heads, 1, hd, 50, F32))
    q, k = torch.ldexp(q, torch.tensor(e, device="cuda")), torch.ldexp(k, torch.tensor(-e, device="cuda"))
    assert torch.isfinite(q).all() and torch.isfinite(k).all()
    _check(nc.packed_attention(ctx, q, k, v, ints([0, 70])), q, k, v, [70], [70], hd**-0.5)


def test_scale(ctx):
    q, k, v = _fused(90, 2, 2, 64, 51, F32)
    for scale in (1.0, 0.0, -0.2):
        _check(nc.packed_attention(ctx, q, k, v, ints([0, 90]), scale=scale), q, k, v, [90], [90], scale)


def test_starts_of_any_value_stay_inside(ctx):
    q, k, v = (x.contiguous() for x in _fused(16, 2, 2, 64, 61, F32))
    guard = torch.full((48, 2, 64), 3.0, device="cuda")
    for start in ([0, 100, 50, 16], [-7, 2, -3, 2**31 - 1], [9, 5, 1, 0], [16] * 4, [-2**31, -1, 8, 2**31 - 1]):
        nc.packed_attention(ctx, q, k, v, ints(start), out=guard[16:32])
        nc.packed_attention(ctx, q, k, v, ints([0, 5, 9, 16]), ints(start), out=guard[16:32])
        assert (guard[:16] == 3).all() and (guard[32:] == 3).all(), start


@pytest.mark.parametrize("seqs", [100, 700])
def test_many_sequences(ctx, seqs):
    rows = np.random.default_rng(seqs).integers(0, 12, seqs).tolist()
    q, k, v = _fused(sum(rows), 2, 1, 64, 71, F32)
    out = nc.packed_attention(ctx, q, k, v, ints(starts(rows)))
    _check(out, q, k, v, rows, rows, 0.125)


@pytest.mark.parametrize("dtype", [F32, F16], ids=ids)
def test_rows_far_apart(ctx, dtype):
    """Row strides that take the last rows past 2^31 elements."""
    n, stride = 300, 1 << 23
    room = torch.empty((n - 1) * stride + 4096, dtype=dtype, device="cuda")
    q, k, v = (torch.as_strided(room, (n, 2, 128), (stride, 128, 1), at) for at in (0, 512, 1024))
    for i, x in enumerate((q, k, v)):
        x.copy_(_randn((n, 2, 128), 81 + i, 1.0, dtype))
    out = nc.packed_attention(ctx, q, k, v, ints([0, n]))
    _check(out, q.contiguous(), k.contiguous(), v.contiguous(), [n], [n], 128**-0.5)


def test_stream_and_graph(ctx):
    q, k, v = (x.contiguous() for x in _fused(300, 4, 2, 128, 91, BF16))
    start = ints([0, 120, 300])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = nc.packed_attention(ctx, q, k, v, start)
    torch.cuda.synchronize()
    assert torch.equal(first, nc.packed_attention(ctx, q, k, v, start))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = nc.packed_attention(ctx, q, k, v, start)
    for i in range(3):
        q.copy_(_randn(q.shape, 95 + i, 1.0, BF16))
        start.copy_(ints([0, 100 + 60 * i, 300 - 10 * i]))
        graph.replay()
        torch.cuda.synchronize()
        eager = nc.packed_attention(ctx, q, k, v, start)
        torch.cuda.synchronize()
        assert torch.equal(out[:300 - 10 * i], eager[:300 - 10 * i]), i


def test_nothing_to_do(ctx):
    none = torch.empty((0, 2, 64), device="cuda")
    assert nc.packed_attention(ctx, none, none, none, ints([0, 0])).shape == (0, 2, 64)
    q = _randn((3, 2, 64), 101)
    assert (nc.packed_attention(ctx, q, none, none, ints([0, 3]), ints([0, 0])) == 0).all()
    out = torch.full_like(q, 2.0)
    nc.packed_attention(ctx, q, q, q, ints([0]), out=out)
    assert (out == 2).all()


@pytest.mark.parametrize("what", ["mixed", "int", "heads", "head_dim", "rows", "start_type", "start_shape", "strided", "unaligned", "cpu", "out", "out_is_q", "out_is_k"])
def test_refusals(ctx, what):
    q, k = _randn((8, 4, 64), 111), _randn((8, 2, 64), 112)
    s, q2 = ints([0, 8]), q.clone()
    calls = {
        "mixed": lambda: nc.packed_attention(ctx, q, k.half(), k, s),
        "int": lambda: nc.packed_attention(ctx, q.int(), k.int(), k.int(), s),
        "heads": lambda: nc.packed_attention(ctx, q[:, :3].contiguous(), k, k, s),
        "head_dim": lambda: nc.packed_attention(ctx, q[..., :48].contiguous(), k[..., :48].contiguous(), k[..., :48].contiguous(), s),
        "rows": lambda: nc.packed_attention(ctx, q, k[:7], k[:7], s),
        "start_type": lambda: nc.packed_attention(ctx, q, k, k, s.long()),
        "start_shape": lambda: nc.packed_attention(ctx, q, k, k, s, ints([0, 4, 8])),
        "strided": lambda: nc.packed_attention(ctx, q, k, q[:, ::2], s),
        "unaligned": lambda: nc.packed_attention(ctx, q, k, _randn((8, 129), 1)[:, 1:].view(8, 2, 64), s),
        "cpu": lambda: nc.packed_attention(ctx, q.cpu(), k.cpu(), k.cpu(), s.cpu()),
        "out": lambda: nc.packed_attention(ctx, q, k, k, s, out=torch.empty((8, 2, 64), device="cuda")),
        "out_is_q": lambda: nc.packed_attention(ctx, q, k, k, s, out=q),
        "out_is_k": lambda: nc.packed_attention(ctx, q, q2, q2, s, out=q2),
    }
    with pytest.raises(nc.NcError) as e:
        calls[what]()
    assert e.value.code == -1
