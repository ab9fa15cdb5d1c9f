"""The paged operators without a GPU: the page arithmetic and bounds that the kernels share with the host, the
C entries' refusals before they touch a device, the angles, and the wrappers' structs."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from nanocamelid_amd import _ffi as F
from tests.test_integration_binding import _c_structs, _layout, _size_align

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

WALK = r"""
#include <cstdio>
#include <cstdlib>
#include <initializer_list>
#include <vector>
#include "nc_paged.h"
using namespace nc;

static void want(bool ok, const char* what, long long a, long long b) {
    if (ok) return;
    std::printf("%s: %lld %lld\n", what, a, b);
    std::exit(1);
}

int main() {
    // every quotient near a multiple of the page size, from 0 to 2^31 - 1
    for (uint32_t d : {1u, 2u, 3u, 5u, 7u, 8u, 16u, 20u, 24u, 100u, 255u, 256u, 257u, 1000u, 65535u, 65537u, 1000003u, 1u << 30, (1u << 30) + 1, 2147483647u}) {
        const PageDiv p = page_div(d);
        for (uint64_t k = 0; k * d < (1ull << 31); k = k < 70000 ? k + 1 : k + k / 1000)
            for (int64_t o = -1; o <= 1; o++) {
                const int64_t n = (int64_t)(k * d) + o;
                if (n >= 0 && n < (1ll << 31)) want(page_of((uint32_t)n, p) == n / d, "quotient", n, d);
            }
        for (int64_t n = 2147483647; n > 2147483600; n--) want(page_of((uint32_t)n, p) == n / d, "quotient", n, d);
    }
    // places inside the pool for every table entry, and none for the others
    PagedPool pool;
    pool.page_stride = 1ll << 33, pool.pos_stride = 256, pool.head_stride = 64, pool.pages = 10, pool.div = page_div(24);
    const std::vector<int32_t> table = {3, 9, -1, 10, 2147483647, -2147483647 - 1, 0};
    for (int p = 0; p < 24 * (int)table.size(); p++) {
        const int64_t at = position_offset(table.data(), pool, p);
        const int32_t id = table[p / 24];
        want(at == (id >= 0 && id < 10 ? id * (1ll << 33) + p % 24 * 256 : -1), "place", p, at);
    }
    // row ranges inside the tensor for any starts
    const std::vector<int32_t> odd = {0, 5, -1, 2147483647, -2147483647 - 1, 7, 100, 3};
    for (int rows : {0, 1, 8, 2147483647})
        for (int a : odd)
            for (int b : odd) {
                const int32_t start[2] = {a, b};
                int begin, n;
                seq_rows(start, 0, rows, begin, n);
                want(begin >= 0 && n >= 0 && (int64_t)begin + n <= rows, "rows", a, b);
                if (a >= 0 && b >= a && b <= rows) want(begin == a && n == b - a, "rows as given", a, b);
            }
    int begin, n;
    seq_rows(nullptr, 4, 5, begin, n);
    want(begin == 4 && n == 1, "one row", begin, n);
    seq_rows(nullptr, 5, 5, begin, n);
    want(n == 0, "no row", begin, n);
    return 0;
}
"""


def test_places_and_rows(tmp_path):
    src, exe = tmp_path / "walk.cpp", tmp_path / "walk"
    src.write_text(WALK)
    subprocess.run(["g++", "-std=c++20", "-O2", "-Wall", "-I", os.path.join(ROOT, "nanocamelid_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout


@pytest.mark.parametrize("name,cls", [("nc_paged_kv", "PagedKVView"), ("nc_paged_batch", "PagedBatchView")])
def test_structs_match_the_header(name, cls):
    st, fields = getattr(F, cls), _c_structs()[name]
    layout, size = _layout(fields)
    assert [f[0] for f in st._fields_] == [f[0] for f in fields] and C.sizeof(st) == size
    for (fname, off, _), (cf, ct) in zip(layout, st._fields_):
        assert getattr(st, fname).offset == off and C.sizeof(ct) == _size_align(dict(fields)[fname])[0]


@pytest.mark.parametrize("dim,base,scaling", [(128, 500000.0, None), (64, 10000.0, None), (74, 10000.0, None), (64, 500000.0, (32.0, 8192.0, 1.0, 4.0))])
def test_rope_table(dim, base, scaling):
    """The angles of the reference's formula, from 64 bits: theta and the angle are rounded to f32 each, so an
    angle is off by at most 3 half steps of itself (powf is allowed one step), and sin and cos by that and their own.
    The exponent -2i / dim, of size e <= 1, is rounded first: base^-(e + d) = base^-e (1 - d ln base + ..) with d <= e 2^-24,
    so theta is off by another ln(base) half steps where dim is no power of two."""
    import nanocamelid_amd as nc
    n = 3000
    table = nc.rope_table(n, dim, base, scaling)
    theta = base ** (-np.arange(0, dim, 2, dtype=np.float64) / dim)
    if scaling:
        factor, orig, low, high = scaling
        wave = 2 * np.pi / theta
        smooth = (orig / wave - low) / (high - low)
        theta = np.where(wave < orig / high, theta, np.where(wave > orig / low, theta / factor, (1 - smooth) * theta / factor + smooth * theta))
    angle = np.arange(n)[:, None] * theta
    # the scaled thetas take a few more roundings, of a blend of terms no larger than theta
    tol = 2.0**-24 * (angle * ((16 if scaling else 5) + np.log(base)) + 2)
    assert table.shape == (n, dim // 2, 2) and table.dtype == np.float32
    assert (np.abs(table[..., 0] - np.sin(angle)) <= tol).all() and (np.abs(table[..., 1] - np.cos(angle)) <= tol).all()
    assert (table[0, :, 0] == 0).all() and (table[0, :, 1] == 1).all()


def test_rope_table_refusals():
    import nanocamelid_amd as nc
    for bad in ((-1, 64, 1e4), (4, 63, 1e4), (4, 64, 0.0), (4, 64, float("nan")), (4, 1 << 20, 1e4)):
        with pytest.raises((nc.NcError, ValueError)):
            nc.rope_table(*bad)
    assert nc.rope_table(0, 64).shape == (0, 32, 2)


# ---------------------------------------------------------------- refusals before a device is touched
KV = dict(k_pages=1 << 20, v_pages=1 << 21, pages=4, page_stride=16 * 2 * 64, pos_stride=2 * 64, head_stride=64, elem_type=F.NC_TYPE_F16,
          page_size=16, kv_heads=2, head_dim=64)
BATCH = dict(table=1 << 12, lens=1 << 13, row_start=1 << 14, table_stride=8, table_pages=8, seqs=3, max_len=0, reserved=0)
ADDRESS = 1 << 22


def _ctx():
    # stands for a context: the calls below are refused, or have nothing to do, before they use it
    return C.create_string_buffer(4096)


def _append(kv=KV, batch=BATCH, **a):
    a = {**dict(type=0, rows=5, k=ADDRESS, ks=128, v=ADDRESS, vs=128, k_out=None, q=ADDRESS, qs=256, heads=4, q_out=ADDRESS, rope=ADDRESS,
                positions=100, dim=64), **a}
    return F.lib().nc_paged_kv_append(_ctx(), C.byref(F.PagedKVView(**kv)), C.byref(F.PagedBatchView(**batch)), a["type"], a["rows"], a["k"],
                                      a["ks"], a["v"], a["vs"], a["k_out"], a["q"], a["qs"], a["heads"], a["q_out"], a["rope"], a["positions"],
                                      a["dim"], None)


def _attend(kv=KV, batch=BATCH, **a):
    a = {**dict(type=0, rows=5, q=ADDRESS, qs=256, heads=4, out=2 * ADDRESS, work=ADDRESS, bytes=1 << 40), **a}
    return F.lib().nc_paged_attention(_ctx(), C.byref(F.PagedKVView(**kv)), C.byref(F.PagedBatchView(**batch)), a["type"], a["rows"], a["q"],
                                      a["qs"], a["heads"], 1.0, a["out"], a["work"], a["bytes"], None)


def _packed(**a):
    a = {**dict(type=0, rows=5, kv_rows=5, q=ADDRESS, qs=256, k=ADDRESS, ks=128, v=ADDRESS, vs=128, heads=4, kv=2, hd=64, start=ADDRESS,
                kv_start=None, seqs=2, out=2 * ADDRESS), **a}
    return F.lib().nc_packed_attention(_ctx(), a["type"], a["rows"], a["kv_rows"], a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["heads"],
                                       a["kv"], a["hd"], a["start"], a["kv_start"], a["seqs"], 1.0, a["out"], None)


@pytest.mark.parametrize("field,value", [("k_pages", 0), ("v_pages", 0), ("k_pages", (1 << 20) + 8), ("pages", 0), ("pages", 1 << 31), ("page_size", 0),
                                         ("page_size", -16), ("kv_heads", 0), ("head_dim", 96), ("head_dim", 0), ("elem_type", F.NC_TYPE_Q8_0),
                                         ("page_stride", 0), ("pos_stride", -128), ("pos_stride", 130), ("head_stride", 32), ("page_stride", 1 << 60)])
def test_bad_caches_are_refused(field, value):
    kv = {**KV, field: value}
    for call in (_append, _attend):
        assert call(kv=kv) == F.NC_EINVAL, field
    assert F.lib().nc_paged_attention_work_bytes(C.byref(F.PagedKVView(**kv)), C.byref(F.PagedBatchView(**BATCH)), 5, 4) == F.NC_EINVAL


@pytest.mark.parametrize("field,value", [("table", 0), ("lens", 0), ("table", 2), ("row_start", 6), ("table_stride", 7), ("table_pages", -1),
                                         ("seqs", -1), ("max_len", -1), ("row_start", 0)])
def test_bad_batches_are_refused(field, value):
    batch = {**BATCH, field: value}
    for call in (_append, _attend):
        assert call(batch=batch) == F.NC_EINVAL, field


@pytest.mark.parametrize("args", [dict(type=2), dict(k=None), dict(v=None), dict(q_out=None), dict(heads=0), dict(ks=127), dict(ks=64), dict(vs=130),
                                  dict(k=ADDRESS + 4), dict(q=ADDRESS + 8), dict(qs=255), dict(k_out=ADDRESS + 4), dict(q_out=ADDRESS + 4), dict(dim=0),
                                  dict(dim=63), dict(dim=128), dict(positions=0), dict(rope=ADDRESS + 2), dict(ks=1 << 40)])
def test_bad_appends_are_refused(args):
    assert _append(**args) == F.NC_EINVAL


@pytest.mark.parametrize("args", [dict(type=F.NC_TYPE_BF16), dict(type=99), dict(q=None), dict(out=None), dict(heads=5), dict(heads=0), dict(qs=128),
                                  dict(q=ADDRESS + 4), dict(out=ADDRESS + 4), dict(out=ADDRESS), dict(qs=1 << 40)])
def test_bad_attentions_are_refused(args):
    assert _attend(**args) == F.NC_EINVAL


@pytest.mark.parametrize("args,code", [(dict(type=8), -1), (dict(hd=80), -1), (dict(heads=5), -1), (dict(kv=0), -1), (dict(heads=0), -1),
                                       (dict(rows=-1), -5), (dict(kv_rows=1 << 31), -5), (dict(seqs=-1), -5), (dict(q=None), -1), (dict(k=None), -1),
                                       (dict(out=None), -1), (dict(start=None), -1), (dict(kv_rows=4), -1), (dict(ks=64), -1), (dict(vs=130), -1),
                                       (dict(q=ADDRESS + 4), -1), (dict(out=ADDRESS + 8), -1), (dict(start=ADDRESS + 2), -1),
                                       (dict(qs=1 << 40), -1), (dict(out=ADDRESS), -1), (dict(q=3 * ADDRESS, out=ADDRESS), -1)])
def test_bad_packed_attentions_are_refused(args, code):
    assert _packed(**args) == code


def test_rows_beyond_an_index_are_refused():
    assert _append(rows=1 << 31) == F.NC_ERANGE and _attend(rows=-1) == F.NC_ERANGE
    assert _attend(rows=1 << 30) == F.NC_ERANGE
    batch = C.byref(F.PagedBatchView(**BATCH))
    assert F.lib().nc_paged_attention_work_bytes(C.byref(F.PagedKVView(**KV)), batch, 1 << 30, 4) == F.NC_ERANGE


def test_nothing_to_do_is_no_error():
    assert _append(rows=0, k=None, v=None, q=None) == 0 and _attend(rows=0, q=None, out=None) == 0 and _packed(rows=0, kv_rows=0, q=None) == 0
    empty = {**BATCH, "seqs": 0}
    assert _append(batch=empty) == 0 and _attend(batch=empty) == 0 and _packed(seqs=0) == 0


def test_null_arguments():
    lib, kv, batch = F.lib(), C.byref(F.PagedKVView(**KV)), C.byref(F.PagedBatchView(**BATCH))
    assert lib.nc_paged_attention_work_bytes(None, batch, 1, 1) == F.NC_EINVAL
    assert lib.nc_paged_attention_work_bytes(kv, None, 1, 1) == F.NC_EINVAL
    assert lib.nc_paged_attention(None, kv, batch, 0, 0, None, 0, 1, 1.0, None, None, 0, None) == F.NC_EINVAL
    assert lib.nc_packed_attention(None, 0, 0, 0, None, 0, None, 0, None, 0, 1, 1, 64, None, None, 0, 1.0, None, None) == F.NC_EINVAL
