// A paged key-value cache for several sequences: the append of new rows with the position rotation on the
// way, and the attention of those rows over the pages.
//
// The cache is the caller's: two pools of pages, [page][position in page][kv head][head_dim] by any strides
// with head_dim contiguous, and a table that names each sequence's pages in order.  Position p of sequence s
// lies in page table[s][p / page_size] at p % page_size.  Row i of a sequence's n new rows stands at position
// len - n + i and sees the positions up to its own.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "nc_internal.h"
#include "nc_paged.h"

namespace nc {

// ---------------------------------------------------------------- append
struct AppendParams {
    PagedSeqs seqs;
    PagedPool pool;
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;  // elements between rows
    void *q_out, *k_out, *k_pages, *v_pages;
    const float* rope;  // [positions][half][2] = (sin, cos)
    int32_t rope_positions, rope_half, heads, kv_heads;
};

// Pairs (2j, 2j + 1) with j < rope_half turn by their position's angle, each product and sum rounded by
// itself as in the sessions' rotation; the cache takes the result rounded once to its type.
//
// Bound by bytes: every value is read and written once.  A thread moves eight values of one row (16 or 32
// bytes each way); their loads go out before the row's place is known, which takes three dependent loads
// (its sequence, the length, the page).  A workgroup takes 256 of a row's units, so a decode batch still
// spreads over many CUs.
template <typename A, typename C, int HD>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendParams a) {
    constexpr int U = HD / 8;  // units of a head
    const int unit = blockIdx.y * 256 + threadIdx.x;
    const int nq = a.q ? a.heads * U : 0, nk = a.kv_heads * U;
    const bool live = unit < nq + 2 * nk;
    const bool is_q = unit < nq, is_k = !is_q && unit < nq + nk;
    const int u = is_q ? unit : is_k ? unit - nq : unit - nq - nk;
    const int d = (u % U) * 8;
    for (int64_t t = blockIdx.x; t < a.seqs.rows; t += gridDim.x) {
        float x[8];
        if (live)
            load8(is_q   ? (const A*)a.q + t * a.q_stride + u * 8
                  : is_k ? (const A*)a.k + t * a.k_stride + u * 8
                         : (const A*)a.v + t * a.v_stride + u * 8,
                  x);
        const int s = seq_of_row(a.seqs.row_start, a.seqs.seqs, (int)t);
        if (s < 0 || !live) continue;
        int begin, n;
        seq_rows(a.seqs.row_start, s, a.seqs.rows, begin, n);
        const int i = (int)t - begin;
        if (i < 0 || i >= n) continue;
        const int64_t p64 = (int64_t)a.seqs.lens[s] - n + i;
        // a row of no position (a padded batch's) stays as it is given; one past the angles has no rotation
        const bool placed = p64 >= 0 && p64 < a.seqs.cap;
        const int p = (int)p64;
        const int64_t at = placed ? position_offset(a.seqs.table + s * a.seqs.table_stride, a.pool, p) : -1;
        const bool turned = !a.rope || p64 < a.rope_positions;
        if ((is_q || is_k) && a.rope && p64 >= 0) {
            const float* angle = a.rope + ((int64_t)(turned ? p : 0) * a.rope_half + d / 2) * 2;
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (d / 2 + j < a.rope_half) {
                    const float sn = angle[2 * j], cs = angle[2 * j + 1];
                    const float x0 = x[2 * j], x1 = x[2 * j + 1];
                    x[2 * j] = turned ? x0 * cs - x1 * sn : __builtin_nanf("");
                    x[2 * j + 1] = turned ? x0 * sn + x1 * cs : __builtin_nanf("");
                }
        }
        if (is_q) {
            store8((A*)a.q_out + (t * a.heads * HD + u * 8), x);
            continue;
        }
        if (is_k && a.k_out) store8((A*)a.k_out + (t * a.kv_heads * HD + u * 8), x);
        if (at >= 0 && turned)
            store8((C*)(is_k ? a.k_pages : a.v_pages) + at + (int64_t)(u / U) * a.pool.head_stride + d, x);
    }
}

// ---------------------------------------------------------------- attention over the pages
struct PagedAttnParams {
    PagedSeqs seqs;
    PagedPool pool;
    const void *q, *k_pages, *v_pages;
    int64_t q_stride;
    void* out;
    int32_t heads, kv_heads;
    float scale;
};

// One wave per (row, head): 64 keys at a time, a key a lane for the scores, a running maximum and sum, then
// the values with head_dim over the lanes.
template <typename A, typename C, int HD>
__global__ __launch_bounds__(64) void paged_attention_kernel(PagedAttnParams a) {
    __shared__ float qs[HD];
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    const int s = seq_of_row(a.seqs.row_start, a.seqs.seqs, t);
    if (s < 0) return;
    int begin, n;
    seq_rows(a.seqs.row_start, s, a.seqs.rows, begin, n);
    const int i = t - begin;
    if (i < 0 || i >= n) return;
    const A* q = (const A*)a.q + (int64_t)t * a.q_stride + h * HD;
    for (int d = lane; d < HD; d += 64) qs[d] = (float)q[d] * a.scale;
    __syncthreads();
    const int64_t seen64 = (int64_t)a.seqs.lens[s] - n + i + 1;
    const int seen = seen64 < 0 ? 0 : seen64 > a.seqs.cap ? a.seqs.cap : (int)seen64;
    const int64_t head = (int64_t)(h / (a.heads / a.kv_heads)) * a.pool.head_stride;
    const int32_t* table = a.seqs.table + s * a.seqs.table_stride;
    float m = -__builtin_inff(), l = seen64 > a.seqs.cap ? __builtin_nanf("") : 0.f, acc[HD / 64] = {};
    for (int base = 0; base < seen; base += 64) {
        const int p = base + lane;
        const int64_t at = p < seen ? position_offset(table, a.pool, p) : -1;
        float score = -__builtin_inff();
        if (p < seen) score = __builtin_nanf("");
        if (at >= 0) {
            score = 0.f;
            const C* k = (const C*)a.k_pages + at + head;
            for (int d = 0; d < HD; d += 8) {
                float x[8];
                load8(k + d, x);
                for (int j = 0; j < 8; j++) score += qs[d + j] * x[j];
            }
        }
        float top = score;
        for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        top = fmaxf(top, m);
        const float base_of = top == -__builtin_inff() ? 0.f : top;
        const float e = p < seen ? expf(score - base_of) : 0.f;
        const float keep = expf(m - base_of);
        float sum = e;
        for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
        l = l * keep + sum;
        m = top;
        for (int c = 0; c < HD / 64; c++) acc[c] *= keep;
        const int count = seen - base < 64 ? seen - base : 64;
        for (int j = 0; j < count; j++) {
            const float w = __shfl(e, j, 64);
            const int64_t vat = __shfl(at, j, 64);
            if (vat < 0) continue;
            const C* v = (const C*)a.v_pages + vat + head;
            for (int c = 0; c < HD / 64; c++) acc[c] += w * (float)v[c * 64 + lane];
        }
    }
    A* out = (A*)a.out + ((int64_t)t * a.heads + h) * HD;
    for (int c = 0; c < HD / 64; c++) out[c * 64 + lane] = (A)(l == 0.f ? 0.f : acc[c] / l);
}

namespace {

int element_size(int type) { return type == NC_TYPE_F32 ? 4 : type == NC_TYPE_F16 || type == NC_TYPE_BF16 ? 2 : 0; }

// The cache and the sequences of a call, or why they are refused.
int read_cache(const char* who, const nc_paged_kv* kv, const nc_paged_batch* b, int64_t rows, PagedSeqs& s, PagedPool& p) {
    const std::string w(who);
    const int size = element_size(kv->elem_type);
    if (!size) return fail(NC_EINVAL, w + ": the cache's type must be F32, F16 or BF16");
    if (kv->head_dim != 64 && kv->head_dim != 128) return fail(NC_EINVAL, w + ": head_dim must be 64 or 128");
    // an empty tensor has no address
    if (!kv->k_pages || !kv->v_pages || (b->seqs > 0 && (!b->lens || (b->table_pages > 0 && !b->table)))) return fail(NC_EINVAL, w + ": null device address");
    if (kv->pages < 1 || kv->pages > INT32_MAX || kv->page_size < 1 || kv->kv_heads < 1)
        return fail(NC_EINVAL, w + ": the cache needs pages, a page size and heads");
    const int64_t strides[3] = {kv->page_stride, kv->pos_stride, kv->head_stride};
    for (int64_t st : strides)
        if (st < kv->head_dim || st > (INT64_MAX >> 34) || st * size % 16)
            return fail(NC_EINVAL, w + ": cache strides must be at least head_dim and multiples of 16 bytes");
    if (kv->k_pages % 16 || kv->v_pages % 16) return fail(NC_EINVAL, w + ": the pools must be 16-byte aligned");
    if (b->seqs < 0 || b->table_pages < 0 || b->table_stride < b->table_pages || b->max_len < 0)
        return fail(NC_EINVAL, w + ": bad table shape");
    if (b->table % 4 || b->lens % 4 || b->row_start % 4) return fail(NC_EINVAL, w + ": misaligned int32 array");
    if (rows < 0 || rows > INT32_MAX) return fail(NC_ERANGE, w + ": too many rows");
    if (!b->row_start && rows != b->seqs) return fail(NC_EINVAL, w + ": without row starts every sequence has one row");
    s.table = (const int32_t*)b->table;
    s.lens = (const int32_t*)b->lens;
    s.row_start = (const int32_t*)b->row_start;
    s.table_stride = b->table_stride;
    s.table_pages = b->table_pages;
    s.seqs = b->seqs;
    s.rows = (int32_t)rows;
    const int64_t named = (int64_t)b->table_pages * kv->page_size;
    // positions stay below 2^31 - 512, so that the kernels' tiles do not overflow
    const int64_t limit = b->max_len ? b->max_len : INT32_MAX;
    s.cap = (int32_t)std::min<int64_t>(std::min(named, limit), INT32_MAX - 512);
    p.page_stride = kv->page_stride;
    p.pos_stride = kv->pos_stride;
    p.head_stride = kv->head_stride;
    p.pages = (int32_t)kv->pages;
    p.div = page_div((uint32_t)kv->page_size);
    return NC_OK;
}

bool bad_rows(const void* p, int64_t stride, int64_t width, int size) {
    return (uintptr_t)p % 16 || stride < width || stride * size % 16;
}

// Calls f with the element types of the activations and the cache.
template <int HD, typename F>
int with_types(int type, int cache, F f) {
    if (cache == NC_TYPE_F32) {
        if (type == NC_TYPE_F32) return f.template operator()<float, float, HD>();
        if (type == NC_TYPE_F16) return f.template operator()<_Float16, float, HD>();
        return f.template operator()<__bf16, float, HD>();
    }
    if (cache == NC_TYPE_F16) {
        if (type == NC_TYPE_F32) return f.template operator()<float, _Float16, HD>();
        if (type == NC_TYPE_F16) return f.template operator()<_Float16, _Float16, HD>();
        return f.template operator()<__bf16, _Float16, HD>();
    }
    if (type == NC_TYPE_F32) return f.template operator()<float, __bf16, HD>();
    if (type == NC_TYPE_F16) return f.template operator()<_Float16, __bf16, HD>();
    return f.template operator()<__bf16, __bf16, HD>();
}

}  // namespace

}  // namespace nc

using namespace nc;

extern "C" int nc_paged_kv_append(nc_ctx* ctx, const nc_paged_kv* kv, const nc_paged_batch* batch, int type, int64_t rows,
                                  const void* k, int64_t k_stride, const void* v, int64_t v_stride, void* k_out,
                                  const void* q, int64_t q_stride, int32_t heads, void* q_out, const float* rope,
                                  int64_t rope_positions, int32_t rope_dim, void* stream) {
    if (!ctx || !kv || !batch) return fail(NC_EINVAL, "nc_paged_kv_append: null argument");
    AppendParams a = {};
    if (int rc = read_cache("nc_paged_kv_append", kv, batch, rows, a.seqs, a.pool)) return rc;
    const int size = element_size(type);
    if (!size) return fail(NC_EINVAL, "nc_paged_kv_append: the rows' type must be F32, F16 or BF16");
    if (rows == 0 || batch->seqs == 0) return NC_OK;
    if (!k || !v || (q && (!q_out || heads < 1))) return fail(NC_EINVAL, "nc_paged_kv_append: null argument");
    const int64_t kw = (int64_t)kv->kv_heads * kv->head_dim, qw = q ? (int64_t)heads * kv->head_dim : 0;
    if (bad_rows(k, k_stride, kw, size) || bad_rows(v, v_stride, kw, size) || (q && bad_rows(q, q_stride, qw, size)) ||
        (uintptr_t)k_out % 16 || (uintptr_t)q_out % 16)
        return fail(NC_EINVAL, "nc_paged_kv_append: rows must be 16-byte aligned and not overlap");
    if (rope && ((uintptr_t)rope % 4 || rope_dim < 2 || rope_dim > kv->head_dim || rope_dim % 2 || rope_positions < 1))
        return fail(NC_EINVAL, "nc_paged_kv_append: the angles need an even width up to head_dim and positions");
    const int64_t units = (qw + 2 * kw) / 8;
    if (units > 65535 * 256ll) return fail(NC_ERANGE, "nc_paged_kv_append: too many heads");
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.q_out = q_out;
    a.k_out = k_out;
    a.k_pages = (void*)kv->k_pages;
    a.v_pages = (void*)kv->v_pages;
    a.rope = rope;
    a.rope_positions = (int32_t)std::min<int64_t>(rope_positions, INT32_MAX);
    a.rope_half = rope_dim / 2;
    a.heads = heads;
    a.kv_heads = kv->kv_heads;
    DeviceGuard guard(ctx->device);
    if (guard.rc) return guard.rc;
    hipStream_t st = stream ? (hipStream_t)stream : ctx->stream;
    const dim3 grid((unsigned)std::min<int64_t>(rows, 1 << 22), (unsigned)((units + 255) / 256));
    auto launch = [&]<typename A, typename C, int HD>() {
        paged_append_kernel<A, C, HD><<<grid, 256, 0, st>>>(a);
        NC_HIP(hipGetLastError());
        return (int)NC_OK;
    };
    return kv->head_dim == 64 ? with_types<64>(type, kv->elem_type, launch) : with_types<128>(type, kv->elem_type, launch);
}

extern "C" int64_t nc_paged_attention_work_bytes(const nc_paged_kv* kv, const nc_paged_batch* batch, int64_t rows,
                                                 int32_t heads) {
    if (!kv || !batch) return fail(NC_EINVAL, "nc_paged_attention_work_bytes: null argument");
    PagedSeqs s;
    PagedPool p;
    if (int rc = read_cache("nc_paged_attention_work_bytes", kv, batch, rows, s, p)) return rc;
    return 0;
}

extern "C" int nc_paged_attention(nc_ctx* ctx, const nc_paged_kv* kv, const nc_paged_batch* batch, int type, int64_t rows,
                                  const void* q, int64_t q_stride, int32_t heads, float scale, void* out, void* work,
                                  int64_t work_bytes, void* stream) {
    if (!ctx || !kv || !batch) return fail(NC_EINVAL, "nc_paged_attention: null argument");
    PagedAttnParams a = {};
    if (int rc = read_cache("nc_paged_attention", kv, batch, rows, a.seqs, a.pool)) return rc;
    const int size = element_size(type);
    if (!size || (type != NC_TYPE_F32 && type != kv->elem_type))
        return fail(NC_EINVAL, "nc_paged_attention: rows must be F32 or of the cache's type");
    if (heads < 1 || heads % kv->kv_heads)
        return fail(NC_EINVAL, "nc_paged_attention: heads must be a multiple of the cache's heads");
    if (rows == 0 || batch->seqs == 0) return NC_OK;
    if (!q || !out) return fail(NC_EINVAL, "nc_paged_attention: null argument");
    if (bad_rows(q, q_stride, (int64_t)heads * kv->head_dim, size) || (uintptr_t)out % 16)
        return fail(NC_EINVAL, "nc_paged_attention: rows must be 16-byte aligned and not overlap");
    if (work_bytes < nc_paged_attention_work_bytes(kv, batch, rows, heads))
        return fail(NC_EINVAL, "nc_paged_attention: the workspace is too small");
    (void)work;
    a.q = q;
    a.k_pages = (const void*)kv->k_pages;
    a.v_pages = (const void*)kv->v_pages;
    a.q_stride = q_stride;
    a.out = out;
    a.heads = heads;
    a.kv_heads = kv->kv_heads;
    a.scale = scale;
    DeviceGuard guard(ctx->device);
    if (guard.rc) return guard.rc;
    hipStream_t st = stream ? (hipStream_t)stream : ctx->stream;
    auto launch = [&]<typename A, typename C, int HD>() {
        if constexpr (std::is_same_v<A, float> || std::is_same_v<A, C>) {
            paged_attention_kernel<A, C, HD><<<dim3((unsigned)rows, heads), 64, 0, st>>>(a);
            NC_HIP(hipGetLastError());
        }
        return (int)NC_OK;
    };
    return kv->head_dim == 64 ? with_types<64>(type, kv->elem_type, launch) : with_types<128>(type, kv->elem_type, launch);
}
