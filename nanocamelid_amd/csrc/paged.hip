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
// spreads over many CUs.  Four prompts of up to 2711 rows, 32 heads over 8 of 128 dimensions, f32 into f16: 244 MB
// in 40 us, 6.1 TB/s, 53 us a call where calls follow each other; 48 sequences of up to 5 rows 5 us, one row 3 us.
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
    float *part_o, *part_ml;  // [row][head][slots][head_dim] and [2] (maximum, sum); null: slots is 1 or all in turn
    int64_t units;  // row groups of all sequences, or more
    int32_t heads, kv_heads, slots, balanced;
    float scale;
};

// A sequence's positions in chunks of four waves, 32 KiB of keys and values a wave, or 16.
template <typename C, int HD>
constexpr int kWaveKeys = HD == 128 && sizeof(C) == 4 ? 32 : 64;
template <typename C, int HD>
constexpr int kChunkKeys = 4 * kWaveKeys<C, HD>;

// What a row has summed over some of its positions: the largest score, and the sums of weights and of weighted
// values relative to it.  Chunks are added in their order, in this form only, whether one workgroup takes them
// in turn or the join kernel reads them: the bits are the same.
template <int N>
struct RowSum {
    float m = -__builtin_inff(), l = 0.f, o[N] = {};
    __device__ __forceinline__ void add(float m2, float l2, float f, float g, const float* o2) {
        m = m2;
        l = __builtin_fmaf(l, f, l2 * g);
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = __builtin_fmaf(o[i], f, o2[i] * g);
    }
    __device__ __forceinline__ void add_chunk(float mc, float lc, const float* oc) {
        const float top = fmaxf(m, mc), base = exp_base(top);
        add(top, lc, exp2_hw(m - base), exp2_hw(mc - base), oc);
    }
    __device__ __forceinline__ float answer(int i) const { return l == 0.f ? 0.f : o[i] / l; }
};

// A barrier that orders LDS alone, so that it does not wait for loads that are in flight.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Attention of the rows of one sequence and kv head over chunks of its positions.
//
// Bound by the cache's bytes, each read once for all rows and heads that share them.  Rows (new row, query
// head of the group) fill the 16 columns of a matrix product, RT tiles of them.  Everything is transposed, so
// that nothing has to cross lanes between the two products: scores^T = K q^T leaves lane (g, r) the scores of
// row r at the keys 4g..4g+3 of each 16, which is where out^T = V^T p^T takes its weights from if its inner
// index counts the keys in that order; maximum, sum and scaling of a row stay in the lanes of its column.
//   16 bits: keys and values go from memory to registers as they lie (16 bytes of a key's dimensions; 16 or 8 of
//   a value's, of the lane's eight keys), the values turned in registers by byte permutes.  f32 queries and the
//   weights are split into 16-bit parts (nc_paged.h); the matrix cores have the room, the bytes are the bound.
//   Weights of 16-bit rows are two parts as well: one alone would round as much as the answer's own rounding.
//   f32: products of 16 x 16 x 4, whose operands need no turning.
// A wave takes 32 or 64 positions at once: all their loads are in flight together, and one maximum serves them.
//
// Measured: 48 rows of 64 heads over 8 of 128 dimensions, bf16, up to 8000 positions: 870 MB in 197 us, 4.4 TB/s (a
// kernel that reads without a table reaches 6.3, a copy 4.8); 16 sequences of up to 5 rows, f32, up to 3000
// positions: 227 MB in 47 us, 4.8 TB/s; one row over 15000 positions in f16: 61 MB in 15 us.  What is lost is lost
// between chunks, where four waves join and the table's next pages are looked up: no byte of the cache is fetched
// twice.  Loads that bypass the caches, 32 positions of 16 bits a wave and keys read in the values' pattern were no
// faster.
template <typename A, typename C, int HD, int RT, bool ONE>
__global__ __launch_bounds__(256, RT == 1 || HD == 64 ? 2 : 1) void paged_attention_kernel(PagedAttnParams a) {
    constexpr bool F32 = sizeof(C) == 4;
    constexpr int KW = kWaveKeys<C, HD>, CH = 4 * KW, KT = KW / 16;
    constexpr bool BF = std::is_same_v<C, __bf16>;
    constexpr int QP = std::is_same_v<A, C> ? 1 : BF ? 3 : 2;  // parts of a query value
    constexpr int PP = BF && QP == 3 ? 3 : 2;                  // parts of a weight
    constexpr bool QSCALE = QP == 2;                           // f16 parts: the row scaled into f16's range
    // f16 weights carry 2^14, which keeps small ones normal numbers and cancels in the answer
    constexpr float PSHIFT = !F32 && !BF ? 14.f : 0.f;
    // A single chunk's keys and values are asked for at once.  Otherwise each half of the values takes the place of that
    // half of the keys, and the next chunk's keys theirs: the next chunk's beside this one's, where registers allow,
    // were slower (24 rows of up to 4000 positions, 64 dimensions, f32: 50 us against 45, bf16: 29 and 27).
    constexpr bool EARLY = RT == 1 && ONE;
    constexpr int JB = RT == 1 && QP < 3 && !ONE ? 2 : 1;  // LDS buffers of the waves' joining
    constexpr int OS = HD + 4;     // LDS row, skewed by four banks
    constexpr int ND = HD / 16;    // dimensions of a thread in the chunk's sum
    __shared__ int64_t s_off[2][4][KW];
    using V8 = typename Vec8<std::conditional_t<F32, _Float16, C>>::type;
    constexpr int QV = F32 ? HD / 16 : HD / 32;  // 16-byte pieces of a lane's queries, and of its key
    __shared__ u32x4 s_q[RT][QP][QV][64];
    __shared__ float s_factor[RT][16];
    __shared__ int64_t s_scan[6];
    __shared__ __attribute__((aligned(8))) float s_ml[JB][4][16][2];
    __shared__ __attribute__((aligned(16))) float s_o[JB][4][16][OS];

    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int G = a.heads / a.kv_heads;
    const int32_t* row_start = a.seqs.row_start;

    // Work comes as (row group, kv head, chunks from, to).  Either the grid names it: groups of all sequences one
    // after the other along z, kv heads along y, chunks along x; or, where there are more chunks than workgroups fit
    // the chip, all chunks of all sequences in one row are cut into equal parts, each of which kv_heads workgroups
    // stream, a kv head each.  Those follow each other in the launch, as their heads do in the usual order of a
    // pool: what lies together is read at one time.  The heads turn from part to part, so that no XCD (workgroups go
    // to the eight in turn) reads one head only, whose rows may all lie in a few channels of its L2.
    int64_t z = blockIdx.z, rest = 0, todo = 0;
    int s = 0;
    auto cost_of = [&](int i, int& begin, int& n, int& chunks) -> int64_t {
        seq_rows(row_start, i, a.seqs.rows, begin, n);
        const int len = a.seqs.lens[i], most = len < a.seqs.cap ? len : a.seqs.cap;
        chunks = most > 0 ? (most - 1) / CH + 1 : 1;
        return (int64_t)((n * G + 16 * RT - 1) / (16 * RT)) * chunks;
    };
    if (!ONE && a.balanced) {
        // the sum over the sequences before the 256 at i0, of theirs up to the thread's own, and the thread's
        int64_t all = 0, upto = 0, mine = 0;
        auto scan = [&](int i0) {
            int begin, n, chunks;
            const int i = i0 + threadIdx.x;
            mine = i < a.seqs.seqs ? cost_of(i, begin, n, chunks) : 0;
            upto = mine;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const int64_t x = __shfl_up(upto, d, 64);
                if (lane >= d) upto += x;
            }
            lds_barrier();
            if (lane == 63) s_scan[w] = upto;
            lds_barrier();
            for (int i = 0; i < w; i++) upto += s_scan[i];
            upto += all;
            all += s_scan[0] + s_scan[1] + s_scan[2] + s_scan[3];
        };
        for (int i0 = 0; i0 < a.seqs.seqs; i0 += 256) scan(i0);
        const int64_t part = blockIdx.x / a.kv_heads, parts = gridDim.x / a.kv_heads;
        const int64_t total = all, first = total * part / parts, past = total * (part + 1) / parts;
        if (first == past) return;
        todo = past - first;
        auto claim = [&](int i0) {
            if (upto - mine <= first && first < upto) s_scan[4] = i0 + threadIdx.x, s_scan[5] = first - (upto - mine);
        };
        if (a.seqs.seqs <= 256) {
            claim(0);
        } else {
            all = 0;
            for (int i0 = 0; i0 < a.seqs.seqs; i0 += 256) {
                scan(i0);
                claim(i0);
            }
        }
        lds_barrier();
        s = __builtin_amdgcn_readfirstlane((int)s_scan[4]);
        rest = s_scan[5];
    }

    for (;;) {
        int begin = 0, n = 0, r0 = 0, kvh = blockIdx.y, c = blockIdx.x, c_to = INT32_MAX;
        if (!ONE && a.balanced) {
            if (todo <= 0 || s >= a.seqs.seqs) return;
            int chunks;
            const int64_t cost = cost_of(s, begin, n, chunks);
            if (rest >= cost) {
                rest -= cost;
                s++;
                continue;
            }
            const int group = (int)(rest / chunks);
            c = (int)(rest - (int64_t)group * chunks);
            kvh = (blockIdx.x + blockIdx.x / a.kv_heads) % a.kv_heads;
            r0 = group * (16 * RT);
            const int take = (int)(todo < chunks - c ? todo : chunks - c);
            c_to = c + take;
            todo -= take;
            rest += take;
        } else if (!row_start) {
            if (z >= a.units) return;
            const int per = (G + 16 * RT - 1) / (16 * RT);
            s = (int)(z / per);
            r0 = (int)(z % per) * (16 * RT);
            begin = s;
            n = 1;
            z += gridDim.z;
        } else {
            if (z >= a.units) return;
            int64_t u = z;
            s = -1;
            for (int s0 = 0; s0 < a.seqs.seqs; s0 += 64) {
                int mb = 0, mn = 0;
                if (s0 + lane < a.seqs.seqs) seq_rows(row_start, s0 + lane, a.seqs.rows, mb, mn);
                const int upto = wave_prefix_sum((mn * G + 16 * RT - 1) / (16 * RT));
                const uint64_t past = __ballot(upto > u);
                if (past) {
                    const int at = __builtin_ctzll(past);
                    s = s0 + at;
                    begin = __builtin_amdgcn_readlane(mb, at);
                    n = __builtin_amdgcn_readlane(mn, at);
                    // counted from the sequence's last group
                    r0 = (__builtin_amdgcn_readlane(upto, at) - 1 - (int)u) * (16 * RT);
                    break;
                }
                u -= __builtin_amdgcn_readlane(upto, 63);
            }
            if (s < 0) return;  // past the last unit, and so is every later one
            s = __builtin_amdgcn_readfirstlane(s);
            z += gridDim.z;
        }
        const int step = a.balanced ? 1 : gridDim.x;
        const int64_t head_off = (int64_t)kvh * a.pool.head_stride;
        const C* kb = (const C*)a.k_pages + head_off;
        const C* vb = (const C*)a.v_pages + head_off;
        const int32_t* table = a.seqs.table + s * a.seqs.table_stride;
        const int64_t before = (int64_t)a.seqs.lens[s] - n;  // positions before the first new row
        const int R = n * G;  // below 2^31: so are all rows' heads
        {
            // the positions that a row sees, at most cap of them
            auto seen_of = [&](int row) {
                const int64_t e = before + row / G + 1;
                return (int)(e < 0 ? 0 : e > a.seqs.cap ? a.seqs.cap : e);
            };
            const int last = R - r0 > 16 * RT ? r0 + 16 * RT - 1 : R - 1;
            const int least = seen_of(r0), most = seen_of(last);
            const int all_chunks = most > 0 ? (most - 1) / CH + 1 : 1, chunks = all_chunks < c_to ? all_chunks : c_to;
            if (c >= chunks) continue;

            // A wave's keys and values of a chunk.  Values are asked for as the scores of their keys are done, the next
            // chunk's keys as the values are summed, so that loads are in flight through the softmax and the waves'
            // joining.  They are issued whether or not there is a next chunk: behind a branch, every wait for an earlier
            // load would have to wait for these as well.
            typedef uint32_t VL __attribute__((ext_vector_type(F32 ? 4 : HD / 32)));  // 16 bytes, or HD / 16 values
            constexpr int KV = QV, NV = F32 ? HD / 64 : 1;
            u32x4 kx[KT][KV];
            VL vx[KT][4][NV];
            // Every lane finds one key's place, for its wave; -1: past the end, or its page is none of the pool's.  The
            // page's number is asked for a chunk ahead, before that chunk's keys: loads return in order, and a later
            // one would be waited for with all of those.
            int32_t page_id = -1;
            bool bad_pages = false;
            auto ask = [&](int c) {
                const int64_t p = (int64_t)c * CH + w * KW + lane;
                page_id = lane < KW && p < a.seqs.cap ? table[page_of((uint32_t)p, a.pool.div)] : -1;
            };
            auto publish = [&](int buf, int c) {
                const int p = c * CH + w * KW + lane;
                const bool live = lane < KW && p < most, good = live && (uint32_t)page_id < (uint32_t)a.pool.pages;
                if (lane < KW) s_off[buf][w][lane] = good ? place_in_page(page_id, p, a.pool) : -1;
                bad_pages = __ballot(live && !good) != 0;
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            };
            // keys without a place read the pool's first row, which is there, and count as nothing
            auto key_at = [&](int buf, int i) {
                const int64_t at = s_off[buf][w][i];
                return at < 0 ? (int64_t)0 : at;
            };
            auto load_keys = [&](int buf, int half) {
#pragma unroll
                for (int j = half * KT / 2; j < (half + 1) * KT / 2; j++) {
                    const C* k = kb + key_at(buf, 16 * j + r) + (F32 ? 4 : 8) * g;
#pragma unroll
                    for (int d = 0; d < KV; d++) kx[j][d] = *(const u32x4*)(k + (F32 ? 16 : 32) * d);
                    __builtin_amdgcn_sched_barrier(0);  // a few addresses at a time: they take two registers each
                }
            };
            auto load_values = [&](int buf, int half) {
#pragma unroll
                for (int j = half * KT / 2; j < (half + 1) * KT / 2; j++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const C* v = vb + key_at(buf, 16 * j + 4 * g + i) + (F32 ? 4 : ND) * r;
#pragma unroll
                        for (int h = 0; h < NV; h++) vx[j][i][h] = *(const VL*)(v + 64 * h);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            };

            ask(c);
            publish(0, c);
            if (!ONE) ask(c + step);
#pragma unroll
            for (int half = 0; half < 2; half++) load_keys(0, half);
            if (EARLY) {
#pragma unroll
                for (int half = 0; half < 2; half++) load_values(0, half);
            }

            // The queries in operand order, in LDS for the four waves: wave t has tile t's.  What scales a row's scores
            // to base 2 goes beside them.
            if (w < RT) {
                const int row = r0 + 16 * w + r, rr = row < R ? row : r0;
                const A* q = (const A*)a.q + (int64_t)(begin + rr / G) * a.q_stride + (kvh * G + rr % G) * HD;
                float factor = a.scale * kLog2e;
                if constexpr (F32 || QP == 1) {
#pragma unroll
                    for (int d = 0; d < QV; d++) s_q[w][0][d][lane] = *(const u32x4*)(q + (F32 ? 16 * d + 4 * g : 32 * d + 8 * g));
                } else {
                    float x[QV][8];
                    float top = 0.f;
#pragma unroll
                    for (int d = 0; d < QV; d++) {
                        load8(q + 32 * d + 8 * g, x[d]);
#pragma unroll
                        for (int e = 0; e < 8; e++) top = fmaxf(top, __builtin_fabsf(x[d][e]));
                    }
                    int shift = 0;
                    if (QSCALE) {  // the row's largest value to [2^9, 2^10)
                        top = max_across<32>(max_across<16>(top));
                        const int ex = (int)(__float_as_uint(top) >> 23);
                        shift = ex == 0 || ex == 255 ? 0 : 136 - ex;
                        factor = __builtin_ldexpf(factor, -shift);
                    }
#pragma unroll
                    for (int d = 0; d < QV; d++) {
                        V8 parts[QP];
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            C part[QP];
                            split_parts(QSCALE ? __builtin_ldexpf(x[d][e], shift) : x[d][e], part);
#pragma unroll
                            for (int p = 0; p < QP; p++) parts[p][e] = part[p];
                        }
#pragma unroll
                        for (int p = 0; p < QP; p++) s_q[w][p][d][lane] = __builtin_bit_cast(u32x4, parts[p]);
                    }
                }
                if (g == 0) s_factor[w][r] = factor;
            }
            int seen[RT];
#pragma unroll
            for (int t = 0; t < RT; t++) seen[t] = r0 + 16 * t + r < R ? seen_of(r0 + 16 * t + r) : 0;
            lds_barrier();

            // The thread's part in joining the waves: of each tile one row, ND dimensions.  Its output row, and its
            // chunks (0: none, there is no such row).
            const int row16 = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * ND;
            RowSum<ND> sum[RT];
            int unit[RT], own[RT];
#pragma unroll
            for (int t = 0; t < RT; t++) {
                const int row = r0 + 16 * t + row16;
                unit[t] = (begin + row / G) * a.heads + kvh * G + row % G;
                own[t] = row >= R ? 0 : seen_of(row) > 0 ? (seen_of(row) - 1) / CH + 1 : 1;
                // a row that needs a position past the last that can be named
                if (before + row / G + 1 > a.seqs.cap) sum[t].l = __builtin_nanf("");
            }
            int buf = 0;
            for (; c < chunks; c += step) {
                const int base = c * CH + w * KW;
                // past the last chunk: no key has a place then
                const int next = chunks - c > step ? c + step : INT32_MAX / CH;
                const bool masked = base + KW > least || bad_pages;

                f32x4 o[RT][ND] = {};
                float m[RT], l[RT];
#pragma unroll
                for (int t = 0; t < RT; t++) m[t] = -__builtin_inff(), l[t] = 0.f;
                {
                    f32x4 sc[RT][KT] = {};
#pragma unroll
                    for (int half = 0; half < 2; half++) {
#pragma unroll
                        for (int t = 0; t < RT; t++)
#pragma unroll
                            for (int d = 0; d < KV; d++) {
                                u32x4 q[QP];
#pragma unroll
                                for (int p = 0; p < QP; p++) q[p] = s_q[t][p][d][lane];
#pragma unroll
                                for (int j = half * KT / 2; j < (half + 1) * KT / 2; j++) {
                                    if constexpr (F32) {
#pragma unroll
                                        for (int e = 0; e < 4; e++)
                                            sc[t][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kx[j][d][e]), __uint_as_float(q[0][e]), sc[t][j], 0, 0, 0);
                                    } else {
#pragma unroll
                                        for (int p = QP - 1; p >= 0; p--)
                                            sc[t][j] = mfma16(__builtin_bit_cast(V8, kx[j][d]), __builtin_bit_cast(V8, q[p]), sc[t][j]);
                                    }
                                }
                            }
                        if (!EARLY) load_values(buf, half);
                    }
                    if (!ONE) {
                        publish(buf ^ 1, next);
                        ask(next + step);
                    }
#pragma unroll
                    for (int t = 0; t < RT; t++) {
                        const float factor = s_factor[t][r];
#pragma unroll
                        for (int j = 0; j < KT; j++) sc[t][j] *= factor;
                    }
                    if (masked) {
#pragma unroll
                        for (int j = 0; j < KT; j++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const int key = 16 * j + 4 * g + i;
                                const bool bad = s_off[buf][w][key] < 0;
#pragma unroll
                                for (int t = 0; t < RT; t++)
                                    sc[t][j][i] = base + key < seen[t] ? (bad ? __builtin_nanf("") : sc[t][j][i])
                                                                       : -__builtin_inff();
                            }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    // scores to weights, in base 2
#pragma unroll
                    for (int t = 0; t < RT; t++) {
                        float top = -__builtin_inff();
#pragma unroll
                        for (int j = 0; j < KT; j++)
#pragma unroll
                            for (int i = 0; i < 4; i++) top = fmaxf(top, sc[t][j][i]);
                        top = max_across<32>(max_across<16>(top));
                        const float lift = exp_base(top) - PSHIFT;
                        float total = 0.f;
#pragma unroll
                        for (int j = 0; j < KT; j++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const float e = exp2_hw(sc[t][j][i] - lift);
                                sc[t][j][i] = e;
                                total += e;
                            }
                        total = sum_across<32>(sum_across<16>(total));
                        m[t] = top;
                        l[t] = total;
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    // A zero weight times an infinity is no zero: in masked tiles values that are not finite, and
                    // those of keys without a place, are left out of the product.
                    bool odd = false;
                    if (masked) {
#pragma unroll
                        for (int j = 0; j < KT; j++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const bool gone = s_off[buf][w][16 * j + 4 * g + i] < 0;
#pragma unroll
                                for (int h = 0; h < NV; h++)
#pragma unroll
                                    for (int d = 0; d < (F32 ? 4 : HD / 32); d++) {
                                        const uint32_t x = vx[j][i][h][d];
                                        if constexpr (F32) {
                                            const bool bad = (x & 0x7f800000u) == 0x7f800000u;
                                            odd |= bad && !gone;
                                            vx[j][i][h][d] = bad || gone ? 0u : x;
                                        } else {
                                            constexpr uint32_t EXP = BF ? 0x7f80u : 0x7c00u;
                                            const bool lo = (x & EXP) == EXP, hi = (x >> 16 & EXP) == EXP;
                                            odd |= (lo || hi) && !gone;
                                            vx[j][i][h][d] = gone ? 0u : (lo ? 0u : x & 0xffffu) | (hi ? 0u : x & 0xffff0000u);
                                        }
                                    }
                            }
                    }
                    if constexpr (F32) {
#pragma unroll
                        for (int j = 0; j < KT; j++) {
                            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                            for (int i = 0; i < 4; i++)
#pragma unroll
                                for (int h = 0; h < NV; h++)
#pragma unroll
                                    for (int e = 0; e < 4; e++)
#pragma unroll
                                        for (int t = 0; t < RT; t++)
                                            o[t][4 * h + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vx[j][i][h][e]), sc[t][j][i], o[t][4 * h + e], 0, 0, 0);
                            if (!ONE && j % (KT / 2) == KT / 2 - 1) load_keys(buf ^ 1, 2 * j / KT);
                        }
                    } else {
#pragma unroll
                        for (int b = 0; b < KT / 2; b++) {
                            __builtin_amdgcn_sched_barrier(0);
                            V8 pv[RT][PP];
#pragma unroll
                            for (int t = 0; t < RT; t++)
#pragma unroll
                                for (int i = 0; i < 8; i++) {
                                    C part[PP];
                                    split_parts(sc[t][2 * b + i / 4][i % 4], part);
#pragma unroll
                                    for (int p = 0; p < PP; p++) pv[t][p][i] = part[p];
                                }
#pragma unroll
                            for (int e = 0; e < ND; e++) {
                                u32x4 x;  // dimension e of the lane's eight keys
#pragma unroll
                                for (int i = 0; i < 4; i++)
                                    x[i] = __builtin_amdgcn_perm(vx[2 * b + i / 2][2 * i % 4 + 1][0][e / 2], vx[2 * b + i / 2][2 * i % 4][0][e / 2],
                                                                 e % 2 ? 0x07060302u : 0x05040100u);
                                const V8 vt = __builtin_bit_cast(V8, x);
#pragma unroll
                                for (int t = 0; t < RT; t++)
#pragma unroll
                                    for (int p = PP - 1; p >= 0; p--) o[t][e] = mfma16(vt, pv[t][p], o[t][e]);
                            }
                            if (!ONE && b % (KT / 4) == KT / 4 - 1) load_keys(buf ^ 1, 4 * b / KT);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    // the values left out go to the rows that see their key
                    if (__ballot(odd)) {
                        const int g4 = kept_here(4 * g);
                        for (int key = 0; key < KW; key++) {
                            const int64_t at = s_off[buf][w][key];
                            if (at < 0) continue;
#pragma unroll
                            for (int e = 0; e < ND; e++)
#pragma unroll
                                for (int i = 0; i < 4; i++) {
                                    const int d = F32 ? 64 * (e / 4) + 4 * g4 + 4 * i + e % 4 : ND * (g4 + i) + e;
                                    const float v = (float)vb[at + d];
                                    if (!__builtin_isfinite(v))
#pragma unroll
                                        for (int t = 0; t < RT; t++)
                                            if (base + key < seen[t]) o[t][e][i] += v;
                                }
                        }
                    }
                }
                buf ^= 1;

                // The four waves' sums to one, in their order.  Two buffers in turn need one barrier: when a buffer is
                // written again, all have passed the barrier of the other, behind their last reading of this one.
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    const int jb = JB == 2 ? buf : 0;
                    if (r0 + 16 * t + r < R) {
                        if (g == 0) *(f32x2*)s_ml[jb][w][r] = f32x2{m[t], l[t]};
#pragma unroll
                        for (int e = 0; e < ND; e += 4)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const int d = F32 ? 16 * e + 16 * g + 4 * i : ND * (4 * g + i) + e;
                                *(f32x4*)&s_o[jb][w][r][d] = f32x4{o[t][e][i], o[t][e + 1][i], o[t][e + 2][i], o[t][e + 3][i]};
                            }
                    }
                    lds_barrier();
                    if (c < own[t]) {
                        f32x2 ml[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) ml[i] = *(const f32x2*)s_ml[jb][i][row16];
                        const float top = fmaxf(fmaxf(ml[0][0], ml[1][0]), fmaxf(ml[2][0], ml[3][0])), lift = exp_base(top);
                        float lc = 0.f, oc[ND] = {};
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float f = exp2_hw(ml[i][0] - lift);
                            lc = __builtin_fmaf(ml[i][1], f, lc);
#pragma unroll
                            for (int d = 0; d < ND; d++) oc[d] = __builtin_fmaf(s_o[jb][i][row16][d0 + d], f, oc[d]);
                        }
                        if (a.slots > 1 && own[t] > 1) {
                            const int64_t at = (int64_t)unit[t] * a.slots + c;
                            if (d0 == 0) *(f32x2*)(a.part_ml + 2 * at) = f32x2{top, lc};
#pragma unroll
                            for (int d = 0; d < ND; d += 4)
                                *(f32x4*)(a.part_o + at * HD + d0 + d) = f32x4{oc[d], oc[d + 1], oc[d + 2], oc[d + 3]};
                        } else {
                            sum[t].add_chunk(top, lc, oc);
                            if (c == own[t] - 1) {
                                A* out = (A*)a.out + (int64_t)unit[t] * HD + d0;
#pragma unroll
                                for (int d = 0; d < ND; d++) out[d] = (A)sum[t].answer(d);
                            }
                        }
                    }
                    if (JB == 1) lds_barrier();
                }
                if (ONE) break;
            }
            lds_barrier();  // before the next unit's queries
        }
    }
}

// The chunks of one (row, head) by a wave, a few dimensions a lane.  The running maxima, which only compare, come
// from a scan over the lanes, 64 chunks at a time, so that the chunks' loads do not wait for each other: 32 are in
// flight while 32 are added.
//
// Bound by latency: few rows, and three loads after each other before a sum is known to count (59 chunks of 32 rows
// 7 us, most of it the start and the loads), by the partial sums' bytes where rows are many (51 MB, 48 rows of 64
// heads of up to 32 chunks: 11 us, 4.6 TB/s).
template <typename A, int HD>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnParams a, int chunk) {
    constexpr int ND = HD / 64;
    const int lane = threadIdx.x & 63;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (unit >= (int64_t)a.seqs.rows * a.heads) return;
    typedef float O __attribute__((ext_vector_type(ND)));
    const float* ml = a.part_ml + unit * a.slots * 2;
    const O* o = (const O*)(a.part_o + unit * a.slots * HD) + lane;
    constexpr int B = 32;
    O x[B], y[B];
    // The first ones are asked for before their number is known: the row's slots are there, written or not
    f32x2 mine = *(const f32x2*)(ml + 2 * (lane < a.slots ? lane : 0));
    auto load = [&](O(&x)[B], int c0, int chunks, int from) {
#pragma unroll
        for (int i = from; i < B; i += 16)
            if (c0 + i < chunks)
#pragma unroll
                for (int j = i; j < i + 16; j++) x[j] = o[(int64_t)(c0 + j < chunks ? c0 + j : chunks - 1) * (HD / ND)];
    };
#pragma unroll
    for (int j = 0; j < 16; j++) x[j] = o[(int64_t)(j < a.slots ? j : a.slots - 1) * (HD / ND)];
    const int t = (int)(unit / a.heads);
    const int s = seq_of_row(a.seqs.row_start, a.seqs.seqs, t);
    if (s < 0) return;
    int begin, n;
    seq_rows(a.seqs.row_start, s, a.seqs.rows, begin, n);
    if (t < begin || t >= begin + n) return;
    const int64_t seen64 = (int64_t)a.seqs.lens[s] - n + (t - begin) + 1;
    const int seen = (int)(seen64 < 0 ? 0 : seen64 > a.seqs.cap ? a.seqs.cap : seen64);
    const int chunks = seen > 0 ? (seen - 1) / chunk + 1 : 1;
    if (chunks == 1) return;  // answered already
    load(x, 0, chunks, 16);
    RowSum<ND> sum;
    if (seen64 > a.seqs.cap) sum.l = __builtin_nanf("");
    for (int c0 = 0; c0 < chunks; c0 += 64) {
        if (c0 + lane >= chunks) mine = f32x2{-__builtin_inff(), 0.f};
        float top = fmaxf(mine[0], sum.m);  // the largest score up to this chunk
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const float y = __shfl_up(top, d, 64);
            if (lane >= d) top = fmaxf(top, y);
        }
        float prev = __shfl_up(top, 1, 64);
        if (lane == 0) prev = sum.m;
        const float base = exp_base(top), f = exp2_hw(prev - base), g = exp2_hw(mine[0] - base), l2 = mine[1];
        sum.m = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(top), 63));
        if (c0 + 64 < chunks) mine = *(const f32x2*)(ml + 2 * (c0 + 64 + lane < chunks ? c0 + 64 + lane : chunks - 1));
        auto of = [](float v, int at) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), at)); };
        for (int b = 0; b < 64 && c0 + b < chunks; b += B) {
            load(y, c0 + b + B, chunks, 0);
#pragma unroll
            for (int j = 0; j < B; j++)
                if (c0 + b + j < chunks) {
                    float z[ND];
#pragma unroll
                    for (int d = 0; d < ND; d++) z[d] = x[j][d];
                    sum.add(sum.m, of(l2, b + j), of(f, b + j), of(g, b + j), z);
                }
#pragma unroll
            for (int j = 0; j < B; j++) x[j] = y[j];
        }
    }
    A* out = (A*)a.out + unit * HD + ND * lane;
#pragma unroll
    for (int d = 0; d < ND; d++) out[d] = (A)sum.answer(d);
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
    return (uintptr_t)p % 16 || stride < width || stride > (INT64_MAX >> 34) || stride * size % 16;
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

// How a call is launched: tiles of 16 rows a workgroup, units of such row groups, workgroups along a unit's chunks,
// and chunk slots of a row's partial sums (1: none are kept).
struct AttnPlan {
    int tiles = 1, chunk = 256, slots = 1, along = 1;
    bool balanced = false;
    bool one = false;  // a workgroup has at most one chunk of a unit: nothing to load ahead
    int64_t units = 1;
    int64_t bytes(int64_t rows, int heads, int hd) const { return slots > 1 ? rows * heads * slots * (hd + 2) * 4 : 0; }
};

AttnPlan plan_attention(const nc_paged_kv& kv, const PagedSeqs& s, int heads) {
    AttnPlan p;
    const int64_t group = heads / kv.kv_heads, seqs = std::max(s.seqs, 1);
    p.chunk = kv.head_dim == 128 && kv.elem_type == NC_TYPE_F32 ? 128 : 256;
    // Two tiles where sequences have more than 16 rows: with one, their keys and values are read twice.  Where they
    // may differ, from an average of 25 on (16 sequences of up to 3000 positions in f32, 4 query heads a kv head: of
    // up to 5 new rows, 10 on average, 62 us with one and 68 with two; up to 8: 65 and 70; up to 16: 109 and 97).
    const int64_t rows = ((int64_t)s.rows + seqs - 1) / seqs * group;
    p.tiles = rows <= (s.row_start ? 24 : 16) ? 1 : 2;
    const int64_t high = 16 * p.tiles;
    p.units = s.row_start ? (int64_t)s.rows * group / high + seqs : seqs * ((group + high - 1) / high);
    const int64_t chunks = std::max<int64_t>(((int64_t)s.cap + p.chunk - 1) / p.chunk, 1);
    // A workgroup takes a chunk, or where there may be more of them than fit the chip at once (two workgroups a CU, one
    // with two tiles of 128 dimensions) an equal part of all, and the chunks are joined afterwards.  A join costs some
    // 7 us, as much as three chunks in turn (8 kv heads, 128 dimensions of 16 bits, chunks of 256; joined and in
    // turn: one row of 700 positions 13.5 and 14.1 us, of 1000 14 and 17, of 15000 23 and 163), and parts
    // stream slower than workgroups that stay with a unit: they are for units that leave CUs idle or of very
    // different lengths (24 rows of up to 2000 positions 33 and 30 us, 40 of up to 3000 62 and 70, 48 of up to 8000
    // 208 and 218; 64 of up to 600, 2000 and 8000 31 and 22, 69 and 70, 235 and 240; 128 of up to 4000 228 and 209).  From 65
    // chunks on they guard more units too against a long sequence among short ones, whose chunks take 2.8 us each in
    // turn, at a cost where lengths are evenly spread (128 rows of up to 16000: 922 and 831 us).
    const int64_t units = kv.kv_heads * p.units, fit = p.tiles == 1 || kv.head_dim == 64 ? 512 : 256;
    const bool fits = units * chunks <= fit;
    if (fits ? chunks > 3 : chunks > 8 && (units < fit * 3 / 2 || (chunks > 64 && units < 2048))) {
        p.slots = (int)std::min<int64_t>(chunks, INT32_MAX);
        p.balanced = !fits;
        p.along = (int)(fits ? chunks : std::max<int64_t>(fit / kv.kv_heads, 1) * kv.kv_heads);
    }
    p.one = p.along == chunks && !p.balanced;
    return p;
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
    if (heads < 1 || heads % kv->kv_heads || kv->kv_heads > 65535)
        return fail(NC_EINVAL, "nc_paged_attention_work_bytes: heads must be a multiple of the cache's heads, those at most 65535");
    if (rows * heads > INT32_MAX - 512) return fail(NC_ERANGE, "nc_paged_attention_work_bytes: too many rows and heads");
    const AttnPlan plan = plan_attention(*kv, s, heads);
    return plan.bytes(rows, heads, kv->head_dim);
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
    if (heads < 1 || heads % kv->kv_heads || kv->kv_heads > 65535)
        return fail(NC_EINVAL, "nc_paged_attention: heads must be a multiple of the cache's heads, those at most 65535");
    if (rows * heads > INT32_MAX - 512) return fail(NC_ERANGE, "nc_paged_attention: too many rows and heads");
    if (rows == 0 || batch->seqs == 0) return NC_OK;
    if (!q || !out) return fail(NC_EINVAL, "nc_paged_attention: null argument");
    if (bad_rows(q, q_stride, (int64_t)heads * kv->head_dim, size) || (uintptr_t)out % 16)
        return fail(NC_EINVAL, "nc_paged_attention: rows must be 16-byte aligned and not overlap");
    if (out == q) return fail(NC_EINVAL, "nc_paged_attention: the output must not be the queries");
    const AttnPlan plan = plan_attention(*kv, a.seqs, heads);
    a.units = plan.units;
    const int64_t need = plan.bytes(rows, heads, kv->head_dim);
    if (need > 0 && (!work || (uintptr_t)work % 16 || work_bytes < need))
        return fail(NC_EINVAL, "nc_paged_attention: the workspace is missing, misaligned or too small");
    a.q = q;
    a.k_pages = (const void*)kv->k_pages;
    a.v_pages = (const void*)kv->v_pages;
    a.q_stride = q_stride;
    a.out = out;
    a.heads = heads;
    a.kv_heads = kv->kv_heads;
    a.scale = scale;
    a.slots = plan.slots;
    a.part_o = (float*)work;
    a.part_ml = (float*)work + (need > 0 ? rows * heads * plan.slots * kv->head_dim : 0);
    const int64_t joins = (rows * heads + 3) / 4;
    if (need > 0 && joins > (1 << 23)) return fail(NC_ERANGE, "nc_paged_attention: too many rows and heads");
    DeviceGuard guard(ctx->device);
    if (guard.rc) return guard.rc;
    hipStream_t st = stream ? (hipStream_t)stream : ctx->stream;
    const dim3 grid((unsigned)plan.along, plan.balanced ? 1 : (unsigned)kv->kv_heads,
                    plan.balanced ? 1 : (unsigned)std::min<int64_t>(plan.units, 65535));
    a.balanced = plan.balanced;
    auto launch = [&]<typename A, typename C, int HD>() {
        if constexpr (std::is_same_v<A, float> || std::is_same_v<A, C>) {
            if (plan.one)
                plan.tiles == 1 ? paged_attention_kernel<A, C, HD, 1, true><<<grid, 256, 0, st>>>(a)
                                : paged_attention_kernel<A, C, HD, 2, true><<<grid, 256, 0, st>>>(a);
            else
                plan.tiles == 1 ? paged_attention_kernel<A, C, HD, 1, false><<<grid, 256, 0, st>>>(a)
                                : paged_attention_kernel<A, C, HD, 2, false><<<grid, 256, 0, st>>>(a);
            NC_HIP(hipGetLastError());
            if (plan.slots > 1) {
                paged_join_kernel<A, HD><<<(unsigned)joins, 256, 0, st>>>(a, plan.chunk);
                NC_HIP(hipGetLastError());
            }
        }
        return (int)NC_OK;
    };
    return kv->head_dim == 64 ? with_types<64>(type, kv->elem_type, launch) : with_types<128>(type, kv->elem_type, launch);
}
