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
    float *part_o, *part_ml;  // [row][head][slots][head_dim] and [2] (maximum, sum); null: slots is 1 or all in turn
    int32_t heads, kv_heads, slots;
    float scale;
};

// A sequence's positions in chunks of four waves, 32 KiB of keys and values a wave, or 16.
template <typename C, int HD>
constexpr int kWaveKeys = sizeof(C) == 4 && HD == 128 ? 32 : 64;
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
        l = l * f + l2 * g;
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = o[i] * f + o2[i] * g;
    }
    __device__ __forceinline__ void add_chunk(float mc, float lc, const float* oc) {
        const float top = fmaxf(m, mc), base = exp_base(top);
        add(top, lc, exp2_hw(m - base), exp2_hw(mc - base), oc);
    }
    __device__ __forceinline__ float answer(int i) const { return l == 0.f ? 0.f : o[i] / l; }
};

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
template <typename A, typename C, int HD, int RT>
__global__ __launch_bounds__(256, RT == 1 ? 2 : 1) void paged_attention_kernel(PagedAttnParams a) {
    constexpr bool F32 = sizeof(C) == 4;
    constexpr int KW = kWaveKeys<C, HD>, CH = 4 * KW, KT = KW / 16;
    constexpr bool BF = std::is_same_v<C, __bf16>;
    constexpr int QP = std::is_same_v<A, C> ? 1 : BF ? 3 : 2;  // parts of a query value
    constexpr int PP = BF && QP == 3 ? 3 : 2;                  // parts of a weight
    constexpr bool QSCALE = QP == 2;                           // f16 parts: the row scaled into f16's range
    // f16 weights carry 2^14, which keeps small ones normal numbers and cancels in the answer
    constexpr float PSHIFT = !F32 && !BF ? 14.f : 0.f;
    constexpr int OS = HD + 4;     // LDS row, skewed by four banks
    constexpr int ND = HD / 16;    // dimensions of a thread in the chunk's sum
    __shared__ int64_t s_off[4][KW];
    __shared__ float s_ml[4][RT][16][2];
    __shared__ float s_o[4][RT][16][OS];

    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int G = a.heads / a.kv_heads, groups = gridDim.y / a.kv_heads;
    const int kvh = blockIdx.y % a.kv_heads;
    const int64_t head_off = (int64_t)kvh * a.pool.head_stride;
    const C* kb = (const C*)a.k_pages + head_off;
    const C* vb = (const C*)a.v_pages + head_off;

    for (int s = blockIdx.z; s < a.seqs.seqs; s += gridDim.z) {
        int begin, n;
        seq_rows(a.seqs.row_start, s, a.seqs.rows, begin, n);
        const int32_t* table = a.seqs.table + s * a.seqs.table_stride;
        const int64_t before = (int64_t)a.seqs.lens[s] - n;  // positions before the first new row
        const int64_t R = (int64_t)n * G;
        for (int64_t r0 = (int64_t)(blockIdx.y / a.kv_heads) * (16 * RT); r0 < R; r0 += (int64_t)groups * (16 * RT)) {
            // the positions that a row sees, at most cap of them
            auto seen_of = [&](int64_t row) {
                const int64_t e = before + row / G + 1;
                return (int)(e < 0 ? 0 : e > a.seqs.cap ? a.seqs.cap : e);
            };
            const int64_t last = r0 + 16 * RT < R ? r0 + 16 * RT - 1 : R - 1;
            const int least = seen_of(r0), most = seen_of(last);
            const int chunks = most > 0 ? (most - 1) / CH + 1 : 1;
            if ((int)blockIdx.x >= chunks) continue;

            // queries in operand order: row r of each tile, as many dimensions a lane as a product takes
            int seen[RT];
            float factor[RT];
            constexpr int QN = F32 ? HD / 4 : 1, QV = F32 ? 1 : HD / 32;
            float qf[RT][QN];
            typename Vec8<std::conditional_t<F32, _Float16, C>>::type qv[RT][QP][QV];
#pragma unroll
            for (int t = 0; t < RT; t++) {
                const int64_t row = r0 + 16 * t + r;
                const bool live = row < R;
                const int64_t rr = live ? row : r0;
                seen[t] = live ? seen_of(row) : 0;
                factor[t] = a.scale * kLog2e;
                const A* q = (const A*)a.q + (begin + rr / G) * a.q_stride + (kvh * G + rr % G) * HD;
                if constexpr (F32) {
#pragma unroll
                    for (int j = 0; j < HD / 16; j++) {
                        const f32x4 x = *(const f32x4*)(q + 16 * j + 4 * g);
#pragma unroll
                        for (int e = 0; e < 4; e++) qf[t][4 * j + e] = x[e];
                    }
                } else if constexpr (QP == 1) {
#pragma unroll
                    for (int j = 0; j < QV; j++)
                        qv[t][0][j] = *(const typename Vec8<C>::type*)(q + 32 * j + 8 * g);
                } else {
                    float x[QV][8];
                    float top = 0.f;
#pragma unroll
                    for (int j = 0; j < QV; j++) {
                        load8(q + 32 * j + 8 * g, x[j]);
#pragma unroll
                        for (int e = 0; e < 8; e++) top = fmaxf(top, __builtin_fabsf(x[j][e]));
                    }
                    int shift = 0;
                    if (QSCALE) {  // the row's largest value to [2^9, 2^10)
                        top = fmaxf(top, __shfl_xor(top, 16, 64));
                        top = fmaxf(top, __shfl_xor(top, 32, 64));
                        const int ex = (int)(__float_as_uint(top) >> 23);
                        shift = ex == 0 || ex == 255 ? 0 : 136 - ex;
                        // applied in two steps: 2^shift alone may overflow, and so may its inverse
                        factor[t] = __builtin_ldexpf(factor[t], -shift);
                    }
#pragma unroll
                    for (int j = 0; j < QV; j++)
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            C part[QP];
                            split_parts(QSCALE ? __builtin_ldexpf(x[j][e], shift) : x[j][e], part);
#pragma unroll
                            for (int p = 0; p < QP; p++) qv[t][p][j][e] = part[p];
                        }
                }
            }

            RowSum<ND> sum[RT];  // of row threadIdx.x / 16 and ND dimensions
            for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
                const int base = c * CH + w * KW;
                // every lane finds one key's place; those past the end and of bad pages read the pool's first
                // row, which is there, and count as nothing
                bool none = false;
                if (lane < KW) {
                    const int p = base + lane;
                    int64_t at = p < most ? position_offset(table, a.pool, p) : -1;
                    none = p < most && at < 0;
                    s_off[w][lane] = at;
                }
                const bool masked = base + KW > least || __ballot(none) != 0;
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");

                f32x4 o[RT][ND] = {};
                float m[RT], l[RT];
#pragma unroll
                for (int t = 0; t < RT; t++) m[t] = -__builtin_inff(), l[t] = 0.f;
                if (base < most) {
                    f32x4 sc[RT][KT] = {};
                    auto key_at = [&](int i) {
                        const int64_t at = s_off[w][i];
                        return at < 0 ? (int64_t)0 : at;
                    };
                    auto mask_scores = [&]() {
                        if (!masked) return;
#pragma unroll
                        for (int j = 0; j < KT; j++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const int key = 16 * j + 4 * g + i;
                                const bool bad = s_off[w][key] < 0;
#pragma unroll
                                for (int t = 0; t < RT; t++)
                                    sc[t][j][i] = base + key < seen[t] ? (bad ? __builtin_nanf("") : sc[t][j][i])
                                                                       : -__builtin_inff();
                            }
                    };
                    // scores to weights, in base 2
                    auto weigh = [&]() {
#pragma unroll
                        for (int t = 0; t < RT; t++) {
                            float top = -__builtin_inff();
#pragma unroll
                            for (int j = 0; j < KT; j++)
#pragma unroll
                                for (int i = 0; i < 4; i++) top = fmaxf(top, sc[t][j][i]);
                            top = fmaxf(top, __shfl_xor(top, 16, 64));
                            top = fmaxf(top, __shfl_xor(top, 32, 64));
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
                            total += __shfl_xor(total, 16, 64);
                            total += __shfl_xor(total, 32, 64);
                            m[t] = top;
                            l[t] = total;
                        }
                    };
                    bool odd = false;  // an infinity or NaN among the values of a masked tile
                    if constexpr (F32) {
                        f32x4 kx[KT][HD / 16], vx[KT][4][HD / 64];
#pragma unroll
                        for (int j = 0; j < KT; j++) {
                            const C* k = kb + key_at(16 * j + r) + 4 * g;
#pragma unroll
                            for (int d = 0; d < HD / 16; d++) kx[j][d] = *(const f32x4*)(k + 16 * d);
                        }
#pragma unroll
                        for (int j = 0; j < KT; j++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const C* v = vb + key_at(16 * j + 4 * g + i) + 4 * r;
#pragma unroll
                                for (int h = 0; h < HD / 64; h++) vx[j][i][h] = *(const f32x4*)(v + 64 * h);
                            }
#pragma unroll
                        for (int j = 0; j < KT; j++)
#pragma unroll
                            for (int d = 0; d < HD / 16; d++)
#pragma unroll
                                for (int e = 0; e < 4; e++)
#pragma unroll
                                    for (int t = 0; t < RT; t++)
                                        sc[t][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[j][d][e], qf[t][4 * d + e], sc[t][j], 0, 0, 0);
#pragma unroll
                        for (int t = 0; t < RT; t++)
#pragma unroll
                            for (int j = 0; j < KT; j++) sc[t][j] *= factor[t];
                        mask_scores();
                        weigh();
                        if (masked) {
#pragma unroll
                            for (int j = 0; j < KT; j++)
#pragma unroll
                                for (int i = 0; i < 4; i++) {
                                    const bool gone = s_off[w][16 * j + 4 * g + i] < 0;
#pragma unroll
                                    for (int h = 0; h < HD / 64; h++)
#pragma unroll
                                        for (int e = 0; e < 4; e++) {
                                            const bool bad = !__builtin_isfinite(vx[j][i][h][e]);
                                            odd |= bad && !gone;
                                            if (bad || gone) vx[j][i][h][e] = 0.f;
                                        }
                                }
                        }
#pragma unroll
                        for (int j = 0; j < KT; j++)
#pragma unroll
                            for (int i = 0; i < 4; i++)
#pragma unroll
                                for (int h = 0; h < HD / 64; h++)
#pragma unroll
                                    for (int e = 0; e < 4; e++)
#pragma unroll
                                        for (int t = 0; t < RT; t++)
                                            o[t][4 * h + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(vx[j][i][h][e], sc[t][j][i], o[t][4 * h + e], 0, 0, 0);
                    } else {
                        using V8 = typename Vec8<C>::type;
                        typedef uint32_t VL __attribute__((ext_vector_type(HD / 32)));  // HD / 16 values
                        V8 kx[KT][QV];
                        VL vx[KT / 2][8];
#pragma unroll
                        for (int j = 0; j < KT; j++) {
                            const C* k = kb + key_at(16 * j + r) + 8 * g;
#pragma unroll
                            for (int d = 0; d < QV; d++) kx[j][d] = *(const V8*)(k + 32 * d);
                        }
#pragma unroll
                        for (int b = 0; b < KT / 2; b++)
#pragma unroll
                            for (int i = 0; i < 8; i++)
                                vx[b][i] = *(const VL*)(vb + key_at(32 * b + 16 * (i / 4) + 4 * g + i % 4) + ND * r);
#pragma unroll
                        for (int j = 0; j < KT; j++)
#pragma unroll
                            for (int d = 0; d < QV; d++)
#pragma unroll
                                for (int t = 0; t < RT; t++)
#pragma unroll
                                    for (int p = QP - 1; p >= 0; p--) sc[t][j] = mfma16(kx[j][d], qv[t][p][d], sc[t][j]);
#pragma unroll
                        for (int t = 0; t < RT; t++)
#pragma unroll
                            for (int j = 0; j < KT; j++) sc[t][j] *= factor[t];
                        mask_scores();
                        weigh();
                        if (masked) {
                            constexpr uint32_t EXP = BF ? 0x7f80u : 0x7c00u;
#pragma unroll
                            for (int b = 0; b < KT / 2; b++)
#pragma unroll
                                for (int i = 0; i < 8; i++) {
                                    const bool gone = s_off[w][32 * b + 16 * (i / 4) + 4 * g + i % 4] < 0;
#pragma unroll
                                    for (int d = 0; d < HD / 32; d++) {
                                        const uint32_t x = vx[b][i][d];
                                        const bool lo = (x & EXP) == EXP, hi = (x >> 16 & EXP) == EXP;
                                        odd |= (lo || hi) && !gone;
                                        vx[b][i][d] = gone ? 0u : (lo ? 0u : x & 0xffffu) | (hi ? 0u : x & 0xffff0000u);
                                    }
                                }
                        }
#pragma unroll
                        for (int b = 0; b < KT / 2; b++) {
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
                                    x[i] = __builtin_amdgcn_perm(vx[b][2 * i + 1][e / 2], vx[b][2 * i][e / 2],
                                                                 e % 2 ? 0x07060302u : 0x05040100u);
                                const V8 vt = __builtin_bit_cast(V8, x);
#pragma unroll
                                for (int t = 0; t < RT; t++)
#pragma unroll
                                    for (int p = PP - 1; p >= 0; p--) o[t][e] = mfma16(vt, pv[t][p], o[t][e]);
                            }
                        }
                    }
                    // A zero weight times an infinity is no zero: in masked tiles such values were left out, and go
                    // to the rows that see their key here.
                    if (__ballot(odd)) {
                        for (int key = 0; key < KW; key++) {
                            const int64_t at = s_off[w][key];
                            if (at < 0) continue;
#pragma unroll
                            for (int e = 0; e < ND; e++)
#pragma unroll
                                for (int i = 0; i < 4; i++) {
                                    const int d = F32 ? 64 * (e / 4) + 16 * g + 4 * i + e % 4 : ND * (4 * g + i) + e;
                                    const float v = (float)vb[at + d];
                                    if (!__builtin_isfinite(v))
#pragma unroll
                                        for (int t = 0; t < RT; t++)
                                            if (base + key < seen[t]) o[t][e][i] += v;
                                }
                        }
                    }
                }

                // the four waves' sums to one, in their order
#pragma unroll
                for (int t = 0; t < RT; t++)
                    if (g == 0) s_ml[w][t][r][0] = m[t], s_ml[w][t][r][1] = l[t];
                __syncthreads();
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    float top = s_ml[0][t][r][0];
#pragma unroll
                    for (int i = 1; i < 4; i++) top = fmaxf(top, s_ml[i][t][r][0]);
                    const float f = exp2_hw(m[t] - exp_base(top));
#pragma unroll
                    for (int e = 0; e < ND; e += 4)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int d = F32 ? 16 * e + 16 * g + 4 * i : ND * (4 * g + i) + e;
                            *(f32x4*)&s_o[w][t][r][d] = f32x4{o[t][e][i], o[t][e + 1][i], o[t][e + 2][i], o[t][e + 3][i]} * f;
                        }
                }
                __syncthreads();
                const int row16 = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * ND;
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    float top = s_ml[0][t][row16][0];
#pragma unroll
                    for (int i = 1; i < 4; i++) top = fmaxf(top, s_ml[i][t][row16][0]);
                    const float lift = exp_base(top);
                    float lc = 0.f, oc[ND] = {};
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        lc += s_ml[i][t][row16][1] * exp2_hw(s_ml[i][t][row16][0] - lift);
#pragma unroll
                        for (int d = 0; d < ND; d++) oc[d] += s_o[i][t][row16][d0 + d];
                    }
                    const int64_t row = r0 + 16 * t + row16;
                    if (row >= R) continue;
                    const int64_t unit = (begin + row / G) * a.heads + kvh * G + row % G;
                    const int mine = seen_of(row), own = mine > 0 ? (mine - 1) / CH + 1 : 1;
                    if (c < own) sum[t].add_chunk(top, lc, oc);
                    if (gridDim.x > 1 && own > 1) {
                        if (c < own) {
                            const int64_t at = unit * a.slots + c;
                            a.part_ml[2 * at] = top;
                            a.part_ml[2 * at + 1] = lc;
#pragma unroll
                            for (int d = 0; d < ND; d++) a.part_o[at * HD + d0 + d] = oc[d];
                        }
                    } else if (c == own - 1) {
                        const bool past = before + row / G + 1 > a.seqs.cap;
                        A* out = (A*)a.out + unit * HD + d0;
#pragma unroll
                        for (int d = 0; d < ND; d++) out[d] = (A)(past ? __builtin_nanf("") : sum[t].answer(d));
                    }
                }
                __syncthreads();
            }
        }
    }
}

// The chunks of one (row, head) by a wave, a few dimensions a lane.  The running maxima, which only compare, come
// from a scan over the lanes, 64 chunks at a time, so that the chunks' loads do not wait for each other.
template <typename A, int HD>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnParams a, int chunk) {
    constexpr int ND = HD / 64;
    const int lane = threadIdx.x & 63;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (unit >= (int64_t)a.seqs.rows * a.heads) return;
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
    const float* ml = a.part_ml + unit * a.slots * 2;
    const float* o = a.part_o + unit * a.slots * HD + ND * lane;
    RowSum<ND> sum;
    for (int c0 = 0; c0 < chunks; c0 += 64) {
        const int c = c0 + lane, count = chunks - c0 < 64 ? chunks - c0 : 64;
        const float mc = c < chunks ? ml[2 * c] : -__builtin_inff(), lc = c < chunks ? ml[2 * c + 1] : 0.f;
        float top = fmaxf(mc, sum.m);  // the largest score up to this chunk
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const float x = __shfl_up(top, d, 64);
            if (lane >= d) top = fmaxf(top, x);
        }
        float prev = __shfl_up(top, 1, 64);
        if (lane == 0) prev = sum.m;
        const float base = exp_base(top), f = exp2_hw(prev - base), g = exp2_hw(mc - base);
        for (int i = 0; i < count; i += 8) {
            float x[8][ND];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int cc = i + j < count ? i + j : count - 1;
#pragma unroll
                for (int d = 0; d < ND; d++) x[j][d] = o[(int64_t)(c0 + cc) * HD + d];
            }
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (i + j < count)
                    sum.add(__shfl(top, i + j, 64), __shfl(lc, i + j, 64), __shfl(f, i + j, 64), __shfl(g, i + j, 64), x[j]);
        }
    }
    A* out = (A*)a.out + unit * HD + ND * lane;
#pragma unroll
    for (int d = 0; d < ND; d++) out[d] = (A)(seen64 > a.seqs.cap ? __builtin_nanf("") : sum.answer(d));
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

// How a call is launched: tiles of 16 rows a workgroup, workgroups along the row groups of a sequence and along
// its chunks, and chunk slots of a row's partial sums (1: none are kept).
struct AttnPlan {
    int tiles = 1, chunk = 256, slots = 1, along = 1;
    int64_t groups = 1;
    int64_t bytes(int64_t rows, int heads, int hd) const { return slots > 1 ? rows * heads * slots * (hd + 2) * 4 : 0; }
};

int plan_attention(const nc_paged_kv& kv, const PagedSeqs& s, int heads, AttnPlan& p) {
    const int64_t group = heads / kv.kv_heads;
    p.chunk = kv.elem_type == NC_TYPE_F32 && kv.head_dim == 128 ? 128 : 256;
    // rows of an average sequence, rounded up, decide the tiles: one where they fit one
    const int64_t rows = s.seqs > 0 ? ((int64_t)s.rows + s.seqs - 1) / s.seqs * group : 1;
    p.tiles = rows <= 16 ? 1 : 2;
    // One sequence may hold nearly all rows: up to all row groups a sequence, as long as the launch stays within
    // some 8192 workgroups or twice what the rows fill (those without rows end at once; the others loop).
    const int64_t all = std::max<int64_t>(((int64_t)s.rows * group + 16 * p.tiles - 1) / (16 * p.tiles), 1);
    const int64_t average = (rows + 16 * p.tiles - 1) / (16 * p.tiles);
    p.groups = !s.row_start ? average : std::min(all, std::max(2 * average, 8192 / ((int64_t)kv.kv_heads * std::max(s.seqs, 1)) + 1));
    const int64_t chunks = std::max<int64_t>(((int64_t)s.cap + p.chunk - 1) / p.chunk, 1);
    // units of work without a split along the positions; from 8 a CU on the chip is full without one
    const int64_t units = kv.kv_heads * std::max<int64_t>(s.seqs, all);
    if (chunks > 1 && units < 2048) {
        p.slots = (int)std::min<int64_t>(chunks, INT32_MAX);
        p.along = (int)std::min<int64_t>(chunks, std::max<int64_t>(2, 16384 / units));
    }
    if (p.groups * kv.kv_heads > 65535) p.groups = std::max<int64_t>(1, 65535 / kv.kv_heads);
    return NC_OK;
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
    AttnPlan plan;
    plan_attention(*kv, s, heads, plan);
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
    if (rows == 0 || batch->seqs == 0) return NC_OK;
    if (!q || !out) return fail(NC_EINVAL, "nc_paged_attention: null argument");
    if (bad_rows(q, q_stride, (int64_t)heads * kv->head_dim, size) || (uintptr_t)out % 16)
        return fail(NC_EINVAL, "nc_paged_attention: rows must be 16-byte aligned and not overlap");
    AttnPlan plan;
    plan_attention(*kv, a.seqs, heads, plan);
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
    if (need > 0 && joins > (1 << 24)) return fail(NC_ERANGE, "nc_paged_attention: too many rows and heads");
    DeviceGuard guard(ctx->device);
    if (guard.rc) return guard.rc;
    hipStream_t st = stream ? (hipStream_t)stream : ctx->stream;
    const dim3 grid((unsigned)plan.along, (unsigned)(plan.groups * kv->kv_heads), (unsigned)std::min(batch->seqs, 65535));
    auto launch = [&]<typename A, typename C, int HD>() {
        if constexpr (std::is_same_v<A, float> || std::is_same_v<A, C>) {
            if (plan.tiles == 1)
                paged_attention_kernel<A, C, HD, 1><<<grid, 256, 0, st>>>(a);
            else
                paged_attention_kernel<A, C, HD, 2><<<grid, 256, 0, st>>>(a);
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
