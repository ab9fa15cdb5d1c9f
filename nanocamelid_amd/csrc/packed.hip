// Causal attention over packed whole prompts: sequences of different lengths end to end in one tensor of
// rows, query heads in groups that share a key-value head.  Row i of a sequence with n query rows and m key
// rows sees its keys 0 .. m - n + i.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "nc_internal.h"
#include "nc_paged.h"

namespace nc {

struct PackedParams {
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    void* out;
    const int32_t *seq_start, *kv_start;
    int32_t seqs, rows, kv_rows, heads, kv_heads;
    int32_t together;  // heads of a workgroup: 4, 2 or 1, as many as divide a group
    float scale;
};

__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

constexpr int kPackedRows = 32;  // query rows of a wave

// The power of two that takes the float of these bits to [2^14, 2^15): the two f16 parts of such a value hold 24
// bits down to 2^-16 of it, and sums of their products are far from infinite.  0 for zero and what is not finite.
__device__ __forceinline__ int shift_of(uint32_t bits) {
    const int ex = (int)(bits >> 23) & 255;
    return ex == 0 || ex == 255 ? 0 : 141 - ex;
}
constexpr uint32_t kInfBits = 0x7f800000u;

// Four keys' values of one dimension: the 16 lanes of a group read four rows of 16 dimensions, eight bytes each,
// and get a column back.
template <typename V4>
__device__ __forceinline__ V4 read_columns(const void* p) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    auto q = (__attribute__((address_space(3))) s16x4*)(p);
    return __builtin_bit_cast(V4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(q));
}

// Attention of 32 query rows of four heads that share a kv head (or 64 of two, 128 of one) over their sequence's
// keys, a tile of keys at a time with a running maximum and sum.  Four heads together end their keys at one place,
// which wastes less of the last tiles than four blocks of rows.
//
// Bound by the matrix products (4 head_dim operations a row and key) and, close behind, by the vector work of
// the softmax.  Everything is transposed: scores^T = K q^T leaves a lane 16 scores of its own row for every 32
// keys, and out^T = V^T p^T takes its weights from just there if its inner index counts the keys in that order,
// so weights never cross lanes.  Keys and values go through LDS, shared by the four waves; rows of 16-byte pieces
// whose order is turned by the row, so that the reads of both products are free of bank conflicts.  The next
// tile's loads are in flight during a tile's products.
//   16 bits: values are read as columns by the transposing LDS read, weights are rounded to the operands' type
//   (as much as the answer's own rounding).
//   f32: keys, values, queries and weights as two f16 parts (nc_paged.h), of whose products the smallest is left
//   out, below 2^-24 of |q||k|.  Parts hold a value's 24 bits down to 2^-16 of what it is scaled by: a row of
//   queries by its largest, a tile's keys by theirs, values by the largest so far, in powers of two that the
//   scores' factor and the answer give back.  The f32 products of the matrix cores run at a sixteenth of the f16
//   rate, these at a third.  Where keys or values of a tile differ in size by more (a huge one that only later rows
//   see, say), or one is not finite, the tile takes the f32 products.
//
// Measured, 32 heads over 8: 8192 rows of 128 dimensions in bf16 630 to 646 us, 850 to 870 TFLOP/s (a large product
// 1039); 4096 rows in f32 462 us, 297 TFLOP/s, of three times as many f16 ones (with f32 products 1159 us, at 118;
// their peak rate would need 938); 24 prompts of up to 700 rows of 64 dimensions in f16 47 us, 350 TFLOP/s: half the
// dimensions have half the products for the same softmax.  A fourth wave a SIMD, of 128 registers, spills: 110 us.
template <typename A, int HD, int NW>
__global__ __launch_bounds__(64 * NW, NW == 8 ? 2 : HD == 64 && sizeof(A) == 2 ? 3 : 2) void packed_attention_kernel(PackedParams a, int64_t units) {
    constexpr bool F32 = sizeof(A) == 4;
    using E = std::conditional_t<F32, _Float16, A>;
    using V8 = typename Vec8<E>::type;
    typedef E V4 __attribute__((ext_vector_type(4)));
    constexpr int NP = F32 ? 2 : 1;        // parts of a value
    constexpr float PSHIFT = F32 ? 14.f : 0.f;  // keeps the parts of small weights normal numbers, cancels in the answer
    constexpr int BN = F32 ? 32 : 64;      // keys of a tile
    constexpr int NB = F32 ? 1 : 2;        // LDS buffers
    constexpr int PC = HD / 8;             // 16-byte pieces of an LDS row
    constexpr int NL = BN * PC / (64 * NW);  // pieces of a tile that a thread moves
    constexpr int KB = BN / 32, DT = HD / 32, KK = HD / 16;
    __shared__ __attribute__((aligned(16))) E s_k[NB][NP][BN][HD], s_v[NB][NP][BN][HD];
    __shared__ int s_odd[2];  // by the tile's parity: the tile (from 1) of whose values some were left out
    __shared__ __attribute__((aligned(16))) uint32_t s_size[NW][4];  // f32: of the next tile's keys and values that a wave moves

    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, r = lane & 31, h = lane >> 5;
    const int G = a.heads / a.kv_heads;
    const float sign = a.scale > 0.f ? 1.f : a.scale < 0.f ? -1.f : a.scale == 0.f ? 0.f : a.scale;
    const float c = a.scale == 0.f ? 1.f : __builtin_fabsf(a.scale) * kLog2e;  // scores to base 2, positive

    for (int64_t b = blockIdx.x; b < units; b += gridDim.x) {
        // the kv heads first, so that one head's workgroups share an XCD's L2
        const int kvh = (int)(b % a.kv_heads), groups = G / a.together;
        const int head = kvh * G + (int)(b / a.kv_heads % groups) * a.together + w % a.together;
        const int high = NW / a.together * kPackedRows;  // rows of the workgroup
        int64_t tile = b / a.kv_heads / groups;
        // Its sequence: tiles of 64 sequences at a time, of them those that see the most first, which keeps the last
        // ones to run short (six prompts of up to 1200 rows, 24 heads over 8: 177 us against 220 sequence by sequence;
        // 24 of up to 700, 16 bits: 46.5 against 48.7).  A tile is the rank-th among the sequences that have a level of it.
        int s = -1, q0 = 0, begin = 0, n = 0;
        for (int s0 = 0; s0 < a.seqs; s0 += 64) {
            int mb = 0, mn = 0;
            if (s0 + lane < a.seqs) seq_rows(a.seq_start, s0 + lane, a.rows, mb, mn);
            const int levels = (mn + high - 1) / high;
            const int all = wave_sum(levels);
            if (tile < all) {
                // the highest level that it and those above have more tiles than `tile`
                int level = 0, over = (int)wave_max((uint32_t)levels), above = 0;
                while (over - level > 1) {
                    const int mid = (level + over) / 2, x = wave_sum(levels > mid ? levels - mid : 0);
                    if (x > tile) level = mid;
                    else over = mid, above = x;
                }
                const uint64_t with = __ballot(levels > level);
                const int rank = __builtin_popcountll(with & ((1ull << lane) - 1));
                const int at = __builtin_ctzll(__ballot(levels > level && rank == (int)tile - above)) & 63;
                s = s0 + at;
                begin = __builtin_amdgcn_readlane(mb, at);
                n = __builtin_amdgcn_readlane(mn, at);
                q0 = level * high;
                break;
            }
            tile -= all;
        }
        if (s < 0) return;  // past the last tile, and so is every later one
        s = __builtin_amdgcn_readfirstlane(s);
        q0 = __builtin_amdgcn_readfirstlane(q0);
        int kbegin, m;
        seq_rows(a.kv_start, s, a.kv_rows, kbegin, m);

        // rows past the sequence's end take the last one's place and are not written
        const int first = q0 + w / a.together * kPackedRows;  // of the wave
        const int row = first + r < n ? first + r : n - 1;
        const int before = m - n;  // may be negative
        const int seen = before + row + 1;
        const int wave_most = before + (first + 31 < n ? first + 31 : n - 1) + 1;  // keys that some row of the wave sees
        const int wave_least = before + (first < n ? first : n - 1) + 1;           // that every row sees
        const int most = before + (q0 + high - 1 < n ? q0 + high - 1 : n - 1) + 1;
        const int tiles = most > 0 ? (most + BN - 1) / BN : 0;
        const A* q = (const A*)a.q + (int64_t)(begin + row) * a.q_stride + head * HD;
        const A* kb = (const A*)a.k + (int64_t)kbegin * a.k_stride + kvh * HD;
        const A* vb = (const A*)a.v + (int64_t)kbegin * a.v_stride + kvh * HD;

        V8 qv[NP][KK];
        int qshift = 0;  // f32: the row of queries is scaled by 2^qshift
        if constexpr (F32) {
            float x[KK][8], top = 0.f;
#pragma unroll
            for (int d = 0; d < KK; d++) {
                load8(q + 16 * d + 8 * h, x[d]);
#pragma unroll
                for (int e = 0; e < 8; e++) top = fmaxf(top, __builtin_fabsf(x[d][e]));
            }
            top = max_across<32>(top);
            qshift = shift_of(__float_as_uint(top));
#pragma unroll
            for (int d = 0; d < KK; d++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    E part[NP];
                    split_parts(__builtin_ldexpf(x[d][e] * sign, qshift), part);
#pragma unroll
                    for (int p = 0; p < NP; p++) qv[p][d][e] = part[p];
                }
        } else {
#pragma unroll
            for (int d = 0; d < KK; d++) {
                float x[8];
                load8(q + 16 * d + 8 * h, x);
#pragma unroll
                for (int e = 0; e < 8; e++) qv[0][d][e] = (E)(x[e] * sign);
            }
        }

        // a thread's pieces of the next tile, as they lie in memory
        typedef A Raw __attribute__((ext_vector_type(8)));
        Raw kx[NL], vx[NL];
        auto load_tile = [&](int t) {
#pragma unroll
            for (int i = 0; i < NL; i++) {
                const int id = tid + 64 * NW * i, key = t * BN + id / PC;
                const int64_t at = key < most ? key : most - 1;
                kx[i] = *(const Raw*)(kb + at * a.k_stride + id % PC * 8);
                vx[i] = *(const Raw*)(vb + at * a.v_stride + id % PC * 8);
            }
        };
        f32x16 o[DT] = {};
        // f32: keys are scaled by 2^kshift, a tile's own, values by 2^vshift, that of the largest so far (1000: none but
        // zeros yet).  A rough tile is one that f16 parts cannot hold together.
        int kshift = 0, vshift = 1000;
        bool rough = false;
        // A zero weight times a value that is not finite is no zero: such values are left out of the product, f32 ones
        // always, 16-bit ones where rows mask keys.
        auto leave_out = [&](int t) {
            bool any = false;
#pragma unroll
            for (int i = 0; i < NL; i++)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (!__builtin_isfinite((float)vx[i][e])) {
                        vx[i][e] = (A)0.f;
                        any = true;
                    }
            if (any) s_odd[t & 1] = t + 1;
        };
        auto look_through = [&](int t) {
            if constexpr (F32) {
                // the largest of every key's and value's dimensions, as bits, which order as the sizes do, infinities
                // and NaN last; of them the wave's largest, and its smallest but zero
                uint32_t km[NL], vm[NL];
                auto sizes = [&]() {
#pragma unroll
                    for (int i = 0; i < NL; i++) {
                        km[i] = vm[i] = 0;
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const uint32_t x = __float_as_uint(kx[i][e]) & 0x7fffffffu, y = __float_as_uint(vx[i][e]) & 0x7fffffffu;
                            km[i] = km[i] > x ? km[i] : x;
                            vm[i] = vm[i] > y ? vm[i] : y;
                        }
                        km[i] = group_max<PC>(km[i]);
                        vm[i] = group_max<PC>(vm[i]);
                    }
                };
                sizes();
                uint32_t big = 0;
#pragma unroll
                for (int i = 0; i < NL; i++) big = big > vm[i] ? big : vm[i];
                if (__ballot(big >= kInfBits)) {
                    leave_out(t);
                    sizes();
                }
                uint32_t kt = 0, vt = 0, kl = ~0u, vl = ~0u;
#pragma unroll
                for (int i = 0; i < NL; i++) {
                    kt = kt > km[i] ? kt : km[i];
                    vt = vt > vm[i] ? vt : vm[i];
                    if (lane % PC == PC - 1) {  // where the group's maximum is
                        kl = km[i] != 0 && km[i] < kl ? km[i] : kl;
                        vl = vm[i] != 0 && vm[i] < vl ? vm[i] : vl;
                    }
                }
                // a smallest is the largest of the complements; both end in the wave's last lane
                kt = wave_max_of_groups<PC>(kt);
                vt = wave_max_of_groups<PC>(vt);
                kl = ~wave_max_of_groups<PC>(~kl);
                vl = ~wave_max_of_groups<PC>(~vl);
                if (lane == 63) *(u32x4*)s_size[w] = u32x4{kt, vt, kl, vl};
            } else if ((t + 1) * BN > before + q0 + 1) {
                float odd = 0.f;  // NaN if there is one
#pragma unroll
                for (int i = 0; i < NL; i++)
#pragma unroll
                    for (int e = 0; e < 8; e++) odd = __builtin_fmaf((float)vx[i][e], 0.f, odd);
                if (__ballot(odd != odd)) leave_out(t);
            }
        };
        auto store_tile = [&](int t) {
            const int buf = NB == 2 ? t & 1 : 0;
            if constexpr (F32) {
                u32x4 size = *(const u32x4*)s_size[0];
#pragma unroll
                for (int i = 1; i < NW; i++) {
                    const u32x4 x = *(const u32x4*)s_size[i];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        size[e] = x[e] > size[e] ? x[e] : size[e];
                        size[2 + e] = x[2 + e] < size[2 + e] ? x[2 + e] : size[2 + e];
                    }
                }
                // one key or value 2^16 times another, or a key that is not finite
                rough = size[0] >= kInfBits || (size[0] != 0 && (size[0] >> 23) - (size[2] >> 23) > 16) ||
                        (size[1] != 0 && (size[1] >> 23) - (size[3] >> 23) > 16);
                kshift = shift_of(size[0]);
                if (size[1] != 0) {
                    const int vs = shift_of(size[1]);
                    if (vs > vshift + 16) {
                        rough = true;  // all far below what came before
                    } else if (vs < vshift) {
                        if (vshift != 1000)
#pragma unroll
                            for (int d = 0; d < DT; d++)
#pragma unroll
                                for (int i = 0; i < 16; i++) o[d][i] = __builtin_ldexpf(o[d][i], vs - vshift);
                        vshift = vs;
                    }
                }
                if (rough) {
                    // the tile as it is, in the same place
#pragma unroll
                    for (int i = 0; i < NL; i++) {
                        const int at = (tid + 64 * NW * i) * 8;
                        *(Raw*)((float*)s_k + at) = kx[i];
                        *(Raw*)((float*)s_v + at) = vx[i];
                    }
                    return;
                }
            }
#pragma unroll
            for (int i = 0; i < NL; i++) {
                const int id = tid + 64 * NW * i, key = id / PC, piece = id % PC;
                const int pk = (piece ^ (key & (PC - 1))) * 8, pv = (piece ^ (2 * key & (PC - 1))) * 8;
                if constexpr (F32) {
                    V8 kp[NP], vp[NP];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        E part[NP];
                        split_finite(__builtin_ldexpf(kx[i][e], kshift), part);
#pragma unroll
                        for (int p = 0; p < NP; p++) kp[p][e] = part[p];
                        split_finite(__builtin_ldexpf(vx[i][e], vshift), part);
#pragma unroll
                        for (int p = 0; p < NP; p++) vp[p][e] = part[p];
                    }
#pragma unroll
                    for (int p = 0; p < NP; p++) {
                        *(V8*)&s_k[buf][p][key][pk] = kp[p];
                        *(V8*)&s_v[buf][p][key][pv] = vp[p];
                    }
                } else {
                    *(Raw*)&s_k[buf][0][key][pk] = kx[i];
                    *(Raw*)&s_v[buf][0][key][pv] = vx[i];
                }
            }
        };

        float top = -__builtin_inff(), l = 0.f;  // of the row; l of the lane's own keys
        if (tid < 2) s_odd[tid] = 0;
        if (tiles > 0) load_tile(0);
        __syncthreads();
        if (tiles > 0) {
            look_through(0);
            if (F32) __syncthreads();
            store_tile(0);
            if (tiles > 1) load_tile(1);
        }
        for (int t = 0; t < tiles; t++) {
            const int buf = NB == 2 ? t & 1 : 0;
            __syncthreads();
            const int base = t * BN;
            if (base < wave_most) {
                f32x16 sc[KB] = {};
                __builtin_amdgcn_s_setprio(1);
                if (F32 && rough) {
                    const float* f = (const float*)s_k + (r * HD + kept_here(h));
#pragma unroll 4
                    for (int d = 0; d < HD; d += 2) sc[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(f[d], (float)q[d + h] * sign, sc[0], 0, 0, 0);
                } else {
#pragma unroll
                    for (int d = 0; d < KK; d++)
#pragma unroll
                        for (int j = 0; j < KB; j++) {
                            const int key = 32 * j + r;
                            V8 kv[NP];
#pragma unroll
                            for (int p = 0; p < NP; p++) kv[p] = *(const V8*)&s_k[buf][p][key][((2 * d + h) ^ (key & (PC - 1))) * 8];
#pragma unroll
                            for (int p = NP - 1; p >= 0; p--)  // the smallest products first
#pragma unroll
                                for (int p2 = NP - 1 - p; p2 >= 0; p2--) sc[j] = mfma32(kv[p], qv[p2][d], sc[j]);
                        }
                }
                __builtin_amdgcn_s_setprio(0);
                if (base + BN > wave_least) {
                    const int own = kept_here(seen - base - 4 * h);  // a branch, not selects in every tile
#pragma unroll
                    for (int j = 0; j < KB; j++)
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            if (32 * j + 8 * (i / 4) + i % 4 >= own) sc[j][i] = -__builtin_inff();
                }
                // kept from 0 and infinity, so that -inf times it stays what it is
                const float to_base2 = !F32 || rough ? c : fminf(fmaxf(__builtin_ldexpf(c, -qshift - kshift), 0x1p-126f), 0x1p127f);
                float next = -__builtin_inff();
#pragma unroll
                for (int j = 0; j < KB; j++)
#pragma unroll
                    for (int i = 0; i < 16; i++) next = fmaxf(next, sc[j][i]);
                next = max_across<32>(next) * to_base2;
                if (__ballot(next > top)) {
                    next = fmaxf(next, top);
                    const float keep = exp2_hw(top - exp_base(next));
                    l *= keep;
#pragma unroll
                    for (int d = 0; d < DT; d++) o[d] *= keep;
                    top = next;
                }
                const float lift = exp_base(top) - PSHIFT;
#pragma unroll
                for (int j = 0; j < KB; j++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        sc[j][i] = exp2_hw(__builtin_fmaf(sc[j][i], to_base2, -lift));
                        l += sc[j][i];
                    }
                if (F32 && rough) {
                    const float* f = (const float*)s_v + (kept_here(4 * h) * HD + r);
#pragma unroll
                    for (int i = 0; i < 16; i++)
#pragma unroll
                        for (int d = 0; d < DT; d++)
                            o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(__builtin_ldexpf(f[(8 * (i / 4) + i % 4) * HD + 32 * d], vshift), sc[0][i], o[d], 0, 0, 0);
                } else {
#pragma unroll
                    for (int j = 0; j < KB; j++)
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            V8 pv[NP];
                            __builtin_amdgcn_s_setprio(1);
#pragma unroll
                            for (int e = 0; e < 8; e++) {
                                E part[NP];
                                split_finite(sc[j][8 * u + e], part);
#pragma unroll
                                for (int p = 0; p < NP; p++) pv[p][e] = part[p];
                            }
                            const int i = lane & 15, key = 32 * j + 16 * u + 4 * h + i / 4;
#pragma unroll
                            for (int d = 0; d < DT; d++) {
                                const int piece = 4 * d + 2 * (lane >> 4 & 1) + (i >> 1 & 1);
                                V8 vt[NP];
#pragma unroll
                                for (int p = 0; p < NP; p++) {
                                    const V4 lo = read_columns<V4>(&s_v[buf][p][key][(piece ^ (2 * key & (PC - 1))) * 8 + 4 * (i & 1)]);
                                    const V4 hi = read_columns<V4>(&s_v[buf][p][key + 8][(piece ^ (2 * (key + 8) & (PC - 1))) * 8 + 4 * (i & 1)]);
                                    vt[p] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                                }
#pragma unroll
                                for (int p = NP - 1; p >= 0; p--)
#pragma unroll
                                    for (int p2 = NP - 1 - p; p2 >= 0; p2--) o[d] = mfma32(vt[p], pv[p2], o[d]);
                            }
                        }
                }
                __builtin_amdgcn_s_setprio(0);
                if (s_odd[t & 1] == t + 1) {
                    // what was left out of the values, to the rows that see it
                    const int h4 = kept_here(4 * h);
                    for (int key = base; key < base + BN; key++)
                        if (key < seen)
#pragma unroll
                            for (int d = 0; d < DT; d++)
#pragma unroll
                                for (int i = 0; i < 16; i++) {
                                    const float x = (float)vb[(int64_t)key * a.v_stride + 32 * d + 8 * (i / 4) + h4 + i % 4];
                                    if (!__builtin_isfinite(x)) o[d][i] += x;
                                }
                }
            }
            if (t + 1 < tiles) {
                look_through(t + 1);
                if (NB == 1) __syncthreads();
                store_tile(t + 1);
                if (t + 2 < tiles) load_tile(t + 2);
            }
        }
        l = sum_across<32>(l);
        if (first + r < n) {
            const float inv = 1.f / l;
            A* out = (A*)a.out + ((int64_t)(begin + row) * a.heads + head) * HD + 4 * h;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    typedef A Out __attribute__((ext_vector_type(4)));
                    Out x;
#pragma unroll
                    for (int e = 0; e < 4; e++) x[e] = (A)(l == 0.f ? 0.f : F32 ? __builtin_ldexpf(o[d][i + e] * inv, -vshift) : o[d][i + e] * inv);
                    *(Out*)(out + 32 * d + 2 * i) = x;
                }
        }
        __syncthreads();
    }
}

}  // namespace nc

using namespace nc;

extern "C" int nc_packed_attention(nc_ctx* ctx, int type, int64_t rows, int64_t kv_rows, const void* q, int64_t q_stride,
                                   const void* k, int64_t k_stride, const void* v, int64_t v_stride, int32_t heads,
                                   int32_t kv_heads, int32_t head_dim, const int32_t* seq_start,
                                   const int32_t* kv_start, int32_t seqs, float scale, void* out, void* stream) {
    if (!ctx) return fail(NC_EINVAL, "nc_packed_attention: null argument");
    const int size = type == NC_TYPE_F32 ? 4 : type == NC_TYPE_F16 || type == NC_TYPE_BF16 ? 2 : 0;
    if (!size) return fail(NC_EINVAL, "nc_packed_attention: the rows' type must be F32, F16 or BF16");
    if (head_dim != 64 && head_dim != 128) return fail(NC_EINVAL, "nc_packed_attention: head_dim must be 64 or 128");
    if (kv_heads < 1 || heads < 1 || heads % kv_heads || heads > 65535)
        return fail(NC_EINVAL, "nc_packed_attention: heads must be a multiple of kv_heads, at most 65535");
    if (rows < 0 || kv_rows < 0 || seqs < 0 || rows > INT32_MAX - 512 || kv_rows > INT32_MAX - 512 || seqs > INT32_MAX - 512)
        return fail(NC_ERANGE, "nc_packed_attention: bad number of rows or sequences");
    if (rows == 0 || seqs == 0) return NC_OK;
    if (!q || !out || !seq_start || (kv_rows > 0 && (!k || !v))) return fail(NC_EINVAL, "nc_packed_attention: null argument");
    if (!kv_start && kv_rows != rows)
        return fail(NC_EINVAL, "nc_packed_attention: without key starts there are as many key rows as query rows");
    const int64_t qw = (int64_t)heads * head_dim, kw = (int64_t)kv_heads * head_dim;
    const void* ptr[3] = {q, k, v};
    const int64_t stride[3] = {q_stride, k_stride, v_stride}, width[3] = {qw, kw, kw};
    for (int i = 0; i < 3; i++)
        if ((uintptr_t)ptr[i] % 16 || stride[i] < width[i] || stride[i] > (INT64_MAX >> 34) || stride[i] * size % 16)
            return fail(NC_EINVAL, "nc_packed_attention: rows must be 16-byte aligned and not overlap");
    if ((uintptr_t)out % 16 || (uintptr_t)seq_start % 4 || (uintptr_t)kv_start % 4)
        return fail(NC_EINVAL, "nc_packed_attention: misaligned output or starts");
    if (out == q || out == k || out == v) return fail(NC_EINVAL, "nc_packed_attention: the output must not be one of the inputs");
    PackedParams a = {q, k, v, q_stride, k_stride, v_stride, out, seq_start, kv_start ? kv_start : seq_start, seqs,
                      (int32_t)rows, (int32_t)kv_rows, heads, kv_heads, 1, scale};
    DeviceGuard guard(ctx->device);
    if (guard.rc) return guard.rc;
    hipStream_t st = stream ? (hipStream_t)stream : ctx->stream;
    const int group = heads / kv_heads;
    a.together = group % 4 == 0 ? 4 : group % 2 == 0 ? 2 : 1;
    // at most a tile more than its rows fill for every sequence; those past the last tile end at once
    auto launch = [&]<typename A, int HD, int NW>() {
        const int64_t units = (rows / (NW / a.together * kPackedRows) + seqs) * (heads / a.together);
        packed_attention_kernel<A, HD, NW><<<(unsigned)std::min<int64_t>(units, 1 << 22), 64 * NW, 0, st>>>(a, units);
        NC_HIP(hipGetLastError());
        return (int)NC_OK;
    };
    if (type == NC_TYPE_F16) return head_dim == 64 ? launch.template operator()<_Float16, 64, 4>() : launch.template operator()<_Float16, 128, 4>();
    if (type == NC_TYPE_BF16) return head_dim == 64 ? launch.template operator()<__bf16, 64, 4>() : launch.template operator()<__bf16, 128, 4>();
    if (head_dim == 64) return launch.template operator()<float, 64, 4>();
    // Eight waves share the splitting of a tile, a third of a wave's vector work, as long as that does not take more
    // than 64 rows of a sequence together (4096 rows, 32 heads over 8: 462 us with eight, 512 with four; six prompts
    // of up to 1200 rows, 24 heads over 8: 232 and 218, both before their order).
    return a.together == 4 ? launch.template operator()<float, 128, 8>() : launch.template operator()<float, 128, 4>();
}
