// What the paged-cache operators (paged.hip, packed.hip) share: where a row stands, where a position
// lies, and how values of the three element types are read and written.
//
// Everything that comes from device memory here (lengths, row starts, page numbers) is checked where
// it is used, so that no value of it makes a kernel leave the tensors: a row outside every sequence is
// left alone, a position outside the table or the pool is not read or written.
#pragma once

#include <cstdint>
#include <type_traits>

#ifdef __HIP__
#define NC_PAGED_HD __host__ __device__ __forceinline__
#else
#define NC_PAGED_HD inline
#endif

namespace nc {

// n / d by a multiplication, for 0 <= n < 2^31 and 1 <= d < 2^31: q = (mulhi(n, magic) + n) >> shift with
// shift = ceil(log2 d) and magic = floor(2^32 (2^shift - d) / d) + 1 (Granlund and Montgomery 1994); the
// sum stays below 2^32 as mulhi(n, magic) <= n < 2^31.
struct PageDiv {
    uint32_t magic = 0, shift = 0, size = 1;
};
NC_PAGED_HD PageDiv page_div(uint32_t d) {
    PageDiv p;
    p.size = d;
    while ((1ull << p.shift) < d) p.shift++;
    p.magic = (uint32_t)((((1ull << p.shift) - d) << 32) / d + 1);
    return p;
}
NC_PAGED_HD uint32_t page_of(uint32_t n, const PageDiv& p) {
    return ((uint32_t)(((uint64_t)n * p.magic) >> 32) + n) >> p.shift;
}

// The last positions that a sequence's length and its table let a row reach.
struct PagedSeqs {
    const int32_t* table = nullptr;      // [seqs][table_stride], table_pages of each row used
    const int32_t* lens = nullptr;       // [seqs] positions, the new rows among them
    const int32_t* row_start = nullptr;  // [seqs + 1], or null: one row a sequence
    int64_t table_stride = 0;
    int32_t table_pages = 0, seqs = 0;
    int32_t cap = 0;  // positions that can be named: min(max_len, table_pages * page size)
    int32_t rows = 0;
};

struct PagedPool {
    int64_t page_stride = 0, pos_stride = 0, head_stride = 0;  // elements, of both pools
    int32_t pages = 0;
    PageDiv div;
};

// Rows [begin, begin + n) of sequence s, inside the tensor whatever row_start holds.
NC_PAGED_HD void seq_rows(const int32_t* start, int s, int rows, int& begin, int& n) {
    if (!start) {
        begin = s;
        n = s < rows ? 1 : 0;
        return;
    }
    const int b = start[s], e = start[s + 1];
    begin = b < 0 ? 0 : (b > rows ? rows : b);
    const int end = e < 0 ? 0 : (e > rows ? rows : e);
    n = end > begin ? end - begin : 0;
}

// Element offset in the pools of position p of a sequence, in page id of the pool.
NC_PAGED_HD int64_t place_in_page(int32_t id, int p, const PagedPool& pool) {
    const uint32_t pg = page_of((uint32_t)p, pool.div);
    return (int64_t)id * pool.page_stride + (int64_t)(p - (int)(pg * pool.div.size)) * pool.pos_stride;
}
// The same by the sequence's row of the table (0 <= p < cap), or -1 where its page is none of the pool's.
NC_PAGED_HD int64_t position_offset(const int32_t* table_row, const PagedPool& pool, int p) {
    const int32_t id = table_row[page_of((uint32_t)p, pool.div)];
    return (uint32_t)id < (uint32_t)pool.pages ? place_in_page(id, p, pool) : -1;
}

#ifdef __HIP__

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The sequence that row t (the same for every lane of the wave) belongs to, or -1: 64 starts at a time.
__device__ __forceinline__ int seq_of_row(const int32_t* start, int seqs, int t) {
    if (!start) return t < seqs ? t : -1;
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base <= seqs; base += 64) {
        const int i = base + lane;
        const bool le = i <= seqs && start[i] <= t;
        const int c = __popcll(__ballot(le));
        before += c;
        if (c < 64) break;
    }
    const int s = before - 1;
    return s >= 0 && s < seqs ? s : -1;
}

// Eight consecutive values, 16-byte aligned.
__device__ __forceinline__ void load8(const float* p, float* v) {
    const f32x4 a = ((const f32x4*)p)[0], b = ((const f32x4*)p)[1];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = a[i], v[4 + i] = b[i];
}
__device__ __forceinline__ void load8(const _Float16* p, float* v) {
    const f16x8 a = *(const f16x8*)p;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = (float)a[i];
}
__device__ __forceinline__ void load8(const __bf16* p, float* v) {
    const bf16x8 a = *(const bf16x8*)p;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = (float)a[i];
}
// One rounding to nearest even where the type is narrower than f32: the result's own type.
__device__ __forceinline__ void store8(float* p, const float* v) {
    ((f32x4*)p)[0] = f32x4{v[0], v[1], v[2], v[3]};
    ((f32x4*)p)[1] = f32x4{v[4], v[5], v[6], v[7]};
}
__device__ __forceinline__ void store8(_Float16* p, const float* v) {
    f16x8 a;
#pragma unroll
    for (int i = 0; i < 8; i++) a[i] = (_Float16)v[i];
    *(f16x8*)p = a;
}
__device__ __forceinline__ void store8(__bf16* p, const float* v) {
    bf16x8 a;
#pragma unroll
    for (int i = 0; i < 8; i++) a[i] = (__bf16)v[i];
    *(bf16x8*)p = a;
}


// ---------------------------------------------------------------- f32 values on 16-bit matrix products
// A 16-bit product of f32 values: the value as a sum of 16-bit parts, each the rest rounded to nearest, so that
// the products of the parts, exact and summed in f32, have f32's accuracy.  Three bf16 parts hold 24 bits at
// any exponent; two f16 parts hold 22 of a value scaled into f16's range.
template <typename T, int N>
__device__ __forceinline__ void split_parts(float x, T (&part)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        part[i] = (T)x;
        // the rest of an infinity is nothing, not NaN
        x = __builtin_isinf((float)part[i]) ? 0.f : x - (float)part[i];
    }
}

// The same of a value that is finite and within the type's range.
template <typename T, int N>
__device__ __forceinline__ void split_finite(float x, T (&part)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        part[i] = (T)x;
        if (i + 1 < N) x = __builtin_fmaf((float)part[i], -1.f, x);  // exact; one instruction takes the 16-bit operand
    }
}

__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

template <typename T>
struct Vec8;
template <>
struct Vec8<_Float16> {
    using type = f16x8;
};
template <>
struct Vec8<__bf16> {
    using type = bf16x8;
};

// The same value, of which the compiler does not know that: what rare branches compute from it stays in them,
// instead of taking registers all along.
__device__ __forceinline__ int kept_here(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// A lane's value and that of the lane 16 or 32 from it, in some order: the swap exchanges every other row of 16
// lanes, or half of 32, of two registers, here of one and the same value.
template <int APART>
__device__ __forceinline__ f32x2 with_lane_across(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto r = APART == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false) : __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return f32x2{__uint_as_float(r[0]), __uint_as_float(r[1])};
}
template <int APART>
__device__ __forceinline__ float max_across(float x) {
    const f32x2 v = with_lane_across<APART>(x);
    return fmaxf(v[0], v[1]);
}
template <int APART>
__device__ __forceinline__ float sum_across(float x) {
    const f32x2 v = with_lane_across<APART>(x);
    return v[0] + v[1];
}

// v or what DPP brings from another lane (0 where there is none), whichever is larger.
template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
    const uint32_t x = __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, false);
    return x > v ? x : v;
}
// The largest of v in each group of 8 or 16 lanes, in the group's last lane (row_shr:1, 2, 4, 8).
template <int LANES>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
    v = max_dpp<0x114>(max_dpp<0x112>(max_dpp<0x111>(v)));
    return LANES == 16 ? max_dpp<0x118>(v) : v;
}
// The largest of the groups' last lanes, in the wave's last lane (row_shr:8, then row_bcast:15 and 31).
template <int LANES>
__device__ __forceinline__ uint32_t wave_max_of_groups(uint32_t v) {
    if (LANES == 8) v = max_dpp<0x118>(v);
    return max_dpp<0x143>(max_dpp<0x142>(v));
}

// The wave's largest of v.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    return __builtin_amdgcn_readlane(wave_max_of_groups<16>(group_max<16>(v)), 63);
}

// The sum of v over the lanes up to the own one: within rows of 16 lanes, then the rows' last ones onto the next.
__device__ __forceinline__ int wave_prefix_sum(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
    return v;
}
// The wave's sum of v.
__device__ __forceinline__ int wave_sum(int v) { return __builtin_amdgcn_readlane(wave_prefix_sum(v), 63); }

constexpr float kLog2e = 1.44269504088896340736f;
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
// A maximum as the base of a row's exponents: 0 where nothing was seen, so that exp2(-inf - base) is 0.
__device__ __forceinline__ float exp_base(float m) { return m == -__builtin_inff() ? 0.f : m; }

#endif

}  // namespace nc
