// Causal attention over packed whole prompts: sequences of different lengths end to end in one tensor of
// rows, query heads in groups that share a key-value head.  Row i of a sequence with n query rows and m key
// rows sees its keys 0 .. m - n + i.
#include <hip/hip_runtime.h>

#include "nc_internal.h"
#include "nc_paged.h"

namespace nc {

struct PackedParams {
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    void* out;
    const int32_t *seq_start, *kv_start;
    int32_t seqs, rows, kv_rows, heads, kv_heads;
    float scale;
};

// One wave per (row, head): 64 keys at a time, a key a lane for the scores, a running maximum and sum, then
// the values with head_dim over the lanes.
template <typename A, int HD>
__global__ __launch_bounds__(64) void packed_attention_kernel(PackedParams a) {
    __shared__ float qs[HD];
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    const int s = seq_of_row(a.seq_start, a.seqs, t);
    if (s < 0) return;
    int begin, n, kbegin, m;
    seq_rows(a.seq_start, s, a.rows, begin, n);
    seq_rows(a.kv_start, s, a.kv_rows, kbegin, m);
    const int i = t - begin;
    if (i < 0 || i >= n) return;
    const A* q = (const A*)a.q + (int64_t)t * a.q_stride + h * HD;
    for (int d = lane; d < HD; d += 64) qs[d] = (float)q[d] * a.scale;
    __syncthreads();
    const int seen = m - n + i + 1;
    const int head = (h / (a.heads / a.kv_heads)) * HD;
    const A* kb = (const A*)a.k + (int64_t)kbegin * a.k_stride + head;
    const A* vb = (const A*)a.v + (int64_t)kbegin * a.v_stride + head;
    float top = -__builtin_inff(), l = 0.f, acc[HD / 64] = {};
    for (int base = 0; base < seen; base += 64) {
        const int p = base + lane;
        float score = -__builtin_inff();
        if (p < seen) {
            score = 0.f;
            for (int d = 0; d < HD; d += 8) {
                float x[8];
                load8(kb + p * a.k_stride + d, x);
                for (int j = 0; j < 8; j++) score += qs[d + j] * x[j];
            }
        }
        float next = score;
        for (int o = 32; o; o >>= 1) next = fmaxf(next, __shfl_xor(next, o, 64));
        next = fmaxf(next, top);
        const float base_of = next == -__builtin_inff() ? 0.f : next;
        const float e = p < seen ? expf(score - base_of) : 0.f;
        const float keep = expf(top - base_of);
        float sum = e;
        for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
        l = l * keep + sum;
        top = next;
        for (int c = 0; c < HD / 64; c++) acc[c] *= keep;
        const int count = seen - base < 64 ? seen - base : 64;
        for (int j = 0; j < count; j++) {
            const float w = __shfl(e, j, 64);
            for (int c = 0; c < HD / 64; c++) acc[c] += w * (float)vb[(base + j) * a.v_stride + c * 64 + lane];
        }
    }
    A* out = (A*)a.out + ((int64_t)t * a.heads + h) * HD;
    for (int c = 0; c < HD / 64; c++) out[c * 64 + lane] = (A)(l == 0.f ? 0.f : acc[c] / l);
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
    PackedParams a = {q, k, v, q_stride, k_stride, v_stride, out, seq_start, kv_start ? kv_start : seq_start, seqs,
                      (int32_t)rows, (int32_t)kv_rows, heads, kv_heads, scale};
    DeviceGuard guard(ctx->device);
    if (guard.rc) return guard.rc;
    hipStream_t st = stream ? (hipStream_t)stream : ctx->stream;
    const dim3 grid((unsigned)rows, heads);
    auto launch = [&]<typename A>() {
        if (head_dim == 64)
            packed_attention_kernel<A, 64><<<grid, 64, 0, st>>>(a);
        else
            packed_attention_kernel<A, 128><<<grid, 64, 0, st>>>(a);
        NC_HIP(hipGetLastError());
        return (int)NC_OK;
    };
    if (type == NC_TYPE_F32) return launch.template operator()<float>();
    if (type == NC_TYPE_F16) return launch.template operator()<_Float16>();
    return launch.template operator()<__bf16>();
}
