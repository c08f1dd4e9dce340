// paged_attention.hip -- attention of new tokens over a paged KV cache.
//
// Row j of request r (j < new_r) stands at position p = len_r - new_r + j and sees
// position i of its request's pages if i <= p, its page is there, and, with a window W,
// i + W > p or i < sinks.  Head h reads kv head h / group:
//   o = sum_i softmax_i(scale * q . k_i) v_i, and 0 where nothing is seen.
#include <hip/hip_fp16.h>
#include <math.h>

#include "kquant.hpp"
#include "paged.hpp"

namespace pk {
namespace {

__device__ __forceinline__ float cache_value(uint32_t type, uint16_t bits) {
    return type == T_F16 ? half_bits_to_float(bits) : __uint_as_float(static_cast<uint32_t>(bits) << 16);
}

// One wave per (token, head): 64 positions at a time, a score per lane, then the values
// with a running maximum and sum.
__global__ __launch_bounds__(64) void k_paged_attention_plain(PagedAttentionArgs a) {
    __shared__ float q[256];
    const uint32_t t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, HD = a.kv.head_dim;
    uint32_t r = a.requests;
    for (uint32_t i = 0; i < a.requests; ++i)
        if (a.query_start[i] <= t && t < a.query_start[i + 1u]) r = i;
    if (r == a.requests || a.query_start[r + 1u] - a.query_start[r] > a.max_new) return;
    const int64_t len = a.lens[r], p = len - (a.query_start[r + 1u] - t);
    const uint64_t at = t * a.q_stride + h * HD;
    for (uint32_t d = lane; d < HD; d += 64u)
        q[d] = a.scale * (a.type == T_F32 ? static_cast<const float*>(a.q)[at + d]
                                          : cache_value(a.type, static_cast<const uint16_t*>(a.q)[at + d]));
    __syncthreads();
    const uint32_t mask = (1u << a.kv.page_shift) - 1u;
    const int64_t cap = static_cast<int64_t>(a.table_stride) << a.kv.page_shift;
    float m = -INFINITY, sum = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t i0 = 0; i0 <= p && i0 < cap; i0 += 64) {
        const int64_t i = i0 + lane;
        bool seen = i <= p && i < cap && (a.window == 0u || i + a.window > p || i < a.sinks);
        const uint32_t page = seen ? a.table[static_cast<uint64_t>(r) * a.table_stride + (i >> a.kv.page_shift)] : kNoSlot;
        seen = page < a.kv.pages;
        const uint64_t row = seen ? page * a.kv.page_stride + (i & mask) * a.kv.slot_stride + (h / a.group) * a.kv.head_stride : 0u;
        float s = -INFINITY;
        if (seen) {
            s = 0.0f;
            for (uint32_t d = 0; d < HD; ++d) s = fmaf(q[d], cache_value(a.kv.type, a.kv.k[row + d]), s);
        }
        float top = s;
        for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
        if (top == -INFINITY) continue;
        const float next = fmaxf(m, top), e = seen ? expf(s - next) : 0.0f, keep = expf(m - next);
        float es = e;
        for (int d = 32; d > 0; d >>= 1) es += __shfl_xor(es, d);
        sum = sum * keep + es;
        for (uint32_t c = 0; c < HD / 64u; ++c) o[c] *= keep;
        for (uint32_t l = 0; l < 64u; ++l) {
            const float w = __shfl(e, l);
            const uint64_t vr = __shfl(row, l);
            if (w == 0.0f) continue;
            for (uint32_t c = 0; c < HD / 64u; ++c) o[c] = fmaf(w, cache_value(a.kv.type, a.kv.v[vr + 64u * c + lane]), o[c]);
        }
        m = next;
    }
    const uint64_t to = t * a.out_stride + h * HD;
    for (uint32_t c = 0; c < HD / 64u; ++c) {
        const float v = sum > 0.0f ? o[c] / sum : 0.0f;
        const uint64_t d = to + 64u * c + lane;
        if (a.type == T_F32) static_cast<float*>(a.out)[d] = v;
        else if (a.type == T_F16) static_cast<_Float16*>(a.out)[d] = static_cast<_Float16>(v);
        else static_cast<__bf16*>(a.out)[d] = static_cast<__bf16>(v);
    }
}

}  // namespace

hipError_t launch_paged_attention(const PagedAttentionArgs& a, hipStream_t s) {
    hipLaunchKernelGGL(k_paged_attention_plain, dim3(a.max_tokens, a.heads), dim3(64), 0, s, a);
    return hipGetLastError();
}

}  // namespace pk
