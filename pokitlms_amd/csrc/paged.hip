// paged.hip -- the paged KV cache's bookkeeping and writer: block tables and slot maps
// from request lengths (k_paged_plan, k_paged_slots), and the head norms, rotation and
// store of new tokens (k_paged_append).  The reference keeps one sequence's ring
// (src/kv_cache.cpp:131-294) and rotates by one position (src/qwen3_moe_runner.cpp:
// 141-172); here many requests share a pool of pages.
#include <hip/hip_fp16.h>
#include <math.h>

#include "kquant.hpp"
#include "paged.hpp"

namespace pk {
namespace {

// ---------------------------------------------------------------------------
// Plan.  With pages(n) = ceil(n / page_size), request r keeps len_r positions (none if
// released) and gets new_r more, so it needs pages(len_r + new_r) - pages(len_r) pages.
// Released pages go on the free stack in request and table order, then the needed ones
// come off it in the same order; exclusive sums over the requests give every request
// its place, so no order depends on timing.  A plan that does not fit changes nothing.
//
// Reads and writes a few words per request and twelve bytes per token: latency bounds
// it.  One workgroup takes the requests (8 of them with a token each 3.4 us); the tokens as
// well while they are few (one launch: 96 requests, 4.8 k tokens 7.7 us), else a second launch
// spreads them over the chip (1024 requests, 96 k tokens 2.8 + 5.8 us).

enum : uint32_t { PLAN_PAGES = 1, PLAN_TABLE = 2, PLAN_TOKENS = 4, PLAN_STATE = 8 };

constexpr uint32_t kPlanThreads = 1024;
// Up to this many tokens one workgroup writes the slot map itself: 8000 tokens of one request
// 6.2 us a call, 9.5 in two launches; 9.6 k of 96 requests 11.7, 9.6 in two.
constexpr uint32_t kPlanFusedTokens = 8192;

struct PlanSums {
    uint32_t tokens, need, back;
};

// Inclusive sums over the lanes.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ void scan_step(PlanSums& v) {
    v.tokens += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v.tokens), CTRL, ROWS, 0xf, false));
    v.need += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v.need), CTRL, ROWS, 0xf, false));
    v.back += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v.back), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ PlanSums wave_scan(PlanSums v) {
    scan_step<0x111>(v);
    scan_step<0x112>(v);
    scan_step<0x114>(v);
    scan_step<0x118>(v);
    scan_step<0x142, 0xa>(v);
    scan_step<0x143, 0xc>(v);
    return v;
}

// f(request, pages in use, lane) for every released request, a wave at a time; neighbours in
// the table go to different waves.
template <typename F>
__device__ __forceinline__ void each_released(const PagedPlanArgs& a, uint32_t tid, F f) {
    constexpr uint32_t WAVES = kPlanThreads / 64u;
    const uint32_t lane = tid & 63u, cap = a.table_stride << a.page_shift;
    for (uint32_t base = tid >> 6; base < a.requests; base += kPlanThreads) {
        const uint32_t r = base + WAVES * lane;
        const uint32_t len = r < a.requests && a.release[r] ? a.lens[r] : 0u;
        uint64_t todo = __ballot(len > 0u && len <= cap);
        while (todo) {
            const uint32_t l = static_cast<uint32_t>(__builtin_ctzll(todo));
            todo &= todo - 1u;
            const uint32_t n = __shfl(len, l);
            f(base + WAVES * l, (n + (1u << a.page_shift) - 1u) >> a.page_shift, lane);
        }
    }
}

// Row j of request r is its position p = len + j.  Its page is an old table entry or the one
// popped for it: where that is read,
__device__ __forceinline__ const uint32_t* plan_page(const PagedPlanArgs& a, uint32_t r, uint32_t len, uint32_t j,
                                                     uint32_t first, uint32_t top) {
    const uint32_t pi = (len + j) >> a.page_shift, have = (len + (1u << a.page_shift) - 1u) >> a.page_shift;
    return pi < have ? a.table + static_cast<uint64_t>(r) * a.table_stride + pi : a.free_pages + (top - 1u - (first + pi - have));
}
// and what becomes of it: the first row of a fresh page writes the table entry.
__device__ __forceinline__ void plan_token(const PagedPlanArgs& a, uint32_t t, uint32_t r, uint32_t len, uint32_t j,
                                           uint32_t page) {
    const uint32_t mask = (1u << a.page_shift) - 1u, p = len + j;
    if ((p & mask) == 0u) a.table[static_cast<uint64_t>(r) * a.table_stride + (p >> a.page_shift)] = page;
    a.positions[t] = p;
    a.slots[t] = page < a.pages ? (page << a.page_shift) | (p & mask) : kNoSlot;
    a.token_request[t] = r;
}

__device__ __forceinline__ void plan_no_token(const PagedPlanArgs& a, uint32_t t) {
    a.positions[t] = 0u;
    a.slots[t] = kNoSlot;
    a.token_request[t] = kNoSlot;
}

// The last r in [lo, hi] with start[r] <= t, where start[lo] <= t.
__device__ __forceinline__ uint32_t plan_search(const uint32_t* start, uint32_t lo, uint32_t hi, uint32_t t) {
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1u) / 2u;
        if (start[mid] <= t) lo = mid;
        else hi = mid - 1u;
    }
    return lo;
}

// NI requests per thread; FUSED (NI = 1): the tokens too, with the requests' data in LDS.
template <uint32_t NI, bool FUSED>
__global__ __launch_bounds__(kPlanThreads) void k_paged_plan(PagedPlanArgs a) {
    static_assert(!FUSED || NI == 1u);
    __shared__ PlanSums wave_total[kPlanThreads / 64];
    __shared__ uint32_t bad;
    __shared__ uint32_t s_start[FUSED ? kPlanThreads + 1u : 1u], s_first[FUSED ? kPlanThreads : 1u],
        s_len[FUSED ? kPlanThreads : 1u], s_back[FUSED ? kPlanThreads : 1u];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint32_t R = a.requests, mask = (1u << a.page_shift) - 1u, cap = a.table_stride << a.page_shift;
    uint32_t* first = FUSED ? s_first : a.work;
    uint32_t* back = FUSED ? s_back : a.work + R;
    const uint32_t count = a.free_count[0];
    if (tid == 0u) bad = 0u;
    if (a.release) {
        for (uint32_t r = tid; r < R; r += kPlanThreads) back[r] = 0u;
        __syncthreads();
        each_released(a, tid, [&](uint32_t r, uint32_t n, uint32_t ln) {
            const uint32_t* row = a.table + static_cast<uint64_t>(r) * a.table_stride;
            uint32_t c = 0;
            for (uint32_t i = ln; i - ln < n; i += 64u)
                c += static_cast<uint32_t>(__popcll(__ballot(i < n && row[i < n ? i : 0u] < a.pages)));
            if (ln == 0u) back[r] = c;
        });
    }
    __syncthreads();
    uint32_t len[NI], fresh[NI], need[NI], rel[NI], flags = 0u;
    PlanSums mine{0, 0, 0};
#pragma unroll
    for (uint32_t i = 0; i < NI; ++i) {
        const uint32_t r = tid * NI + i;
        len[i] = fresh[i] = need[i] = rel[i] = 0u;
        if (r >= R) continue;
        len[i] = a.lens[r];
        fresh[i] = a.new_lens[r];
        if (len[i] > cap) {
            flags |= PLAN_STATE;
            len[i] = 0u;
        }
        if (a.release && a.release[r]) {
            len[i] = 0u;
            rel[i] = back[r];
        }
        if (fresh[i] > a.max_tokens) {
            flags |= PLAN_TOKENS;
            fresh[i] = 0u;
        }
        if (fresh[i] > cap - len[i]) {
            flags |= PLAN_TABLE;
            fresh[i] = 0u;
        }
        need[i] = ((len[i] + fresh[i] + mask) >> a.page_shift) - ((len[i] + mask) >> a.page_shift);
        mine.tokens += fresh[i];
        mine.need += need[i];
        mine.back += rel[i];
    }
    // a sum past max_tokens only has to stay past it
    if (mine.tokens > kMaxPagedTokens + 1u) mine.tokens = kMaxPagedTokens + 1u;
    PlanSums at = wave_scan(mine);
    if (lane == 63u) wave_total[wave] = at;
    at.tokens -= mine.tokens;
    at.need -= mine.need;
    at.back -= mine.back;
    if (flags) atomicOr(&bad, flags);
    __syncthreads();
    PlanSums total{0, 0, 0};
    uint64_t tokens_sum = 0;
#pragma unroll
    for (uint32_t w = 0; w < kPlanThreads / 64; ++w) {
        const PlanSums s = wave_total[w];
        if (w < wave) {
            at.tokens += s.tokens;
            at.need += s.need;
            at.back += s.back;
        }
        tokens_sum += s.tokens;
        total.need += s.need;
        total.back += s.back;
    }
    flags = bad;
    if (count > a.pages || total.back > a.pages - count) flags |= PLAN_STATE;
    else if (total.need > count + total.back) flags |= PLAN_PAGES;
    if (tokens_sum > a.max_tokens) flags |= PLAN_TOKENS;
    const uint32_t tokens = flags ? 0u : static_cast<uint32_t>(tokens_sum);
    const uint32_t top = count + total.back;
    if (!flags && total.back) {
        for (uint32_t i = 0; i < NI; ++i)
            if (tid * NI + i < R) {
                back[tid * NI + i] = at.back;
                at.back += rel[i];
            }
        __syncthreads();
        each_released(a, tid, [&](uint32_t r, uint32_t n, uint32_t ln) {
            const uint32_t* row = a.table + static_cast<uint64_t>(r) * a.table_stride;
            uint32_t to = count + back[r];
            for (uint32_t i = ln; i - ln < n; i += 64u) {
                const uint32_t page = i < n ? row[i] : kNoSlot;
                const uint64_t there = __ballot(page < a.pages);
                if (page < a.pages) a.free_pages[to + __popcll(there & ((1ull << ln) - 1u))] = page;
                to += static_cast<uint32_t>(__popcll(there));
            }
        });
    }
    __syncthreads();  // every read of lens and free_count is done: the outputs may be the inputs
    uint32_t start = at.tokens;
#pragma unroll
    for (uint32_t i = 0; i < NI; ++i) {
        const uint32_t r = tid * NI + i;
        if (r >= R) continue;
        if (flags) {
            if (a.lens_out != a.lens) a.lens_out[r] = a.lens[r];
            a.query_start[r] = 0u;
            continue;
        }
        a.lens_out[r] = len[i] + fresh[i];
        a.query_start[r] = start;
        first[r] = at.need;
        if constexpr (FUSED) {
            s_start[r] = start;
            s_len[r] = len[i];
        }
        start += fresh[i];
        at.need += need[i];
    }
    if (tid == 0u) {
        a.query_start[R] = tokens;
        a.free_count_out[0] = flags ? count : top - total.need;
        a.status[0] = flags;
        a.status[1] = tokens;
        a.status[2] = flags ? 0u : total.need;
        a.status[3] = flags ? 0u : total.back;
    }
    if constexpr (FUSED) {
        __syncthreads();
        // four tokens a thread at a time: their searches and page reads wait together
        constexpr uint32_t U = 4u;
        uint32_t widest = 1u;
        while (2u * widest < R) widest *= 2u;
        for (uint32_t t0 = tid; t0 < a.max_tokens; t0 += U * kPlanThreads) {
            uint32_t r[U], page[U];
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) r[u] = 0u;
            for (uint32_t step = R > 1u ? widest : 0u; step > 0u; step /= 2u)
#pragma unroll
                for (uint32_t u = 0; u < U; ++u) {
                    const uint32_t next = r[u] + step;
                    if (next < R && s_start[next] <= t0 + u * kPlanThreads) r[u] = next;
                }
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                const uint32_t t = t0 + u * kPlanThreads;
                page[u] = t < tokens ? *plan_page(a, r[u], s_len[r[u]], t - s_start[r[u]], s_first[r[u]], top) : kNoSlot;
            }
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                const uint32_t t = t0 + u * kPlanThreads;
                if (t < tokens) plan_token(a, t, r[u], s_len[r[u]], t - s_start[r[u]], page[u]);
                else if (t < a.max_tokens) plan_no_token(a, t);
            }
        }
    }
}

// The tokens of a plan whose requests k_paged_plan has settled.  A workgroup's tokens
// belong to few requests: one search for its first and last token narrows each lane's.
__global__ __launch_bounds__(256) void k_paged_slots(PagedPlanArgs a) {
    const uint32_t t0 = blockIdx.x * 256u, t = t0 + threadIdx.x, tokens = a.status[1];
    const uint32_t top = a.free_count_out[0] + a.status[2];
    uint32_t lo = 0u, hi = 0u;
    if (t0 < tokens) {
        lo = plan_search(a.query_start, 0u, a.requests - 1u, t0);
        hi = plan_search(a.query_start, lo, a.requests - 1u, t0 + 255u < tokens ? t0 + 255u : tokens - 1u);
    }
    if (t >= a.max_tokens) return;
    if (t >= tokens) {
        plan_no_token(a, t);
        return;
    }
    const uint32_t r = plan_search(a.query_start, lo, hi, t), start = a.query_start[r];
    const uint32_t len = a.lens_out[r] - (a.query_start[r + 1u] - start);
    plan_token(a, t, r, len, t - start, *plan_page(a, r, len, t - start, a.work[r], top));
}

// ---------------------------------------------------------------------------
// Append.  Per token and head row x of HD values: q and k rows are normed,
//   x <- x / sqrt(mean(x^2) + eps) * w,
// and the pairs (i, i + pairs), i < pairs, turned by the angle of the token's position on
// the pair's axis; then q goes to q_out, k and v to the pages.  Every value is read and
// written once: HBM bounds it.  Angles are taken in double as a fraction of a turn and
// brought to an eighth of a turn around zero before the float sine and cosine, so a far
// position costs no accuracy; a token's are computed once, in LDS, for all of its heads.
// 16,384 BF16 tokens of 16 + 2 heads of 256: 66 us (5.1 TB/s, a copy reaches 5.2); 8 F32 tokens
// of 32 + 4 heads of 128: 5.2 us, the latency of angles, then rows.

template <uint32_t T> struct Row8;
template <> struct Row8<T_F32> {
    using E = float;
    static __device__ __forceinline__ void load(const E* p, float* v) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    static __device__ __forceinline__ void store(E* p, const float* v) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
};
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
template <typename V, typename S>
struct Row8Half {
    using E = uint16_t;
    static __device__ __forceinline__ void load(const E* p, float* v) {
        const V x = *reinterpret_cast<const V*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(x[i]);
    }
    static __device__ __forceinline__ void store(E* p, const float* v) {  // nearest even
        V x;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = static_cast<S>(v[i]);
        *reinterpret_cast<V*>(p) = x;
    }
};
template <> struct Row8<T_F16> : Row8Half<h16x8, _Float16> {};
template <> struct Row8<T_BF16> : Row8Half<b16x8, __bf16> {};

// Cosine and sine of `turns` full turns: the quarter turn next to it is taken off in
// double, the rest is within an eighth of a turn.
__device__ __forceinline__ void turn_cos_sin(double turns, float& c, float& s) {
    const double f = turns - rint(turns), q = rint(4.0 * f);
    float sn, cs;
    sincosf(static_cast<float>((f - 0.25 * q) * 6.283185307179586), &sn, &cs);
    const int k = static_cast<int>(q) & 3;
    c = k == 0 ? cs : k == 1 ? -sn : k == 2 ? -cs : sn;
    s = k == 0 ? sn : k == 1 ? cs : k == 2 ? -sn : -cs;
}

// A workgroup takes NT tokens; a row sits on HD / 16 lanes, eight values and their
// rotation partners (or eight more unrotated ones) each.
template <uint32_t T, uint32_t HD, uint32_t NT>
__global__ __launch_bounds__(256) void k_paged_append(PagedAppendArgs a) {
    using Row = Row8<T>;
    using E = typename Row::E;
    constexpr uint32_t LP = HD / 16u, ROWS = 256u / LP;
    __shared__ float cs[NT][HD / 2u], sn[NT][HD / 2u];
    const uint32_t tid = threadIdx.x, t0 = blockIdx.x * NT, pairs = a.rotary_pairs;
    for (uint32_t i = tid; i < NT * pairs; i += 256u) {
        const uint32_t t = t0 + i / pairs, p = i % pairs;
        if (t >= a.tokens) continue;
        const uint32_t pos = a.positions[a.axis[p] * a.position_stride + t];
        turn_cos_sin(static_cast<double>(pos) * a.turns[p], cs[i / pairs][p], sn[i / pairs][p]);
    }
    __syncthreads();
    const uint32_t rows = a.heads + 2u * a.kv.kv_heads, l = tid % LP, rc = pairs / 8u;
    // this lane's two chunks of eight values: rotation partners, or one of each half of the rest
    const bool turned = l < rc;
    const uint32_t c0 = turned ? l : l + rc, c1 = turned ? l + rc : l + LP;
    for (uint32_t i = tid / LP; i < NT * rows; i += ROWS) {
        const uint32_t t = t0 + i / rows, row = i % rows;
        if (t >= a.tokens) break;
        const uint32_t slot = a.slots[t];
        if ((slot >> a.kv.page_shift) >= a.kv.pages) continue;
        const bool isq = row < a.heads, isv = row >= a.heads + a.kv.kv_heads;
        const uint32_t head = isq ? row : row - a.heads - (isv ? a.kv.kv_heads : 0u);
        const E* src = isq ? static_cast<const E*>(a.q) + t * a.q_stride
                           : isv ? static_cast<const E*>(a.v) + t * a.v_stride
                                 : static_cast<const E*>(a.k) + t * a.k_stride;
        float x[8], y[8];
        Row::load(src + head * HD + 8u * c0, x);
        Row::load(src + head * HD + 8u * c1, y);
        if constexpr (T == T_F32) {
            const uint64_t step = isq ? a.q_part : a.kv_part;
            for (uint32_t k = 1; k < a.parts; ++k) {
                float u[8], v[8];
                Row::load(src + k * step + head * HD + 8u * c0, u);
                Row::load(src + k * step + head * HD + 8u * c1, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] += u[e];
                    y[e] += v[e];
                }
            }
        }
        const float* w = isv ? nullptr : isq ? a.q_norm : a.k_norm;
        if (w) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss += x[e] * x[e] + y[e] * y[e];
#pragma unroll
            for (uint32_t d = 1; d < LP; d *= 2) ss += __shfl_xor(ss, d);
            const float scale = 1.0f / sqrtf(ss / static_cast<float>(HD) + a.eps);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = x[e] * scale * w[8u * c0 + e];
                y[e] = y[e] * scale * w[8u * c1 + e];
            }
        }
        if (!isv && turned) {
            const uint32_t ti = i / rows;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float c = cs[ti][8u * l + e], s = sn[ti][8u * l + e], u = x[e];
                x[e] = u * c - y[e] * s;
                y[e] = y[e] * c + u * s;
            }
        }
        if (isq) {
            E* dst = static_cast<E*>(a.q_out) + t * a.q_out_stride + head * HD;
            Row::store(dst + 8u * c0, x);
            Row::store(dst + 8u * c1, y);
        } else {
            const uint32_t page = slot >> a.kv.page_shift, in_page = slot & ((1u << a.kv.page_shift) - 1u);
            uint16_t* dst = (isv ? a.kv.v : a.kv.k) + page * a.kv.page_stride + in_page * a.kv.slot_stride +
                            head * a.kv.head_stride;
            if (a.kv.type == T_F16) {
                Row8<T_F16>::store(dst + 8u * c0, x);
                Row8<T_F16>::store(dst + 8u * c1, y);
            } else {
                Row8<T_BF16>::store(dst + 8u * c0, x);
                Row8<T_BF16>::store(dst + 8u * c1, y);
            }
        }
    }
}

// From this many tokens on a workgroup takes four, which spreads its start over more rows; with
// fewer, more workgroups wait at once.  One token a workgroup or four, us: 32 + 4 heads of 128,
// F16, 1024 tokens 6.7 and 9.0, 2048 10.0 and 11.8, 4096 17.2 and 16.6, 8192 28.5 and 28.7;
// 16 + 2 of 256, BF16, 2048 9.8 and 12.0, 4096 16.8 and 16.8; 8 + 2 of 128, F16, 2048 5.1 and
// 5.7, 4096 8.5 and 7.6, 8192 14.8 and 11.5.
constexpr uint32_t kAppendManyTokens = 4096;

template <uint32_t T, uint32_t HD>
hipError_t append_t(const PagedAppendArgs& a, hipStream_t s) {
    if (a.tokens < kAppendManyTokens) hipLaunchKernelGGL((k_paged_append<T, HD, 1>), dim3(a.tokens), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_paged_append<T, HD, 4>), dim3((a.tokens + 3u) / 4u), dim3(256), 0, s, a);
    return hipGetLastError();
}

template <uint32_t T>
hipError_t append_hd(const PagedAppendArgs& a, hipStream_t s) {
    switch (a.kv.head_dim) {
        case 64: return append_t<T, 64>(a, s);
        case 128: return append_t<T, 128>(a, s);
        case 256: return append_t<T, 256>(a, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

void rotary_turns(PagedAppendArgs& a, float theta) {
    for (uint32_t i = 0; i < a.rotary_pairs; ++i)
        a.turns[i] = pow(static_cast<double>(theta), -static_cast<double>(i) / a.rotary_pairs) / 6.283185307179586;
}

size_t paged_plan_work_words(uint32_t requests, uint32_t max_tokens) {
    return requests <= kPlanThreads && max_tokens <= kPlanFusedTokens ? 0u : 2u * static_cast<size_t>(requests);
}

hipError_t launch_paged_plan(const PagedPlanArgs& a, hipStream_t s) {
    if (!paged_plan_work_words(a.requests, a.max_tokens)) {
        hipLaunchKernelGGL((k_paged_plan<1, true>), dim3(1), dim3(kPlanThreads), 0, s, a);
        return hipGetLastError();
    }
    if (a.requests <= kPlanThreads) hipLaunchKernelGGL((k_paged_plan<1, false>), dim3(1), dim3(kPlanThreads), 0, s, a);
    else hipLaunchKernelGGL((k_paged_plan<kMaxPagedRequests / kPlanThreads, false>), dim3(1), dim3(kPlanThreads), 0, s, a);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    hipLaunchKernelGGL(k_paged_slots, dim3((a.max_tokens + 255u) / 256u), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t s) {
    switch (a.type) {
        case T_F32: return append_hd<T_F32>(a, s);
        case T_F16: return append_hd<T_F16>(a, s);
        case T_BF16: return append_hd<T_BF16>(a, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace pk
