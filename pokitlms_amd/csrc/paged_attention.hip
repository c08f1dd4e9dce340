// paged_attention.hip -- attention of new tokens over a paged KV cache.
//
// Row j of request r (j < new_r) stands at position p = len_r - new_r + j and sees
// position i of its request's pages if i <= p, its page is there, and, with a window W,
// i + W > p or i < sinks.  Head h reads kv head h / group:
//   o = sum_i softmax_i(scale * q . k_i) v_i, and 0 where nothing is seen.
//
// One pass over K and V with a running maximum m and sum l per row (in units of log 2):
// o <- o * 2^(m - m') + sum_i 2^(c s_i - m') v_i, with c = scale * log2(e).  Rows of one
// kv head's query heads share a tile, so K and V are read once for all of them.  Both
// products run on the matrix cores as S^T = K Q^T and O^T = V^T P^T: a lane then holds
// scores of one row only, maximum, sum and rescaling stay in the lane (and the few that
// share its row), and the weights are in the layout that the second product takes, with
// the keys of a tile in the order in which the first left them.
//
// FP32 rows enter the 16-bit products as parts, q = q0 + q1 (+ q2) and likewise the weights:
// two F16 parts hold 22 bits (q under a power of two per row, weights times 2^12, so that
// small ones keep them), three BF16 parts 24.  16-bit rows round the weights once to
// the cache's type, half a step each at most, so the output is off by half a step of
// sum_i w_i |v_i| at most and then rounds to the same type itself.  Over BF16 the mean error
// is 0.0022 of the output's, 0.0017 with unrounded weights; a second part of the weights
// would take half as many matrix instructions again.
#include <hip/hip_fp16.h>
#include <math.h>

#include "kquant.hpp"
#include "paged.hpp"

namespace pk {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <uint32_t T> struct Mat;
template <> struct Mat<T_F16> {
    using E = _Float16;
    typedef _Float16 V8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 mma16(V8 a, V8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mma32(V8 a, V8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
template <> struct Mat<T_BF16> {
    using E = __bf16;
    typedef __bf16 V8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 mma16(V8 a, V8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mma32(V8 a, V8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};

constexpr uint32_t parts_of(uint32_t T, bool f32) { return !f32 ? 1u : T == T_F16 ? 2u : 3u; }

// The maximum moves (and o and l are rescaled) only when it has grown by 2^3, and weights carry
// 2^bias: at most 2^(bias + 3).  F16: 2^15, so that small ones keep their bits, and with V at
// most 2^16 FP32 holds any sum.  BF16, whose V may be as large as FP32's values: over the
// len positions of a request, len 2^(bias + 3) is at most 1, so that no sum is above V's
// largest, as with a softmax's weights.
constexpr float kSlack = 3.0f;
template <uint32_t T>
__device__ __forceinline__ float weight_bias(int32_t len) {
    if (T == T_F16) return 12.0f;
    const float b = static_cast<float>(__builtin_clz(static_cast<uint32_t>(len) | 1u)) - 32.0f - kSlack;
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(b)));  // the same for all lanes
}

// 8 values as NP parts: v = parts[0] + parts[1] + ...
template <typename M, uint32_t NP>
__device__ __forceinline__ void split8(const float* v, typename M::V8* parts) {
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) {
        float rest = v[e];
#pragma unroll
        for (uint32_t i = 0; i < NP; ++i) {
            const auto h = static_cast<typename M::E>(rest);
            parts[i][e] = h;
            rest -= static_cast<float>(h);
        }
    }
}

__device__ __forceinline__ float cache_value(uint32_t type, uint16_t bits) {
    return type == T_F16 ? half_bits_to_float(bits) : __uint_as_float(static_cast<uint32_t>(bits) << 16);
}

// A launch's share of the rows, and its scratch: parts of split tiles (BM rows of head_dim
// sums, then their m and l), the split tiles, and their number.
struct RowWork {
    uint32_t min_rows, max_rows, log_target, least;
    float* part;
    uint32_t* head;   // per split tile kHeadWords: parts, first row's q row, tokens, tile, first part's place
    uint32_t* count;  // [1]
    // of more than kWaveRequests requests: k_paged_schedule's pieces and split tiles, then per
    // request its first unit and its first part and split tile (null: every wave counts)
    uint32_t* schedule;
};
// Counted by every wave, or by a launch before (single tokens of 32 heads over 4 of 128, 200
// positions each): 65 requests 10.5 us or 13.8, 128 16.0 or 19.2, 193 28.4 or 26.9, 256 31.7 or
// 29.8, 1024 262 or 111, 8192 (100 positions) 14,525 or 587.
constexpr uint32_t kWaveRequests = 192u;
constexpr uint32_t schedule_words(uint32_t requests) { return 4u + 2u * (requests + 1u); }

// One workgroup's piece: part `part` of `parts` of row tile `tile` of request r; its place
// among the parts and its tile's among the split tiles, both per kv head.
struct Piece {
    uint32_t r, q0, fresh, tile, part, parts, slot, split;
    int32_t len;
};

template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t dpp_from(uint32_t v) {  // 0 where there is no lane to read
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ uint32_t wave_prefix(uint32_t v) {  // inclusive sums over the lanes
    v += dpp_from<0x111>(v);
    v += dpp_from<0x112>(v);
    v += dpp_from<0x114>(v);
    v += dpp_from<0x118>(v);
    v += dpp_from<0x142, 0xa>(v);
    v += dpp_from<0x143, 0xc>(v);
    return v;
}

__device__ __forceinline__ uint32_t lane_value(uint32_t v, uint32_t lane) {
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), static_cast<int>(lane)));
}

// A request's rows and work, from the lengths.
struct Request {
    uint32_t q0, q1, len;
    RequestWork work;
};
__device__ __forceinline__ Request request_of(const PagedAttentionArgs& a, const RowWork& w, uint32_t bm, uint32_t r) {
    const uint32_t at = r < a.requests ? r : 0u, positions = a.table_stride << a.kv.page_shift;
    Request q{a.query_start[at], a.query_start[at + 1u], a.lens[at], {0u, 0u}};
    const uint32_t fresh = r < a.requests ? paged_new(q.q0, q.q1, a.max_new, a.max_tokens) : 0u;
    q.work = request_work(fresh, q.len, a.group, bm, w.min_rows, w.max_rows, a.window, a.sinks, positions);
    return q;
}
// Its units, and its parts of split tiles and split tiles in one word (over all requests at
// most 2 * target and target).
__device__ __forceinline__ uint32_t units_of(const RequestWork& q, uint32_t pieces, uint32_t& cut) {
    const uint32_t n = request_parts(q.keys, pieces);
    cut = n > 1u ? q.tiles * (n + 0x10000u) : 0u;
    return q.tiles * n;
}

// The piece of unit u.  Up to kWaveRequests every wave finds it by itself from the lengths,
// its lanes taking a 64th of the requests each: exclusive sums give each its units.  With
// more, a launch before has left those sums, and two looks of 64 lanes find the request.
// splits: split tiles per kv head.
__device__ __forceinline__ bool find_piece(const PagedAttentionArgs& a, const RowWork& w, uint32_t bm, uint32_t u,
                                           Piece& p, uint32_t& splits) {
    const uint32_t lane = threadIdx.x & 63u, positions = a.table_stride << a.kv.page_shift;
    Request q;
    uint32_t pieces, left, before;
    if (!w.schedule) {
        const uint32_t per = (a.requests + 63u) / 64u;
        q = request_of(a, w, bm, lane * per);
        double work = static_cast<double>(q.work.tiles) * q.work.keys;  // exact below 2^53
        for (uint32_t i = 1; i < per; ++i) {
            q = request_of(a, w, bm, lane * per + i);
            work += static_cast<double>(q.work.tiles) * q.work.keys;
        }
        work = lane63(group_sum<64>(work));
        pieces = part_pieces(static_cast<uint64_t>(work) * a.kv.kv_heads, w.log_target, w.least);
        uint32_t units = 0u, cut = 0u, c;
        for (uint32_t i = 0; i < per; ++i) {
            if (per > 1u) q = request_of(a, w, bm, lane * per + i);
            units += units_of(q.work, pieces, c);
            cut += c;
        }
        uint32_t eu = wave_prefix(units), ec = wave_prefix(cut);
        splits = lane_value(ec, 63u) >> 16;
        eu -= units;
        ec -= cut;
        const uint64_t mine = __ballot(u >= eu && u - eu < units);
        if (!mine) return false;
        uint32_t r = lane * per;
        left = u - eu;
        for (uint32_t i = 0; per > 1u && i < per; ++i) {  // only the owner's walk matters
            q = request_of(a, w, bm, lane * per + i);
            r = lane * per + i;
            const uint32_t n = units_of(q.work, pieces, c);
            if (left < n || i + 1u == per) break;
            left -= n;
            ec += c;
        }
        const uint32_t owner = static_cast<uint32_t>(__builtin_ctzll(mine));
        p.r = lane_value(r, owner);
        left = lane_value(left, owner);
        before = lane_value(ec, owner);
        q.q0 = lane_value(q.q0, owner);
        q.q1 = lane_value(q.q1, owner);
        q.len = lane_value(q.len, owner);
        q.work = {lane_value(q.work.tiles, owner), lane_value(q.work.keys, owner)};
    } else {
        const uint32_t R = a.requests, step = (R + 63u) / 64u;
        const uint32_t *start = w.schedule + 4u, *cuts = start + R + 1u;
        pieces = w.schedule[0];
        splits = w.schedule[1];
        // the last request that starts at u or before
        const uint32_t at = lane * step < R ? lane * step : R;
        const uint32_t k = static_cast<uint32_t>(__popcll(__ballot(at < R && start[at] <= u))) - 1u;
        if (u >= start[R]) return false;
        const uint32_t base = k * step;
        uint32_t count = 0;
        for (uint32_t i = 0; i < step; i += 64u) {
            const uint32_t r = base + i + lane;
            count += static_cast<uint32_t>(__popcll(__ballot(i + lane < step && r < R && start[r < R ? r : R] <= u)));
        }
        p.r = base + count - 1u;
        left = u - start[p.r];
        before = cuts[p.r];
        q = request_of(a, w, bm, p.r);
    }
    p.parts = request_parts(q.work.keys, pieces);
    p.tile = q.work.tiles - 1u - left / p.parts;  // the tiles that see most keys first
    p.part = left % p.parts;
    p.slot = (before & 0xffffu) + left;
    p.split = (before >> 16) + left / p.parts;
    p.q0 = q.q0;
    p.fresh = q.q1 - q.q0;
    p.len = static_cast<int32_t>(q.len < positions ? q.len : positions);
    // (sums of a query_start that decreases may leave their words and the scratch)
    return left < q.work.tiles * p.parts &&
           (p.parts == 1u || split_fits(p.split, p.slot, a.kv.kv_heads, 1u << w.log_target));
}

// What find_piece needs where there are more than kWaveRequests requests: a workgroup per kind of
// tile, its threads a 1024th of the requests each.
__global__ __launch_bounds__(1024) void k_paged_schedule(PagedAttentionArgs a, RowWork few, RowWork many) {
    __shared__ double s_work[16];
    __shared__ uint32_t s_units[16], s_cut[16];
    const RowWork& w = blockIdx.x ? many : few;
    const uint32_t bm = blockIdx.x ? 128u : 16u, R = a.requests;
    if (!w.schedule) return;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, per = (R + 1023u) / 1024u;
    double work = 0.0;
    for (uint32_t i = 0; i < per; ++i) {
        const RequestWork q = request_of(a, w, bm, tid * per + i).work;
        work += static_cast<double>(q.tiles) * q.keys;
    }
    work = group_sum<64>(work);
    if (lane == 63u) s_work[wave] = work;
    __syncthreads();
    work = 0.0;
    for (uint32_t i = 0; i < 16u; ++i) work += s_work[i];
    const uint32_t pieces = part_pieces(static_cast<uint64_t>(work) * a.kv.kv_heads, w.log_target, w.least);
    uint32_t units = 0u, cut = 0u;
    for (uint32_t i = 0; i < per; ++i) {
        uint32_t c;
        units += units_of(request_of(a, w, bm, tid * per + i).work, pieces, c);
        cut += c;
    }
    uint32_t eu = wave_prefix(units), ec = wave_prefix(cut);
    if (lane == 63u) {
        s_units[wave] = eu;
        s_cut[wave] = ec;
    }
    __syncthreads();
    eu -= units;
    ec -= cut;
    for (uint32_t i = 0; i < wave; ++i) {
        eu += s_units[i];
        ec += s_cut[i];
    }
    uint32_t *start = w.schedule + 4u, *cuts = start + R + 1u;
    for (uint32_t i = 0; i < per && tid * per + i < R; ++i) {
        const uint32_t r = tid * per + i;
        uint32_t c;
        start[r] = eu;
        cuts[r] = ec;
        eu += units_of(request_of(a, w, bm, r).work, pieces, c);
        ec += c;
    }
    if (tid == 1023u) {  // behind every request's
        start[R] = eu;
        w.schedule[0] = pieces;
        w.schedule[1] = ec >> 16;
    }
}

// 4 values of a row of q's type.
__device__ __forceinline__ void store4(uint32_t type, void* out, uint64_t at, f32x4 v) {
    if (type == T_F32) {
        *reinterpret_cast<f32x4*>(static_cast<float*>(out) + at) = v;
    } else if (type == T_F16) {
        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<h4*>(static_cast<uint16_t*>(out) + at) = __builtin_convertvector(v, h4);
    } else {
        typedef __bf16 b4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<b4*>(static_cast<uint16_t*>(out) + at) = __builtin_convertvector(v, b4);
    }
}

// Where a row's result goes: its output, or its place among the parts.
struct RowTo {
    void* out;
    uint64_t at;
    float* part;  // [HD] sums, or null
    float* ml;
};
__device__ __forceinline__ RowTo row_to(const PagedAttentionArgs& a, const RowWork& w, const Piece& p, uint32_t bm,
                                        uint32_t hk, uint32_t row) {
    const uint32_t f = p.tile * bm + row, HD = a.kv.head_dim;
    RowTo to{a.out, (p.q0 + a.group(f)) * a.out_stride + (hk * a.group.by + a.group.rest(f)) * HD, nullptr, nullptr};
    if (p.parts > 1u) {
        float* base = w.part + static_cast<uint64_t>(p.slot * a.kv.kv_heads + hk) * bm * (HD + 2u);
        to.part = base + row * HD;
        to.ml = base + bm * HD + 2u * row;
    }
    return to;
}
__device__ __forceinline__ void store_row4(const PagedAttentionArgs& a, const RowTo& to, uint32_t d, f32x4 o, float m,
                                           float l) {
    if (to.part) {
        *reinterpret_cast<f32x4*>(to.part + d) = o;
        if (d == 0u) {
            to.ml[0] = m;
            to.ml[1] = l;
        }
    } else {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        store4(a.type, to.out, to.at + d, f32x4{o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv});
    }
}

// The split tile's entry, written by its first part.
constexpr uint32_t kHeadWords = 8u;
__device__ __forceinline__ void write_head(const PagedAttentionArgs& a, const RowWork& w, const Piece& p, uint32_t hk) {
    if (p.parts == 1u || p.part) return;
    u32x4* h = reinterpret_cast<u32x4*>(w.head + kHeadWords * (p.split * a.kv.kv_heads + hk));
    h[0] = u32x4{p.parts, p.q0, p.fresh, p.tile};
    h[1] = u32x4{p.slot, 0u, 0u, 0u};
}

// Whether any of a lane's sums is NaN.
template <uint32_t N, typename V>
__device__ __forceinline__ bool any_nan(const V (&o)[N]) {
    constexpr uint32_t W = sizeof(V) / sizeof(float);
    bool nan = false;
#pragma unroll
    for (uint32_t d = 0; d < N; ++d)
#pragma unroll
        for (uint32_t x = 0; x < W; x += 2) nan = nan || __builtin_isunordered(o[d][x], o[d][x + 1]);
    return nan;
}

// Where the products make NaN and the definition does not.  V is loaded for all rows of a tile, so
// a row that does not see a NaN or an infinity there takes it with weight 0.  And a part of
// q or of a weight can be 0, or of the other sign than the whole: an infinity that a row does
// see, times the parts, is NaN where the score is -inf or the output infinite.  (So can a
// weight that its type rounds to 0.)  Rows whose sums are NaN in the end are rare; then one
// more look at V, for F32 rows at K too, finds the positions that hold NaN or infinities, and
// the rows that do not see all of them, those whose own q has an infinite part, or all if
// there is an infinity, are done again by themselves.  Sums that are NaN because of a NaN that a row sees are right, and cost that look.
constexpr uint32_t kNoPosition = 0x7fffffffu;
struct OddValues {
    uint32_t first, end;  // V's first position that a window can hide (or kNoPosition), its last one's + 1 (or 0)
    uint32_t infinite;    // whether there is an infinity
};
// Of the key tiles t, t + step, .. below t1, loaded from lo on and for sinks up to p_last.
__device__ __forceinline__ OddValues odd_values(const PagedAttentionArgs& a, const Piece& p, const KeyTiles& keys,
                                                uint32_t kt, uint32_t t, uint32_t t1, uint32_t step, uint32_t hk,
                                                uint32_t lo, int32_t p_last) {
    constexpr uint32_t U = 8u;
    const uint32_t lane = threadIdx.x & 63u, lanes = a.kv.head_dim / 8u, rows = 64u / lanes;
    const uint32_t positions = a.table_stride << a.kv.page_shift, mask = (1u << a.kv.page_shift) - 1u;
    const uint32_t infinity = a.kv.type == T_F16 ? 0x7c00u : 0x7f80u;
    const uint32_t* table = a.table + static_cast<uint64_t>(p.r) * a.table_stride;
    const bool f32 = a.type == T_F32;
    OddValues odd{kNoPosition, 0u, 0u};
    for (; t < t1; t += step) {
        const uint32_t base = keys.base(t, kt), at = base + lane;
        const bool in = lane < kt && static_cast<int32_t>(at) <= p_last && at < positions && (at >= lo || at < a.sinks);
        const uint32_t page = in ? table[at >> a.kv.page_shift] : kNoSlot;
        for (uint32_t r0 = lane / lanes; r0 < kt; r0 += U * rows) {
            u32x4 x[U], y[U];
            bool there[U];
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                const uint32_t r = r0 + u * rows, pg = __shfl(page, r & 63u);
                there[u] = r < kt && pg < a.kv.pages;
                const uint64_t row = pg * a.kv.page_stride + ((base + r) & mask) * a.kv.slot_stride + hk * a.kv.head_stride;
                x[u] = *reinterpret_cast<const u32x4*>(a.kv.v + (there[u] ? row + 8u * (lane % lanes) : 0u));
                if (f32) y[u] = *reinterpret_cast<const u32x4*>(a.kv.k + (there[u] ? row + 8u * (lane % lanes) : 0u));
            }
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                bool bad = false, infinite = false;
#pragma unroll
                for (uint32_t d = 0; d < 4; ++d)
#pragma unroll
                    for (uint32_t half = 0; half < 32u; half += 16u) {
                        const uint32_t v = (x[u][d] >> half) & 0x7fffu;
                        bad = bad || v >= infinity;
                        infinite = infinite || v == infinity || (f32 && ((y[u][d] >> half) & 0x7fffu) == infinity);
                    }
                if (infinite && there[u]) odd.infinite = 1u;
                const uint32_t i = base + r0 + u * rows;
                if (bad && there[u]) {
                    odd.end = odd.end > i ? odd.end : i + 1u;
                    if (i >= a.sinks && i < odd.first) odd.first = i;
                }
            }
        }
    }
    return odd;
}
// Of the rows f0 + i whose bit i of `nan` is set, those that have to be done again.
__device__ __forceinline__ uint32_t rows_again(const PagedAttentionArgs& a, const Piece& p, uint32_t hk, uint32_t f0,
                                               uint32_t nan, const OddValues& odd) {
    const uint32_t i = threadIdx.x & 31u, token = a.group(f0 + i), HD = a.kv.head_dim;
    const int32_t pos = p.len - static_cast<int32_t>(p.fresh) + static_cast<int32_t>(token);
    const bool mine = (nan >> i) & 1u;
    bool again = odd.infinite || static_cast<int32_t>(odd.end) > pos + 1 ||
                 (a.window && odd.first + a.window <= static_cast<uint32_t>(pos));
    if (a.type == T_F32 && mine && !again) {
        const float* q = static_cast<const float*>(a.q) + (p.q0 + token) * a.q_stride +
                         (hk * a.group.by + a.group.rest(f0 + i)) * HD;
        // (values from here on are infinite as BF16; F16's parts come under a power of two)
        for (uint32_t d = 0; d < HD; ++d) again = again || fabsf(q[d]) >= 0x1.ffp127f;
    }
    return static_cast<uint32_t>(__ballot(mine && again));
}

// One row over the key tiles t0 .. t1 - 1 by one wave, reading only what the row sees, in FP32.
__device__ __forceinline__ void row_alone(const PagedAttentionArgs& a, const Piece& p, const KeyTiles& keys,
                                          uint32_t kt, uint32_t t0, uint32_t t1, uint32_t hk, uint32_t f, float bias,
                                          const RowTo& to) {
    constexpr uint32_t U = 8u;
    const uint32_t lane = threadIdx.x & 63u, HD = a.kv.head_dim, token = p.q0 + a.group(f);
    const int32_t pos = p.len - static_cast<int32_t>(p.fresh) + static_cast<int32_t>(a.group(f));
    const uint64_t at = token * a.q_stride + (hk * a.group.by + a.group.rest(f)) * HD;
    const float c = a.scale * 1.4426950408889634f;
    const uint32_t mask = (1u << a.kv.page_shift) - 1u, column = 4u * lane % HD;
    const uint32_t* table = a.table + static_cast<uint64_t>(p.r) * a.table_stride;
    float m = -INFINITY, l = 0.0f;
    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t t = t0; t < t1 && l == l; ++t) {  // a sum that is NaN stays so
        const uint32_t i = keys.base(t, kt) + lane;
        uint32_t page = kNoSlot;
        if (lane < kt && row_sees(pos, i, a.window, a.sinks) && (i >> a.kv.page_shift) < a.table_stride)
            page = table[i >> a.kv.page_shift];
        const bool seen = page < a.kv.pages;
        const uint64_t row = seen ? page * a.kv.page_stride + (i & mask) * a.kv.slot_stride + hk * a.kv.head_stride : 0u;
        const uint64_t all = __ballot(seen);
        if (!all) continue;
        float s = 0.0f;
        for (uint32_t d = 0; d < HD; d += 8u) {
            const u32x4 k = *reinterpret_cast<const u32x4*>(a.kv.k + row + d);
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) {
                const float q = a.type == T_F32 ? static_cast<const float*>(a.q)[at + d + e]
                                                : cache_value(a.type, static_cast<const uint16_t*>(a.q)[at + d + e]);
                s = fmaf(q, cache_value(a.kv.type, static_cast<uint16_t>(k[e / 2u] >> (16u * (e % 2u)))), s);
            }
        }
        s = seen ? s * c : -INFINITY;
        float top = s;
        for (uint32_t d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
        const float next = fmaxf(m, top), ref = next == -INFINITY ? 0.0f : next;
        const float e = exp2f(s - ref + bias), keep = exp2f(m - ref);
        float es = e;
        for (uint32_t d = 32; d > 0; d >>= 1) es += __shfl_xor(es, d);
        l = l * keep + es;
        for (uint32_t k = 0; k < 4u; ++k) o[k] *= keep;
        for (uint32_t j = 0; j < kt; j += U) {
            u32x2 v[U];
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) v[u] = *reinterpret_cast<const u32x2*>(a.kv.v + __shfl(row, j + u) + column);
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                const float x = __shfl(e, j + u);
                if (!((all >> (j + u)) & 1u)) continue;
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k)
                    o[k] = fmaf(x, cache_value(a.kv.type, static_cast<uint16_t>(v[u][k / 2u] >> (16u * (k % 2u)))), o[k]);
            }
        }
        m = next;
    }
    if (4u * lane < HD) store_row4(a, to, 4u * lane, f32x4{o[0], o[1], o[2], o[3]}, m, l);
}

__device__ __forceinline__ float max_over(float v, uint32_t d) { return fmaxf(v, __shfl_xor(v, d)); }
// The maximum with the lane 32 (16) lanes away.
__device__ __forceinline__ float max_32(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto w = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
}
__device__ __forceinline__ float max_16(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto w = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
}

// A lane's part of its row: 8 values at q + at + STEP * k of each k, as parts.  F16 parts of
// FP32 rows come under a power of two, which goes to c; the row's other lanes are MIN, 2 MIN ..
// lanes away.
template <uint32_t T, bool F32, uint32_t KK, uint32_t STEP, uint32_t MIN>
__device__ __forceinline__ void load_q(const PagedAttentionArgs& a, uint64_t at, bool live,
                                       typename Mat<T>::V8 (*q)[KK], float& c) {
    using M = Mat<T>;
    constexpr uint32_t NP = parts_of(T, F32);
    if constexpr (!F32) {
#pragma unroll
        for (uint32_t k = 0; k < KK; ++k) {
            u32x4 x = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + at + STEP * k);
            if (!live) x = u32x4{0u, 0u, 0u, 0u};
            q[0][k] = __builtin_bit_cast(typename M::V8, x);
        }
    } else {
        float v[KK][8], top = 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < KK; ++k) {
            const f32x4* src = reinterpret_cast<const f32x4*>(static_cast<const float*>(a.q) + at + STEP * k);
            const f32x4 x = src[0], y = src[1];
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) {
                v[k][e] = !live ? 0.0f : e < 4u ? x[e & 3u] : y[e & 3u];
                top = fmaxf(top, fabsf(v[k][e]));
            }
        }
        if constexpr (T == T_F16) {
#pragma unroll
            for (uint32_t d = MIN; d < 64u; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
            // the largest value to [2^14, 2^15)
            const int ex = top > 0.0f && top < INFINITY ? static_cast<int>(__float_as_uint(top) >> 23) - 127 - 14 : 0;
            const float up = ldexpf(1.0f, -ex / 2), up2 = ldexpf(1.0f, -ex - (-ex / 2));
#pragma unroll
            for (uint32_t k = 0; k < KK; ++k)
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) v[k][e] = v[k][e] * up * up2;
            c = fmaxf(ldexpf(c, ex), 1.1754944e-38f);
        }
#pragma unroll
        for (uint32_t k = 0; k < KK; ++k) {
            typename M::V8 part[NP];
            split8<M, NP>(v[k], part);
#pragma unroll
            for (uint32_t i = 0; i < NP; ++i) q[i][k] = part[i];
        }
    }
}

// ---------------------------------------------------------------------------
// Few rows (single tokens): one tile of 16 rows, four waves that take the tile's keys in
// turn, 32 at a time, straight from memory into the matrix operands.
//
// K rows are the first product's A operand as they lie (8 values of a row per lane).  V is
// the second product's A operand transposed, a value of 8 rows per lane: a lane loads the
// same HD / 16 columns of 8 rows and exchanges halves of its own registers, and column
// (l % 16) * HD / 16 + e is row l % 16 of product e.  Reading K and V bounds it: the next
// K is on its way while the weights are taken, the next V while the next scores are.  32
// heads over 4 of 128, F16: 131,072 positions 42.5 us (6.3 TB/s); 64 requests up to 8192
// positions, BF16, 70 us (4.8 TB/s, uneven requests); eight of 512, F32, 10.4 us, where the
// 64 KB of a workgroup's 128 keys take a CU 1.3 us (50 GB/s).  Eight waves share out the same
// reading: eight requests of 500 10.2 -> 10.0 us, one of 131,072 57.9 -> 56.6, 64 up to 8192
// 79 -> 89.
template <uint32_t HD>
struct RowsLds {
    alignas(16) uint64_t off[4][32];
    alignas(16) float o[4][16][HD + 4u];
    float m[4][16], l[4][16];
    uint32_t nan, first, end, infinite;
};

template <uint32_t T, uint32_t HD, bool F32>
__device__ __forceinline__ void rows_piece(const PagedAttentionArgs& a, const RowWork& w, uint32_t block, RowsLds<HD>& lds) {
    using M = Mat<T>;
    using V8 = typename M::V8;
    constexpr uint32_t NP = parts_of(T, F32), KK = HD / 32u, DPL = HD / 16u, BM = 16u, KT = 32u;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, g = lane >> 4, j = lane & 15u;
    const uint32_t hk = block % a.kv.kv_heads;
    Piece p;
    uint32_t splits;
    const bool live_piece = find_piece(a, w, BM, block / a.kv.kv_heads, p, splits);
    if (w.count && block == 0u && tid == 0u) w.count[0] = splits * a.kv.kv_heads;
    if (!live_piece) return;
    if (tid == 0u) {
        write_head(a, w, p, hk);
        lds.nan = lds.end = lds.infinite = 0u;
        lds.first = kNoPosition;
    }
    const uint32_t rows = p.fresh * a.group.by - p.tile * BM < BM ? p.fresh * a.group.by - p.tile * BM : BM;
    const uint32_t positions = a.table_stride << a.kv.page_shift, mask = (1u << a.kv.page_shift) - 1u;
    const int32_t p0 = p.len - static_cast<int32_t>(p.fresh);
    const int32_t p_first = p0 + static_cast<int32_t>(a.group(p.tile * BM));
    const int32_t p_last = p0 + static_cast<int32_t>(a.group(p.tile * BM + rows - 1u));
    const KeyTiles keys = key_tiles(p_first, p_last, a.window, a.sinks, positions, KT);
    uint32_t b0, b1;
    part_range(keys.tiles, p.part, p.parts, b0, b1);
    // this lane's row: q parts and position
    const uint32_t f = p.tile * BM + j;
    const bool live = j < rows;
    const int32_t pos = live ? p0 + static_cast<int32_t>(a.group(f)) : -1;
    V8 q[NP][KK];
    float c = a.scale * 1.4426950408889634f;
    const float bias = weight_bias<T>(p.len);
    load_q<T, F32, KK, 32u, 16u>(a, (p.q0 + (live ? a.group(f) : 0u)) * a.q_stride +
                                    (hk * a.group.by + (live ? a.group.rest(f) : 0u)) * HD + 8u * g, live, q, c);
    const uint32_t* table = a.table + static_cast<uint64_t>(p.r) * a.table_stride;
    const uint16_t* kbase = a.kv.k + hk * a.kv.head_stride + 8u * g;
    const uint16_t* vbase = a.kv.v + hk * a.kv.head_stride + DPL * j;
    const uint32_t lo = a.window && p_first >= 0 && static_cast<uint32_t>(p_first) + 1u > a.window
                            ? static_cast<uint32_t>(p_first) + 1u - a.window : 0u;
    // the table entry of position base(b) + lane % 32, where any row may see it
    auto entry = [&](uint32_t b) -> uint32_t {
        const uint32_t i = keys.base(b, KT) + (lane & 31u);
        const bool in = static_cast<int32_t>(i) <= p_last && i < positions && (i >= lo || i < a.sinks);
        return in ? table[i >> a.kv.page_shift] : kNoSlot;
    };
    uint32_t there = 0u;
    auto place = [&](uint32_t b, uint32_t page) {
        const uint32_t i = keys.base(b, KT) + (lane & 31u);
        const bool in = page < a.kv.pages;
        there = static_cast<uint32_t>(__ballot(in));
        lds.off[wave][lane & 31u] = in ? page * a.kv.page_stride + (i & mask) * a.kv.slot_stride : 0u;
        __builtin_amdgcn_wave_barrier();
    };
    u32x4 kr[2][KK];
    constexpr uint32_t VW = DPL / 2u;  // dwords of a V row per lane
    uint32_t vr[8][VW];
    auto load_k = [&] {
#pragma unroll
        for (uint32_t t = 0; t < 2; ++t) {
            const uint16_t* src = kbase + lds.off[wave][16u * t + j];
#pragma unroll
            for (uint32_t k = 0; k < KK; ++k) kr[t][k] = *reinterpret_cast<const u32x4*>(src + 32u * k);
        }
    };
    auto load_v = [&] {
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            const uint16_t* src = vbase + lds.off[wave][16u * (e / 4u) + 4u * g + e % 4u];
            if constexpr (VW == 2u) {
                const u32x2 x = *reinterpret_cast<const u32x2*>(src);
                vr[e][0] = x[0];
                vr[e][1] = x[1];
            } else {
#pragma unroll
                for (uint32_t h = 0; h < VW / 4u; ++h) {
                    const u32x4 x = reinterpret_cast<const u32x4*>(src)[h];
#pragma unroll
                    for (uint32_t y = 0; y < 4; ++y) vr[e][4u * h + y] = x[y];
                }
            }
        }
    };
    f32x4 o[DPL];
#pragma unroll
    for (uint32_t e = 0; e < DPL; ++e) o[e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    uint32_t b = b0 + wave, next_page = kNoSlot;
    if (b < b1) {
        place(b, entry(b));
        load_k();
        load_v();
        if (b + 4u < b1) next_page = entry(b + 4u);
    }
    for (; b < b1; b += 4u) {
        const uint32_t base = keys.base(b, KT), here = there;
        f32x4 s[2];
#pragma unroll
        for (uint32_t t = 0; t < 2; ++t) {
            s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (uint32_t k = 0; k < KK; ++k)
#pragma unroll
                for (uint32_t i = 0; i < NP; ++i) s[t] = M::mma16(__builtin_bit_cast(V8, kr[t][k]), q[i][k], s[t]);
        }
        const bool more = b + 4u < b1;
        if (more) {
            place(b + 4u, next_page);
            load_k();
            if (b + 8u < b1) next_page = entry(b + 8u);
        }
        __builtin_amdgcn_sched_barrier(0);
        // every row sees the whole tile, or each score asks
        const bool cut = here != 0xffffffffu || static_cast<int32_t>(base + KT) - 1 > p_first ||
                         (a.window && base + a.window <= static_cast<uint32_t>(p_last) && base + KT > a.sinks);
        if (cut) {
#pragma unroll
            for (uint32_t t = 0; t < 2; ++t)
#pragma unroll
                for (uint32_t x = 0; x < 4; ++x) {
                    const uint32_t at = 16u * t + 4u * g + x;
                    if (!((here >> at) & 1u) || !row_sees(pos, base + at, a.window, a.sinks)) s[t][x] = -INFINITY;
                }
            if (here != 0xffffffffu)
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e)
                    if (!((here >> (16u * (e / 4u) + 4u * g + e % 4u)) & 1u))
#pragma unroll
                        for (uint32_t y = 0; y < VW; ++y) vr[e][y] = 0u;
        }
        float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                          fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        top = max_32(max_16(top)) * c;
        if (__any(top > m + kSlack)) {
            const float mm = fmaxf(m, top), keep = mm == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mm);
            m = mm;
            l *= keep;
#pragma unroll
            for (uint32_t e = 0; e < DPL; ++e) o[e] = o[e] * keep;
        }
        const float ref = m == -INFINITY ? 0.0f : m - bias;
        float pw[8];
#pragma unroll
        for (uint32_t x = 0; x < 8; ++x) {
            pw[x] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x / 4u][x % 4u], c, -ref));
            l += pw[x];
        }
        V8 pp[NP];
        split8<M, NP>(pw, pp);
#pragma unroll
        for (uint32_t e = 0; e < DPL; ++e) {
            u32x4 x;
#pragma unroll
            for (uint32_t y = 0; y < 4; ++y)
                x[y] = __builtin_amdgcn_perm(vr[2u * y + 1u][e / 2u], vr[2u * y][e / 2u],
                                             e % 2u ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (uint32_t i = 0; i < NP; ++i) o[e] = M::mma16(__builtin_bit_cast(V8, x), pp[i], o[e]);
        }
        if (more) load_v();
        __builtin_amdgcn_sched_barrier(0);
    }
    // the four waves' parts
    l += __shfl_xor(l, 16u);
    l += __shfl_xor(l, 32u);
    if (g == 0u) {
        lds.m[wave][j] = m;
        lds.l[wave][j] = l;
    }
    __syncthreads();  // lds.nan is 0 as well
    if (j < rows && (l == l ? any_nan(o) : F32)) atomicOr(&lds.nan, 1u << j);
    {
        const float mm = fmaxf(fmaxf(lds.m[0][j], lds.m[1][j]), fmaxf(lds.m[2][j], lds.m[3][j]));
        const float keep = mm == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mm);
#pragma unroll
        for (uint32_t x = 0; x < 4; ++x)
#pragma unroll
            for (uint32_t e = 0; e < DPL; e += 4)
                *reinterpret_cast<f32x4*>(&lds.o[wave][j][(4u * g + x) * DPL + e]) =
                    f32x4{o[e][x] * keep, o[e + 1][x] * keep, o[e + 2][x] * keep, o[e + 3][x] * keep};
    }
    __syncthreads();
    const uint32_t row = tid / 16u;
    const float mm = fmaxf(fmaxf(lds.m[0][row], lds.m[1][row]), fmaxf(lds.m[2][row], lds.m[3][row]));
    float sum = 0.0f;
#pragma unroll
    for (uint32_t v = 0; v < 4; ++v) sum += mm == -INFINITY ? lds.l[v][row] : lds.l[v][row] * __builtin_amdgcn_exp2f(lds.m[v][row] - mm);
    uint32_t again = lds.nan;
    if (again) {
        const OddValues odd = odd_values(a, p, keys, KT, b0 + wave, b1, 4u, hk, lo, p_last);
        atomicMax(&lds.end, odd.end);
        atomicMin(&lds.first, odd.first);
        atomicOr(&lds.infinite, odd.infinite);
        __syncthreads();
        again = rows_again(a, p, hk, p.tile * BM, again, {lds.first, lds.end, lds.infinite});
    }
    if (row < rows && !((again >> row) & 1u)) {
        const RowTo to = row_to(a, w, p, BM, hk, row);
#pragma unroll
        for (uint32_t k = 0; k < HD / 64u; ++k) {
            const uint32_t d = 64u * k + 4u * (tid % 16u);
            f32x4 r = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (uint32_t v = 0; v < 4; ++v) r = r + *reinterpret_cast<const f32x4*>(&lds.o[v][row][d]);
            store_row4(a, to, d, r, mm, sum);
        }
    }
    if (again)
        for (uint32_t i = wave; i < rows; i += 4u)
            if ((again >> i) & 1u) row_alone(a, p, keys, KT, b0, b1, hk, p.tile * BM + i, bias, row_to(a, w, p, BM, hk, i));
}

// ---------------------------------------------------------------------------
// Many rows (chunks of prompts): tiles of 128 rows, 32 per wave, over tiles of 64 keys that
// all four waves read from LDS, two tiles of K and V in turn: one is read while the other's
// loads go straight into LDS.  A row of a tile is HD / 8 pieces of 16 bytes; piece c of row r
// lies at c ^ swizzle(r), so that neither the 32 rows that the first product reads side by
// side nor the 4 rows by 32 columns of the transposing reads of the second meet in a bank (the
// counter of bank conflicts is 0).  32 heads over 4 of 128, BF16: a prompt of 8192 tokens
// 555 us (991 TFLOP/s, 75% of a large library product's rate); the matrix cores are busy half of
// the cycles and the softmax's vector instructions are issued in the other half.  Four waves of
// 32 rows rather than eight: two workgroups of them fit a CU and hide each other's barriers.
constexpr uint32_t kTileRows = 128u, kTileKeys = 64u;

template <uint32_t HD>
__device__ __forceinline__ uint32_t swizzle(uint32_t r) {
    return HD == 64u ? (((r >> 1) & 1u) << 2) | ((r >> 2) & 3u) : ((r & 3u) << 2) | ((r >> 2) & 3u);
}

// What a row that is not there is read from.
__device__ __attribute__((aligned(16))) uint16_t g_no_row[256];

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef s16x4 __attribute__((address_space(3))) * lds_s16x4;
typedef uint8_t __attribute__((address_space(3))) * lds_ptr;

// 16 bytes per lane from src (+ a lane's offset) into LDS, lane after lane from `to` (the
// same for all lanes), which the instruction takes in m0.  Written out, since the builtin
// makes every later LDS read wait for it: the loop waits itself, once per tile, before the
// barrier that lets the tile be read.
__device__ __forceinline__ void load_to_lds(const void* src, uint32_t to) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "{m0}"(to) : "memory");
}
__device__ __forceinline__ void load_to_lds(const void* src, uint32_t offset, uint32_t to) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(src), "{m0}"(to) : "memory");
}

template <uint32_t HD>
struct TilesLds {
    alignas(1024) uint8_t k[2][kTileKeys * 2u * HD], v[2][kTileKeys * 2u * HD];
    uint32_t nan, first, end, infinite;
};

template <uint32_t T, uint32_t HD, bool F32>
__device__ __forceinline__ void tiles_piece(const PagedAttentionArgs& a, const RowWork& w, uint32_t block, TilesLds<HD>& lds) {
    using M = Mat<T>;
    using V8 = typename M::V8;
    constexpr uint32_t NP = parts_of(T, F32), KK = HD / 16u, DT = HD / 32u, BM = kTileRows, KT = kTileKeys;
    constexpr uint32_t ROWB = 2u * HD, CH = HD / 8u, RPI = 1024u / ROWB, NI = KT / RPI / 4u;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t h = lane >> 5, j = lane & 31u, hk = block % a.kv.kv_heads;
    Piece p;
    uint32_t splits;
    const bool live_piece = find_piece(a, w, BM, block / a.kv.kv_heads, p, splits);
    if (w.count && block == 0u && tid == 0u) w.count[0] = splits * a.kv.kv_heads;
    if (!live_piece) return;
    if (tid == 0u) {
        write_head(a, w, p, hk);
        lds.nan = lds.end = lds.infinite = 0u;
        lds.first = kNoPosition;
    }
    const uint32_t left = p.fresh * a.group.by - p.tile * BM, rows = left < BM ? left : BM;
    const uint32_t positions = a.table_stride << a.kv.page_shift, mask = (1u << a.kv.page_shift) - 1u;
    const int32_t p0 = p.len - static_cast<int32_t>(p.fresh);
    const int32_t p_first = p0 + static_cast<int32_t>(a.group(p.tile * BM));
    const int32_t p_last = p0 + static_cast<int32_t>(a.group(p.tile * BM + rows - 1u));
    const KeyTiles keys = key_tiles(p_first, p_last, a.window, a.sinks, positions, KT);
    uint32_t t0, t1;
    part_range(keys.tiles, p.part, p.parts, t0, t1);
    const uint32_t lo = a.window && p_first >= 0 && static_cast<uint32_t>(p_first) + 1u > a.window
                            ? static_cast<uint32_t>(p_first) + 1u - a.window : 0u;
    // this wave's rows and this lane's
    const uint32_t f0 = p.tile * BM + 32u * wave, f = f0 + j;
    const bool live = 32u * wave + j < rows, wave_live = 32u * wave < rows;
    const uint32_t wrows = wave_live ? (rows - 32u * wave < 32u ? rows - 32u * wave : 32u) : 0u;
    const int32_t w_first = p0 + static_cast<int32_t>(a.group(f0));
    const int32_t w_last = wave_live ? p0 + static_cast<int32_t>(a.group(f0 + wrows - 1u)) : -1;
    const int32_t pos = live ? p0 + static_cast<int32_t>(a.group(f)) : -1;
    V8 q[NP][KK];
    float c = a.scale * 1.4426950408889634f;
    const float bias = weight_bias<T>(p.len);
    load_q<T, F32, KK, 16u, 32u>(a, (p.q0 + (live ? a.group(f) : 0u)) * a.q_stride +
                                    (hk * a.group.by + (live ? a.group.rest(f) : 0u)) * HD + 8u * h, live, q, c);
    // Loads: the wave brings 16 rows, a lane 16 bytes of a row at a time.  Lane i asks the table
    // for position i of the tile; where all of them are there and pages hold 16 rows or more,
    // the rest is scalar: the address of the wave's rows and fixed offsets.
    const uint32_t* table = a.table + static_cast<uint64_t>(p.r) * a.table_stride;
    const uint32_t in_row = lane / CH;
    const uint32_t lds_k = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_ptr)&lds.k[0][0]));
    const uint32_t lds_v = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_ptr)&lds.v[0][0]));
    const bool plain = a.kv.page_shift >= 4u && a.kv.slot_stride < (1u << 26);
    uint32_t offset[NI];
#pragma unroll
    for (uint32_t n = 0; n < NI; ++n)
        offset[n] = 2u * ((n * RPI + in_row) * static_cast<uint32_t>(a.kv.slot_stride) +
                          8u * ((lane % CH) ^ swizzle<HD>((wave * NI + n) * RPI + in_row)));
    auto entry = [&](uint32_t t) -> uint32_t {
        const uint32_t i = keys.base(t, KT) + lane;
        const bool in = static_cast<int32_t>(i) <= p_last && i < positions && (i >= lo || i < a.sinks);
        return in ? table[i >> a.kv.page_shift] : kNoSlot;
    };
    auto load = [&](uint32_t t, uint32_t page, uint32_t buf) -> uint64_t {
        const uint32_t base = keys.base(t, KT);
        const uint64_t there = __ballot(page < a.kv.pages);
        if (plain && there == ~0ull) {
            const uint32_t pg = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(page), static_cast<int>(16u * wave)));
            const uint64_t off = pg * a.kv.page_stride + ((base + 16u * wave) & mask) * a.kv.slot_stride + hk * a.kv.head_stride;
            const uint32_t to = buf * KT * ROWB + wave * NI * 1024u;
#pragma unroll
            for (uint32_t n = 0; n < NI; ++n) {
                load_to_lds(a.kv.k + off, offset[n], lds_k + to + n * 1024u);
                load_to_lds(a.kv.v + off, offset[n], lds_v + to + n * 1024u);
            }
        } else {
#pragma unroll
            for (uint32_t n = 0; n < NI; ++n) {
                const uint32_t row = (wave * NI + n) * RPI + in_row, to = buf * KT * ROWB + (wave * NI + n) * 1024u;
                const uint32_t piece = 8u * ((lane % CH) ^ swizzle<HD>(row)), pg = __shfl(page, row);
                const uint64_t off = pg * a.kv.page_stride + ((base + row) & mask) * a.kv.slot_stride + hk * a.kv.head_stride;
                const bool in = pg < a.kv.pages;
                load_to_lds((in ? a.kv.k + off : g_no_row) + piece, lds_k + to);
                load_to_lds((in ? a.kv.v + off : g_no_row) + piece, lds_v + to);
            }
        }
        return there;
    };
    // where this lane reads: K row j, its piece 2 k + h; V rows 4 h + 8 second + (lane % 16) / 4,
    // columns 32 dt + 16 ((lane / 16) % 2) + 4 (lane % 4)
    const uint32_t kf = swizzle<HD>(j) ^ h;
    uint32_t vat[2][DT];
#pragma unroll
    for (uint32_t second = 0; second < 2; ++second)
#pragma unroll
        for (uint32_t dt = 0; dt < DT; ++dt) {
            const uint32_t row = 4u * h + 8u * second + (lane & 15u) / 4u;
            const uint32_t piece = 4u * dt + 2u * ((lane >> 4) & 1u) + (lane & 3u) / 2u;
            vat[second][dt] = row * ROWB + 16u * (piece ^ swizzle<HD>(row)) + 8u * (lane & 1u);
        }
    f32x16 o[DT];
#pragma unroll
    for (uint32_t d = 0; d < DT; ++d)
#pragma unroll
        for (uint32_t x = 0; x < 16; ++x) o[d][x] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    uint64_t next_there = 0;
    uint32_t page = kNoSlot;
    if (t0 < t1) {
        next_there = load(t0, entry(t0), 0u);
        if (t0 + 1u < t1) page = entry(t0 + 1u);
    }
    for (uint32_t t = t0; t < t1; ++t) {
        const uint32_t buf = (t - t0) & 1u, base = keys.base(t, KT);
        const uint64_t there = next_there;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's loads of the tile have landed
        __syncthreads();                                  // and everyone's; the other buffer has been read
        if (t + 1u < t1) {
            next_there = load(t + 1u, page, buf ^ 1u);
            if (t + 2u < t1) page = entry(t + 2u);
        }
        // nothing of the tile for this wave's rows
        if (static_cast<int32_t>(base) > w_last ||
            (a.window && w_first >= 0 && base + (KT - 1u) + a.window <= static_cast<uint32_t>(w_first) && base >= a.sinks))
            continue;
        f32x16 s[2];
#pragma unroll
        for (uint32_t ks = 0; ks < 2; ++ks)
#pragma unroll
            for (uint32_t x = 0; x < 16; ++x) s[ks][x] = 0.0f;
        const uint8_t* kb = lds.k[buf] + j * ROWB;
#pragma unroll
        for (uint32_t k = 0; k < KK; ++k)
#pragma unroll
            for (uint32_t ks = 0; ks < 2; ++ks) {
                const V8 x = *reinterpret_cast<const V8*>(kb + 32u * ks * ROWB + 16u * (kf ^ (2u * k)));
#pragma unroll
                for (uint32_t i = 0; i < NP; ++i) s[ks] = M::mma32(x, q[i][k], s[ks]);
            }
        // LDS answers late: six reads ahead of the products
        __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
        for (uint32_t k = 0; k < 2u * KK - 6u; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x008, NP, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 6u * NP, 0);
        const bool cut = there != ~0ull || static_cast<int32_t>(base + KT) - 1 > w_first ||
                         (a.window && base + a.window <= static_cast<uint32_t>(w_last) && base + KT > a.sinks);
        if (cut) {
            const uint64_t mine = there >> (4u * h);
#pragma unroll
            for (uint32_t ks = 0; ks < 2; ++ks)
#pragma unroll
                for (uint32_t x = 0; x < 16; ++x) {
                    const uint32_t i = 32u * ks + 8u * (x / 4u) + x % 4u;  // + 4 h: the key in its tile
                    if (!((mine >> i) & 1u) || !row_sees(pos, base + i + 4u * h, a.window, a.sinks)) s[ks][x] = -INFINITY;
                }
        }
        float top = -INFINITY;
#pragma unroll
        for (uint32_t ks = 0; ks < 2; ++ks)
#pragma unroll
            for (uint32_t x = 0; x < 16; ++x) top = fmaxf(top, s[ks][x]);
        top = max_32(top) * c;
        if (__any(top > m + kSlack)) {
            const float mm = fmaxf(m, top), keep = mm == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mm);
            m = mm;
            l *= keep;
#pragma unroll
            for (uint32_t d = 0; d < DT; ++d) o[d] = o[d] * keep;
        }
        const float ref = m == -INFINITY ? 0.0f : m - bias;
#pragma unroll
        for (uint32_t ks = 0; ks < 2; ++ks)
#pragma unroll
            for (uint32_t t16 = 0; t16 < 2; ++t16) {
                float pw[8];
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) {
                    pw[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ks][8u * t16 + e], c, -ref));
                    l += pw[e];
                }
                V8 pp[NP];
                split8<M, NP>(pw, pp);
#pragma unroll
                for (uint32_t d = 0; d < DT; ++d) {
                    struct { s16x4 a, b; } x;
                    uint8_t* vb = lds.v[buf] + (32u * ks + 16u * t16) * ROWB;
                    x.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(vb + vat[0][d]));
                    x.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(vb + vat[1][d]));
#pragma unroll
                    for (uint32_t i = 0; i < NP; ++i) o[d] = M::mma32(__builtin_bit_cast(V8, x), pp[i], o[d]);
                }
            }
    }
    l += __shfl_xor(l, 32u);
    const uint64_t either = __ballot(live && (l == l ? any_nan(o) : F32));
    const uint32_t nan = static_cast<uint32_t>(either | (either >> 32));
    if (nan && lane == 0u) atomicOr(&lds.nan, 1u);  // (a barrier of the loop ago it was set to 0)
    if (live) {
        const RowTo to = row_to(a, w, p, BM, hk, 32u * wave + j);
#pragma unroll
        for (uint32_t d = 0; d < DT; ++d)
#pragma unroll
            for (uint32_t x = 0; x < 16; x += 4)
                store_row4(a, to, 32u * d + 2u * x + 4u * h, f32x4{o[d][x], o[d][x + 1], o[d][x + 2], o[d][x + 3]}, m, l);
    }
    __syncthreads();
    if (!lds.nan) return;
    const OddValues odd = odd_values(a, p, keys, KT, t0 + wave, t1, 4u, hk, lo, p_last);
    atomicMax(&lds.end, odd.end);
    atomicMin(&lds.first, odd.first);
    atomicOr(&lds.infinite, odd.infinite);
    __syncthreads();
    // (the stores of the rows that are done again came before the barrier)
    uint32_t again = rows_again(a, p, hk, f0, nan, {lds.first, lds.end, lds.infinite});
    while (again) {
        const uint32_t i = static_cast<uint32_t>(__builtin_ctz(again));
        again &= again - 1u;
        row_alone(a, p, keys, KT, t0, t1, hk, f0 + i, bias, row_to(a, w, p, BM, hk, 32u * wave + i));
    }
}

// At most 256 registers up to head_dim 128 (two workgroups a CU): given 512, the compiler keeps
// operands in the accumulator half and moves them over for every tile.  F32 rows, four chunks
// of 512 over 2048, 16 heads over 4: of 128 over F16 118 us, with 256 88, over BF16 135 and 110
// (a few spills), of 64 over F16 65 and 59.  At 256 the LDS holds one workgroup; its single
// tokens, held to 256 registers, would spill (16 of 2000, F32: 30 us, 57).
// One launch: the tiles' workgroups first, they take longest.
template <uint32_t T, uint32_t HD, bool F32>
__global__ __launch_bounds__(256, HD <= 128u ? 2 : 1) void k_paged_chunks(PagedAttentionArgs a, RowWork many,
                                                                                RowWork few, uint32_t tile_blocks) {
    __shared__ union Lds {
        TilesLds<HD> tiles;
        RowsLds<HD> rows;
    } lds;
    if (blockIdx.x < tile_blocks) tiles_piece<T, HD, F32>(a, many, blockIdx.x, lds.tiles);
    else rows_piece<T, HD, F32>(a, few, blockIdx.x - tile_blocks, lds.rows);
}

template <uint32_t T, uint32_t HD, bool F32>
__global__ __launch_bounds__(256, HD <= 128u ? 2 : 1) void k_paged_rows(PagedAttentionArgs a, RowWork few) {
    __shared__ RowsLds<HD> lds;
    rows_piece<T, HD, F32>(a, few, blockIdx.x, lds);
}

// ---------------------------------------------------------------------------
// Joins the parts of split tiles: o = sum_i o_i 2^(m_i - m), m the parts' maximum, and l
// likewise.  HD / 4 lanes hold a row.  Parts come from other XCDs' caches, so latency bounds
// it: several parts' loads are on the way at once.  128 parts of four tiles 5.4 us, 1024 parts
// of 16-row tiles 6.8, 500 of 128-row ones 11.6.
constexpr uint32_t kMostParts = 2048u;

struct SplitTile {
    Piece p;
    uint32_t parts, rows;
    uint64_t stride;  // floats from a part to the next
    const float* base;
};
// Entry i, if there is one (entries past the last hold what an earlier call left, and so do
// those of tiles that no workgroup took, where query_start decreases).
__device__ __forceinline__ bool split_tile(const PagedAttentionArgs& a, const RowWork& w, uint32_t bm, uint32_t i, SplitTile& t) {
    const u32x4* h = reinterpret_cast<const u32x4*>(w.head + kHeadWords * i);
    const uint32_t HD = a.kv.head_dim, hk = i % a.kv.kv_heads, count = w.count[0];
    const u32x4 x = h[0];
    const uint32_t slot = h[1][0];
    if (i >= count || !split_entry_fits(x[0], slot, x[1], x[2], x[3], a.group.by, bm, a.max_new, a.max_tokens,
                                        a.kv.kv_heads, 1u << w.log_target))
        return false;
    t.p = Piece{};
    t.parts = x[0];
    t.p.parts = 1u;
    t.p.q0 = x[1];
    t.p.fresh = x[2];
    t.p.tile = x[3];
    const uint32_t left = t.p.fresh * a.group.by - t.p.tile * bm;
    t.rows = left < bm ? left : bm;
    t.stride = static_cast<uint64_t>(a.kv.kv_heads) * bm * (HD + 2u);
    t.base = w.part + static_cast<uint64_t>(slot * a.kv.kv_heads + hk) * bm * (HD + 2u);
    return true;
}

// 16-row tiles: few rows of up to kMostParts parts.  A workgroup takes rows y, y + step, ..;
// HD / 4 lanes hold a row's sums, the others other parts, the first JU of them on the way
// before the maxima are known.
template <uint32_t HD>
__device__ __forceinline__ void join_rows(const PagedAttentionArgs& a, const RowWork& w, uint32_t i, uint32_t y, uint32_t step) {
    constexpr uint32_t BM = 16u, LANES = HD / 4u, GROUPS = 256u / LANES, JU = 8u;
    __shared__ __attribute__((aligned(16))) float s_o[GROUPS][HD];
    __shared__ float s_w[kMostParts], s_red[2][4];
    const uint32_t tid = threadIdx.x, lane = tid % LANES, grp = tid / LANES, wave = tid >> 6;
    SplitTile t;
    if (!split_tile(a, w, BM, i, t)) return;
    for (uint32_t row = y; row < t.rows; row += step) {
        const float* ml = t.base + BM * HD + 2u * row;
        const float* at = t.base + row * HD + 4u * lane;
        f32x4 x[JU];
        auto load = [&](uint32_t k0) {
#pragma unroll
            for (uint32_t k = 0; k < JU; ++k) {
                const uint32_t n = k0 + GROUPS * k;
                x[k] = *reinterpret_cast<const f32x4*>(at + (n < t.parts ? n : 0u) * t.stride);
            }
        };
        float m = tid < t.parts ? ml[tid * t.stride] : -INFINITY, l = tid < t.parts ? ml[tid * t.stride + 1u] : 0.0f;
        const float m0 = m, l0 = l;
        load(grp);
        for (uint32_t k = tid + 256u; k < t.parts; k += 256u) m = fmaxf(m, ml[k * t.stride]);
        for (uint32_t d = 1; d < 16u; d *= 2) m = max_over(m, d);
        m = max_32(max_16(m));
        if ((tid & 63u) == 0u) s_red[0][wave] = m;
        __syncthreads();
        m = fmaxf(fmaxf(s_red[0][0], s_red[0][1]), fmaxf(s_red[0][2], s_red[0][3]));
        // m = -inf: nothing seen, or NaN alone, which has to stay
        auto weight = [&](float part_m) { return m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(part_m - m); };
        s_w[tid] = weight(m0);
        l = l0 * s_w[tid];
        if (tid >= t.parts) l = 0.0f;
        for (uint32_t k = tid + 256u; k < t.parts; k += 256u) {
            const float f = weight(ml[k * t.stride]);
            s_w[k] = f;
            l += ml[k * t.stride + 1u] * f;
        }
        l = group_sum<64>(l);
        if ((tid & 63u) == 63u) s_red[1][wave] = l;
        __syncthreads();
        l = (s_red[1][0] + s_red[1][1]) + (s_red[1][2] + s_red[1][3]);
        f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t k0 = grp;;) {
#pragma unroll
            for (uint32_t k = 0; k < JU; ++k)
                if (k0 + GROUPS * k < t.parts) o = o + x[k] * s_w[k0 + GROUPS * k];
            k0 += GROUPS * JU;
            if (k0 >= t.parts) break;
            load(k0);
        }
        *reinterpret_cast<f32x4*>(&s_o[grp][4u * lane]) = o;
        __syncthreads();
        if (grp == 0u) {
            const uint32_t used = t.parts < GROUPS ? t.parts : GROUPS;
            for (uint32_t k = 1; k < used; ++k) o = o + *reinterpret_cast<const f32x4*>(&s_o[k][4u * lane]);
            store_row4(a, row_to(a, w, t.p, BM, i % a.kv.kv_heads, row), 4u * lane, o, m, l);
        }
        __syncthreads();
    }
}

// 128-row tiles: many rows of few parts.  Every HD / 4 lanes take a row of their own.
template <uint32_t HD>
__device__ __forceinline__ void join_tiles(const PagedAttentionArgs& a, const RowWork& w, uint32_t i, uint32_t y, uint32_t step) {
    constexpr uint32_t BM = kTileRows, LANES = HD / 4u, GROUPS = 256u / LANES, JU = 4u;
    SplitTile t;
    if (!split_tile(a, w, BM, i, t)) return;
    const uint32_t lane = threadIdx.x % LANES;
    for (uint32_t row = y * GROUPS + threadIdx.x / LANES; row < t.rows; row += step * GROUPS) {
        const float* at = t.base + row * HD + 4u * lane;
        const float* ml = t.base + BM * HD + 2u * row;
        float m = -INFINITY, l = 0.0f;
        f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t k0 = 0; k0 < t.parts; k0 += JU) {
            f32x4 x[JU];
            float pm[JU], pl[JU], top = m;
#pragma unroll
            for (uint32_t k = 0; k < JU; ++k) {
                const uint64_t to = (k0 + k < t.parts ? k0 + k : k0) * t.stride;
                x[k] = *reinterpret_cast<const f32x4*>(at + to);
                pm[k] = ml[to];
                pl[k] = ml[to + 1u];
            }
#pragma unroll
            for (uint32_t k = 0; k < JU; ++k) top = fmaxf(top, pm[k]);
            const bool none = top == -INFINITY;  // nothing seen yet, or NaN alone, which has to stay
            const float keep = none ? 1.0f : __builtin_amdgcn_exp2f(m - top);
            o = o * keep;
            l *= keep;
            m = top;
#pragma unroll
            for (uint32_t k = 0; k < JU; ++k)
                if (k0 + k < t.parts) {
                    const float f = none ? 1.0f : __builtin_amdgcn_exp2f(pm[k] - m);
                    o = o + x[k] * f;
                    l += pl[k] * f;
                }
        }
        store_row4(a, row_to(a, w, t.p, BM, i % a.kv.kv_heads, row), 4u * lane, o, m, l);
    }
}

template <uint32_t HD>
__global__ __launch_bounds__(256) void k_paged_join(PagedAttentionArgs a, RowWork many, RowWork few, uint32_t many_tiles,
                                                    uint32_t many_step, uint32_t few_tiles, uint32_t few_step) {
    const uint32_t b = blockIdx.x, n = many_tiles * many_step;
    if (b < n) join_tiles<HD>(a, many, b / many_step, b % many_step, many_step);
    else join_rows<HD>(a, few, (b - n) / few_step, (b - n) % few_step, few_step);
}

// Rows of a request (new tokens times group) up to which the 16-row tiles take it.
constexpr uint32_t kFewRows = 32u;

// How far long rows are cut: workgroups that split tiles are spread over (the logarithm) and
// a part's least work in kScheduleKeys positions.  Measured with 32 heads over 4 of 128:
// 64 requests of up to 8192 positions in 1024 parts of 16-row tiles 78.5 us, in 512 81.7
// (512 workgroups are resident, but requests are uneven); one request of 131,072 in 1024
// 61.7 us, in 512 57.7 (all alike, and half the parts to join), so calls of few tiles take
// 512.  128-row tiles (24 requests, six chunks of 512): 512 parts 120 us, 256 132, 1024 141.
// Least work of 8 pieces: eight requests of 512 in one part each 10.9 us, in two (least 4)
// 13.9; 16 chunks under a window of 1024 in two or three parts 40 us, whole (least 16) 59.
constexpr uint32_t kRowsTarget = 10u, kFewTilesTarget = 9u, kTilesTarget = 9u, kLeast = 8u;
constexpr uint64_t kFewTiles = 64u;
static_assert(most_parts(1u << kRowsTarget) <= kMostParts && most_parts(1u << kTilesTarget) <= kMostParts);

// The two kinds of row tiles of a call, their scratch and what they need of it.
struct Half {
    RowWork w;
    uint32_t bm;
    bool used, splits;
    uint64_t tiles;  // at most, over all kv heads
    uint32_t keys;   // pieces that a tile sees at most
    uint32_t target() const { return 1u << w.log_target; }
    uint64_t part_floats() const { return splits ? most_parts(target()) * bm : 0u; }
    uint64_t words() const { return splits ? target() * kHeadWords + 4u : 0u; }  // a split tile has two parts
    uint32_t schedule_words(uint32_t requests) const {
        return used && requests > kWaveRequests ? (pk::schedule_words(requests) + 3u) / 4u * 4u : 0u;
    }
    uint64_t units(uint32_t kv_heads) const {
        return (splits ? most_units_seen(tiles / kv_heads, kv_heads, target(), keys, w.least) : tiles / kv_heads) * kv_heads;
    }
    uint32_t split_tiles() const { return !splits ? 0u : tiles < target() ? static_cast<uint32_t>(tiles) : target(); }
};
void halves(const PagedAttentionArgs& a, Half& few, Half& many) {
    const uint64_t positions = static_cast<uint64_t>(a.table_stride) << a.kv.page_shift;
    const uint32_t group = a.group.by;
    // a request of the 16-row tiles has at most kFewRows rows
    const uint64_t n = a.requests < a.max_tokens ? a.requests : a.max_tokens;
    const uint64_t tokens = n * (kFewRows / group ? kFewRows / group : 1u);
    few = Half{{1u, kFewRows, kRowsTarget, kLeast, nullptr, nullptr, nullptr, nullptr}, 16u, group <= kFewRows, false,
               most_tiles(tokens < a.max_tokens ? tokens : a.max_tokens, a.requests, group, 16u) * a.kv.kv_heads,
               most_keys(a.group, 16u, a.window, a.sinks, positions)};
    if (few.tiles < kFewTiles) few.w.log_target = kFewTilesTarget;
    many = Half{{kFewRows + 1u, 0xffffffffu, kTilesTarget, kLeast, nullptr, nullptr, nullptr, nullptr}, kTileRows,
                static_cast<uint64_t>(a.max_new) * group > kFewRows, false,
                most_tiles(a.max_tokens, a.requests, group, kTileRows) * a.kv.kv_heads,
                most_keys(a.group, kTileRows, a.window, a.sinks, positions)};
    few.splits = few.used && request_parts(few.keys, kLeast) > 1u;
    many.splits = many.used && request_parts(many.keys, kLeast) > 1u;
}

template <uint32_t T, uint32_t HD, bool F32>
hipError_t attention_t(const PagedAttentionArgs& a, const Half& few, const Half& many, hipStream_t s) {
    const uint64_t fu = few.used ? few.units(a.kv.kv_heads) : 0u, mu = many.used ? many.units(a.kv.kv_heads) : 0u;
    const dim3 g(static_cast<uint32_t>(fu + mu)), b(256);
    if (few.w.schedule || many.w.schedule)
        hipLaunchKernelGGL(k_paged_schedule, dim3(2), dim3(1024), 0, s, a, few.w, many.w);
    if (many.used)
        hipLaunchKernelGGL((k_paged_chunks<T, HD, F32>), g, b, 0, s, a, many.w, few.w, static_cast<uint32_t>(mu));
    else
        hipLaunchKernelGGL((k_paged_rows<T, HD, F32>), g, b, 0, s, a, few.w);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess || !(many.splits || few.splits)) return err;
    // workgroups enough for the split tiles' rows: about 2048 of each kind
    const uint32_t mn = many.split_tiles(), fn = few.split_tiles();
    const uint32_t my = kTileRows * HD / 1024u, fy = fn <= 128u ? 16u : 2048u / fn;
    hipLaunchKernelGGL(k_paged_join<HD>, dim3(mn * my + fn * fy), b, 0, s, a, many.w, few.w, mn, my, fn, fy);
    return hipGetLastError();
}

template <uint32_t T, bool F32>
hipError_t attention_hd(const PagedAttentionArgs& a, const Half& few, const Half& many, hipStream_t s) {
    switch (a.kv.head_dim) {
        case 64: return attention_t<T, 64, F32>(a, few, many, s);
        case 128: return attention_t<T, 128, F32>(a, few, many, s);
        case 256: return attention_t<T, 256, F32>(a, few, many, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

uint64_t paged_attention_workgroups(const PagedAttentionArgs& a) {
    Half few, many;
    halves(a, few, many);
    return (few.used ? few.units(a.kv.kv_heads) : 0u) + (many.used ? many.units(a.kv.kv_heads) : 0u);
}

uint32_t paged_attention_launches(const PagedAttentionArgs& a) {
    Half few, many;
    halves(a, few, many);
    return (few.splits || many.splits ? 2u : 1u) + (a.requests > kWaveRequests ? 1u : 0u);
}

size_t paged_attention_work_floats(const PagedAttentionArgs& a) {
    Half few, many;
    halves(a, few, many);
    return (few.part_floats() + many.part_floats()) * (a.kv.head_dim + 2u) + few.words() + many.words() +
           few.schedule_words(a.requests) + many.schedule_words(a.requests);
}

hipError_t launch_paged_attention(const PagedAttentionArgs& a, float* work, hipStream_t s) {
    Half few, many;
    halves(a, few, many);
    float* at = work;
    for (Half* half : {&few, &many}) {
        if (half->schedule_words(a.requests)) half->w.schedule = reinterpret_cast<uint32_t*>(at);
        at += half->schedule_words(a.requests);
        if (!half->splits) continue;
        half->w.part = at;
        at += half->part_floats() * (a.kv.head_dim + 2u);
        half->w.head = reinterpret_cast<uint32_t*>(at);
        half->w.count = half->w.head + half->target() * kHeadWords;
        at += half->words();
    }
    const bool f32 = a.type == T_F32;
    if (a.kv.type == T_F16) return f32 ? attention_hd<T_F16, true>(a, few, many, s) : attention_hd<T_F16, false>(a, few, many, s);
    return f32 ? attention_hd<T_BF16, true>(a, few, many, s) : attention_hd<T_BF16, false>(a, few, many, s);
}

}  // namespace pk
