// paged_check.hpp -- the argument checks of the paged-cache entry points and their
// launch arguments (host only, no device call: refusals do not need a GPU).
#pragma once

#include <cmath>
#include <cstdint>

#include "../../include/pokit_hip.h"
#include "paged.hpp"

namespace pk {

// What is wrong with a call (null: nothing) and whether it is a size or type that no
// kernel covers rather than a mistake.
struct PagedCheck {
    const char* error = nullptr;
    bool unsupported = false;
};

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
inline bool paged_float(uint32_t type) { return type == 0u || type == 1u || type == 30u; }
inline uint32_t paged_shift(uint32_t page_size) {
    uint32_t s = 0;
    while ((1u << s) < page_size) ++s;
    return s;
}
inline bool page_size_ok(uint32_t n) { return n >= 1u && n <= kMaxPageSize && (n & (n - 1u)) == 0u; }

inline PagedCheck check_pages(uint32_t pages, uint32_t page_size) {
    if (!page_size_ok(page_size)) return {"page_size must be a power of two up to 1024"};
    if (pages == 0u || static_cast<uint64_t>(pages) * page_size >= (1ull << 31))
        return {"the cache needs 1 or more pages and fewer than 2^31 slots"};
    return {};
}

inline PagedCheck check_table(uint32_t requests, uint32_t table_stride, uint32_t page_size) {
    if (requests == 0u || requests > kMaxPagedRequests) return {"requests must be between 1 and 8192"};
    if (table_stride == 0u || static_cast<uint64_t>(table_stride) * page_size > kMaxPagedPositions)
        return {"a block table row holds 1 to 2^30 positions"};
    return {};
}

inline PagedCheck check_kv(const pk_hip_paged_kv& c, PagedKv& out) {
    if (!c.k || !c.v) return {"the cache needs k and v"};
    if (!aligned16(c.k) || !aligned16(c.v)) return {"the cache must be 16-byte aligned"};
    if (const PagedCheck e = check_pages(c.pages, c.page_size); e.error) return e;
    if (c.type != 1u && c.type != 30u) return {"a paged cache is F16 or BF16", true};
    if (c.head_dim != 64u && c.head_dim != 128u && c.head_dim != 256u)
        return {"a paged cache covers head_dim 64, 128 and 256", true};
    if (c.kv_heads == 0u || c.kv_heads > 4096u) return {"kv_heads must be between 1 and 4096"};
    out = PagedKv{static_cast<uint16_t*>(c.k), static_cast<uint16_t*>(c.v), c.type, c.pages,
                  paged_shift(c.page_size), c.kv_heads, c.head_dim, c.page_stride, c.slot_stride,
                  c.head_stride};
    if (!c.page_stride && !c.slot_stride && !c.head_stride) {
        out.head_stride = c.head_dim;
        out.slot_stride = out.head_stride * c.kv_heads;
        out.page_stride = out.slot_stride * c.page_size;
    }
    if (out.page_stride % 8u || out.slot_stride % 8u || out.head_stride % 8u)
        return {"cache strides must be multiples of 8 elements"};
    constexpr uint64_t most = 1ull << 40;
    if (out.page_stride > most || out.slot_stride > most || out.head_stride > most)
        return {"cache strides are out of range"};
    if ((c.kv_heads > 1u && out.head_stride < c.head_dim) || (c.page_size > 1u && out.slot_stride < c.head_dim) ||
        (c.pages > 1u && out.page_stride < c.head_dim))
        return {"cache strides are shorter than a row"};
    return {};
}

// A row stride in elements of `type` (0: `width`).
inline PagedCheck check_stride(uint64_t stride, uint64_t width, uint32_t type, uint64_t& out) {
    out = stride ? stride : width;
    if (out < width) return {"row strides are shorter than a row"};
    if (out > (1ull << 40)) return {"row strides are out of range"};
    if (out % (type == 0u ? 4u : 8u)) return {"row strides must be multiples of 16 bytes"};
    return {};
}

inline PagedCheck check_plan(const pk_hip_paged_plan* p, PagedPlanArgs& a) {
    if (!p) return {"a plan is required"};
    if (const PagedCheck e = check_pages(p->pages, p->page_size); e.error) return e;
    if (const PagedCheck e = check_table(p->requests, p->table_stride, p->page_size); e.error) return e;
    if (p->max_tokens == 0u || p->max_tokens > kMaxPagedTokens) return {"max_tokens must be between 1 and 2^24"};
    for (const void* q : {static_cast<const void*>(p->lens), static_cast<const void*>(p->new_lens),
                          static_cast<const void*>(p->block_table), static_cast<const void*>(p->free_pages),
                          static_cast<const void*>(p->free_count), static_cast<const void*>(p->lens_out),
                          static_cast<const void*>(p->free_count_out), static_cast<const void*>(p->query_start),
                          static_cast<const void*>(p->positions), static_cast<const void*>(p->slots),
                          static_cast<const void*>(p->token_request), static_cast<const void*>(p->status)})
        if (!q || !aligned4(q)) return {"a plan's device buffers are required, 4-byte aligned"};
    if (!aligned4(p->release)) return {"a plan's device buffers are required, 4-byte aligned"};
    if (p->lens_out == p->new_lens || p->lens_out == p->release || p->query_start == p->lens ||
        p->query_start == p->new_lens)
        return {"a plan's outputs may not be its inputs, but lens_out lens and free_count_out free_count"};
    a = PagedPlanArgs{p->requests, paged_shift(p->page_size), p->pages, p->table_stride, p->max_tokens,
                      p->lens, p->new_lens, p->release, p->free_count, p->block_table, p->free_pages,
                      p->lens_out, p->free_count_out, p->query_start, p->positions, p->slots,
                      p->token_request, p->status, nullptr};
    return {};
}

// Fills all of a but the angles.
inline PagedCheck check_append(const pk_hip_paged_append* p, PagedAppendArgs& a) {
    if (!p) return {"an append is required"};
    a = PagedAppendArgs{};
    if (const PagedCheck e = check_kv(p->cache, a.kv); e.error) return e;
    if (!paged_float(p->type)) return {"rows are F32, F16 or BF16", true};
    if (p->tokens == 0u || p->tokens > kMaxPagedTokens) return {"tokens must be between 1 and 2^24"};
    if (p->heads > 4096u) return {"heads must be at most 4096"};
    if (!p->k || !p->v || !p->slots || (p->heads && (!p->q || !p->q_out)))
        return {"q, k, v, q_out and slots are required"};
    if (!aligned16(p->q) || !aligned16(p->k) || !aligned16(p->v) || !aligned16(p->q_out))
        return {"rows must be 16-byte aligned"};
    if (!aligned4(p->q_norm) || !aligned4(p->k_norm) || !aligned4(p->positions) || !aligned4(p->slots))
        return {"norm weights, positions and slots must be 4-byte aligned"};
    const uint64_t qd = static_cast<uint64_t>(p->heads) * p->cache.head_dim,
                   kd = static_cast<uint64_t>(p->cache.kv_heads) * p->cache.head_dim;
    for (const PagedCheck e : {check_stride(p->q_stride, qd, p->type, a.q_stride),
                               check_stride(p->k_stride, kd, p->type, a.k_stride),
                               check_stride(p->v_stride, kd, p->type, a.v_stride),
                               check_stride(p->q_out_stride, qd, p->type, a.q_out_stride)})
        if (e.error) return e;
    if (p->heads && p->q_out == p->q && a.q_out_stride != a.q_stride)
        return {"q_out may be q only with q's stride"};
    if ((p->q_norm || p->k_norm) && !(p->rms_eps > 0.0f && std::isfinite(p->rms_eps)))
        return {"invalid norm epsilon"};
    if (p->rotary_dim % 16u || p->rotary_dim > p->cache.head_dim)
        return {"rotary_dim must be a multiple of 16 up to head_dim"};
    if (p->rotary_dim) {
        if (!p->positions) return {"positions are required"};
        if (p->axes == 0u || p->axes > kMaxRotaryAxes) return {"axes must be between 1 and 4"};
        if (!(p->rope_theta > 0.0f && std::isfinite(p->rope_theta))) return {"invalid RoPE base"};
        if (p->position_stride && p->position_stride < p->tokens) return {"position_stride is shorter than tokens"};
        if (p->position_stride > (1ull << 40)) return {"position_stride is out of range"};
        for (uint32_t i = 0; p->pair_axis && i < p->rotary_dim / 2u; ++i) {
            if (p->pair_axis[i] >= p->axes) return {"pair_axis names an axis that is not there"};
            a.axis[i] = p->pair_axis[i];
        }
    }
    a.type = p->type;
    a.tokens = p->tokens;
    a.heads = p->heads;
    a.rotary_pairs = p->rotary_dim / 2u;
    a.axes = p->axes;
    a.parts = 1u;
    a.eps = p->rms_eps;
    a.q = p->q;
    a.k = p->k;
    a.v = p->v;
    a.q_out = p->q_out;
    a.q_norm = p->q_norm;
    a.k_norm = p->k_norm;
    a.positions = p->positions;
    a.position_stride = p->position_stride ? p->position_stride : p->tokens;
    a.slots = p->slots;
    return {};
}

inline PagedCheck check_attention(const pk_hip_paged_attention* p, PagedAttentionArgs& a) {
    if (!p) return {"an attention is required"};
    a = PagedAttentionArgs{};
    if (const PagedCheck e = check_kv(p->cache, a.kv); e.error) return e;
    if (const PagedCheck e = check_table(p->requests, p->table_stride, p->cache.page_size); e.error) return e;
    if (!paged_float(p->type) || (p->type != 0u && p->type != p->cache.type))
        return {"q and out are F32 or of the cache's type", true};
    if (p->heads == 0u || p->heads > 4096u || p->heads % p->cache.kv_heads)
        return {"query heads must be evenly grouped over KV heads"};
    if (p->max_tokens == 0u || p->max_tokens > kMaxPagedTokens) return {"max_tokens must be between 1 and 2^24"};
    if (static_cast<uint64_t>(p->max_tokens) * p->heads >= (1ull << 31))
        return {"max_tokens times heads must be below 2^31"};
    if (!p->q || !p->out || !p->query_start || !p->lens || !p->block_table)
        return {"q, out, query_start, lens and block_table are required"};
    if (!aligned16(p->q) || !aligned16(p->out)) return {"rows must be 16-byte aligned"};
    if (!aligned4(p->query_start) || !aligned4(p->lens) || !aligned4(p->block_table))
        return {"query_start, lens and block_table must be 4-byte aligned"};
    if (p->q == p->out) return {"out may not be q"};
    if (!(p->scale >= 0.0f && std::isfinite(p->scale))) return {"invalid attention scale"};
    const uint64_t width = static_cast<uint64_t>(p->heads) * p->cache.head_dim;
    for (const PagedCheck e : {check_stride(p->q_stride, width, p->type, a.q_stride),
                               check_stride(p->out_stride, width, p->type, a.out_stride)})
        if (e.error) return e;
    a.type = p->type;
    a.heads = p->heads;
    a.group = divide_by(p->heads / p->cache.kv_heads);
    a.requests = p->requests;
    a.max_tokens = p->max_tokens;
    a.max_new = p->max_new && p->max_new < p->max_tokens ? p->max_new : p->max_tokens;
    a.table_stride = p->table_stride;
    a.q = p->q;
    a.out = p->out;
    a.query_start = p->query_start;
    a.lens = p->lens;
    a.table = p->block_table;
    a.scale = p->scale > 0.0f ? p->scale : 1.0f / std::sqrt(static_cast<float>(p->cache.head_dim));
    // a window over every position a row can hold hides none
    a.window = p->window < kMaxPagedPositions ? p->window : 0u;
    a.sinks = p->sinks < kMaxPagedPositions ? p->sinks : kMaxPagedPositions;
    return {};
}

}  // namespace pk
