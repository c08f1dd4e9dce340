// paged.hpp -- host-side entry points of the paged KV cache's kernels (paged.hip,
// paged_attention.hip): many requests share one pool of pages per layer.
//
// A request's position p lies in slot p % page_size of page table[p / page_size] of
// its row of the block table.  A table entry that is not below `pages` is a page that
// is not there: attention takes its positions as masked, append writes nothing.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "paged_index.hpp"

namespace pk {

constexpr uint32_t kNoSlot = 0xffffffffu;
constexpr uint32_t kMaxPagedRequests = 8192;
constexpr uint32_t kMaxPagedTokens = 1u << 24;  // rows of one call
constexpr uint32_t kMaxPagedPositions = 1u << 30;  // positions a table row can hold
constexpr uint32_t kMaxPageSize = 1024;

struct PagedKv {
    uint16_t *k, *v;          // row (page, slot, head) at their strides, in elements
    uint32_t type;            // T_F16 or T_BF16
    uint32_t pages, page_shift, kv_heads, head_dim;
    uint64_t page_stride, slot_stride, head_stride;
};

// Plan: see pk_hip_paged_plan in pokit_hip.h.  work: 2 * requests words of scratch
// where the plan takes two launches (paged_plan_work_words).
struct PagedPlanArgs {
    uint32_t requests, page_shift, pages, table_stride, max_tokens;
    const uint32_t *lens, *new_lens, *release, *free_count;
    uint32_t *table, *free_pages;
    uint32_t *lens_out, *free_count_out, *query_start, *positions, *slots, *token_request, *status;
    uint32_t* work;
};
size_t paged_plan_work_words(uint32_t requests, uint32_t max_tokens);
hipError_t launch_paged_plan(const PagedPlanArgs& a, hipStream_t stream);

// Append: head norms, rotation and the store into the pages (pk_hip_paged_append).
constexpr uint32_t kMaxRotaryPairs = 128;
constexpr uint32_t kMaxRotaryAxes = 4;
struct PagedAppendArgs {
    PagedKv kv;
    uint32_t type;            // of q, k, v and q_out: T_F32, T_F16 or T_BF16
    uint32_t tokens, heads, rotary_pairs, axes;
    float eps;
    const void *q, *k, *v;
    void* q_out;
    uint64_t q_stride, k_stride, v_stride, q_out_stride;  // elements between tokens' rows
    const float *q_norm, *k_norm;                         // [head_dim], or null: no norm
    const uint32_t* positions;                            // [axes][position_stride]
    uint64_t position_stride;
    const uint32_t* slots;
    // F32 rows as sums of `parts` partial ones (a projection's K split), in order, these
    // strides apart
    uint32_t parts;
    uint64_t q_part, kv_part;
    double turns[kMaxRotaryPairs];    // theta^(-i / pairs) / 2 pi
    uint8_t axis[kMaxRotaryPairs];
};
void rotary_turns(PagedAppendArgs& a, float theta);
hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t stream);

// Attention over the pages (pk_hip_paged_attention).
struct PagedAttentionArgs {
    PagedKv kv;
    uint32_t type;            // of q and out
    uint32_t heads;
    Divide group;             // heads / kv_heads
    uint32_t requests, max_tokens, max_new, table_stride;
    const void* q;
    void* out;
    uint64_t q_stride, out_stride;  // elements between tokens' rows
    const uint32_t *query_start, *lens, *table;
    float scale;
    uint32_t window, sinks;   // window 0: none
};
// work: paged_attention_work_floats(a) floats of scratch, 16-byte aligned.
size_t paged_attention_work_floats(const PagedAttentionArgs& a);
uint32_t paged_attention_launches(const PagedAttentionArgs& a);
// Of 256 threads, in the call's largest launch; a launch holds fewer than 2^32 threads.
uint64_t paged_attention_workgroups(const PagedAttentionArgs& a);
constexpr uint64_t kMaxPagedWorkgroups = (1ull << 24) - 1u;
hipError_t launch_paged_attention(const PagedAttentionArgs& a, float* work, hipStream_t stream);

// One step of a batched generation (prompt.hip): `rows` rows of plan.requests slots, whose
// selected ones get logits and a next token.  Device memory throughout.
struct BatchArgs {
    PagedPlanArgs plan;               // rows: max_tokens
    PagedAppendArgs append;           // k, v, q and norms per layer
    PagedAttentionArgs attention;
    uint32_t rows, selected, head_batch;  // rows of logits per pass over the head
    uint16_t* kv;                     // per layer K pages, then V pages
    uint64_t layer_kv;                // elements of one of them
    uint32_t *tokens, *row_tokens;    // every request's tokens, this step's rows'
    const uint32_t* token_start;      // per request: where its tokens start
    const uint32_t* slot_request;     // per slot: its request
    const uint32_t* select;           // per selected row: row, request
    uint32_t *zero, *flags;           // a zero word; non-finite logits, a refused plan
    float *att, *normed, *logits, *head_work, *attention_work;
};

}  // namespace pk
