// paged_index.hpp -- which rows, keys and pieces of work the paged attention's kernels
// take: plain arithmetic, for the device and for the host's tests.
//
// A request's rows are its (token, head of one kv head) pairs, token by token, `group`
// per token; a row tile is BM of them in order.  A tile's keys lie in tiles of KT
// positions: those of the sinks, then those from the window's start (or 0) to its last
// row's position.  A request whose tiles see many keys is split along them: all of its
// row tiles into the same number of parts, joined afterwards.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define PK_BOTH __host__ __device__ __forceinline__
#else
#define PK_BOTH inline
#endif

namespace pk {

constexpr uint32_t kScheduleKeys = 64;  // positions of a unit of the schedule's work

// n / d for n below 2^31 by a multiplication: with s = ceil(log2 d) and m = floor(2^(31 + s) /
// d) + 1, n m / 2^(31 + s) is above n / d by less than 1 / d.
struct Divide {
    uint32_t by, magic, shift;
    PK_BOTH uint32_t operator()(uint32_t n) const {
        return static_cast<uint32_t>((static_cast<uint64_t>(n) * magic) >> shift);
    }
    PK_BOTH uint32_t rest(uint32_t n) const { return n - (*this)(n) * by; }
};
inline Divide divide_by(uint32_t d) {
    uint32_t s = 0;
    while ((1u << s) < d) ++s;
    return {d, static_cast<uint32_t>((1ull << (31u + s)) / d + 1u), 31u + s};
}

// A request's new tokens (group rows each for one kv head), 0 for one that is left out.
PK_BOTH uint32_t paged_new(uint32_t q0, uint32_t q1, uint32_t max_new, uint32_t max_tokens) {
    return q1 > q0 && q1 <= max_tokens && q1 - q0 <= max_new ? q1 - q0 : 0u;
}

// Key tiles of rows at positions p_first .. p_last (negative positions see nothing).
struct KeyTiles {
    uint32_t sink_tiles, first_tile, tiles;
    PK_BOTH uint32_t base(uint32_t t, uint32_t kt) const {
        return (t < sink_tiles ? t : first_tile + (t - sink_tiles)) * kt;
    }
};
PK_BOTH KeyTiles key_tiles(int32_t p_first, int32_t p_last, uint32_t window, uint32_t sinks,
                           uint32_t positions, uint32_t kt) {
    if (p_last < 0) return {0u, 0u, 0u};
    uint32_t end = static_cast<uint32_t>(p_last) + 1u;
    if (end > positions) end = positions;
    uint32_t lo = 0u;
    if (window && p_first >= 0 && static_cast<uint32_t>(p_first) + 1u > window)
        lo = static_cast<uint32_t>(p_first) + 1u - window;
    const uint32_t first = lo / kt, last = (end + kt - 1u) / kt, seen = sinks < lo ? sinks : lo;
    uint32_t sink_tiles = (seen + kt - 1u) / kt;
    if (sink_tiles > first) sink_tiles = first;
    if (sink_tiles > last) sink_tiles = last;
    return {sink_tiles, first, sink_tiles + (last > first ? last - first : 0u)};
}

// Whether the row at position p sees position i (its page aside).
PK_BOTH bool row_sees(int32_t p, uint32_t i, uint32_t window, uint32_t sinks) {
    return static_cast<int32_t>(i) <= p &&
           (window == 0u || i + window > static_cast<uint32_t>(p) || i < sinks);
}

// A request's share of one launch.
struct RequestWork {
    uint32_t tiles;  // row tiles
    uint32_t keys;   // kScheduleKeys-sized pieces that its last row tile sees
};
PK_BOTH RequestWork request_work(uint32_t fresh, uint32_t len, const Divide& group, uint32_t bm, uint32_t min_rows,
                                 uint32_t max_rows, uint32_t window, uint32_t sinks, uint32_t positions) {
    const uint64_t rows = static_cast<uint64_t>(fresh) * group.by;
    if (rows == 0u || rows < min_rows || rows > max_rows) return {0u, 0u};
    if (len > positions) len = positions;
    const int32_t last = static_cast<int32_t>(len) - 1;
    const uint32_t tokens = group(bm) + 1u;  // of one row tile, at most
    const int32_t first = last - static_cast<int32_t>(tokens < fresh ? tokens : fresh) + 1;
    return {static_cast<uint32_t>((rows + bm - 1u) / bm),
            key_tiles(first < 0 ? 0 : first, last, window, sinks, positions, kScheduleKeys).tiles};
}

// Pieces per part where the launch's work (sum of tiles * keys * kv_heads, below 2^53) is
// spread over 2^log_target workgroups, at least `least`; and the parts of a request's row
// tiles.  A request has fewer than 2^25 pieces, so more per part need not be told apart.
PK_BOTH uint32_t part_pieces(uint64_t work, uint32_t log_target, uint32_t least) {
    const uint64_t n = (work + (1ull << log_target) - 1u) >> log_target;
    return n > (1u << 28) ? 1u << 28 : n > least ? static_cast<uint32_t>(n) : least;
}
PK_BOTH uint32_t request_parts(uint32_t keys, uint32_t pieces) {
    return keys <= pieces + pieces / 4u ? 1u : (keys + pieces - 1u) / pieces;
}
// Part `part` of `parts` of a tile's key tiles.
PK_BOTH void part_range(uint32_t tiles, uint32_t part, uint32_t parts, uint32_t& t0, uint32_t& t1) {
    const uint32_t n = (tiles + parts - 1u) / parts;
    t0 = part * n < tiles ? part * n : tiles;
    t1 = t0 + n < tiles ? t0 + n : tiles;
}

// Bounds on the host, which knows no lengths.  Row tiles of max_tokens tokens of `requests`
// requests:
PK_BOTH uint64_t most_tiles(uint64_t max_tokens, uint64_t requests, uint64_t group, uint64_t bm) {
    return max_tokens * group / bm + (max_tokens < requests ? max_tokens : requests);
}
// Workgroups per kv head: a tile's parts beyond its first are fewer than keys / pieces, and
// the sum of keys over all tiles is at most target * pieces / kv_heads.
PK_BOTH uint64_t most_units(uint64_t tiles, uint32_t kv_heads, uint32_t target) {
    return tiles + (target + kv_heads - 1u) / kv_heads;
}
// Pieces that a row tile sees at most: those of a table row, or of a window, the tile's own
// tokens and the sinks.
PK_BOTH uint32_t most_keys(const Divide& group, uint32_t bm, uint32_t window, uint32_t sinks, uint64_t positions) {
    const uint64_t all = (positions + kScheduleKeys - 1u) / kScheduleKeys;
    const uint64_t seen = (static_cast<uint64_t>(window) + group(bm) + 1u) / kScheduleKeys + 2u +
                          (static_cast<uint64_t>(sinks) + kScheduleKeys - 1u) / kScheduleKeys;
    return static_cast<uint32_t>(window && seen < all ? seen : all);
}
// Workgroups per kv head where a tile sees at most `keys` pieces: its parts are then few.
PK_BOTH uint64_t most_units_seen(uint64_t tiles, uint32_t kv_heads, uint32_t target, uint32_t keys, uint32_t least) {
    const uint64_t a = most_units(tiles, kv_heads, target), b = tiles * ((keys + least - 1u) / least);
    return b < a ? b : a;
}
// Parts of split tiles, over all kv heads: a split tile sees more than 1.25 pieces, so its
// parts are fewer than 1.8 keys / pieces.
PK_BOTH constexpr uint64_t most_parts(uint32_t target) { return 2ull * target; }

// Whether a split tile's entry and the last of its parts, both counted per kv head, lie in
// the scratch that these bounds give.  They always do where query_start does not decrease;
// where it does, rows can be more than max_tokens and the bounds do not hold.
PK_BOTH bool split_fits(uint32_t split, uint32_t last_part, uint32_t kv_heads, uint32_t target) {
    return (split + 1ull) * kv_heads <= target && (last_part + 1ull) * kv_heads <= most_parts(target);
}
// Whether an entry of the split tiles' list, as read back, is one of this call's size.
PK_BOTH bool split_entry_fits(uint32_t parts, uint32_t first_part, uint32_t q0, uint32_t fresh, uint32_t tile,
                              uint32_t group, uint32_t bm, uint32_t max_new, uint32_t max_tokens, uint32_t kv_heads,
                              uint32_t target) {
    const uint64_t most = most_parts(target);
    return parts > 1u && parts <= most && first_part < most && (0ull + first_part + parts) * kv_heads <= most &&
           fresh && paged_new(q0, q0 + fresh, max_new, max_tokens) == fresh &&
           static_cast<uint64_t>(tile) * bm < static_cast<uint64_t>(fresh) * group;
}

}  // namespace pk
