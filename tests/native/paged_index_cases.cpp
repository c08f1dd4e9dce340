// The paged attention's index arithmetic (csrc/paged_index.hpp) against plain loops, on the
// host: which keys a tile visits, how a launch's work is cut, and that neither workgroups
// nor scratch are ever short.  Prints "ok" and the number of cases.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../pokitlms_amd/csrc/paged_index.hpp"

namespace {

uint64_t state = 1;
uint32_t draw(uint32_t n) {
    state = state * 6364136223846793005ull + 1442695040888963407ull;
    return static_cast<uint32_t>((state >> 33) % n);
}

#define CHECK(x)                                                        \
    do {                                                                \
        if (!(x)) {                                                     \
            std::printf("line %d: %s (case %u)\n", __LINE__, #x, at);   \
            std::exit(1);                                               \
        }                                                               \
    } while (0)

// Every position that a row of the tile sees is visited once, in order, below `positions`
// rounded up to a tile; no tile lies outside [0, p_last].
void keys(uint32_t at) {
    const uint32_t kt = draw(2) ? 32 : 64, positions = 1 + draw(600);
    const int32_t p_first = static_cast<int32_t>(draw(650)) - 40, p_last = p_first + static_cast<int32_t>(draw(40));
    const uint32_t window = draw(2) ? 0 : 1 + draw(300), sinks = draw(2) ? draw(5) : draw(400);
    const pk::KeyTiles t = pk::key_tiles(p_first, p_last, window, sinks, positions, kt);
    std::vector<int> seen(positions + kt, 0);
    uint32_t last = 0;
    for (uint32_t i = 0; i < t.tiles; ++i) {
        const uint32_t base = t.base(i, kt);
        CHECK(base % kt == 0 && base < positions && static_cast<int32_t>(base) <= p_last);
        CHECK(i == 0 || base > last);
        last = base;
        for (uint32_t k = 0; k < kt; ++k) ++seen[base + k];
    }
    for (int32_t p = p_first; p <= p_last; ++p)
        for (uint32_t i = 0; i < positions; ++i) {
            const bool want = p >= 0 && static_cast<int64_t>(i) <= p &&
                              (!window || static_cast<int64_t>(i) + window > p || i < sinks);
            CHECK(pk::row_sees(p, i, window, sinks) == want);
            if (want) CHECK(seen[i] == 1);
        }
    // the parts of a tile are its tiles in order, each once
    const uint32_t parts = 1 + draw(9);
    uint32_t next = 0;
    for (uint32_t i = 0; i < parts; ++i) {
        uint32_t t0, t1;
        pk::part_range(t.tiles, i, parts, t0, t1);
        CHECK(t0 == next && t1 >= t0 && t1 <= t.tiles);
        next = t1;
    }
    CHECK(next == t.tiles);
}

void schedule(uint32_t at) {
    const uint32_t bm = draw(2) ? 16 : 128, group = 1 + draw(draw(2) ? 9 : 70), kv_heads = 1 + draw(8);
    const uint32_t log_target = draw(11), target = 1u << log_target, least = 1 + draw(8), requests = 1 + draw(40);
    const uint32_t min_rows = draw(2) ? 1 : 33, max_rows = draw(2) ? 32 : 0xffffffffu;
    const uint32_t window = draw(3) ? 0 : 1 + draw(3000), sinks = draw(200), positions = 64 + draw(40000);
    const uint32_t tokens = 1 + draw(3000), max_new = 1 + draw(tokens);
    std::vector<uint32_t> start(requests + 1, 0), lens(requests);
    for (uint32_t r = 0; r < requests; ++r) {
        uint32_t n = draw(3) ? draw(3) : draw(1 + draw(800));
        if (start[r] + n > tokens) n = tokens - start[r];
        start[r + 1] = start[r] + n;
        lens[r] = draw(4) ? draw(positions + 1) : draw(0x80000000u);  // beyond the table too
    }
    uint64_t work = 0;
    std::vector<pk::RequestWork> all;
    for (uint32_t r = 0; r < requests; ++r) {
        const uint32_t fresh = pk::paged_new(start[r], start[r + 1], max_new, tokens);
        CHECK(fresh == (start[r + 1] - start[r] > max_new ? 0 : start[r + 1] - start[r]));
        all.push_back(pk::request_work(fresh, lens[r], pk::divide_by(group), bm, min_rows, max_rows, window, sinks, positions));
        const uint64_t rows = uint64_t(fresh) * group;
        CHECK(all[r].tiles == (rows >= min_rows && rows <= max_rows ? (rows + bm - 1) / bm : 0));
        work += uint64_t(all[r].tiles) * all[r].keys;
    }
    const uint32_t pieces = pk::part_pieces(work * kv_heads, log_target, least);
    CHECK(pieces >= least && uint64_t(pieces) * target >= work * kv_heads);
    uint64_t units = 0, parts = 0;
    for (const pk::RequestWork& r : all) {
        const uint32_t n = pk::request_parts(r.keys, pieces);
        CHECK(n >= 1);
        units += uint64_t(r.tiles) * n;
        if (n > 1) parts += uint64_t(r.tiles) * n;
    }
    CHECK(units <= pk::most_units(pk::most_tiles(tokens, requests, group, bm), kv_heads, target));
    CHECK(parts * kv_heads <= pk::most_parts(target));
    // a cache whose rows are too short to be split has no parts
    if (positions / pk::kScheduleKeys + 2 <= least + least / 4) CHECK(parts == 0);
}

// Tiles of any length see no more pieces than most_keys says, with that the workgroups
// suffice, and a call without a tile that could be cut has none that is.
void windows(uint32_t at) {
    const uint32_t bm = draw(2) ? 16 : 128, group = 1 + draw(draw(2) ? 9 : 200), kv_heads = 1 + draw(8);
    const uint32_t log_target = 3 + draw(8), target = 1u << log_target, least = 1 + draw(9), requests = 1 + draw(30);
    const uint32_t window = draw(4) ? 1 + draw(draw(2) ? 3000 : 200) : 0, sinks = draw(3) ? draw(300) : 0;
    const uint32_t positions = 1 + draw(draw(2) ? 20000 : 900);
    const pk::Divide by = pk::divide_by(group);
    const uint32_t most = pk::most_keys(by, bm, window, sinks, positions);
    uint64_t work = 0, tiles = 0, units = 0, split = 0;
    std::vector<pk::RequestWork> all;
    for (uint32_t r = 0; r < requests; ++r) {
        const uint32_t fresh = draw(3) ? 1 + draw(3) : 1 + draw(700);
        const uint32_t len = draw(4) ? draw(positions + 1) : fresh + draw(positions);
        all.push_back(pk::request_work(fresh, len, by, bm, 1, 0xffffffffu, window, sinks, positions));
        CHECK(all[r].keys <= most);
        work += uint64_t(all[r].tiles) * all[r].keys;
        tiles += all[r].tiles;
    }
    const uint32_t pieces = pk::part_pieces(work * kv_heads, log_target, least);
    for (const pk::RequestWork& r : all) {
        const uint32_t n = pk::request_parts(r.keys, pieces);
        units += uint64_t(r.tiles) * n;
        split += n > 1 ? r.tiles : 0;
    }
    if (pk::request_parts(most, least) == 1) CHECK(split == 0 && units == tiles);
    else CHECK(units <= pk::most_units_seen(tiles, kv_heads, target, most, least));
}

void divide(uint32_t at) {
    const uint32_t d = 1 + draw(at % 2 ? 40 : 5000);
    const pk::Divide by = pk::divide_by(d);
    for (const uint32_t n : {0u, 1u, d - 1, d, d + 1, draw(0x7fffffff), 0x7fffffffu, 0x7fffffffu / d * d,
                             0x7fffffffu / d * d - 1, draw(100000)})
        CHECK(by(n) == n / d && by.rest(n) == n % d);
}

void bad_lengths(uint32_t at) {
    const uint32_t q0 = draw(100), q1 = draw(100), most = 1 + draw(100), tokens = 1 + draw(100);
    const uint32_t n = pk::paged_new(q0, q1, most, tokens);
    CHECK(n <= most && (n == 0 || (q0 + n == q1 && q1 <= tokens)));
}

// What the kernels do with the sums and entries of any query_start, in their 32-bit words:
// nothing that is taken lies outside the scratch or the rows.
void broken_starts(uint32_t at) {
    const uint32_t target = 1u << (9 + at % 2), kv_heads = 1 + draw(at % 3 ? 16 : 4096), group = 1 + draw(16);
    const uint32_t bm = at % 2 ? 16 : 128, max_tokens = 1 + draw(5000), max_new = 1 + draw(max_tokens);
    const uint32_t most = 2 * target;
    for (int i = 0; i < 20; ++i) {
        const uint32_t split = draw(i % 2 ? 2000 : 0xffffffffu), part = draw(i % 3 ? 4000 : 0xffffffffu);
        if (pk::split_fits(split, part, kv_heads, target))
            CHECK(uint64_t(split) * kv_heads + kv_heads <= target && uint64_t(part) * kv_heads + kv_heads <= most);
        const bool any = i % 4 == 0;
        const uint32_t parts = draw(any ? 0xffffffffu : 40), first = draw(any ? 0xffffffffu : 3000);
        const uint32_t q0 = draw(any ? 0xffffffffu : 6000), fresh = draw(any ? 0xffffffffu : 6000);
        const uint32_t tile = draw(any ? 0xffffffffu : 600);
        if (pk::split_entry_fits(parts, first, q0, fresh, tile, group, bm, max_new, max_tokens, kv_heads, target)) {
            CHECK(parts >= 2 && (uint64_t(first) + parts) * kv_heads <= most && uint64_t(q0) + fresh <= max_tokens);
            CHECK(uint64_t(tile) * bm < uint64_t(fresh) * group);
        }
    }
    // an entry that a call without a fault writes is taken
    const uint32_t fresh = 1 + draw(max_new), q0 = draw(max_tokens - fresh + 1);
    const uint32_t tile = draw((fresh * group + bm - 1) / bm), kvh = 1 + draw(target / 2);
    CHECK(pk::split_entry_fits(2, most / kvh - 2, q0, fresh, tile, group, bm, max_new, max_tokens, kvh, target));
    CHECK(pk::split_fits(target / kvh - 1, most / kvh - 1, kvh, target));
}

}  // namespace

int main() {
    uint32_t at = 0;
    for (; at < 3000; ++at) keys(at);
    for (; at < 60000; ++at) schedule(at);
    for (; at < 80000; ++at) bad_lengths(at);
    for (; at < 100000; ++at) divide(at);
    for (; at < 130000; ++at) broken_starts(at);
    for (; at < 190000; ++at) windows(at);
    std::printf("ok %u\n", at);
    return 0;
}
