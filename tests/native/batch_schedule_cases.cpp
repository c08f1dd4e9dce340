// The steps of a batched generation (csrc/batch_schedule.hpp): every request's positions go
// through in order, once, within the budget, and no more pages are held than are counted.
#include <cstdio>
#include <cstdlib>

#include "../../pokitlms_amd/csrc/batch_schedule.hpp"

#define CHECK(x)                                                       \
    do {                                                               \
        if (!(x)) {                                                    \
            std::printf("line %d: %s (case %u)\n", __LINE__, #x, at); \
            std::exit(1);                                              \
        }                                                              \
    } while (0)

int main() {
    uint64_t state = 7;
    auto draw = [&](uint32_t n) {
        state = state * 6364136223846793005ull + 1442695040888963407ull;
        return static_cast<uint32_t>((state >> 33) % n);
    };
    for (uint32_t at = 0; at < 400; ++at) {
        const uint32_t n = 1 + draw(30), budget = 1 + draw(at % 2 ? 600 : 40), page = 16;
        const uint32_t slots = std::min(std::min(n, budget), 1 + draw(12));
        std::vector<uint32_t> prompt, fresh;
        for (uint32_t r = 0; r < n; ++r) {
            prompt.push_back(1 + draw(draw(3) ? 20 : 900));
            fresh.push_back(draw(12));
        }
        const pk::BatchSchedule s = pk::batch_schedule(prompt, fresh, slots, budget, page);
        std::vector<uint64_t> done(n, 0), selected(n, 0);
        std::vector<uint32_t> held(slots, 0xffffffffu);
        uint32_t most = 0, width = 0, most_selected = 0;
        for (const pk::BatchStep& step : s.steps) {
            const uint32_t *w = s.words.data() + step.at, *release = w + slots, *request = release + slots,
                           *select = request + slots;
            CHECK(step.at + 3ull * slots + 2ull * step.selected <= s.words.size());
            uint32_t rows = 0, big = 0, used = 0, taken = 0;
            for (uint32_t i = 0; i < slots; ++i) {
                if (release[i]) {  // only what is done is let go
                    CHECK(held[i] < n && done[held[i]] == pk::batch_positions(prompt[held[i]], fresh[held[i]]));
                    held[i] = 0xffffffffu;
                }
                if (held[i] == 0xffffffffu) held[i] = request[i];
                CHECK(held[i] == request[i]);
                if (request[i] == 0xffffffffu) {
                    CHECK(w[i] == 0);
                    continue;
                }
                const uint32_t r = request[i];
                // prompt rows and decoded ones do not share a step
                if (done[r] < prompt[r]) CHECK(done[r] + w[i] <= prompt[r]);
                else CHECK(w[i] <= 1);
                done[r] += w[i];
                rows += w[i];
                big = std::max(big, w[i]);
                used += static_cast<uint32_t>((done[r] + page - 1) / page);
                if (w[i] && done[r] >= prompt[r]) {
                    CHECK(select[2 * taken] == rows - 1 && select[2 * taken + 1] == r);
                    ++selected[r];
                    ++taken;
                }
            }
            CHECK(rows == step.rows && rows >= 1 && rows <= budget && big == step.most_new && taken == step.selected);
            most = std::max(most, used);
            most_selected = std::max(most_selected, taken);
        }
        for (uint32_t r = 0; r < n; ++r) {
            CHECK(done[r] == pk::batch_positions(prompt[r], fresh[r]));
            CHECK(selected[r] == (fresh[r] ? fresh[r] : 1));
            width = std::max(width, static_cast<uint32_t>((done[r] + page - 1) / page));
        }
        CHECK(most == s.pages && width == s.width && most_selected == s.most_selected);
    }
    std::printf("ok\n");
    return 0;
}
