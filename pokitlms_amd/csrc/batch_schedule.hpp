// batch_schedule.hpp -- the steps of a batched generation, all known beforehand (host only):
// greedy generation without an end token takes as many positions as it is asked for, so
// which request brings how many rows to which step follows from the lengths.
//
// Requests wait for one of `slots` rows of the block table.  A step takes one row of each
// request that decodes, then rows of prompts in slot order while the step's budget lasts.
// A request that has all of its positions gives its slot (and, by the plan, its pages)
// to the next one in the step after.
#pragma once

#include <stdint.h>

#include <algorithm>
#include <vector>

namespace pk {

struct BatchStep {
    uint32_t rows, most_new, selected;
    uint64_t at;  // words: new rows [slots], release [slots], request [slots], then per selected
                  // row (the last of a prompt, or a decoded one): row, request
};
struct BatchSchedule {
    std::vector<uint32_t> words;
    std::vector<BatchStep> steps;
    uint32_t pages = 0;  // at most in use at once
    uint32_t width = 0;  // pages of the longest request
    uint32_t most_selected = 0;
};

// Positions of a request that go through the model: the last token is never fed back.
inline uint64_t batch_positions(uint32_t n_prompt, uint32_t n_new) {
    return uint64_t(n_prompt) + (n_new ? n_new - 1u : 0u);
}

inline BatchSchedule batch_schedule(const std::vector<uint32_t>& n_prompt, const std::vector<uint32_t>& n_new,
                                    uint32_t slots, uint32_t budget, uint32_t page_size) {
    constexpr uint32_t none = 0xffffffffu;
    BatchSchedule s;
    const uint32_t n = static_cast<uint32_t>(n_prompt.size());
    std::vector<uint32_t> held(slots, none);
    std::vector<uint64_t> done(n, 0), total(n);
    for (uint32_t r = 0; r < n; ++r) total[r] = batch_positions(n_prompt[r], n_new[r]);
    uint32_t next = 0;
    auto pages = [&](uint64_t len) { return static_cast<uint32_t>((len + page_size - 1u) / page_size); };
    for (;;) {
        BatchStep step{0, 0, 0, s.words.size()};
        s.words.resize(s.words.size() + 3ull * slots, 0u);
        uint32_t* fresh = s.words.data() + step.at;
        uint32_t *release = fresh + slots, *request = release + slots, decoding = 0;
        for (uint32_t i = 0; i < slots; ++i) {
            if (held[i] != none && done[held[i]] == total[held[i]]) {
                release[i] = 1u;
                held[i] = none;
            }
            if (held[i] == none && next < n) held[i] = next++;
            request[i] = held[i];
            if (held[i] != none && done[held[i]] >= n_prompt[held[i]]) ++decoding;
        }
        uint32_t left = budget - decoding;
        for (uint32_t i = 0; i < slots; ++i) {
            const uint32_t r = held[i];
            if (r == none) continue;
            if (done[r] >= n_prompt[r]) {
                fresh[i] = 1u;
            } else {
                fresh[i] = static_cast<uint32_t>(std::min<uint64_t>(left, n_prompt[r] - done[r]));
                left -= fresh[i];
            }
        }
        std::vector<uint32_t> selected;
        uint32_t used = 0;
        for (uint32_t i = 0; i < slots; ++i) {
            const uint32_t r = held[i];
            if (r == none) continue;
            done[r] += fresh[i];
            step.rows += fresh[i];
            step.most_new = std::max(step.most_new, fresh[i]);
            used += pages(done[r]);
            s.width = std::max(s.width, pages(total[r]));
            if (fresh[i] && done[r] >= n_prompt[r]) {
                selected.push_back(step.rows - 1u);
                selected.push_back(r);
            }
        }
        if (step.rows == 0u) {
            s.words.resize(step.at);
            return s;
        }
        step.selected = static_cast<uint32_t>(selected.size() / 2u);
        s.most_selected = std::max(s.most_selected, step.selected);
        s.pages = std::max(s.pages, used);
        s.words.insert(s.words.end(), selected.begin(), selected.end());
        s.steps.push_back(step);
    }
}

}  // namespace pk
