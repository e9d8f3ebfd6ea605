// Replays how decode attention over the 8-bit cache hands its slices out (csrc/kv8.h, included, not copied). Each line of
// the input: kv_heads seq_pages budget seqs, then the sequences' lengths. Each line of the output, for one kv head:
//   waves stream blocks   the cut's
//   slices                of all sequences
//   counts                how many blocks count a slice of several while they hold a further one
//   joins                 sequences whose every slice is counted so: whichever block counts last joins them there
//   rounds                the most tiles that one wavefront takes of one slice
#include <algorithm>
#include <cstdio>
#include <vector>

#include "kv8.h"

int main() {
    uint32_t kv_heads, seq_pages, budget, seqs;
    while (std::scanf("%u %u %u %u", &kv_heads, &seq_pages, &budget, &seqs) == 4) {
        const Kv8Cut cut = kv8_cut(kv_heads, seqs, seq_pages, budget);
        uint32_t slices = 0, counts = 0, joins = 0, rounds = 0;
        struct Sequence {
            uint32_t keys, active, held;  // held: slices with a further one behind them
        };
        for (uint32_t s0 = 0; s0 < seqs; s0 += 64) {
            std::vector<Sequence> group(std::min(64u, seqs - s0));
            for (Sequence& s : group) {
                uint32_t len, per;
                if (std::scanf("%u", &len) != 1) return 1;
                s.keys = kv8_keys(len, seq_pages);
                const uint32_t pages = (s.keys + KV8_PAGE - 1) / KV8_PAGE, np = budget ? std::min(budget, pages) : pages;
                s.active = kv8_slices((np + KV8_TILE - 1) / KV8_TILE, cut.waves, cut.slices, cut.rounds, per);
                s.held = 0;
                rounds = std::max(rounds, per / cut.waves);
            }
            std::vector<uint32_t> of;  // the sequence of every slice
            auto list = [&] {
                of.clear();
                for (uint32_t i = 0; i < group.size(); ++i) of.insert(of.end(), group[i].active, i);
            };
            list();
            if (of.size() > cut.blocks) {  // longest first
                std::stable_sort(group.begin(), group.end(), [](const Sequence& a, const Sequence& b) { return a.keys > b.keys; });
                list();
            }
            std::vector<bool> taken(of.size());
            for (uint32_t block = 0; block < cut.blocks; ++block)
                for (uint32_t r = 0, at; (at = kv8_turn(r, block, cut.blocks)) < of.size(); ++r) {
                    if (taken[at]) return 1;
                    taken[at] = true;
                    Sequence& s = group[of[at]];
                    if (s.active > 1 && kv8_turn(r + 1, block, cut.blocks) < of.size()) ++s.held;
                }
            if (!std::all_of(taken.begin(), taken.end(), [](bool t) { return t; })) return 1;
            for (const Sequence& s : group) {
                counts += s.held;
                joins += s.active > 1 && s.held == s.active;
            }
            slices += (uint32_t)of.size();
        }
        std::printf("%u %d %u %u %u %u %u\n", cut.waves, cut.stream, cut.blocks, slices, counts, joins, rounds);
    }
}
