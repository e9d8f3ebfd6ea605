// How the rows of log probabilities are cut (logprobs.hip): plain arithmetic, which a test replays on the host.
#pragma once
#include <algorithm>
#include <cstdint>

constexpr uint32_t LOGPROBS_MOST_TOP = 64;

// So many alternatives a block of these threads picks by the largest of 16 (up to 12 of them) or 32 groups of its threads; more
// by its wavefronts' sorted threads.
constexpr uint32_t logprobs_in_groups(uint32_t threads) { return threads >= 512 ? 24 : 12; }

struct LogprobsCut {
    uint32_t threads, each;   // of a block, logits to a thread
    uint32_t count, length;   // slices of a row, logits of one
    uint32_t join;            // keys to a thread where slices are joined
    uint32_t at_once;         // rows of a launch
};

// A launch has so many rows and slices at most (fewer than 2^32 threads), and the workspace is a launch's: more are further launches.
constexpr uint64_t LOGPROBS_MOST_ROWS = 65536, LOGPROBS_MOST_SLICES = 1u << 22;
// Blocks up to which long rows are cut into slices of 4096.
constexpr uint64_t LOGPROBS_FEW = 768;

// Measured on MI355X (us; threads x logits). A row in one slice needs no second kernel: 8000 logits, one row with 20 alternatives
// 5.5 with 512 x 16, 9.2 in two slices; 16000: 6.9 with 512 x 32, 9.8 in four; 32001: 8.6 with 1024 x 32, 10.6 in eight, while
// there are up to 2 rows to a CU (512 rows with 5: 17.1, 19.1 in slices; 1024 rows 33.4, 28.8). Many short rows: 256 x 32
// (4096 of 8000 with 5: 24.7; 31.0 with 512 x 16).
// Longer rows: 256 x 16 while there are up to 3 blocks to a CU (one row of 151936, 20 alternatives: 10.7; 11.4 with 256 x 32),
// then 256 x 32, which selects once for twice the logits (512 rows, 20: 63.1; 77.7 with 256 x 16, 74.0 with 512 x 16), but f32
// without selection, which is bound by its loads: 512 x 16 (1024 rows of 151936: 107.3; 110.7 with 256 x 32, 112.4 with 256 x 16).
inline LogprobsCut logprobs_cut(uint32_t rows, uint32_t vocab, uint32_t top, bool bf16) {
    const auto cut = [&](uint32_t threads, uint32_t each) {
        LogprobsCut c = {threads, each, (vocab + threads * each - 1) / (threads * each)};
        c.length = ((vocab + c.count - 1) / c.count + 15) / 16 * 16;  // even slices, whose ends would leave groups of lanes empty
        // Shorter code is over sooner: 760 keys at 4 to a thread 12.2 us for one row, at 16 13.2; more than 1024 in one go.
        c.join = (uint64_t)c.count * top > 1024 ? 16 : 4;
        c.at_once = (uint32_t)std::min(LOGPROBS_MOST_ROWS, LOGPROBS_MOST_SLICES / c.count);
        return c;
    };
    if (vocab <= 4096) return cut(256, 16);
    if (vocab <= 8192) return rows > 512 ? cut(256, 32) : cut(512, 16);
    if (vocab <= 16384) return cut(512, 32);
    if (vocab <= 32768 && rows <= 512) return cut(1024, 32);
    const LogprobsCut few = cut(256, 16);
    if ((uint64_t)rows * few.count <= LOGPROBS_FEW) return few;
    return top <= 1 && !bf16 ? cut(512, 16) : cut(256, 32);
}

// Slices that the workspace has room for: enough for fewer rows too, which may be cut into more of them, up to LOGPROBS_FEW.
inline uint64_t logprobs_most_slices(uint32_t rows, uint32_t vocab, uint32_t top, bool bf16) {
    const uint64_t some = std::min<uint64_t>(rows, LOGPROBS_MOST_ROWS);
    return std::max(std::min(some * logprobs_cut(rows, vocab, top, bf16).count, LOGPROBS_MOST_SLICES),
                    std::min(some * ((vocab + 4095) / 4096), LOGPROBS_FEW));
}
