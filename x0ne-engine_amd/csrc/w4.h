// How a launch of the product with 4-bit weights is cut (w4.hip): plain arithmetic, which a test replays on the host.
#pragma once
#include <algorithm>
#include <cstdint>

// Counters that a launch whose units are cut may use, and bytes of their sums.
constexpr uint64_t W4_COUNTERS = 65536, W4_PARTS_BYTES = 64ull << 20;

// Rows of X that a launch takes.
inline uint32_t w4_rows_at_once(uint32_t cols) { return std::min<uint32_t>(512, (uint32_t)(0xFFFFFFF0ull / (2 * (uint64_t)cols)) / 32 * 32); }

struct W4Plan {
    uint32_t xl;      // loads of 4 rows of X to a wavefront's tile: 1, 2, 4 or 8
    uint32_t panels;  // panels of 16 rows of W to a unit
    uint32_t waves;   // wavefronts to a block
    bool even;        // blocks take even runs of rounds, over the ends of units; else a unit each
    uint32_t units, rounds, groups;  // rounds of a tile to each wavefront in a unit, groups of 4 xl rows of X
    uint32_t run, blocks;            // rounds to a block, blocks to a group
};

// Measured on MI355X, weights from memory, back to back in a captured graph, in us (panels and wavefronts; "even": 4 and 8, one
// block to a CU). Against every kernel that a shape can take, over 77 matrices from 256 x 512 to 151936 x 8192, the plan's
// takes 1.3 % longer than the fastest on average for one row and 4, 4.3 % for 8, 2.5 % for 16, 2 % for 32, 2.5 % for 64. Where
// it is furthest off: one row of 2048 columns, 1.13 times the 8 wavefronts' time; 8 rows of 24576 and 12288 x 6400, 1.2 times
// that of a unit to a block; 32 rows of 12288 x 25600, 1.2 times that of even runs of 8.
//  - One to 4 rows of X: blocks of a unit each, as many as there are. 8 wavefronts have a row of 4096 columns in flight at once
//    (6144 x 4096: 5.5 with 8, 6.0 with 4); 4 do for short rows (4096 x 1024: 2.8 with 4, 3.3 with 8) and where blocks come in
//    many rounds (151936 x 4096: 49.3 with 4, 54.2 with 8; 51200 x 5120 SwiGLU 24.3 and 25.8); 16 for long rows of a matrix with
//    a panel to a CU at most (4096 x 12288: 7.1 with 16, 8.2 with 8; 1024 x 8192: 5.4 and 5.9).
//  - More rows: X passes the L2 once for every unit, at about 20 bytes a clock and CU, so the more panels share it the better,
//    while each CU has a block: 4096 x 4096, 16 rows: 5.7 with 1 panel (256 blocks), 6.4 with 2, 8.0 with 4; 6144 x 4096: 6.6
//    with 2 (192 blocks), 8.3 with 1; 6150 x 4104, 61 rows: 12.5 with 4 (194), 15.9 with 2; 24576 x 4096 SwiGLU, 32 rows: 16.8
//    with 8 (192), 20.2 with 4.
//  - Where that is more than a block to a CU, or long, even runs, whose cut units cost 3 us to join, of 8 panels or, where those
//    were fewer than the CUs, 4: 51200 x 5120 SwiGLU, 32 rows: 37.2 with 8, 42.5 with 4, 48.7 a unit to a block; 151936 x 4096, 16
//    rows: 59.3, 61.3, 62.7; 5120 x 25600, 16 rows: 20.7 with 8, 19.9 with 4, 29.1 a unit of 2 to a block; 4096 x 12288: 9.9 with
//    4, 11.9 a unit of 1 to a block.
inline W4Plan w4_plan(uint32_t rows, uint32_t cols, uint32_t n, bool swiglu, uint32_t cus, bool parts) {
    W4Plan p = {};
    const uint32_t all = (rows + 15) / 16, tiles = (cols + 127) / 128, pair = swiglu ? 2 : 1;
    p.xl = n <= 4 ? 1 : n <= 8 ? 2 : n <= 16 ? 4 : 8;
    p.groups = (n + 4 * p.xl - 1) / (4 * p.xl);
    auto units = [&](uint32_t panels) { return (all + panels - 1) / panels; };
    p.waves = 8;
    if (p.xl == 1) {
        p.panels = pair;
        if (tiles <= 16 || units(pair) > 4 * cus)
            p.waves = 4;
        else if (tiles >= 64 && units(pair) <= cus)
            p.waves = 16;
    } else {
        const uint32_t most = p.xl == 2 ? 4 : 8;
        p.panels = p.xl == 8 ? 2 : pair;
        while (p.panels < most && units(p.panels) * (uint64_t)p.groups > cus) p.panels *= 2;
        p.even = tiles > 48 || units(p.panels) * (uint64_t)p.groups > cus;
        if (p.even) p.panels = units(8) * (uint64_t)p.groups >= cus ? most : 4;
    }
    p.units = units(p.panels);
    p.rounds = (tiles + p.waves - 1) / p.waves;
    p.run = p.rounds;
    // Blocks to a group: whole rounds of the 8 XCDs, so that none gets a block more than it has CUs (96 rows of 24576 x 4096:
    // 65 us with 85 blocks to each of three groups, 39 with 80).
    const uint64_t each = std::max<uint64_t>(1, cus / p.groups >= 8 ? cus / 8 / p.groups * 8 : cus / p.groups);
    p.even = p.even && parts && (uint64_t)p.units * p.groups <= W4_COUNTERS &&
             each * p.groups * 2 * p.panels * ((p.xl + 3) / 4) * 1024 <= W4_PARTS_BYTES;
    if (p.even) p.run = (uint32_t)(((uint64_t)p.units * p.rounds + each - 1) / each);
    p.blocks = (uint32_t)(((uint64_t)p.units * p.rounds + p.run - 1) / p.run);
    return p;
}
