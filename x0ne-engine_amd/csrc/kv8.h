// The 8-bit paged K/V cache: its layout, its rounding rule and its page lookup, for the kernels
// (kv8.hip) and for host programs.
//
// A row x of 128 bf16 values (a key after norm and rotation, or a value) is held as 128 e4m3 codes
// of x 2^-e (to nearest, ties to even) and one scale byte e + 127. e is the smallest exponent from
// KV8_LOWEST on with 448 2^e >= the largest finite |x| (448: e4m3's largest value), so the largest
// code is above 224: e4m3's own exponent serves the smaller values, and a scale that is a power of
// two makes code 2^e exact in bf16. A value that is not finite is held as NaN (e4m3 has no
// infinity). The lowest exponent keeps e4m3's smallest step, 2^-9, a normal bf16 value.
//
// codes  [pool][kv_heads][4096]: the keys of 16 positions [16][128], then their values dim-major
//        [128][16] (the 16 positions of one dim contiguous: the operand order of P V)
// scales [pool][kv_heads][32]: the 16 keys' scale bytes, then the 16 values'
// bounds [pool][kv_heads][2][128] bf16: the smallest and the largest value of each dim over the 16
//        keys of a complete page (exact: the values are bf16; zeros are +0; NaN where a key holds one)
#pragma once
#include <stddef.h>
#include <stdint.h>

#ifdef __HIPCC__
#define KV8_BOTH __host__ __device__ __forceinline__
#else
#define KV8_BOTH inline
#endif

constexpr uint32_t KV8_HEAD = 128, KV8_PAGE = 16;
constexpr uint32_t KV8_PART = KV8_HEAD * KV8_PAGE;  // bytes of a page's keys (or values) of one head
constexpr uint32_t KV8_RECORD = 2 * KV8_PART, KV8_SCALES = 2 * KV8_PAGE, KV8_BOUNDS = 2 * KV8_HEAD;
constexpr uint32_t KV8_NONE = 0xFFFFFFFFu;
constexpr int KV8_LOWEST = -117;

// Physical page of a sequence's logical page; KV8_NONE where there is none: a sequence or page
// outside the table, or an entry outside the pool.
KV8_BOTH uint32_t kv8_page(const uint32_t* table, uint32_t seqs, uint32_t seq_pages, uint32_t pool, uint32_t seq,
                           uint32_t page) {
    if (seq >= seqs || page >= seq_pages) return KV8_NONE;
    const uint32_t p = table[(size_t)seq * seq_pages + page];
    return p < pool ? p : KV8_NONE;
}

// First byte of a page's record of kv head h: 64 bits, a pool may pass 4 GiB.
KV8_BOTH size_t kv8_record(uint32_t page, uint32_t kv_heads, uint32_t h) {
    return ((size_t)page * kv_heads + h) * KV8_RECORD;
}
KV8_BOTH size_t kv8_scale(uint32_t page, uint32_t kv_heads, uint32_t h) {
    return ((size_t)page * kv_heads + h) * KV8_SCALES;
}
KV8_BOTH size_t kv8_bound(uint32_t page, uint32_t kv_heads, uint32_t h) {
    return ((size_t)page * kv_heads + h) * KV8_BOUNDS;
}

// Keys of sequence length len that a table of seq_pages pages holds.
KV8_BOTH uint32_t kv8_keys(uint32_t len, uint32_t seq_pages) {
    const uint64_t room = (uint64_t)seq_pages * KV8_PAGE;
    return len < room ? len : (uint32_t)room;
}

// The scale exponent of a row whose largest finite magnitude has these bf16 bits: 448 is 1.75 2^8,
// so a mantissa of at most 0.75 (0x60 of 0x80) fits under it eight exponents down.
KV8_BOTH int kv8_exponent(uint32_t magnitude) {
    const int e = (int)(magnitude >> 7) - 127 - ((magnitude & 0x7Fu) <= 0x60u ? 8 : 7);
    return e < KV8_LOWEST ? KV8_LOWEST : e;
}

// Radix selection of 64-bit keys over the range lo .. hi (lo < hi) that holds the undecided ones: its keys fall into
// 2048 bins, (key - lo) >> shift; then one bin's range takes its place. The range loses 11 bits each time, so KV8_PASSES
// of them end at a single key. The bin's end is not computed where it would pass hi (it can pass 2^64 there).
constexpr int KV8_PASSES = 6;
KV8_BOTH int kv8_shift(uint64_t lo, uint64_t hi) {
    const int bits = 64 - __builtin_clzll(hi - lo);
    return bits > 11 ? bits - 11 : 0;
}
KV8_BOTH void kv8_narrow(uint64_t& lo, uint64_t& hi, int shift, uint32_t bin) {
    const uint64_t span = (1ull << shift) - 1;
    lo += (uint64_t)bin << shift;
    if (hi - lo > span) hi = lo + span;
}

// How decode attention cuts sequences: at most `slices` slices of at least `rounds` rounds (a tile of KV8_TILE pages for
// each of a block's `waves` wavefronts), over `blocks` blocks for each kv head and 64 sequences.
//  - Few pairs of sequence and kv head: slices for one block on each of 256 CUs; more bring more states to join than
//    overlap gains (us, 32768 keys, 8 pairs, blocks of 4, 16 / 32 / 64 slices: 27.2 / 21.7 / 26.8).
//  - Many: blocks that fill the card walk the slices, longest first. A slice of one round costs about four (its lookups
//    are waited for, its states and count are not hidden), so slices are two thirds of what a block has to do if every
//    sequence fills its table, or 8192 positions of it (pairs / 24), and up to 16: known before the lengths are, and the
//    same under tables far wider than the sequences (16 sequences of up to 8192 keys 35 us under 513, 2048 and 8192 pages;
//    16 rounds 67). An estimate: where the slices happen to fill the blocks evenly, fewer or more rounds are faster. us
//    by rounds, 8 kv heads, lengths spread evenly up to 8192 (64: 6000), the estimate's in brackets:
//      rounds           2     3     4     5     6     8    12    16
//       8 sequences  [25.7]  18.5  19.7  22.0  24.4  29.1  36.8  46.5
//      13             33.9   38.1 [36.1] 30.7  32.7  37.2  43.2  57.0
//      16             46.3   41.7  44.6 [35.0] 36.7  42.5  53.2  66.8
//      20             47.9   47.1  50.1  49.7 [55.8] 44.8  54.9  68.0
//      32 ([10] 67.3) 75.5   70.3  70.0  63.5  66.3  68.8  63.7  74.5
//      64            107.6   99.7  94.1  97.0  92.5  86.3  72.7 [72.6]
//    and it does not see one long sequence among short ones: 32768 keys among 63 of 200 under 2048 pages takes 16 rounds, 4
//    slices, and 77.7 us; 4 rounds 36.5.
//  - Blocks of 8 wavefronts, one on a CU, join fewer states than two of 4 and start fewer slices (us with 4 / 8: 32768
//    keys 21.1 / 19.0, 64 sequences 84 / 73, 16 sequences 35 / 35); where the pages, all attended, are less than two
//    rounds of 8 for each CU, 4 (128 pages for each of 8 pairs, with their selection, 21.9 / 24.1).
//  - Loads of more than the Infinity Cache holds, by the tables' width, bypass it (64 sequences of up to 6000 keys 76.6 ->
//    72.9 us); 67 MB, read again before 256 MB of others, come from it (32768 keys 19 us with it, 22 without).
constexpr uint64_t KV8_STREAM = 256ull << 20;  // the Infinity Cache's bytes
constexpr uint32_t KV8_TILE = 4;               // pages of a wavefront's tile
constexpr uint32_t KV8_SLICES = 64;            // the most slices of a sequence
struct Kv8Cut {
    uint32_t waves, slices, rounds, blocks;
    bool stream;
};
inline Kv8Cut kv8_cut(uint32_t kv_heads, uint32_t seqs, uint32_t seq_pages, uint32_t budget) {
    auto least = [](uint64_t a, uint64_t b) { return a < b ? a : b; };
    auto most_of = [](uint64_t a, uint64_t b) { return a > b ? a : b; };
    const uint64_t pairs = most_of(1, (uint64_t)seqs * kv_heads), parts = (seqs + 63) / 64, together = least(seqs, 64);
    const uint32_t most = budget && budget < seq_pages ? budget : seq_pages;  // pages a sequence attends
    Kv8Cut cut;
    cut.waves = pairs * ((most + 31) / 32) >= 512 ? 8 : 4;
    cut.stream = pairs * most * (KV8_RECORD + KV8_SCALES) > KV8_STREAM;  // 8 wavefronts then
    cut.slices = (uint32_t)least(KV8_SLICES, most_of(16, 256 / pairs));
    cut.blocks = (uint32_t)most_of(1, 2048 / cut.waves / most_of(1, parts * kv_heads));
    const uint64_t fullest = (uint64_t)((most + KV8_TILE * cut.waves - 1) / (KV8_TILE * cut.waves)) * together;
    cut.rounds = (uint32_t)most_of(1, least(least(16, pairs / 24), 2 * fullest / (3 * cut.blocks)));
    cut.blocks = (uint32_t)most_of(1, least(cut.blocks, cut.slices * together));
    return cut;
}
// The slices of a sequence of `tiles` tiles, and the tiles of each: at least one slice, by its own length and the cut only.
KV8_BOTH uint32_t kv8_slices(uint32_t tiles, uint32_t waves, uint32_t slices, uint32_t cut_rounds, uint32_t& per) {
    const uint32_t rounds = (tiles + waves - 1) / waves, wanted = (rounds + cut_rounds - 1) / cut_rounds;
    const uint32_t few = wanted < slices ? wanted : slices, active = few > 1 ? few : 1, each = (rounds + active - 1) / active;
    per = waves * (each > 1 ? each : 1);
    const uint32_t n = (tiles + per - 1) / per;
    return n > 1 ? n : 1;
}
// The slice that a block takes in its turn r, among those of its kv head and 64 sequences: to and fro over the blocks.
KV8_BOTH uint32_t kv8_turn(uint32_t r, uint32_t block, uint32_t blocks) {
    return r * blocks + (r & 1 ? blocks - 1 - block : block);
}
