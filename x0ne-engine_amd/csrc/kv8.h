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
