// The 8-bit cache's own rules (csrc/kv8.h, included, not copied) on the host: the scale exponent of every
// magnitude against its definition, page lookup with entries that are not there, offsets past 4 GiB, lengths
// past the table, the selection's ranges. Exit status 0: all hold.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "kv8.h"

#define CHECK(c, ...)                                       \
    do {                                                    \
        if (!(c)) {                                         \
            std::fprintf(stderr, __VA_ARGS__);              \
            std::fprintf(stderr, " (line %d)\n", __LINE__); \
            std::exit(1);                                   \
        }                                                   \
    } while (0)

int main() {
    for (uint32_t m = 0; m < 0x7F80; ++m) {
        const uint32_t b = m << 16;
        float top;
        std::memcpy(&top, &b, 4);
        const int e = kv8_exponent(m);
        CHECK(e >= KV8_LOWEST && e + 127 >= 10 && e + 127 <= 247, "%g: exponent %d", top, e);
        CHECK(std::ldexp(448.0, e) >= top, "%g: 448 2^%d is below it", top, e);
        CHECK(e == KV8_LOWEST || std::ldexp(448.0, e - 1) < top, "%g: 2^%d is not the smallest", top, e);
        CHECK(127 - e >= 1 && 127 - e <= 254, "%g: 2^-%d is no normal f32", top, e);
    }
    const uint32_t table[6] = {5, 9, 10, 0xFFFFFFFFu, 0, 7};  // [2][3], a pool of 10
    CHECK(kv8_page(table, 2, 3, 10, 0, 0) == 5 && kv8_page(table, 2, 3, 10, 0, 1) == 9 && kv8_page(table, 2, 3, 10, 1, 2) == 7, "entries");
    CHECK(kv8_page(table, 2, 3, 10, 0, 2) == KV8_NONE && kv8_page(table, 2, 3, 10, 1, 0) == KV8_NONE, "outside the pool");
    CHECK(kv8_page(nullptr, 2, 3, 10, 2, 0) == KV8_NONE && kv8_page(nullptr, 2, 3, 10, KV8_NONE, 0) == KV8_NONE, "no such sequence");
    CHECK(kv8_page(nullptr, 2, 3, 10, 1, 3) == KV8_NONE && kv8_page(nullptr, 2, 3, 10, 0, KV8_NONE) == KV8_NONE, "no such page");
    CHECK(kv8_record(0xFFFFFFFEu, 1024, 1023) == (0xFFFFFFFEull * 1024 + 1023) * 4096, "64-bit records");
    CHECK(kv8_scale(1u << 31, 8, 3) == ((1ull << 34) + 3) * 32 && kv8_bound(1u << 31, 8, 3) == ((1ull << 34) + 3) * 256, "64-bit offsets");
    CHECK(kv8_keys(0, 4) == 0 && kv8_keys(64, 4) == 64 && kv8_keys(65, 4) == 64 && kv8_keys(0xFFFFFFFFu, (1u << 24) - 1) == 16 * ((1u << 24) - 1), "lengths");
    // The selection's passes over keys at both ends of 64 bits, equal ones among them: as a sort takes them.
    uint64_t seed = 1;
    auto random = [&] { return seed = seed * 6364136223846793005ull + 1442695040888963407ull, seed ^ seed >> 29; };
    for (int round = 0; round < 3000; ++round) {
        std::vector<uint64_t> keys(2 + random() % 60);
        for (uint64_t& x : keys) {
            const uint64_t r = random();
            x = r % 7 == 0 ? ~0ull : r % 7 == 1 ? 0 : r % 7 == 2 ? ~0ull - random() % 5 : r % 7 == 3 ? random() % 3 : random() >> random() % 64;
        }
        const uint32_t take = 1 + random() % (keys.size() - 1);
        uint64_t lo = *std::min_element(keys.begin(), keys.end()), hi = *std::max_element(keys.begin(), keys.end());
        uint32_t need = take;
        bool ties = true;
        for (int pass = 0; pass < KV8_PASSES && lo != hi; ++pass) {
            const int shift = kv8_shift(lo, hi);
            std::vector<uint32_t> bin(2048, 0);
            for (uint64_t x : keys)
                if (x >= lo && x <= hi) {
                    CHECK((x - lo) >> shift < 2048, "bin of %llx", (unsigned long long)x);
                    ++bin[(x - lo) >> shift];
                }
            uint32_t above = 0;
            int b = 2047;
            while (above + bin[b] < need) above += bin[b--];
            need -= above;
            kv8_narrow(lo, hi, shift, (uint32_t)b);
            CHECK(lo <= hi, "range %llx .. %llx", (unsigned long long)lo, (unsigned long long)hi);
            if (bin[b] == need) {
                ties = false;
                break;
            }
        }
        CHECK(!ties || lo == hi, "%d passes end at one key", KV8_PASSES);
        std::vector<uint64_t> got, want = keys;
        for (uint64_t x : keys)
            if (ties ? x > lo || (x == lo && need && need--) : x >= lo) got.push_back(x);
        std::sort(want.rbegin(), want.rend());
        want.resize(take);
        std::sort(got.rbegin(), got.rend());
        CHECK(got == want, "%zu of %u keys", got.size(), take);
    }
    std::puts("ok");
}
