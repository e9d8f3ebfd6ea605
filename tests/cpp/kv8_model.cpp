// The 8-bit cache's own rules (csrc/kv8.h, included, not copied) on the host: the scale exponent of every
// magnitude against its definition, page lookup with entries that are not there, offsets past 4 GiB, lengths
// past the table. Exit status 0: all hold.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>

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
    std::puts("ok");
}
