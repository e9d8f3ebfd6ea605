// The 8-bit paged K/V cache (kv8.h): its write behind QK-norm and RoPE, its read-back into bf16
// pages, decode attention over it, and the selection of pages by their bounds.
#include <algorithm>
#include <string>

#include "device.h"
#include "internal.h"
#include "kv8.h"

using namespace x0ne;

namespace {

struct Table {
    const uint32_t* pages;
    uint32_t seqs, seq_pages, pool, kv_heads;
    __device__ __forceinline__ uint32_t page(uint32_t seq, uint32_t p) const {
        return kv8_page(pages, seqs, seq_pages, pool, seq, p);
    }
};

// The value of a code under a scale byte: exact in f32 and in bf16.
__device__ __forceinline__ float kv8_value(uint32_t code, uint32_t scale) {
    return __builtin_amdgcn_cvt_f32_fp8((int)code, 0) * __uint_as_float(scale << 23);
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)lo, (__bf16)hi});
}
__device__ __forceinline__ float half_of(const u32x4& x, int e) { return e & 1 ? bf_hi(x[e / 2]) : bf_lo(x[e / 2]); }

// Values moved within a row of 16 lanes by DPP (0xB1, 0x4E: xor 1 and 2; 0x141: lane 7 - i of each half row; 0x124, 0x128:
// 4 and 8 lanes round): every lane has a source, so no old value is kept.
template <int CTRL>
__device__ __forceinline__ uint32_t row_move(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true);
}
template <int CTRL>
__device__ __forceinline__ uint64_t row_move_u(uint64_t v) {
    return (uint64_t)row_move<CTRL>((uint32_t)(v >> 32)) << 32 | row_move<CTRL>((uint32_t)v);
}
template <int CTRL>
__device__ __forceinline__ double row_move_d(double v) {
    return __longlong_as_double((long long)row_move_u<CTRL>((uint64_t)__double_as_longlong(v)));
}
// The sums of lanes 0 .. i, by DPP: within the rows of 16, then lane 15 of rows 0 and 2, then lane 31.
__device__ __forceinline__ uint32_t wave_up_to(uint32_t x) {
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xF, 0xF, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xF, 0xF, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xF, 0xF, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xF, 0xF, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xA, 0xF, false);
    return x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xC, 0xF, false);
}
__device__ __forceinline__ float row_max(float v) {
    v = fmaxf(v, __uint_as_float(row_move<0xB1>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(row_move<0x4E>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(row_move<0x141>(__float_as_uint(v))));
    return fmaxf(v, __uint_as_float(row_move<0x128>(__float_as_uint(v))));
}
__device__ __forceinline__ float row_sum(float v) {
    v += __uint_as_float(row_move<0xB1>(__float_as_uint(v)));
    v += __uint_as_float(row_move<0x4E>(__float_as_uint(v)));
    v += __uint_as_float(row_move<0x141>(__float_as_uint(v)));
    return v + __uint_as_float(row_move<0x128>(__float_as_uint(v)));
}
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max_u16(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

// The codes of a lane's 8 bf16 values of a row that lies in 16 lanes, and the row's scale byte. The largest magnitude
// is that of the bit patterns, two at a time; infinities and NaN, whose patterns are above all finite ones, are taken
// out (and their codes set: the conversion's own NaN has either sign) only where a wavefront meets one.
__device__ __forceinline__ u32x2 quantise(u32x4 x, uint32_t& scale) {
    auto largest = [](u32x4 m) {
        uint32_t top = max_u16(max_u16(m[0], m[1]), max_u16(m[2], m[3]));
        top = max(top & 0xFFFFu, top >> 16);
        top = max(top, row_move<0xB1>(top));
        top = max(top, row_move<0x4E>(top));
        top = max(top, row_move<0x141>(top));
        return max(top, row_move<0x128>(top));
    };
    const u32x4 mag = x & 0x7FFF7FFFu;
    uint32_t top = largest(mag);
    const bool poison = __any(top >= 0x7F80u);
    if (poison) {
        u32x4 m = mag;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            m[j] &= ((m[j] & 0xFFFFu) >= 0x7F80u ? 0u : 0xFFFFu) | (m[j] >> 16 >= 0x7F80u ? 0u : 0xFFFF0000u);
        }
        top = largest(m);
    }
    const int e = kv8_exponent(top);
    scale = (uint32_t)(e + 127);
    const float power = __uint_as_float(scale << 23);
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    u32x2 w;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t first = x[2 * j], second = x[2 * j + 1];  // an element of a vector is no object to cast
        s16x2 c = {0, 0};
        c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, __builtin_bit_cast(bf16x2, first), power, false);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, __builtin_bit_cast(bf16x2, second), power, true);
        w[j] = __builtin_bit_cast(uint32_t, c);
    }
    if (poison) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t code = 0xFFu << 8 * (j % 4);
            w[j / 4] = (mag[j / 2] >> 16 * (j % 2) & 0xFFFFu) >= 0x7F80u ? (w[j / 4] & ~code) | (0x7F7F7F7Fu & code) : w[j / 4];
        }
    }
    return w;
}

constexpr uint32_t WRITE_ROWS = 16;   // rows of a block, one to 16 lanes
constexpr uint32_t WRITE_HEADS = 4;   // heads of q or k that a block takes, where there are blocks enough
constexpr uint32_t WRITE_VALUES = 4;  // kv heads whose values a block takes

struct Write {
    Table t;
    uint8_t *codes, *scales;
    const bf16_t *qkv, *q_norm, *k_norm;
    const double2* cs;
    const uint32_t *row_seq, *row_pos;
    bf16_t *q_out, *bounds;
    uint32_t rows, q_heads, positions;
    float eps;
};

// A lane's part of a head: dims 4 n .. + 3 and the same 64 dims on, so that a dim and the one it is rotated with are in
// one lane.
__device__ __forceinline__ u32x4 load_head(const bf16_t* head, uint32_t n) {
    const u32x2 a = *reinterpret_cast<const u32x2*>(head + 4 * n), b = *reinterpret_cast<const u32x2*>(head + 64 + 4 * n);
    return u32x4{a[0], a[1], b[0], b[1]};
}
// The sum of a head's squares, every lane of its 16 with it: pairs (i, i + 64) first, then the bits of i from the
// lowest, the tree of x0ne_qk_norm_rope_kv_write_rows_bf16 (the squares are exact, so the pairs' sums are one fma).
__device__ __forceinline__ double square_sum(u32x4 x) {
    double s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const double a = (double)half_of(x, j), b = (double)half_of(x, 4 + j);
        s[j] = fma(b, b, a * a);
    }
    double sum = (s[0] + s[1]) + (s[2] + s[3]);
    sum += row_move_d<0xB1>(sum);
    sum += row_move_d<0x4E>(sum);
    sum += row_move_d<0x141>(sum);
    return sum + row_move_d<0x128>(sum);
}
// The head normed (scale: 1 over its root mean square) and rotated, as bf16.
__device__ __forceinline__ u32x4 turn_head(u32x4 x, double scale, u32x4 w, const double2 (&c)[4]) {
    float a[4], b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const double na = (double)half_of(x, j) * scale * (double)half_of(w, j);
        const double nb = (double)half_of(x, 4 + j) * scale * (double)half_of(w, 4 + j);
        a[j] = (float)(na * c[j].x - nb * c[j].y);
        b[j] = (float)(nb * c[j].x + na * c[j].y);
    }
    return u32x4{pack(a[0], a[1]), pack(a[2], a[3]), pack(b[0], b[1]), pack(b[2], b[3])};
}
__device__ __forceinline__ double root_of(double sum, float eps) { return 1.0 / sqrt(sum / (double)KV8_HEAD + (double)eps); }

// The bounds of a page whose key of slot r lies as codes w (dims as load_head's) and a scale byte in the 16 lanes r of
// the block: the keys through LDS, then a thread per dim and side.
typedef float KeyValues[KV8_PAGE][KV8_HEAD + 4];
__device__ __forceinline__ void put_bounds(u32x2 w, uint32_t byte, bf16_t* to, KeyValues& keys) {
    const uint32_t n = threadIdx.x & 15, r = threadIdx.x >> 4;
#pragma unroll
    for (int j = 0; j < 2; ++j)
        *reinterpret_cast<f32x4*>(&keys[r][64 * j + 4 * n]) = f32x4{kv8_value(w[j] & 0xFFu, byte), kv8_value(w[j] >> 8 & 0xFFu, byte),
                                                                    kv8_value(w[j] >> 16 & 0xFFu, byte), kv8_value(w[j] >> 24, byte)};
    lds_barrier();
    const uint32_t d = threadIdx.x % KV8_HEAD;
    const float sign = threadIdx.x < KV8_HEAD ? -1.f : 1.f;  // the smallest is the largest of the negatives
    float top = -INFINITY;
    bool nan = false;
#pragma unroll
    for (uint32_t i = 0; i < KV8_PAGE; ++i) {
        const float v = sign * keys[i][d];
        nan |= v != v;
        top = fmaxf(top, v);
    }
    to[threadIdx.x] = f2bf(nan ? __uint_as_float(0x7FC00000u) : sign * top + 0.f);  // a zero of either sign is +0
    lds_barrier();  // the keys are read
}

// RMSNorm of each head of q and k, rotate-half RoPE from the table, q to q_out as bf16, k and v quantised into their
// page: the arithmetic of x0ne_qk_norm_rope_kv_write_rows_bf16, so q_out has its bits and the codes are those of its k
// row. A block takes 16 rows, 16 lanes to a row, and by blockIdx.y
//  - HEADS heads of q, or of k behind those: their loads are all requested at once, cos and sin are read once, and the
//    f64 square roots and divisions are one for all (lane i computes head i's). Of k, and of values, the page lookups of a
//    thread's row and of row n (to tell a whole page) come one after the other, each waited for, behind those loads;
//  - then the values of WRITE_VALUES kv heads, turned dim-major in LDS: where the block's rows are one whole page, as in
//    a prompt, that is stored as such, else byte by byte.
// A row of no sequence, or past the sequence's pages or the rope table, writes nothing.
// Bounds of a page belong to the blocks of the row of its last slot. Rows that are one whole page have its keys at
// hand; else each 16 lanes take a slot, whose codes are this block's own (through LDS) or of an earlier call (from the
// cache); a row of this call before the block's, whose codes another block writes meanwhile, is computed again (all of the
// call's rows computed again: 64 rows of 64 sequences 9.6 us for 7.4, 777 rows 13.1 for 12.8).
template <int HEADS>
__global__ void __launch_bounds__(256) kv8_write_kernel(const Write a) {
    constexpr uint32_t HD = KV8_HEAD;
    __shared__ union {
        uint32_t turned[WRITE_VALUES][KV8_PART / 4];
        struct {
            KeyValues keys;
            uint32_t code[HEADS][WRITE_ROWS][HD / 4], byte[HEADS][WRITE_ROWS];
        };
    } sh;
    const uint32_t n = threadIdx.x & 15, r = threadIdx.x >> 4, r0 = blockIdx.x * WRITE_ROWS, last = a.rows - 1;
    const uint32_t kvh = a.t.kv_heads, heads = a.q_heads + kvh;
    const uint32_t q_parts = (a.q_heads + HEADS - 1) / HEADS, parts = q_parts + (kvh + HEADS - 1) / HEADS;
    const size_t stride = (size_t)(heads + kvh) * HD;
    auto live_at = [&](uint32_t row, uint32_t seq, uint32_t pos) {
        return row <= last && seq < a.t.seqs && pos < a.positions && pos / KV8_PAGE < a.t.seq_pages;
    };
    const uint32_t row = r0 + r, seq = a.row_seq[min(row, last)], pos = a.row_pos[min(row, last)], slot = pos % KV8_PAGE;
    const bool live = live_at(row, seq, pos);
    // Row n of the block, in every 16 lanes: what the block as a whole goes by.
    const uint32_t row_n = r0 + n, seq_n = a.row_seq[min(row_n, last)], pos_n = a.row_pos[min(row_n, last)];
    auto page_at = [&](uint32_t row, uint32_t seq, uint32_t pos) {
        return live_at(row, seq, pos) ? a.t.page(seq, pos / KV8_PAGE) : KV8_NONE;
    };
    const bf16_t* line = a.qkv + min(row, last) * stride;
    if (blockIdx.y < parts) {
        const bool is_q = blockIdx.y < q_parts;
        // Heads of q, or (the same code on other numbers) of k, which lie behind them.
        const uint32_t h0 = (is_q ? blockIdx.y : blockIdx.y - q_parts) * HEADS, count = min((uint32_t)HEADS, (is_q ? a.q_heads : kvh) - h0);
        const size_t first = (size_t)(is_q ? h0 : a.q_heads + h0) * HD;
        u32x4 x[HEADS];
#pragma unroll
        for (uint32_t i = 0; i < HEADS; ++i) x[i] = load_head(line + first + min(i, count - 1) * HD, n);
        const u32x4 w = load_head(is_q ? a.q_norm : a.k_norm, n);
        double2 c[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = a.cs[(size_t)(live ? pos : 0) * (HD / 2) + 4 * n + j];
        const uint32_t page = is_q ? KV8_NONE : page_at(row, seq, pos), page_n = is_q ? KV8_NONE : page_at(row_n, seq_n, pos_n);
        double square = 0.0;
#pragma unroll
        for (uint32_t i = 0; i < HEADS; ++i) {
            const double sum = square_sum(x[i]);
            if (n == i) square = sum;
        }
        const double root = root_of(square, a.eps);
#pragma unroll
        for (uint32_t i = 0; i < HEADS; ++i) x[i] = turn_head(x[i], __shfl(root, (threadIdx.x & 48) + i, 64), w, c);
        if (is_q) {
            bf16_t* to = a.q_out + ((size_t)row * a.q_heads + h0) * HD;
#pragma unroll
            for (uint32_t i = 0; i < HEADS; ++i)
                if (live && i < count) {
                    *reinterpret_cast<u32x2*>(to + i * HD + 4 * n) = u32x2{x[i][0], x[i][1]};
                    *reinterpret_cast<u32x2*>(to + i * HD + 64 + 4 * n) = u32x2{x[i][2], x[i][3]};
                }
            return;
        }
        const bool whole = __all(page_n != KV8_NONE && pos_n % KV8_PAGE == n && page_n == __builtin_amdgcn_readfirstlane(page_n));
        u32x2 code[HEADS];
        uint32_t byte[HEADS];
#pragma unroll
        for (uint32_t i = 0; i < HEADS; ++i) {
            code[i] = quantise(x[i], byte[i]);
            if (page == KV8_NONE || i >= count) continue;
            uint8_t* to = a.codes + kv8_record(page, kvh, h0 + i) + slot * HD;
            *reinterpret_cast<uint32_t*>(to + 4 * n) = code[i][0];
            *reinterpret_cast<uint32_t*>(to + 64 + 4 * n) = code[i][1];
            if (n == 0) a.scales[kv8_scale(page, kvh, h0 + i) + slot] = (uint8_t)byte[i];
        }
        if (!a.bounds) return;
        if (whole) {
#pragma unroll
            for (uint32_t i = 0; i < HEADS; ++i)
                if (i < count) put_bounds(code[i], byte[i], a.bounds + kv8_bound(page_n, kvh, h0 + i), sh.keys);
            return;
        }
        uint64_t ends = __ballot(page_n != KV8_NONE && pos_n % KV8_PAGE == KV8_PAGE - 1) & 0xFFFFu;
        if (!ends) return;
#pragma unroll
        for (uint32_t i = 0; i < HEADS; ++i) {
            sh.code[i][r][n] = code[i][0];
            sh.code[i][r][16 + n] = code[i][1];
            if (n == 0) sh.byte[i][r] = byte[i];
        }
        lds_barrier();
        for (; ends; ends &= ends - 1) {
            const uint32_t at = (uint32_t)__builtin_ctzll(ends), end = r0 + at;
            const uint32_t its_seq = __builtin_amdgcn_readlane(seq_n, at), its_pos = __builtin_amdgcn_readlane(pos_n, at);
            const uint32_t its_page = __builtin_amdgcn_readlane(page_n, at);
            const uint32_t from = end + r - 15, from_pos = its_pos + r - 15;  // slot r's row, if it is of this call
            const bool fresh = end + r >= 15 && a.row_seq[min(from, last)] == its_seq && a.row_pos[min(from, last)] == from_pos;
            const bool here = fresh && from >= r0;
#pragma unroll 1
            for (uint32_t i0 = 0; i0 < count; i0 += 2) {
                u32x2 v[2];
                uint32_t b[2];
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i) {
                    const uint32_t h = h0 + min(i0 + i, count - 1);
                    const uint8_t* rec = a.codes + kv8_record(its_page, kvh, h) + r * HD;
                    v[i] = u32x2{*reinterpret_cast<const uint32_t*>(rec + 4 * n), *reinterpret_cast<const uint32_t*>(rec + 64 + 4 * n)};
                    b[i] = a.scales[kv8_scale(its_page, kvh, h) + r];
                }
                if (__any(fresh && !here)) {
                    u32x4 was[2];
#pragma unroll
                    for (uint32_t i = 0; i < 2; ++i) was[i] = load_head(a.qkv + min(from, last) * stride + first + min(i0 + i, count - 1) * HD, n);
#pragma unroll
                    for (int j = 0; j < 4; ++j) c[j] = a.cs[(size_t)from_pos * (HD / 2) + 4 * n + j];
#pragma unroll
                    for (uint32_t i = 0; i < 2; ++i) {
                        uint32_t again;
                        const u32x2 x = quantise(turn_head(was[i], root_of(square_sum(was[i]), a.eps), w, c), again);
                        if (fresh) {
                            v[i] = x;
                            b[i] = again;
                        }
                    }
                }
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i) {
                    if (i0 + i >= count) break;
                    if (here) {
                        v[i] = u32x2{sh.code[i0 + i][from - r0][n], sh.code[i0 + i][from - r0][16 + n]};
                        b[i] = sh.byte[i0 + i][from - r0];
                    }
                    put_bounds(v[i], b[i], a.bounds + kv8_bound(its_page, kvh, h0 + i0 + i), sh.keys);
                }
            }
        }
        return;
    }
    const uint32_t k0 = (blockIdx.y - parts) * WRITE_VALUES;
    u32x4 x[WRITE_VALUES];
#pragma unroll
    for (uint32_t i = 0; i < WRITE_VALUES; ++i) x[i] = *reinterpret_cast<const u32x4*>(line + (heads + min(k0 + i, kvh - 1)) * HD + 8 * n);
    const uint32_t page = page_at(row, seq, pos), page_n = page_at(row_n, seq_n, pos_n);
    const bool whole = __all(page_n != KV8_NONE && pos_n % KV8_PAGE == n && page_n == __builtin_amdgcn_readfirstlane(page_n));
#pragma unroll
    for (uint32_t i = 0; i < WRITE_VALUES; ++i) {
        uint32_t byte;
        const u32x2 w = quantise(x[i], byte);
        uint8_t* to = reinterpret_cast<uint8_t*>(sh.turned[i]) + 8 * n * WRITE_ROWS + r;
#pragma unroll
        for (int j = 0; j < 8; ++j) to[j * WRITE_ROWS] = (uint8_t)(w[j / 4] >> 8 * (j % 4));
        if (n == 0 && page != KV8_NONE && k0 + i < kvh) a.scales[kv8_scale(page, kvh, k0 + i) + KV8_PAGE + slot] = (uint8_t)byte;
    }
    lds_barrier();
#pragma unroll
    for (uint32_t i = 0; i < WRITE_VALUES; ++i) {
        if (k0 + i >= kvh) break;
        if (whole) {
            uint8_t* to = a.codes + kv8_record(page_n, kvh, k0 + i) + KV8_PART;
            reinterpret_cast<u32x2*>(to)[threadIdx.x] = reinterpret_cast<const u32x2*>(sh.turned[i])[threadIdx.x];
        } else if (page_n != KV8_NONE) {
            uint8_t* to = a.codes + kv8_record(page_n, kvh, k0 + i) + KV8_PART + pos_n % KV8_PAGE;
            for (uint32_t d = r; d < HD; d += 16) to[d * KV8_PAGE] = reinterpret_cast<const uint8_t*>(sh.turned[i])[d * WRITE_ROWS + n];
        }
    }
}

// A load or store of what is too much for the Infinity Cache to hold until it is read again (STREAM: not kept there).
template <bool STREAM, class T>
__device__ __forceinline__ T take(const T* p) {
    if constexpr (STREAM) return __builtin_nontemporal_load(p);
    return *p;
}
template <bool STREAM, class T>
__device__ __forceinline__ void put(T* p, T x) {
    if constexpr (STREAM)
        __builtin_nontemporal_store(x, p);
    else
        *p = x;
}

// Eight codes as bf16, times the power of two `scale`: exact.
__device__ __forceinline__ u32x4 decode(uint32_t lo, uint32_t hi, float scale) {
    u32x4 r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
    return r;
}

// Positions below a sequence's length as bf16: the codes' order is the bf16 pages' order, so a wavefront streams one
// page of one head, 8 codes per lane and load and 16 bytes per lane and store. Slots past the length are zero; a page
// that is not there reads as zeros, an output page outside its pool is not written.
template <bool STREAM>
__global__ void __launch_bounds__(256)
    kv8_read_kernel(Table t, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                    const uint32_t* __restrict__ lens, bf16_t* __restrict__ k_out, bf16_t* __restrict__ v_out,
                    const uint32_t* __restrict__ out_table, uint32_t out_pool) {
    const uint32_t s = blockIdx.y, i = threadIdx.x & 63;
    const uint32_t keys = kv8_keys(lens[s], t.seq_pages);
    const uint64_t records = (uint64_t)((keys + KV8_PAGE - 1) / KV8_PAGE) * t.kv_heads;
    for (uint64_t id = (uint64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); id < records; id += (uint64_t)gridDim.x * 4) {
        const uint32_t p = (uint32_t)(id / t.kv_heads), kh = (uint32_t)(id % t.kv_heads);
        const uint32_t to = kv8_page(out_table, t.seqs, t.seq_pages, out_pool, s, p), page = t.page(s, p);
        if (to == KV8_NONE) continue;
        const uint32_t valid = page == KV8_NONE ? 0u : min(keys - p * KV8_PAGE, KV8_PAGE), from = page == KV8_NONE ? 0u : page;
        const u32x2* rec = reinterpret_cast<const u32x2*>(codes + kv8_record(from, t.kv_heads, kh)) + i;
        const uint8_t* sc = scales + kv8_scale(from, t.kv_heads, kh);
        u32x2 k[4], v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) k[j] = take<STREAM>(rec + 64 * j);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = take<STREAM>(rec + KV8_PART / 8 + 64 * j);
        // Keys 4 j + i / 16; the values of positions 8 (i % 2) .. + 7.
        const u32x4 ks = *reinterpret_cast<const u32x4*>(sc);
        const u32x2 vs = *reinterpret_cast<const u32x2*>(sc + KV8_PAGE + 8 * (i & 1));
        u32x4 *kd = reinterpret_cast<u32x4*>(k_out + ((size_t)to * t.kv_heads + kh) * KV8_PART) + i,
              *vd = reinterpret_cast<u32x4*>(v_out + ((size_t)to * t.kv_heads + kh) * KV8_PART) + i;
        float power[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) power[e] = __uint_as_float((vs[e / 4] >> 8 * (e % 4) & 0xFFu) << 23);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u32x4 x = decode(k[j][0], k[j][1], __uint_as_float((ks[j] >> 8 * (i >> 4) & 0xFFu) << 23));
            if (4 * j + (i >> 4) >= valid) x = u32x4{0, 0, 0, 0};
            put<STREAM>(kd + 64 * j, x);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const auto two = (e & 2) ? __builtin_amdgcn_cvt_pk_f32_fp8((int)v[j][e / 4], true)
                                         : __builtin_amdgcn_cvt_pk_f32_fp8((int)v[j][e / 4], false);
                f[e] = 8 * (i & 1) + e < valid ? two[0] * power[e] : 0.f;
                f[e + 1] = 8 * (i & 1) + e + 1 < valid ? two[1] * power[e + 1] : 0.f;
            }
            put<STREAM>(vd + 64 * j, u32x4{pack(f[0], f[1]), pack(f[2], f[3]), pack(f[4], f[5]), pack(f[6], f[7])});
        }
    }
}

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// Partial states go between blocks through agent-scope accesses, coherent across the XCDs' caches.
__device__ __forceinline__ void put2(float* p, float a, float b) {
    __hip_atomic_store((uint64_t*)p, (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get2(const float* p) {
    const uint64_t v = __hip_atomic_load((const uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}
// A state without a key has the maximum -inf. One whose keys all score -inf (an infinity in the query) has the lowest
// finite value and no weight: its softmax is 0 / 0.
constexpr float LOWEST = -3.402823466e+38f;
__device__ __forceinline__ float share(float top, float l) { return l != 0.f ? 1.f / l : top == -INFINITY ? 0.f : NAN; }
// 2^(m - top), 0 for a state without a key.
__device__ __forceinline__ float factor(float m, float top) {
    return __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.f : top));
}

constexpr uint32_t STATE = KV8_HEAD + 4;  // floats of a partial state: m, l, two unused, o
constexpr uint32_t MAX_GROUP = 16;

struct Attend {
    Table t;
    const uint8_t *codes, *scales;
    const bf16_t* q;
    const uint32_t *lens, *list;
    bf16_t* out;
    float* state;
    uint32_t* counter;
    uint32_t budget, q_heads, group, slices, rounds;
    float scale2;  // the scale times log2 e: a weight is one exp2
};

template <uint32_t WAVES>
struct Shared {
    float wm[WAVES][MAX_GROUP], wl[WAVES][MAX_GROUP];
    float wo[WAVES][MAX_GROUP][KV8_HEAD + 4];
    float m[MAX_GROUP][KV8_SLICES], l[MAX_GROUP][KV8_SLICES];  // the join's: each slice's maximum (then factor) and sum
    uint32_t last;
};

// The slices' states of a group's heads joined, in slice order within each part: a thread has four dims of one head
// and, where a group's 32 threads a head are at most a quarter or half of the block (2 and 4 heads for 4 wavefronts, 4 and 8
// for 8), every fourth or second slice (the parts meet in LDS). All of a thread's loads of up to JOIN_AHEAD slices are
// requested before the maxima are known, so they cost one round trip.
constexpr uint32_t JOIN_AHEAD = 8;
template <uint32_t WAVES>
__device__ __forceinline__ void join(const Attend& a, const float* __restrict__ st, bf16_t* __restrict__ out,
                                     uint32_t active, Shared<WAVES>& sh) {
    constexpr uint32_t THREADS = 64 * WAVES;
    const uint32_t t = threadIdx.x, quads = a.group * (KV8_HEAD / 4);
    const uint32_t parts = quads <= THREADS / 4 ? 4 : quads <= THREADS / 2 ? 2 : 1;
    const uint32_t part = t / (THREADS / parts), first = t % (THREADS / parts);
    auto request = [&](uint32_t e, uint32_t z0, f32x4 (&x)[JOIN_AHEAD]) {
        const float* p = st + (size_t)(e / (KV8_HEAD / 4)) * a.slices * STATE + 4 + 4 * (e % (KV8_HEAD / 4));
#pragma unroll
        for (uint32_t i = 0; i < JOIN_AHEAD; ++i) {
            const uint32_t z = z0 + i * parts;
            if (z < active && e < quads) {
                const float2 u = get2(p + z * STATE), v = get2(p + z * STATE + 2);
                x[i] = f32x4{u.x, u.y, v.x, v.y};
            }
        }
    };
    f32x4 ahead[JOIN_AHEAD];
    request(first, part, ahead);
    for (uint32_t i = t; i < a.group * active; i += THREADS) {
        const uint32_t h = i / active, z = i % active;
        const float2 ml = get2(st + ((size_t)h * a.slices + z) * STATE);
        sh.m[h][z] = ml.x;
        sh.l[h][z] = ml.y;
    }
    lds_barrier();
    // Each head's factors and sum by one wavefront, a lane per slice.
    for (uint32_t h = t / 64; h < a.group; h += WAVES) {
        const uint32_t z = t % 64;
        const float m = z < active ? sh.m[h][z] : -INFINITY, top = rows_max(row_max(m)), f = factor(m, top);
        if (z < active) sh.m[h][z] = f;
        const float l = rows_sum(row_sum(z < active ? f * sh.l[h][z] : 0.f));
        if (z == 0) sh.wl[0][h] = share(top, l);
    }
    lds_barrier();
    auto sum = [&](uint32_t e) -> f32x4 {
        const uint32_t h = e / (KV8_HEAD / 4);
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t z0 = part; z0 < active; z0 += JOIN_AHEAD * parts) {
            if (e != first || z0 != part) request(e, z0, ahead);
#pragma unroll
            for (uint32_t i = 0; i < JOIN_AHEAD; ++i)
                if (z0 + i * parts < active) x += sh.m[h][z0 + i * parts] * ahead[i];
        }
        return x;
    };
    auto store = [&](uint32_t e, f32x4 x) {
        const uint32_t h = e / (KV8_HEAD / 4);
        const float r = sh.wl[0][h];
        *reinterpret_cast<uint2*>(out + 4 * e) = make_uint2(pack(x[0] * r, x[1] * r), pack(x[2] * r, x[3] * r));
    };
    if (parts == 1) {
        for (uint32_t e = first; e < quads; e += THREADS) store(e, sum(e));  // twice for more than 8 heads of 4 wavefronts
        return;
    }
    float* mine = &sh.wo[0][0][0] + 4 * t;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    if (first < quads) x = sum(first);
    *reinterpret_cast<f32x4*>(mine) = x;
    lds_barrier();
    if (part || first >= quads) return;
    for (uint32_t w = 1; w < parts; ++w) x += *reinterpret_cast<const f32x4*>(mine + 4 * w * (THREADS / parts));
    store(first, x);
}

// A slice of a sequence: its tiles are cut into `active` slices of `per` tiles, by its own length and the call's `slices`
// and `rounds` only. A block walks slices of its kv head and its 64 sequences: lane l of each wavefront holds a sequence's
// length, its slices' number and size (the divisions, once for all lanes) and the slices up to and with it.
struct Item {
    uint32_t s, y, keys, pages, np, per, active, t0, t_end;  // sequence and slice; this wavefront's tiles t0, t0 + WAVES ..
    __device__ __forceinline__ bool any() const { return t0 < t_end; }
};

// Decode attention. A block takes slices of the sequences' tiles for the q heads of one kv head, one after the other,
// its wavefront w of WAVES a slice's tiles w, w + WAVES, ...; a tile is 4 pages. The products are S^T = K Q^T and
// O^T = V^T P^T on the matrix cores (16 x 16 x 32, bf16 with f32 sums), the group's heads the 16 columns: lane
// (n = lane % 16, g = lane / 16) holds column n, so the softmax of a head is lane-local but for the four lanes n,
// n + 16, n + 32, n + 48. Codes become bf16 in one conversion, keys times their scale (exact); a value's scale goes
// into its weight (exact).
//  - Product m's row r = 4 g' + i is key 4 m + i of the tile's page g': its 16 outputs per lane are then the 16 keys of
//    page g, and with the value of dim 16 c + n at those keys as row n of product c (one 16-byte load: V is dim-major)
//    the weights are an operand as they lie, without a move between lanes.
//  - Dims of a product's k step j are 32 g + 8 j ..: a lane's keys come as two 16-byte loads.
//  - Weights enter as bf16 hi + lo (2^-17 of the weight, 2^-134 where its value's power of two is tiny): one bf16 would add
//    as much error as the output's rounding. Their sum takes them whole.
// The next tile's keys are requested behind the scores, its values behind the value products; the next slice's first
// tile and queries likewise, so the memory is busy while a slice's states are joined. It is not at a slice's start: the
// list and table entries of the slice after it are waited for there, one behind the other, and with them this slice's
// first tile, before its first product. The running maximum and sum are f32, and the sums of weighted values, not yet
// divided: values near bf16's largest over several keys pass f32. A slice's state (m, l, o) is joined by the last block
// of its (sequence, kv head) to count itself, slices in order; a sequence of one slice is written at once. Keys past the
// length, entries behind a list and pages that are not there weigh 0, their values are taken as 0.
template <uint32_t WAVES, bool STREAM>
__global__ void __launch_bounds__(64 * WAVES, 2) kv8_attention_kernel(const Attend a) {
    constexpr uint32_t THREADS = 64 * WAVES;
    __shared__ Shared<WAVES> sh;
    const uint32_t kh = blockIdx.x, s0 = blockIdx.z * 64, step = WAVES;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    auto shape = [&](uint32_t keys) -> Item {  // all but its slices
        Item it = {};
        it.keys = keys;
        it.pages = (keys + KV8_PAGE - 1) / KV8_PAGE;
        it.np = a.list ? min(a.budget, it.pages) : it.pages;
        it.t_end = (it.np + KV8_TILE - 1) / KV8_TILE;
        return it;
    };
    uint32_t my_keys = s0 + lane < a.t.seqs ? kv8_keys(a.lens[s0 + lane], a.t.seq_pages) : 0u, my_seq = lane;
    uint32_t per, active = kv8_slices(shape(my_keys).t_end, WAVES, a.slices, a.rounds, per);
    if (s0 + lane >= a.t.seqs) active = 0;
    uint32_t upto = wave_up_to(active);
    const uint32_t total = __builtin_amdgcn_readlane(upto, 63), blocks = gridDim.y;
    if (total > blocks) {  // several slices per block: the longest sequences' first
        uint32_t rank = 0;
        const uint32_t there = min(64u, a.t.seqs - s0);
#pragma unroll 1
        for (uint32_t j = 0; j < there; ++j) {
            const uint32_t other = __builtin_amdgcn_readlane(my_keys, j);
            rank += other > my_keys || (other == my_keys && j < lane);
        }
        my_seq = (uint32_t)__builtin_amdgcn_ds_permute((int)(4 * rank), (int)lane);
        my_keys = (uint32_t)__builtin_amdgcn_ds_permute((int)(4 * rank), (int)my_keys);
        per = (uint32_t)__builtin_amdgcn_ds_permute((int)(4 * rank), (int)per);
        active = (uint32_t)__builtin_amdgcn_ds_permute((int)(4 * rank), (int)active);
        upto = wave_up_to(active);
    }
    // A block's slice of round r, the rounds to and fro over the blocks.
    auto item = [&](uint32_t r) -> Item {
        const uint32_t i = kv8_turn(r, blockIdx.y, blocks);
        if (i >= total) return Item{};
        const uint32_t at = (uint32_t)__popcll(__ballot(upto <= i));
        Item it = shape(__builtin_amdgcn_readlane(my_keys, at));
        it.s = s0 + __builtin_amdgcn_readlane(my_seq, at);
        it.per = __builtin_amdgcn_readlane(per, at);
        it.active = __builtin_amdgcn_readlane(active, at);
        it.y = i - (__builtin_amdgcn_readlane(upto, at) - it.active);
        it.t0 = it.y * it.per + wave;
        it.t_end = min(it.t_end, (it.y + 1) * it.per);
        return it;
    };

    // A lane's page of a tile is the one at index 4 t + g: its logical number (from the list two tiles ahead), its
    // table entry (one tile ahead), and then the physical page with how many of its keys count.
    struct Place {
        uint32_t page, valid;
    };
    auto logical_at = [&](const Item& it, uint32_t t) -> uint32_t {
        const uint32_t at = KV8_TILE * t + g;
        if (t >= it.t_end || at >= it.np) return KV8_NONE;
        return a.list ? a.list[((size_t)it.s * a.t.kv_heads + kh) * a.budget + at] : at;
    };
    auto entry_of = [&](const Item& it, uint32_t logical) -> uint32_t {
        return logical < it.pages ? a.t.pages[(size_t)it.s * a.t.seq_pages + logical] : KV8_NONE;
    };
    auto place = [&](const Item& it, uint32_t logical, uint32_t entry) -> Place {
        if (entry >= a.t.pool) return Place{0u, 0u};
        return Place{entry, (uint32_t)min(it.keys - logical * KV8_PAGE, KV8_PAGE)};
    };
    u32x4 k[4][2], v[8], ks, vs, qb[4];
    auto key_at = [&](uint32_t page) -> const uint8_t* {
        return a.codes + kv8_record(page, a.t.kv_heads, kh) + (n & 3) * KV8_HEAD + 32 * g;
    };
    auto key_scales = [&](uint32_t page) { return reinterpret_cast<const u32x4*>(a.scales + kv8_scale(page, a.t.kv_heads, kh)); };
    auto value_at = [&](uint32_t page) -> const uint8_t* {
        return a.codes + kv8_record(page, a.t.kv_heads, kh) + KV8_PART + n * KV8_PAGE;
    };
    // The lanes of row n of a key product take page n / 4, the page of the lanes 16 (n / 4) ...
    auto key_page = [&](uint32_t page) -> uint32_t { return __shfl(page, 16 * (n >> 2), 64); };
    auto load_k = [&](const uint8_t* p, int m) {
        k[m][0] = take<STREAM>(reinterpret_cast<const u32x4*>(p + m * 4 * KV8_HEAD));
        k[m][1] = take<STREAM>(reinterpret_cast<const u32x4*>(p + m * 4 * KV8_HEAD + 16));
    };
    auto load_v = [&](const uint8_t* p, int c) { v[c] = take<STREAM>(reinterpret_cast<const u32x4*>(p + c * 16 * KV8_PAGE)); };
    // Columns past the group repeat its last head: their results are not used.
    auto load_q = [&](const Item& it) {
        const bf16_t* p = a.q + ((size_t)it.s * a.q_heads + kh * a.group + min(n, a.group - 1)) * KV8_HEAD + 32 * g;
#pragma unroll
        for (int j = 0; j < 4; ++j) qb[j] = reinterpret_cast<const u32x4*>(p)[j];
    };
    auto load_first = [&](const Item& it, const Place& at) {
        const uint32_t page = key_page(at.page);
        const uint8_t *kp = key_at(page), *vp = value_at(at.page);
        ks = *key_scales(page);
#pragma unroll
        for (int m = 0; m < 4; ++m) load_k(kp, m);
        vs = key_scales(at.page)[1];
#pragma unroll
        for (int c = 0; c < 8; ++c) load_v(vp, c);
        load_q(it);
    };

    Item it = item(0);
    if (!it.active) return;
    // A slice whose states are written but not counted: its sequence and how many slices that has. The block that
    // counts the last one joins them.
    struct Waiting {
        uint32_t s, active;
    };
    auto counter_of = [&](const Waiting& w) { return a.counter + (size_t)w.s * a.t.kv_heads + kh; };
    auto finish = [&](const Waiting& w) {
        if (threadIdx.x == 0) __hip_atomic_store(counter_of(w), 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next call
        const size_t head = (size_t)w.s * a.q_heads + kh * a.group;
        join(a, a.state + head * a.slices * STATE, a.out + head * KV8_HEAD, w.active, sh);
    };
    uint32_t l0 = logical_at(it, it.t0), l1 = logical_at(it, it.t0 + step), l2 = logical_at(it, it.t0 + 2 * step);
    uint32_t e0 = entry_of(it, l0), e1 = entry_of(it, l1);
    Place here = place(it, l0, e0);
    if (it.any()) load_first(it, here);
    Waiting waiting = {};
    for (uint32_t r = 1;; ++r) {
        const Item next = item(r);
        const uint32_t n0 = logical_at(next, next.t0), n1 = logical_at(next, next.t0 + step), n2 = logical_at(next, next.t0 + 2 * step);
        const uint32_t f0 = entry_of(next, n0), f1 = entry_of(next, n1);
        float m_run = -INFINITY, lsum = 0.f;
        f32x4 o[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (uint32_t t = it.t0; t < it.t_end; t += step) {
            const uint32_t e2 = entry_of(it, l2), l3 = logical_at(it, t + 3 * step);
            // The tile behind this one: of this slice, the first of the next, or (behind the last) page 0, without use.
            const bool more = t + step < it.t_end;
            const Place then = more ? place(it, l1, e1) : place(next, n0, f0);
            const uint32_t then_page = key_page(then.page);
            const uint8_t *kp = key_at(then_page), *vp = value_at(then.page);
            float sc[4][4];
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const float scale = __uint_as_float(((ks[m] >> (8 * (n & 3))) & 0xFFu) << 23);
                f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < 4; ++j) acc = mfma(decode(k[m][j >> 1][2 * (j & 1)], k[m][j >> 1][2 * (j & 1) + 1], scale), qb[j], acc);
                load_k(kp, m);
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[m][e] = acc[e] * a.scale2;
            }
            ks = *key_scales(then_page);
            if (!more && next.any()) load_q(next);
            const bool whole = __all(here.valid == KV8_PAGE);
            uint32_t keep[4];
            if (!whole) {
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const int left = (int)here.valid - 4 * m;
                    keep[m] = left >= 4 ? 0xFFFFFFFFu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e >= left) sc[m][e] = -INFINITY;
                    vs[m] &= keep[m];
#pragma unroll
                    for (int c = 0; c < 8; ++c) v[c][m] &= keep[m];
                }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = fmaxf(mx, sc[m][e]);
            mx = fmaxf(m_run, rows_max(mx));
            if (whole || __any(here.valid != 0)) mx = fmaxf(mx, LOWEST);
            if (__any(mx > m_run)) {
                const float alpha = factor(m_run, mx);
                lsum *= alpha;
#pragma unroll
                for (int c = 0; c < 8; ++c) o[c] *= alpha;
                m_run = mx;
            }
            const float ref = m_run == -INFINITY ? 0.f : m_run;  // a tile without a key
            u32x4 hi[2], lo[2];
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = __builtin_amdgcn_exp2f(sc[m][e] - ref);
                    lsum += p;
                    w[e] = p * __uint_as_float(((vs[m] >> (8 * e)) & 0xFFu) << 23);
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t h = pack(w[2 * e], w[2 * e + 1]);
                    hi[m >> 1][2 * (m & 1) + e] = h;
                    lo[m >> 1][2 * (m & 1) + e] = pack(w[2 * e] - bf_lo(h), w[2 * e + 1] - bf_hi(h));
                }
            }
            vs = key_scales(then.page)[1];
#pragma unroll
            for (int c = 0; c < 8; ++c) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const u32x4 x = decode(v[c][2 * j], v[c][2 * j + 1], 1.f);
                    o[c] = mfma(x, hi[j], o[c]);
                    o[c] = mfma(x, lo[j], o[c]);
                }
                load_v(vp, c);
            }
            here = then;
            l1 = l2;
            e1 = e2;
            l2 = l3;
        }
        if (!it.any() && next.any()) {
            here = place(next, n0, f0);
            load_first(next, here);
        }
        lsum = rows_sum(lsum);

        // The block's states meet; then the output, or the slice's state. The states of the slice before are
        // counted here: this wavefront's stores of them are older than the loads of at least one tile.
        if (n < a.group) {
            if (g == 0) {
                sh.wm[wave][n] = m_run;
                sh.wl[wave][n] = lsum;
            }
#pragma unroll
            for (int c = 0; c < 8; ++c) *reinterpret_cast<f32x4*>(&sh.wo[wave][n][16 * c + 4 * g]) = o[c];
        }
        if (waiting.active) {
            if (it.any() && next.any())
                asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
            else
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        lds_barrier();
        uint32_t before = 0;
        if (waiting.active && threadIdx.x == 0)
            before = __hip_atomic_fetch_add(counter_of(waiting), 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        bf16_t* out = a.out + ((size_t)it.s * a.q_heads + kh * a.group) * KV8_HEAD;
        float* state = a.state + ((size_t)it.s * a.q_heads + kh * a.group) * a.slices * STATE;
        for (uint32_t e = threadIdx.x; e < a.group * (KV8_HEAD / 4); e += THREADS) {
            const uint32_t h = e / (KV8_HEAD / 4), d = 4 * (e % (KV8_HEAD / 4));
            float top = sh.wm[0][h], l = 0.f;
            f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (uint32_t w = 1; w < WAVES; ++w) top = fmaxf(top, sh.wm[w][h]);
#pragma unroll
            for (uint32_t w = 0; w < WAVES; ++w) {
                const float f = factor(sh.wm[w][h], top);
                l += f * sh.wl[w][h];
                x += f * *reinterpret_cast<const f32x4*>(&sh.wo[w][h][d]);
            }
            if (it.active == 1) {
                const float r = share(top, l);
                *reinterpret_cast<uint2*>(out + h * KV8_HEAD + d) = make_uint2(pack(x[0] * r, x[1] * r), pack(x[2] * r, x[3] * r));
            } else {
                float* st = state + ((size_t)h * a.slices + it.y) * STATE;
                put2(st + 4 + d, x[0], x[1]);
                put2(st + 6 + d, x[2], x[3]);
                if (d == 0) put2(st, top, l);
            }
        }
        if (waiting.active) {
            if (threadIdx.x == 0) sh.last = before == waiting.active - 1;
            lds_barrier();
            if (sh.last) finish(waiting);
        }
        waiting = it.active > 1 ? Waiting{it.s, it.active} : Waiting{};
        if (!next.active) break;
        lds_barrier();  // the states in LDS are read
        it = next;
        l1 = n1;
        e1 = f1;
        l2 = n2;
    }
    if (!waiting.active) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();
    if (threadIdx.x == 0)
        sh.last = __hip_atomic_fetch_add(counter_of(waiting), 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == waiting.active - 1;
    lds_barrier();
    if (sh.last) finish(waiting);
}

// The order of scores as whole numbers: larger scores larger, zeros of either sign equal, NaN above all, 0 below all
// (for a page that is not there).
__device__ __forceinline__ uint64_t score_key(double x) {
    if (x != x) return ~0ull;
    const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

constexpr uint32_t SELECT_THREADS = 256, SELECT_WAVES = SELECT_THREADS / 64;
constexpr uint32_t SELECT_KEYS = 64 / SELECT_WAVES;  // keys that a thread holds while a block selects: 4096 pages at once
constexpr uint32_t SELECT_BINS = 2048;
constexpr uint32_t SELECT_PAGES = 4 * 4 * SELECT_WAVES;  // pages that a block scores: 16 lanes have 4

struct SelectShared {
    uint32_t bin[SELECT_BINS];
    uint64_t key[SELECT_PAGES];  // of a pair whose pages one block scores
    uint64_t low[SELECT_WAVES], high[SELECT_WAVES];
    uint32_t part[SELECT_WAVES], count[SELECT_KEYS * SELECT_WAVES], equal[SELECT_KEYS * SELECT_WAVES];
    uint32_t found, above, inside, last;
};

// The `take` largest of the n keys that get(index) gives (0 < take < n; ties to the lower index), their indices ascending
// in `to`. Radix selection over the range of the keys that are still undecided, 11 bits at a time: the range is that of
// the keys and not of all numbers, so scores of one sign and size are told apart in a pass or two. A thread holds keys
// t, t + 256, ...; more than 4096 are read again in each pass.
template <class Get>
__device__ __forceinline__ void select_keys(Get&& get, uint32_t n, uint32_t take, uint32_t* __restrict__ to, SelectShared& sh) {
    constexpr uint32_t AT_ONCE = SELECT_KEYS * SELECT_THREADS, EACH = SELECT_BINS / SELECT_THREADS;
    const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6;
    uint64_t key[SELECT_KEYS];
    auto rows = [&](uint32_t first, auto&& f) {  // f(row, whether this thread has a key of it), of rows that hold one
#pragma unroll
        for (uint32_t j = 0; j < SELECT_KEYS; ++j) {
            if (first + SELECT_THREADS * j >= n) break;
            f(j, first + SELECT_THREADS * j + t < n);
        }
    };
    auto load = [&](uint32_t first) {
        rows(first, [&](uint32_t j, bool in) {
            if (in) key[j] = get(first + SELECT_THREADS * j + t);
        });
    };
    auto each = [&](auto&& f) {  // f(key) of every key
        for (uint32_t first = 0; first < n; first += AT_ONCE) {
            if (n > AT_ONCE) load(first);
            rows(first, [&](uint32_t j, bool in) {
                if (in) f(key[j]);
            });
        }
    };
    if (n <= AT_ONCE) load(0);
    uint64_t lo = ~0ull, hi = 0;
    each([&](uint64_t x) {
        lo = min(lo, x);
        hi = max(hi, x);
    });
    lo = min(lo, row_move_u<0xB1>(lo));
    hi = max(hi, row_move_u<0xB1>(hi));
    lo = min(lo, row_move_u<0x4E>(lo));
    hi = max(hi, row_move_u<0x4E>(hi));
    lo = min(lo, row_move_u<0x141>(lo));
    hi = max(hi, row_move_u<0x141>(hi));
    lo = min(lo, row_move_u<0x128>(lo));
    hi = max(hi, row_move_u<0x128>(hi));
#pragma unroll
    for (int d = 16; d < 64; d <<= 1) {
        lo = min(lo, (uint64_t)__shfl_xor((unsigned long long)lo, d, 64));
        hi = max(hi, (uint64_t)__shfl_xor((unsigned long long)hi, d, 64));
    }
    if (lane == 0) {
        sh.low[wave] = lo;
        sh.high[wave] = hi;
    }
    for (uint32_t j = t; j < SELECT_BINS; j += SELECT_THREADS) sh.bin[j] = 0;
    lds_barrier();
#pragma unroll
    for (uint32_t w = 0; w < SELECT_WAVES; ++w) {
        lo = min(lo, sh.low[w]);
        hi = max(hi, sh.high[w]);
    }
    uint32_t need = take;  // of the keys from lo to hi; those above are taken
    bool ties = true;      // all keys from lo to hi are equal: the first `need` of them
    for (int pass = 0; pass < KV8_PASSES && lo != hi; ++pass) {
        const int shift = kv8_shift(lo, hi);
        if (pass) {
            for (uint32_t j = t; j < SELECT_BINS; j += SELECT_THREADS) sh.bin[j] = 0;
            lds_barrier();
        }
        each([&](uint64_t x) {
            if (x >= lo && x <= hi) atomicAdd(&sh.bin[(uint32_t)((x - lo) >> shift)], 1u);
        });
        lds_barrier();
        // Bins from the top, EACH to a thread: the one in which the count reaches `need`.
        uint32_t bin[EACH], mine = 0;
#pragma unroll
        for (uint32_t j = 0; j < EACH; ++j) mine += bin[j] = sh.bin[SELECT_BINS - 1 - EACH * t - j];
        const uint32_t upto = wave_up_to(mine);
        if (lane == 63) sh.part[wave] = upto;
        lds_barrier();
        uint32_t above = upto - mine;
#pragma unroll
        for (uint32_t w = 0; w < SELECT_WAVES; ++w) above += w < wave ? sh.part[w] : 0u;
        if (above < need && above + mine >= need) {
            uint32_t j = 0, inside = bin[0];
#pragma unroll
            for (uint32_t b = 1; b < EACH; ++b) {  // past the bins that end before `need`
                if (above + inside >= need) continue;
                above += inside;
                inside = bin[b];
                j = b;
            }
            sh.found = SELECT_BINS - 1 - EACH * t - j;
            sh.above = above;
            sh.inside = inside;
        }
        lds_barrier();
        need -= sh.above;
        kv8_narrow(lo, hi, shift, sh.found);
        if (sh.inside == need) {
            ties = false;
            break;
        }
        lds_barrier();  // found, above and inside are read
    }
    // Indices in order: per row of 256 keys and wavefront the number taken, then its place.
    uint32_t placed = 0, equals = 0;
    for (uint32_t first = 0; first < n; first += AT_ONCE) {
        if (n > AT_ONCE) load(first);
        uint32_t equal_before[SELECT_KEYS];
        const uint64_t below = (1ull << lane) - 1;
        if (t < SELECT_KEYS * SELECT_WAVES) sh.count[t] = sh.equal[t] = 0;
        lds_barrier();
        if (ties) {
            rows(first, [&](uint32_t j, bool in) {
                const uint64_t m = __ballot(in && key[j] == lo);
                equal_before[j] = (uint32_t)__popcll(m & below);
                if (lane == 0) sh.equal[SELECT_WAVES * j + wave] = (uint32_t)__popcll(m);
            });
            lds_barrier();
            const uint32_t own = sh.equal[lane], upto = wave_up_to(own);
            rows(first, [&](uint32_t j, bool) { equal_before[j] += equals + __builtin_amdgcn_readlane(upto - own, SELECT_WAVES * j + wave); });
            equals += __builtin_amdgcn_readlane(upto, 63);
        }
        uint64_t taken[SELECT_KEYS];
        rows(first, [&](uint32_t j, bool in) {
            taken[j] = __ballot(in && (ties ? key[j] > lo || (key[j] == lo && equal_before[j] < need) : key[j] >= lo));
            if (lane == 0) sh.count[SELECT_WAVES * j + wave] = (uint32_t)__popcll(taken[j]);
        });
        lds_barrier();
        const uint32_t own = sh.count[lane], upto = wave_up_to(own);
        rows(first, [&](uint32_t j, bool) {
            const uint32_t at = placed + __builtin_amdgcn_readlane(upto - own, SELECT_WAVES * j + wave);
            if (taken[j] >> lane & 1) to[at + (uint32_t)__popcll(taken[j] & below)] = first + SELECT_THREADS * j + t;
        });
        placed += __builtin_amdgcn_readlane(upto, 63);
        if (n > AT_ONCE) lds_barrier();  // the counts are read
    }
}

// The pages of (sequence, kv head). A block scores 64 pages, a wavefront 16 of them as 4 x 4: lane l has dims 8 (l / 4) ..
// of page l % 4 of each four (two 16-byte loads of bounds each, all in flight at once; one four to a wavefront, with 4
// times the blocks to count: 33.6 us for 24.2, 2048 pages of 8 pairs) and of query l % 4, so element d of the 8 is an
// operand of a product of 4 pages and 4 queries over 4 dims, 4 of which (4 x 4 x 4, four blocks) the f64 matrix
// instruction sums: max(q lo, q hi) = q+ hi + q- lo, q+ and q- being q where it is not below and where it is below 0, else
// 0 (a NaN is in q+). Products of bf16 are exact and sums f64, in one order for all pages, so equal pages score equal and
// near ones in their order (with 16 lanes to a page and vector f64: 33.5 us for 29.7, 16 sequences of up to 16000 keys).
// The last block of its (sequence, kv head) to count itself selects; a block that has them all need not count. The last
// page stands outside: it is always kept.
__global__ void __launch_bounds__(SELECT_THREADS)
    kv8_select_kernel(Table t, const bf16_t* __restrict__ bounds, const bf16_t* __restrict__ q,
                      const uint32_t* __restrict__ lens, uint32_t budget, uint32_t* __restrict__ list,
                      uint64_t* __restrict__ keys_of, uint32_t* __restrict__ counter_of, uint32_t group) {
    __shared__ SelectShared sh;
    const uint32_t kh = blockIdx.x, s = blockIdx.z, i = threadIdx.x;
    const uint32_t lane = i & 63, wave = __builtin_amdgcn_readfirstlane(i >> 6), n = lane & 15, g = lane >> 4;
    const size_t pair = (size_t)s * t.kv_heads + kh;
    uint32_t* to = list + pair * budget;
    const uint32_t first = blockIdx.y * SELECT_PAGES;
    const uint32_t pages = (kv8_keys(lens[s], t.seq_pages) + KV8_PAGE - 1) / KV8_PAGE;
    if (pages <= budget || budget == 1) {
        if (blockIdx.y == 0)
            for (uint32_t j = i; j < budget; j += SELECT_THREADS) to[j] = j >= pages ? KV8_NONE : budget == 1 ? pages - 1 : j;
        return;
    }
    const uint32_t scored = pages - 1;
    if (first >= scored) return;
    // Behind the length, the table's entries and the first queries at once; behind the entries, the bounds. Nothing is
    // read for pages past the sequence's block of 64: a table may be far wider than its sequence. Queries past the group
    // repeat its last one, which leaves the maximum as it is.
    auto entry_at = [&](uint32_t p) { return t.pages[(size_t)s * t.seq_pages + min(p, t.seq_pages - 1)]; };
    uint32_t entry[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) entry[j] = entry_at(first + 16 * wave + 4 * j + (lane & 3));
    const uint32_t at = 16 * wave + 4 * (n >> 2) + g, its_entry = entry_at(first + at);
    const bf16_t* head = q + pair * group * KV8_HEAD + 8 * (lane >> 2);
    auto query = [&](uint32_t h) { return *reinterpret_cast<const u32x4*>(head + min(h + (lane & 3), group - 1) * KV8_HEAD); };
    u32x4 x = query(0), lo[4], hi[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
        const u32x4* b = reinterpret_cast<const u32x4*>(bounds + kv8_bound(entry[j] < t.pool ? entry[j] : 0u, t.kv_heads, kh)) + (lane >> 2);
        lo[j] = b[0];
        hi[j] = b[KV8_HEAD / 8];
    }
    uint64_t best = 0;
#pragma unroll 1
    for (uint32_t h = 0; h < group; h += 4) {
        // Converted again for every 4 queries: kept, the bounds' 64 doubles are half the registers (30.7 us for 29.7).
#pragma unroll
        for (int j = 0; j < 4; ++j) asm("" : "+v"(lo[j]), "+v"(hi[j]));
        double sum[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            const float v = half_of(x, d);
            const double up = v < 0.f ? 0.0 : (double)v, down = v < 0.f ? (double)v : 0.0;
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[j] = __builtin_amdgcn_mfma_f64_4x4x4f64((double)half_of(hi[j], d), up, sum[j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[j] = __builtin_amdgcn_mfma_f64_4x4x4f64((double)half_of(lo[j], d), down, sum[j], 0, 0, 0);
        }
        if (h + 4 < group) x = query(h + 4);
        // The result of page i, query j, block b is in lane 16 i + 4 b + j: the blocks' sum, in all four; lane n then takes
        // the pages of four n / 4, so its page is 4 (n / 4) + g of the wavefront's.
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            sum[j] += row_move_d<0x128>(sum[j]);
            sum[j] += row_move_d<0x124>(sum[j]);
        }
        best = max(best, score_key(n & 8 ? n & 4 ? sum[3] : sum[2] : n & 4 ? sum[1] : sum[0]));
    }
    best = max(best, row_move_u<0xB1>(best));
    best = max(best, row_move_u<0x4E>(best));
    uint64_t* key = keys_of + pair * t.seq_pages;
    if (its_entry >= t.pool) best = 0;
    const bool puts = (n & 3) == 0 && first + at < scored;
    if (scored > SELECT_PAGES) {
        if (puts) __hip_atomic_store(key + first + at, best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        // The keys acknowledged, then the count: the block that completes it selects.
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        uint32_t* counter = counter_of + pair;
        if (i == 0) {
            const uint32_t before = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            sh.last = before == (scored - 1) / SELECT_PAGES;
        }
        __syncthreads();
        if (!sh.last) return;
        if (i == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next call
    } else {
        if (puts) sh.key[at] = best;
        __syncthreads();
    }
    if (i == 0) to[budget - 1] = pages - 1;
    auto key_of = [&](uint32_t x) {
        return scored > SELECT_PAGES ? __hip_atomic_load(key + x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : sh.key[x];
    };
    select_keys(key_of, scored, budget - 1, to, sh);
}

// ---- host ----

// The Gpu's device is current while a call launches, whatever the caller's is.
struct OnDevice {
    int before = -1;
    explicit OnDevice(int device) {
        int now = device;
        if (hipGetDevice(&now) == hipSuccess && now != device && hipSetDevice(device) == hipSuccess) before = now;
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

x0ne_status bad(const char* what, const std::string& why) { return fail(X0NE_ERR_FORMAT, std::string(what) + ": " + why); }

x0ne_status check_shape(const char* what, const x0ne_kv8* c) {
    if (!c) return bad(what, "no cache");
    if (c->pool == 0 || c->kv_heads == 0 || c->kv_heads > 1024 || c->seqs > 65535 || c->seq_pages == 0 ||
        c->seq_pages >= (1u << 24))
        return bad(what, std::to_string(c->pool) + " pages of " + std::to_string(c->kv_heads) + " kv heads, " +
                             std::to_string(c->seqs) + " sequences of " + std::to_string(c->seq_pages) +
                             " pages (1 to 1024 kv heads, up to 65535 sequences, 1 to 2^24 - 1 pages)");
    return X0NE_OK;
}

x0ne_status check_cache(const char* what, const x0ne_kv8* c) {
    X0NE_TRY(check_shape(what, c));
    if (!c->codes || !c->scales || !c->page_table || c->codes % 16 || c->scales % 16 || c->page_table % 4)
        return bad(what, "codes and scales (16-byte aligned) and page_table are required");
    return X0NE_OK;
}

x0ne_status check_heads(const char* what, const x0ne_kv8* c, uint32_t q_heads) {
    if (q_heads == 0 || q_heads % c->kv_heads != 0 || q_heads / c->kv_heads > 16)
        return bad(what, std::to_string(q_heads) + " q heads for " + std::to_string(c->kv_heads) +
                             " kv heads (1 to 16 per kv head)");
    return X0NE_OK;
}

Table whole_table(const x0ne_kv8* c) {
    return Table{(const uint32_t*)c->page_table, c->seqs, c->seq_pages, c->pool, c->kv_heads};
}

}  // namespace

extern "C" x0ne_status x0ne_gpu_kv8_write(x0ne_gpu* g, const x0ne_kv8* c, uint64_t qkv, uint64_t rows, uint32_t q_heads,
                                          uint64_t q_norm, uint64_t k_norm, float eps, uint64_t rope_cs,
                                          uint32_t positions, uint64_t row_seq, uint64_t row_pos, uint64_t q_out,
                                          uint64_t bounds) {
    const char* what = "kv8 write";
    X0NE_TRY(check_cache(what, c));
    if (q_heads == 0 || q_heads > 16384 || rows >= (1u << 24))
        return bad(what, std::to_string(q_heads) + " q heads, " + std::to_string(rows) + " rows");
    if (!qkv || !q_norm || !k_norm || !rope_cs || !row_seq || !row_pos || !q_out || qkv % 16 || q_norm % 16 ||
        k_norm % 16 || rope_cs % 16 || row_seq % 4 || row_pos % 4 || q_out % 16 || bounds % 16)
        return bad(what, "qkv, q_norm, k_norm, rope_cs and q_out (16-byte aligned), row_seq and row_pos are required");
    if (!g) return fail(X0NE_ERR_GPU, "no device");
    if (rows == 0 || c->seqs == 0 || positions == 0) return X0NE_OK;
    const OnDevice on(g->device);
    Write a = {whole_table(c),
               (uint8_t*)c->codes,
               (uint8_t*)c->scales,
               (const bf16_t*)qkv,
               (const bf16_t*)q_norm,
               (const bf16_t*)k_norm,
               (const double2*)rope_cs,
               (const uint32_t*)row_seq,
               (const uint32_t*)row_pos,
               (bf16_t*)q_out,
               (bf16_t*)bounds,
               (uint32_t)rows,
               q_heads,
               positions,
               eps};
    // 4 heads to a block read cos and sin, and take square roots, half as often as 2, which are over sooner and, with
    // bounds, keep the blocks of a row that ends a page short (us with 2 / 4: 64 rows of 64 sequences, 40 blocks of 4, 7.4 /
    // 10.9; 777 rows of 72 heads, 882 blocks, 12.8 / 13.9; 2048 rows of 40 heads, 1280 blocks, 15.0 / 13.8; 8 heads 16.3).
    const uint32_t tiles = (a.rows + WRITE_ROWS - 1) / WRITE_ROWS;
    const bool many = (uint64_t)tiles * ((q_heads + c->kv_heads) / WRITE_HEADS) >= 1024;
    const uint32_t each = many ? WRITE_HEADS : 2;
    const dim3 grid(tiles, (q_heads + each - 1) / each + (c->kv_heads + each - 1) / each + (c->kv_heads + WRITE_VALUES - 1) / WRITE_VALUES);
    g->counts.launches++;
    hipLaunchKernelGGL(many ? kv8_write_kernel<WRITE_HEADS> : kv8_write_kernel<2>, grid, dim3(256), 0, g->stream, a);
    X0NE_HIP(hipGetLastError(), what);
    return X0NE_OK;
}

extern "C" x0ne_status x0ne_gpu_kv8_read(x0ne_gpu* g, const x0ne_kv8* c, uint64_t lens, uint64_t k, uint64_t v,
                                         uint64_t out_table, uint32_t out_pool) {
    const char* what = "kv8 read";
    X0NE_TRY(check_cache(what, c));
    if (!lens || !k || !v || !out_table || lens % 4 || k % 16 || v % 16 || out_table % 4 || out_pool == 0)
        return bad(what, "lens, k and v (16-byte aligned), out_table and an out_pool are required");
    if (!g) return fail(X0NE_ERR_GPU, "no device");
    if (c->seqs == 0) return X0NE_OK;
    const OnDevice on(g->device);
    g->counts.launches++;
    const uint64_t blocks = std::min<uint64_t>(65536, ((uint64_t)c->seq_pages * c->kv_heads + 3) / 4);
    // Bypassing the Infinity Cache with more than it holds: 16 sequences of up to 8192 positions 88.5 -> 85.3 us.
    const bool stream = (uint64_t)c->seqs * c->seq_pages * c->kv_heads * (3 * KV8_RECORD) > KV8_STREAM;
    hipLaunchKernelGGL(stream ? kv8_read_kernel<true> : kv8_read_kernel<false>, dim3((uint32_t)blocks, c->seqs), dim3(256), 0, g->stream,
                       whole_table(c), (const uint8_t*)c->codes, (const uint8_t*)c->scales, (const uint32_t*)lens,
                       (bf16_t*)k, (bf16_t*)v, (const uint32_t*)out_table, out_pool);
    X0NE_HIP(hipGetLastError(), what);
    return X0NE_OK;
}

static Kv8Cut cut_of(const x0ne_kv8* c, uint32_t budget = 0) { return kv8_cut(c->kv_heads, c->seqs, c->seq_pages, budget); }

// The workspace: a counter per (sequence, kv head), then the states of attention or the scores of selection. The counters
// are as many for every cache, so that no call's states lie where another's counters are: caches of any shapes share a
// workspace. Sequences beyond 65536 pairs are further launches, which come upon the counters left at zero.
static constexpr uint64_t COUNTERS = 65536, COUNTER_BYTES = 4 * COUNTERS;
static uint32_t seqs_at_once(const x0ne_kv8* c) { return (uint32_t)(COUNTERS / c->kv_heads) / 64 * 64; }
static Table table_of(const x0ne_kv8* c, uint64_t first) {  // of a launch's sequences
    return Table{(const uint32_t*)c->page_table + first * c->seq_pages, (uint32_t)std::min<uint64_t>(c->seqs - first, seqs_at_once(c)),
                 c->seq_pages, c->pool, c->kv_heads};
}

extern "C" uint64_t x0ne_kv8_work_bytes(const x0ne_kv8* c, uint32_t q_heads) {
    if (check_shape("kv8 workspace", c) != X0NE_OK || check_heads("kv8 workspace", c, q_heads) != X0NE_OK) return 0;
    const uint64_t states = (uint64_t)c->seqs * q_heads * cut_of(c).slices * STATE * 4;
    const uint64_t scores = (uint64_t)c->seqs * c->kv_heads * c->seq_pages * 8;
    return COUNTER_BYTES + std::max(states, scores);
}

extern "C" x0ne_status x0ne_gpu_kv8_attention(x0ne_gpu* g, const x0ne_kv8* c, uint64_t q, uint32_t q_heads, uint64_t lens,
                                              uint64_t page_list, uint32_t budget, uint64_t out, float scale,
                                              uint64_t work, uint64_t work_bytes) {
    const char* what = "kv8 attention";
    X0NE_TRY(check_cache(what, c));
    X0NE_TRY(check_heads(what, c, q_heads));
    if (budget >= (1u << 24)) return bad(what, "a budget of " + std::to_string(budget) + " pages");
    if (!q || !lens || !out || q % 16 || lens % 4 || out % 16 || page_list % 4 || !page_list != !budget)
        return bad(what, "q and out (16-byte aligned) and lens are required; a page list has a budget, and no other call has one");
    if (!work || work % 256 || work_bytes < x0ne_kv8_work_bytes(c, q_heads))
        return bad(what, "a workspace of x0ne_kv8_work_bytes (256-byte aligned) is required");
    if (!g) return fail(X0NE_ERR_GPU, "no device");
    if (c->seqs == 0) return X0NE_OK;
    const OnDevice on(g->device);
    const Kv8Cut cut = cut_of(c, budget);
    const auto kernel = cut.waves == 4 ? kv8_attention_kernel<4, false> : cut.stream ? kv8_attention_kernel<8, true> : kv8_attention_kernel<8, false>;
    for (uint64_t s = 0; s < c->seqs; s += seqs_at_once(c)) {
        Attend a = {};
        a.t = table_of(c, s);
        a.codes = (const uint8_t*)c->codes;
        a.scales = (const uint8_t*)c->scales;
        a.q = (const bf16_t*)q + s * q_heads * KV8_HEAD;
        a.lens = (const uint32_t*)lens + s;
        a.list = page_list ? (const uint32_t*)page_list + s * c->kv_heads * budget : nullptr;
        a.out = (bf16_t*)out + s * q_heads * KV8_HEAD;
        a.counter = (uint32_t*)work;
        a.state = (float*)(work + COUNTER_BYTES);
        a.budget = budget;
        a.q_heads = q_heads;
        a.group = q_heads / c->kv_heads;
        a.slices = cut.slices;
        a.rounds = cut.rounds;
        a.scale2 = scale * 1.44269504088896340736f;
        g->counts.launches++;
        hipLaunchKernelGGL(kernel, dim3(c->kv_heads, cut.blocks, (a.t.seqs + 63) / 64), dim3(64 * cut.waves), 0, g->stream, a);
        X0NE_HIP(hipGetLastError(), what);
    }
    return X0NE_OK;
}

extern "C" x0ne_status x0ne_gpu_kv8_select(x0ne_gpu* g, const x0ne_kv8* c, uint64_t bounds, uint64_t q, uint32_t q_heads,
                                           uint64_t lens, uint32_t budget, uint64_t page_list, uint64_t work,
                                           uint64_t work_bytes) {
    const char* what = "kv8 select";
    X0NE_TRY(check_cache(what, c));
    X0NE_TRY(check_heads(what, c, q_heads));
    if (budget == 0 || budget >= (1u << 24)) return bad(what, "a budget of " + std::to_string(budget) + " pages");
    if (!bounds || !q || !lens || !page_list || bounds % 16 || q % 16 || lens % 4 || page_list % 4)
        return bad(what, "bounds and q (16-byte aligned), lens and page_list are required");
    if (!work || work % 256 || work_bytes < x0ne_kv8_work_bytes(c, q_heads))
        return bad(what, "a workspace of x0ne_kv8_work_bytes (256-byte aligned) is required");
    const uint32_t blocks = (c->seq_pages + SELECT_PAGES - 1) / SELECT_PAGES;
    if (blocks > 65535) return bad(what, std::to_string(c->seq_pages) + " pages of a sequence (up to 65535 x 64)");
    if (!g) return fail(X0NE_ERR_GPU, "no device");
    if (c->seqs == 0) return X0NE_OK;
    const OnDevice on(g->device);
    for (uint64_t s = 0; s < c->seqs; s += seqs_at_once(c)) {
        const Table t = table_of(c, s);
        g->counts.launches++;
        hipLaunchKernelGGL(kv8_select_kernel, dim3(c->kv_heads, blocks, t.seqs), dim3(SELECT_THREADS), 0, g->stream, t,
                           (const bf16_t*)bounds, (const bf16_t*)q + s * q_heads * KV8_HEAD, (const uint32_t*)lens + s, budget,
                           (uint32_t*)page_list + s * c->kv_heads * budget, (uint64_t*)(work + COUNTER_BYTES), (uint32_t*)work,
                           q_heads / c->kv_heads);
        X0NE_HIP(hipGetLastError(), what);
    }
    return X0NE_OK;
}
