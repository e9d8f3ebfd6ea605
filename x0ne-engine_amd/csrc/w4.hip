// Weights in 4 bits: a bf16 matrix brought into that form, read back, and the products of a few rows with it.
//
// A group of 32, 64 or 128 weights of a row is held as e2m1 codes of w / s and one bf16 scale s. Codes lie in tiles of
// 16 rows and 128 columns, 1 KiB each, in the order of a matrix instruction's lanes: lane l's 16 bytes are row l % 16,
// byte 4 s + b of them columns 32 s + 8 (l / 16) + 2 b and the next, so that a lane's word s is its operand of the
// product over columns 32 s to 32 s + 31, two conversions (v_cvt_scalef32_pk_bf16_fp4) to a register of it.
#include <algorithm>
#include <string>

#include "device.h"
#include "internal.h"
#include "w4.h"

using namespace x0ne;

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t TILE_ROWS = 16, TILE_COLS = 128, TILE_BYTES = 1024;

struct Form {
    uint8_t* codes;
    bf16_t* scales;
    uint32_t rows, cols, tiles;  // tiles of a panel of 16 rows
};

// 2^-126: a group's smallest scale, so that its reciprocal is finite and codes times scales are as exact as bf16.
constexpr uint32_t LEAST = 0x0080;

// The two values of byte b of a word of codes, exact.
template <int B>
__device__ __forceinline__ uint32_t decode2(uint32_t codes) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.0f, B));
}
__device__ __forceinline__ bf16x8 decode8(uint32_t codes) {
    return __builtin_bit_cast(bf16x8, u32x4{decode2<0>(codes), decode2<1>(codes), decode2<2>(codes), decode2<3>(codes)});
}

// A wavefront's tile of bf16 values between memory, where it is 16 rows of 256 bytes, and the lanes of a matrix instruction: of
// a load or store four neighbouring lanes on the 64 bytes of four rows became 16 on the 256 of one, through the wavefront's own
// LDS, 16-byte pieces placed by an XOR of the row. Piece p of row r is at tile_at(r, p); the instruction's lane l takes piece
// 4 s + l / 16 of row l % 16 as its word s.
__device__ __forceinline__ uint32_t tile_at(uint32_t r, uint32_t p) { return r * 16 + ((p ^ r) & 15); }
// What a wavefront's lanes exchange through LDS: its LDS operations go in order, so that only the compiler has to keep them.
__device__ __forceinline__ void wave_lds() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// s = max |w| / 6 of each group, codes of w / s. A wavefront takes a tile. The four lanes of a row hold 8 columns of each 32: a
// group's largest magnitude is theirs, found with two shuffles, and each lane's codes are 16 bytes as they lie in memory.
// Measured on MI355X (back to back in a captured graph, matrices in turn past the Infinity Cache): 47.2 us for 24576 x 4096
// (201 MB read and 52 written: 5.4 TB/s; a copy of 1 GiB reaches 5.1); 4.7 for 1000 x 1096, which is a launch and one trip to
// memory.
template <int G, bool STREAM>
__global__ void __launch_bounds__(256) w4_quantise_kernel(const bf16_t* __restrict__ from, Form f) {
    const uint32_t lane = threadIdx.x & 63, t = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= f.tiles) return;
    __shared__ u32x4 lds[4][256];
    u32x4* mine = lds[threadIdx.x >> 6];
    u32x4 in[4], w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t row = blockIdx.y * TILE_ROWS + 4 * j + (lane >> 4), col = t * TILE_COLS + 8 * (lane & 15);
        const u32x4* p = reinterpret_cast<const u32x4*>(from + (size_t)row * f.cols + col);
        in[j] = u32x4{0, 0, 0, 0};
        if (row < f.rows && col < f.cols) in[j] = STREAM ? __builtin_nontemporal_load(p) : *p;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) mine[tile_at(4 * j + (lane >> 4), lane)] = in[j];
    wave_lds();
    uint32_t top[4];  // magnitudes as bits: infinities and NaN are above all others
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        w[s] = mine[tile_at(lane & 15, 4 * s + (lane >> 4))];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, max(w[s][i] & 0x7FFFu, w[s][i] >> 16 & 0x7FFFu));
        top[s] = m;
    }
    constexpr int STEPS = G / 32;  // words to a group
    uint32_t out[4], scale[4 / STEPS];
#pragma unroll
    for (int g = 0; g < 4 / STEPS; ++g) {
        uint32_t m = 0;
#pragma unroll
        for (int s = g * STEPS; s < (g + 1) * STEPS; ++s) m = max(m, top[s]);
        m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
        m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
        const bool finite = m < 0x7F80;
        // A third of a value of 8 bits is that far from the middle of two of them that one rounding to f32 before the one to
        // bf16 changes nothing.
        const uint32_t sc = max((uint32_t)f2bf(bf2f((bf16_t)m) / 6.0f), LEAST);
        scale[g] = finite ? sc : 0x7FC0u;
        // w / s is at a middle of two codes or 2^-12.4 of it away (8 bits against 8 and 3). So the quotient by a reciprocal,
        // which is a few 2^-24 off, is rounded to 15 bits, which brings it back to a middle that it stands for, and then to a code.
        const float inv = finite ? __builtin_amdgcn_rcpf(bf2f((bf16_t)sc)) : 0.f;
#pragma unroll
        for (int s = g * STEPS; s < (g + 1) * STEPS; ++s) {
            uint32_t c = 0;
            float q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = finite ? (i & 1 ? bf_hi(w[s][i / 2]) : bf_lo(w[s][i / 2])) * inv : 0.f;
                q[i] = __uint_as_float((__float_as_uint(x) + 0x80u) & 0xFFFFFF00u);
            }
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, q[0], q[1], 1.0f, 0);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, q[2], q[3], 1.0f, 1);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, q[4], q[5], 1.0f, 2);
            out[s] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, q[6], q[7], 1.0f, 3);
        }
    }
    const size_t tile = (size_t)blockIdx.y * f.tiles + t;
    *reinterpret_cast<u32x4*>(f.codes + tile * TILE_BYTES + 16 * lane) = u32x4{out[0], out[1], out[2], out[3]};
    if (lane < 16) {
        bf16_t* to = f.scales + (tile * TILE_ROWS + lane) * (4 / STEPS);
#pragma unroll
        for (int g = 0; g < 4 / STEPS; ++g) to[g] = (bf16_t)scale[g];
    }
}

// The scale of word s of lane l's codes of a tile.
template <int G>
__device__ __forceinline__ float scale_of(const bf16_t* scales, size_t tile, uint32_t row, int s) {
    return bf2f(scales[(tile * TILE_ROWS + row) * (TILE_COLS / G) + s * 32 / G]);
}

// Codes times scales, rounded once to bf16. A wavefront takes a tile and stores whole rows of its 256 bytes. Measured on
// MI355X, as above: 109.9 us for 51200 x 5120 (147 MB read, 524 written: 6.1 TB/s), 42.6 for 24576 x 4096 (37.1 behind its
// quantising, whose codes the cache still has), 4.1 for 4096 x 1024.
template <int G, bool STREAM>
__global__ void __launch_bounds__(256) w4_read_kernel(Form f, bf16_t* __restrict__ to) {
    const uint32_t lane = threadIdx.x & 63, t = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= f.tiles) return;
    __shared__ u32x4 lds[4][256];
    u32x4* mine = lds[threadIdx.x >> 6];
    const size_t tile = (size_t)blockIdx.y * f.tiles + t;
    const u32x4 c = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(f.codes + tile * TILE_BYTES + 16 * lane));
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const float scale = scale_of<G>(f.scales, tile, lane & 15, s);
        const u32x4 v = __builtin_bit_cast(u32x4, decode8(c[s]));
        u32x4 out;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            out[i] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)(bf_lo(v[i]) * scale), (__bf16)(bf_hi(v[i]) * scale)});
        mine[tile_at(lane & 15, 4 * s + (lane >> 4))] = out;
    }
    wave_lds();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const u32x4 v = mine[tile_at(4 * j + (lane >> 4), lane)];
        const uint32_t row = blockIdx.y * TILE_ROWS + 4 * j + (lane >> 4), col = t * TILE_COLS + 8 * (lane & 15);
        u32x4* p = reinterpret_cast<u32x4*>(to + (size_t)row * f.cols + col);
        if (row >= f.rows || col >= f.cols) continue;
        if (STREAM)
            __builtin_nontemporal_store(v, p);
        else
            *p = v;
    }
}

// Word 3 of a raw buffer's descriptor (gfx9: 32-bit data format). A load at or past its bytes gives zeros.
constexpr uint32_t RSRC_WORD3 = 0x00020000, OFF_NONE = 0xFFFFFFF0u;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, (int)RSRC_WORD3);
}
// The cache policy of what is read once (non-temporal).
constexpr int NT = 2;
template <int POLICY = 0>
__device__ __forceinline__ u32x4 load16(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, POLICY));
}

// A tile of a panel in flight: a lane's codes and its row's scales.
template <int G>
struct Piece {
    u32x4 codes;
    uint32_t scales[G == 32 ? 2 : 1];
};

// x / (1 + e^-x), by an exponential that does not overflow for far gates.
__device__ __forceinline__ float silu(float x) {
    const float e = expf(-fabsf(x));
    return x * ((x < 0.f ? e : 1.f) / (1.f + e));
}

// How a launch's blocks share the work: a unit is `rounds` rounds of a tile to each wavefront, and block b takes the rounds
// from b run to (b + 1) run - 1 of all units' one behind the other.
struct Cut {
    uint32_t all, rounds, run, blocks, groups;
    float* parts;        // [blocks][2][P TT][4][64]: of a block's first unit, and of its last, where they are cut
    uint32_t* counters;  // one per unit: zero, left at zero
};

// Y = X W^T: y[t][r] is the sum over the groups g of s[r][g] times the sum over g's columns c of x[t][c] code[r][c]. Codes are
// exact as bf16, so a group's sum is formed on them as they are and scaled once.
// A block of V wavefronts takes a run of the tiles of units of P panels (SwiGLU: half of them gate, the others up) and 4 XL
// rows of X; its wavefronts take the run's tiles in turn, so that it reads V KiB in a row. X is the A operand, W the B operand:
// a lane's four sums are four tokens of one row of W, whose scale of a group is one value. A load of X takes 4 rows of a tile's
// 256 bytes, neighbouring lanes on one row, and passes through the wavefront's own LDS into the operand's order (loaded in
// that order, four lanes to each of 16 rows, 54 us for the 16 rows below): there is no barrier until a unit's end.
// Measured on MI355X, as above: one row is bound by the weights: 50.6 us for 151936 x 4096 (322 MB, 6.4 TB/s); 11.3 for 24576 x
// 4096 SwiGLU (54 MB, 4.7 TB/s; 9.7 from the cache), of which 2 pass before the first product; 3.0 for 4096 x 1024 (3.4 by a
// kernel trace), which is that and one trip to memory. More rows by X's way through the L2, once to a unit, and by the joins of
// cut units: 16 rows of 5120 x 25600 (82 MB) 20.4 (20.1 from the cache, with first products after 2.1, 8 rounds of 1.5, the cut
// units' parts joined by 18.6); 61 rows of 6150 x 4104 13.2 (12.2) in 194 blocks of 5 rounds (208 launched, for whole rounds of
// the XCDs).
template <int G, bool SWIGLU, int XL, int P, int V, int U, bool EVEN>
__global__ void __launch_bounds__(64 * V) w4_gemv_kernel(Form f, const bf16_t* __restrict__ x, uint32_t n, void* __restrict__ y,
                                                         uint32_t out_f32, Cut cut) {
    constexpr int PAIR = SWIGLU ? 2 : 1, POLICY = NT, PER = 128 / G, TT = (XL + 3) / 4, TOKENS = XL < 4 ? 4 * XL : 16 * TT;
    // A wavefront's X tile, then its sums of a unit.
    constexpr int OWN = XL * 64 > P * TT * 64 ? XL * 64 : P * TT * 64;
    __shared__ u32x4 lds[V][OWN];
    __shared__ uint32_t last;
    // Blocks go round the 8 XCDs in the order of their ids: those of a run for the groups of rows of X are neighbours on one,
    // so that its weights come from memory once.
    const uint32_t group = (blockIdx.x >> 3) % cut.groups, block = (blockIdx.x >> 3) / cut.groups * 8 + (blockIdx.x & 7);
    const uint32_t first = block * cut.run, end = min(first + cut.run, cut.all);
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t token0 = group * TOKENS, panels = (f.rows + 15) / 16;
    const __amdgpu_buffer_rsrc_t xr = rsrc(x, n * f.cols * 2);
    u32x4* mine = lds[wave];
    // Panel p of unit u: SwiGLU's odd ones are the up rows of the even ones.
    auto panel_of = [&](uint32_t u, int p) { return u * (P / PAIR) + p / PAIR + p % PAIR * (panels / 2); };

    Piece<G> w[U][P];
    u32x4 a[U][XL];
    auto load = [&](int slot, bool more, uint32_t u, uint32_t t) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const uint32_t panel = panel_of(u, p);
            const bool there = more && panel < panels;
            const size_t tile = (size_t)panel * f.tiles;
            const auto cr = rsrc(f.codes + (there ? tile * TILE_BYTES : 0), there ? f.tiles * TILE_BYTES : 0);
            const auto sr = rsrc(f.scales + (there ? tile * (16 * PER) : 0), there ? f.tiles * (32 * PER) : 0);
            w[slot][p].codes = load16<POLICY>(cr, t * TILE_BYTES + 16 * lane);
            const int at = (int)((t * 16 + (lane & 15)) * 2 * PER);
            if (PER == 4) {
                const auto v = __builtin_amdgcn_raw_buffer_load_b64(sr, at, 0, POLICY);
                w[slot][p].scales[0] = v[0];
                w[slot][p].scales[PER / 4] = v[1];
            } else if (PER == 2)
                w[slot][p].scales[0] = __builtin_amdgcn_raw_buffer_load_b32(sr, at, 0, POLICY);
            else
                w[slot][p].scales[0] = (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(sr, at, 0, POLICY);
        }
        const uint32_t col = t * TILE_COLS + 8 * (lane & 15);
#pragma unroll
        for (int i = 0; i < XL; ++i) {
            const uint32_t token = token0 + 4 * i + (lane >> 4);
            a[slot][i] = load16(xr, more && token < n && col < f.cols ? (token * f.cols + col) * 2 : OFF_NONE);
        }
    };

    f32x4 sum[P][TT] = {};
    auto multiply = [&](int slot) {
#pragma unroll
        for (int i = 0; i < XL; ++i) {
            mine[tile_at(4 * i + (lane >> 4), lane)] = a[slot][i];
        }
        wave_lds();
        bf16x8 frag[TT][4];
#pragma unroll
        for (int i = 0; i < TT; ++i)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const uint32_t r = (16 * i + (lane & 15)) & (4 * XL - 1);
                frag[i][s] = __builtin_bit_cast(bf16x8, mine[tile_at(r, 4 * s + (lane >> 4))]);
            }
        wave_lds();
#pragma unroll
        for (int p = 0; p < P; ++p) {
            f32x4 acc[TT] = {};
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const bf16x8 b = decode8(w[slot][p].codes[s]);
#pragma unroll
                for (int i = 0; i < TT; ++i) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(frag[i][s], b, acc[i], 0, 0, 0);
                if ((s + 1) % (G / 32) == 0) {
                    const int g = s * 32 / G;
                    const uint32_t word = w[slot][p].scales[PER == 4 ? g / 2 : 0];
                    const float scale = g & 1 ? bf_hi(word) : bf_lo(word);
#pragma unroll
                    for (int i = 0; i < TT; ++i) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) sum[p][i][j] = fmaf(acc[i][j], scale, sum[p][i][j]);
                        acc[i] = f32x4{};
                    }
                }
            }
        }
    };

    auto write = [&](uint32_t u, uint32_t o, const f32x4* r) {
        const uint32_t p = o / TT * PAIR, i = o % TT;
        const uint32_t row = panel_of(u, p) * 16 + (lane & 15), out_rows = f.rows / PAIR;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t to = token0 + 16 * i + 4 * (lane >> 4) + j;
            if (row >= out_rows || to >= min(n, token0 + TOKENS)) continue;
            const size_t at = (size_t)to * out_rows + row;
            if (SWIGLU)
                static_cast<bf16_t*>(y)[at] = f2bf(silu(r[0][j]) * r[PAIR - 1][j]);
            else if (out_f32)
                static_cast<float*>(y)[at] = r[0][j];
            else
                static_cast<bf16_t*>(y)[at] = f2bf(r[0][j]);
        }
    };
    // The wavefronts' sums of a unit, and those of the other blocks that have tiles of it: each leaves its part, and the
    // last to count itself adds them in the blocks' order.
    auto finish = [&](uint32_t u) {
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int i = 0; i < TT; ++i) {
                mine[(p * TT + i) * 64 + lane] = __builtin_bit_cast(u32x4, sum[p][i]);
                sum[p][i] = f32x4{};
            }
        lds_barrier();
        const uint32_t begin = u * cut.rounds, behind = begin + cut.rounds;
        const bool whole = !EVEN || (begin >= first && behind <= end);
        float* parts = cut.parts + (size_t)group * cut.blocks * (2 * P * TT * 256);
        float* part = parts + (size_t)(2 * block + (begin > first)) * (P * TT * 256);
        for (uint32_t o = wave; o < P / PAIR * TT; o += V) {
            const uint32_t p = o / TT * PAIR, i = o % TT;
            f32x4 r[PAIR] = {};
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int k = 0; k < PAIR; ++k) r[k] += __builtin_bit_cast(f32x4, lds[v][((p + k) * TT + i) * 64 + lane]);
            if (whole) {
                write(u, o, r);
                continue;
            }
#pragma unroll
            for (int k = 0; k < PAIR; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    __hip_atomic_store(part + (((p + k) * TT + i) * 4 + j) * 64 + lane, r[k][j], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        if (whole) {
            lds_barrier();
            return;
        }
        const uint32_t b1 = begin / cut.run, b2 = (behind - 1) / cut.run;
        // The parts acknowledged, then the count.
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        uint32_t* counter = cut.counters + group * (cut.all / cut.rounds) + u;
        if (threadIdx.x == 0) last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == b2 - b1;
        __syncthreads();
        if (!last) return;
        if (threadIdx.x == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next call
        for (uint32_t o = wave; o < P / PAIR * TT; o += V) {
            const uint32_t p = o / TT * PAIR, i = o % TT;
            f32x4 r[PAIR] = {};
            for (uint32_t b = b1; b <= b2; ++b) {
                const float* from = parts + (size_t)(2 * b + (b == b1 && begin > b * cut.run)) * (P * TT * 256);
#pragma unroll
                for (int k = 0; k < PAIR; ++k)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        r[k][j] += __hip_atomic_load(from + (((p + k) * TT + i) * 4 + j) * 64 + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            write(u, o, r);
        }
    };

    if (first >= end) return;
    // U rounds in flight, over the ends of units too. A round past the run's end is one of zeros, so that the loop has no
    // other way out: with one, the compiler moved the loads' registers and waited for all of them.
    uint32_t unit = first / cut.rounds, round = first % cut.rounds, next = first, next_u = unit, next_round = round;
    auto load_next = [&](int slot) {
        load(slot, next < end, next_u, next_round * V + wave);
        ++next;
        const bool over = ++next_round == cut.rounds;
        next_u += over;
        next_round = over ? 0 : next_round;
    };
#pragma unroll
    for (int slot = 0; slot < U; ++slot) load_next(slot);
    for (uint32_t at = first; at < end; at += U) {
#pragma unroll
        for (int slot = 0; slot < U; ++slot) {
            multiply(slot);
            load_next(slot);
            const bool over = ++round == cut.rounds;
            if (over || at + slot + 1 == end) {
                if (at + slot < end) finish(unit);
                unit += over;
                round = over ? 0 : round;
            }
        }
    }
}

// ---- host ----

x0ne_status bad(const char* what, const std::string& why) { return fail(X0NE_ERR_FORMAT, std::string(what) + ": " + why); }

static_assert(W4_COUNTERS <= GPU_COUNTERS && W4_PARTS_BYTES <= TILE_PARTS_BYTES, "the Gpu's workspaces");

constexpr uint32_t MOST = 1u << 24;
constexpr uint64_t MOST_WEIGHTS = 1ull << 40;  // more than memory holds; tiles are counted in 32 bits

x0ne_status check_shape(const char* what, const x0ne_w4* w) {
    if (!w) return bad(what, "no matrix");
    if (w->rows == 0 || w->rows > MOST || w->cols == 0 || w->cols > MOST || w->cols % 8 || (uint64_t)w->rows * w->cols > MOST_WEIGHTS ||
        (w->group != 32 && w->group != 64 && w->group != 128))
        return bad(what, std::to_string(w->rows) + " rows of " + std::to_string(w->cols) + " columns in groups of " +
                             std::to_string(w->group) + " (1 to 2^24 rows and columns and up to 2^40 weights, columns a multiple of 8, groups of 32, 64 or 128)");
    return X0NE_OK;
}

x0ne_status check_matrix(const char* what, const x0ne_w4* w) {
    X0NE_TRY(check_shape(what, w));
    if (!w->codes || !w->scales || w->codes % 16 || w->scales % 16) return bad(what, "codes and scales (16-byte aligned) are required");
    return X0NE_OK;
}

uint64_t tiles_of(const x0ne_w4* w) { return (uint64_t)((w->rows + 15) / 16) * ((w->cols + 127) / 128); }

Form form_of(const x0ne_w4* w) {
    return Form{(uint8_t*)w->codes, (bf16_t*)w->scales, w->rows, w->cols, (w->cols + TILE_COLS - 1) / TILE_COLS};
}

// Whether a matrix's bf16 form bypasses the Infinity Cache: one of more than half of it, which is seldom there alone (24576 x
// 4096, 201 MB, quantised and read back into another 201 MB: 101 us through it, 81 past it; alone and quantised again and again
// 43 through it, 48 past it; 51200 x 5120 read back 116 and 108).
constexpr uint64_t INFINITY_CACHE = 256ull << 20;
bool streams(const x0ne_w4* w) { return (uint64_t)w->rows * w->cols * 2 > INFINITY_CACHE / 2; }

// grid y holds at most 65535 panels: a taller matrix is several launches.
template <class Launch>
x0ne_status by_panels(x0ne_gpu* g, const char* what, const x0ne_w4* w, Launch launch) {
    Form f = form_of(w);
    const uint32_t panels = (w->rows + 15) / 16;
    for (uint32_t first = 0; first < panels; first += 65535) {
        const uint32_t some = std::min(panels - first, 65535u);
        Form part = f;
        part.codes += (size_t)first * f.tiles * TILE_BYTES;
        part.scales += (size_t)first * f.tiles * TILE_ROWS * (TILE_COLS / w->group);
        part.rows = f.rows - first * TILE_ROWS;
        g->counts.launches++;
        launch(dim3((f.tiles + 3) / 4, some), part, (size_t)first * TILE_ROWS * f.cols);
        X0NE_HIP(hipGetLastError(), what);
    }
    return X0NE_OK;
}

}  // namespace

extern "C" uint64_t x0ne_w4_code_bytes(const x0ne_w4* w) { return check_shape("w4 codes", w) == X0NE_OK ? tiles_of(w) * TILE_BYTES : 0; }

extern "C" uint64_t x0ne_w4_scale_bytes(const x0ne_w4* w) {
    return check_shape("w4 scales", w) == X0NE_OK ? tiles_of(w) * TILE_ROWS * (TILE_COLS / w->group) * 2 : 0;
}

extern "C" x0ne_status x0ne_gpu_w4_quantise(x0ne_gpu* g, const x0ne_w4* w, uint64_t from) {
    const char* what = "w4 quantise";
    X0NE_TRY(check_matrix(what, w));
    if (!from || from % 16) return bad(what, "a bf16 matrix (16-byte aligned) is required");
    if (!g) return fail(X0NE_ERR_GPU, "no device");
    const OnDevice on(g->device);
    const bool past = streams(w);
    const auto kernel = w->group == 32   ? past ? w4_quantise_kernel<32, true> : w4_quantise_kernel<32, false>
                        : w->group == 64 ? past ? w4_quantise_kernel<64, true> : w4_quantise_kernel<64, false>
                                         : past ? w4_quantise_kernel<128, true> : w4_quantise_kernel<128, false>;
    return by_panels(g, what, w, [&](dim3 grid, const Form& f, size_t at) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, g->stream, (const bf16_t*)from + at, f);
    });
}

extern "C" x0ne_status x0ne_gpu_w4_read(x0ne_gpu* g, const x0ne_w4* w, uint64_t to) {
    const char* what = "w4 read";
    X0NE_TRY(check_matrix(what, w));
    if (!to || to % 16) return bad(what, "a bf16 matrix (16-byte aligned) is required");
    if (!g) return fail(X0NE_ERR_GPU, "no device");
    const OnDevice on(g->device);
    // Stores past the cache want whole pieces of 64 bytes (24576 x 4104: 74 us with them, 45 without).
    const bool past = streams(w) && w->cols % 32 == 0;
    const auto kernel = w->group == 32   ? past ? w4_read_kernel<32, true> : w4_read_kernel<32, false>
                        : w->group == 64 ? past ? w4_read_kernel<64, true> : w4_read_kernel<64, false>
                                         : past ? w4_read_kernel<128, true> : w4_read_kernel<128, false>;
    return by_panels(g, what, w, [&](dim3 grid, const Form& f, size_t at) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, g->stream, f, (bf16_t*)to + at);
    });
}

template <bool SWIGLU, int XL, int P, int V, int U, bool EVEN>
static void launch_as(const x0ne_gpu* g, const x0ne_w4* w, const W4Plan& p, const bf16_t* x, uint32_t n, void* y, uint32_t out_f32, float* parts) {
    const auto kernel = w->group == 32   ? w4_gemv_kernel<32, SWIGLU, XL, P, V, U, EVEN>
                        : w->group == 64 ? w4_gemv_kernel<64, SWIGLU, XL, P, V, U, EVEN>
                                         : w4_gemv_kernel<128, SWIGLU, XL, P, V, U, EVEN>;
    const Cut cut = {p.units * p.rounds, p.rounds, p.run, p.blocks, p.groups, parts, g->counters};
    hipLaunchKernelGGL(kernel, dim3((p.blocks + 7) / 8 * 8 * p.groups), dim3(64 * V), 0, g->stream, form_of(w), x, n, y, out_f32, cut);
}

// The kernel of a plan; false for one that has none.
template <bool SWIGLU>
static bool launch_plan(const x0ne_gpu* g, const x0ne_w4* w, const W4Plan& p, const bf16_t* x, uint32_t n, void* y, uint32_t out_f32, float* parts) {
    constexpr uint32_t PAIR = SWIGLU ? 2 : 1;
    const auto go = [&](auto launch) {
        launch(g, w, p, x, n, y, out_f32, parts);
        return true;
    };
    if (p.xl == 1 && p.panels == PAIR && !p.even) {
        if (p.waves == 4) return go(launch_as<SWIGLU, 1, PAIR, 4, 2, false>);
        if (p.waves == 8) return go(launch_as<SWIGLU, 1, PAIR, 8, 2, false>);
        if (p.waves == 16) return go(launch_as<SWIGLU, 1, PAIR, 16, 2, false>);
    }
    if (p.waves != 8) return false;
    if (p.panels == 1 && !SWIGLU && !p.even) {
        if (p.xl == 2) return go(launch_as<false, 2, 1, 8, 1, false>);
        if (p.xl == 4) return go(launch_as<false, 4, 1, 8, 1, false>);
    }
    if (p.panels == 2 && !p.even) {
        if (p.xl == 2) return go(launch_as<SWIGLU, 2, 2, 8, 1, false>);
        if (p.xl == 4) return go(launch_as<SWIGLU, 4, 2, 8, 1, false>);
        if (p.xl == 8) return go(launch_as<SWIGLU, 8, 2, 8, 1, false>);
    }
    if (p.panels == 4) {
        if (p.xl == 2) return go(p.even ? launch_as<SWIGLU, 2, 4, 8, 1, true> : launch_as<SWIGLU, 2, 4, 8, 1, false>);
        if (p.xl == 4) return go(p.even ? launch_as<SWIGLU, 4, 4, 8, 1, true> : launch_as<SWIGLU, 4, 4, 8, 1, false>);
        if (p.xl == 8) return go(p.even ? launch_as<SWIGLU, 8, 4, 8, 1, true> : launch_as<SWIGLU, 8, 4, 8, 1, false>);
    }
    if (p.panels == 8) {
        if (p.xl == 4) return go(p.even ? launch_as<SWIGLU, 4, 8, 8, 1, true> : launch_as<SWIGLU, 4, 8, 8, 1, false>);
        if (p.xl == 8) return go(p.even ? launch_as<SWIGLU, 8, 8, 8, 1, true> : launch_as<SWIGLU, 8, 8, 8, 1, false>);
    }
    return false;
}

extern "C" x0ne_status x0ne_gpu_w4_gemv(x0ne_gpu* g, const x0ne_w4* w, uint64_t x, uint64_t n, uint64_t y, uint32_t out) {
    const char* what = "w4 gemv";
    X0NE_TRY(check_matrix(what, w));
    if (out > X0NE_W4_SWIGLU) return bad(what, "no output " + std::to_string(out));
    if (out == X0NE_W4_SWIGLU && w->rows % 32) return bad(what, std::to_string(w->rows) + " rows of gate and up (a multiple of 32)");
    if (n > MOST) return bad(what, std::to_string(n) + " rows of x (up to 2^24)");
    if (!x || !y || x % 16 || y % 4) return bad(what, "x (16-byte aligned) and y (4-byte aligned) are required");
    if (!g) return fail(X0NE_ERR_GPU, "no device");
    if (n == 0) return X0NE_OK;
    const OnDevice on(g->device);
    const bool swiglu = out == X0NE_W4_SWIGLU;
    const uint64_t out_row = (swiglu ? w->rows / 2 : w->rows) * (out == X0NE_W4_F32 ? 4ull : 2ull);
    // X in pieces of which a launch's offsets are below 4 GiB and its threads below 2^32.
    for (uint64_t first = 0, some; first < n; first += some) {
        some = std::min<uint64_t>(n - first, w4_rows_at_once(w->cols));
        W4Plan p = w4_plan(w->rows, w->cols, (uint32_t)some, swiglu, g->cus, true);
        float* parts = p.even ? own_parts(g) : nullptr;
        if (p.even && !parts) p = w4_plan(w->rows, w->cols, (uint32_t)some, swiglu, g->cus, false);
        if (!(swiglu ? launch_plan<true> : launch_plan<false>)(g, w, p, (const bf16_t*)x + first * w->cols, (uint32_t)some, (uint8_t*)y + first * out_row,
                                                               out == X0NE_W4_F32, parts))
            return fail(X0NE_ERR_GPU, std::string(what) + ": no kernel for its plan");
        g->counts.launches++;
        X0NE_HIP(hipGetLastError(), what);
    }
    return X0NE_OK;
}
