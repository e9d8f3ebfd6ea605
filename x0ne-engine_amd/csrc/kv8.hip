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

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }

// The scale exponent and the two codes of a lane's values a and b of a row that lies in the 64 lanes.
__device__ __forceinline__ uint32_t quantise_pair(float a, float b, int& e) {
    const float top = wave_max(fmaxf(finite(a) ? fabsf(a) : 0.f, finite(b) ? fabsf(b) : 0.f));
    e = kv8_exponent(__float_as_uint(top) >> 16);
    const float down = __uint_as_float((uint32_t)(127 - e) << 23);
    // The conversion's own NaN has either sign: 0x7F stands for all that is not finite.
    const uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a * down, b * down, 0, false);
    return (finite(a) ? w & 0xFFu : 0x7Fu) | (finite(b) ? w & 0xFF00u : 0x7F00u);
}

// RMSNorm of each head of q and k, rotate-half RoPE from the table, q to q_out as bf16, k and v
// quantised into their page: the arithmetic of x0ne_qk_norm_rope_kv_write_rows_bf16, so q_out has its
// bits and the codes are those of its k row. One wavefront per (row, head of q and k), lane i the pair
// (i, i + 64). A row of no sequence, or past the sequence's pages or the rope table, writes nothing.
__global__ void __launch_bounds__(256)
    kv8_write_kernel(Table t, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, const bf16_t* __restrict__ qkv,
                     const bf16_t* __restrict__ q_norm, const bf16_t* __restrict__ k_norm, const double* __restrict__ cs,
                     const uint32_t* __restrict__ row_seq, const uint32_t* __restrict__ row_pos,
                     bf16_t* __restrict__ q_out, uint32_t q_heads, uint32_t positions, float eps) {
    constexpr uint32_t HD = KV8_HEAD, HALF = HD / 2;
    const uint32_t head = blockIdx.y * 4 + (threadIdx.x >> 6), row = blockIdx.x, i = threadIdx.x & 63;
    if (head >= q_heads + t.kv_heads) return;
    const uint32_t seq = row_seq[row], pos = row_pos[row];
    if (seq >= t.seqs || pos >= positions || pos / KV8_PAGE >= t.seq_pages) return;
    const bool is_q = head < q_heads;
    const uint32_t kh = is_q ? 0 : head - q_heads;
    const bf16_t* line = qkv + (size_t)row * (q_heads + 2 * t.kv_heads) * HD;
    const bf16_t *src = line + (size_t)head * HD, *nw = is_q ? q_norm : k_norm;
    const double2 c = reinterpret_cast<const double2*>(cs)[(size_t)pos * HALF + i];
    const float a = bf2f(src[i]), b = bf2f(src[i + HALF]);
    const double ss = wave_sum_d((double)a * (double)a + (double)b * (double)b);
    const double scale = 1.0 / sqrt(ss / (double)HD + (double)eps);
    const double na = (double)a * scale * (double)bf2f(nw[i]), nb = (double)b * scale * (double)bf2f(nw[i + HALF]);
    const bf16_t ra = f2bf((float)(na * c.x - nb * c.y)), rb = f2bf((float)(nb * c.x + na * c.y));
    if (is_q) {
        bf16_t* d = q_out + ((size_t)row * q_heads + head) * HD;
        d[i] = ra;
        d[i + HALF] = rb;
        return;
    }
    const uint32_t page = t.page(seq, pos / KV8_PAGE), slot = pos % KV8_PAGE;
    if (page == KV8_NONE) return;
    uint8_t *rec = codes + kv8_record(page, t.kv_heads, kh), *sc = scales + kv8_scale(page, t.kv_heads, kh);
    int e;
    uint32_t w = quantise_pair(bf2f(ra), bf2f(rb), e);
    rec[slot * HD + i] = (uint8_t)w;
    rec[slot * HD + i + HALF] = (uint8_t)(w >> 8);
    if (i == 0) sc[slot] = (uint8_t)(e + 127);
    const bf16_t* vs = line + (size_t)(q_heads + t.kv_heads + kh) * HD;
    w = quantise_pair(bf2f(vs[i]), bf2f(vs[i + HALF]), e);
    rec[KV8_PART + i * KV8_PAGE + slot] = (uint8_t)w;
    rec[KV8_PART + (i + HALF) * KV8_PAGE + slot] = (uint8_t)(w >> 8);
    if (i == 0) sc[KV8_PAGE + slot] = (uint8_t)(e + 127);
}

// The bounds of the pages that the rows complete (slot 15), from the codes; a wavefront per (row, kv
// head), lane i dims 2i and 2i + 1.
__global__ void __launch_bounds__(256)
    kv8_bounds_kernel(Table t, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                      const uint32_t* __restrict__ row_seq, const uint32_t* __restrict__ row_pos, uint32_t positions,
                      bf16_t* __restrict__ bounds) {
    const uint32_t kh = blockIdx.y * 4 + (threadIdx.x >> 6), row = blockIdx.x, i = threadIdx.x & 63;
    if (kh >= t.kv_heads) return;
    const uint32_t pos = row_pos[row];
    if (pos % KV8_PAGE != KV8_PAGE - 1 || pos >= positions) return;
    const uint32_t page = t.page(row_seq[row], pos / KV8_PAGE);
    if (page == KV8_NONE) return;
    const uint8_t *rec = codes + kv8_record(page, t.kv_heads, kh), *sc = scales + kv8_scale(page, t.kv_heads, kh);
    float lo[2] = {INFINITY, INFINITY}, hi[2] = {-INFINITY, -INFINITY};
    bool nan[2] = {false, false};
    for (uint32_t s = 0; s < KV8_PAGE; ++s) {
        const uint32_t w = *reinterpret_cast<const uint16_t*>(rec + s * KV8_HEAD + 2 * i);
        for (int j = 0; j < 2; ++j) {
            const float v = kv8_value(j ? w >> 8 : w, sc[s]);
            nan[j] |= v != v;
            lo[j] = fminf(lo[j], v);
            hi[j] = fmaxf(hi[j], v);
        }
    }
    const float q = __uint_as_float(0x7FC00000u);
    bf16_t* d = bounds + kv8_bound(page, t.kv_heads, kh);
    for (int j = 0; j < 2; ++j) {
        d[2 * i + j] = f2bf(nan[j] ? q : lo[j]);
        d[KV8_HEAD + 2 * i + j] = f2bf(nan[j] ? q : hi[j]);
    }
}

// Positions below a sequence's length as bf16, page by page: the codes' order is the bf16 pages' order, so
// a wavefront streams one page of one head. Slots past the length are zero; a page that is not there reads
// as zeros, an output page outside its pool is not written.
__global__ void __launch_bounds__(256)
    kv8_read_kernel(Table t, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                    const uint32_t* __restrict__ lens, bf16_t* __restrict__ k_out, bf16_t* __restrict__ v_out,
                    const uint32_t* __restrict__ out_table, uint32_t out_pool) {
    const uint32_t p = blockIdx.x, s = blockIdx.z, i = threadIdx.x & 63, kh = blockIdx.y * 4 + (threadIdx.x >> 6);
    const uint32_t keys = kv8_keys(lens[s], t.seq_pages);
    if (kh >= t.kv_heads || p * KV8_PAGE >= keys) return;
    const uint32_t to = kv8_page(out_table, t.seqs, t.seq_pages, out_pool, s, p);
    if (to == KV8_NONE) return;
    const uint32_t page = t.page(s, p), valid = page == KV8_NONE ? 0u : min(keys - p * KV8_PAGE, KV8_PAGE);
    const uint8_t *rec = codes + kv8_record(page == KV8_NONE ? 0 : page, t.kv_heads, kh),
                  *sc = scales + kv8_scale(page == KV8_NONE ? 0 : page, t.kv_heads, kh);
    bf16_t *kd = k_out + ((size_t)to * t.kv_heads + kh) * KV8_PART, *vd = v_out + ((size_t)to * t.kv_heads + kh) * KV8_PART;
    for (uint32_t j = i; j < KV8_PART; j += 64) {
        const uint32_t ks = j / KV8_HEAD, vs = j % KV8_PAGE;
        kd[j] = ks < valid ? f2bf(kv8_value(rec[j], sc[ks])) : 0;
        vd[j] = vs < valid ? f2bf(kv8_value(rec[KV8_PART + j], sc[KV8_PAGE + vs])) : 0;
    }
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)lo, (__bf16)hi});
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

// Partial states go between blocks through agent-scope accesses, coherent across the XCDs' caches.
__device__ __forceinline__ void put2(float* p, float a, float b) {
    __hip_atomic_store((uint64_t*)p, (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get2(const float* p) {
    const uint64_t v = __hip_atomic_load((const uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}
// 2^(m - top), 0 for a state without a key.
__device__ __forceinline__ float factor(float m, float top) {
    return __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.f : top));
}

constexpr uint32_t ATTEND_WAVES = 4, TILE_PAGES = 4;
constexpr uint32_t MAX_SLICES = 64;
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
    uint32_t budget, q_heads, group, slices;
    float scale2;  // the scale times log2 e: a weight is one exp2
};

// Decode attention. A block of 4 wavefronts takes a slice of one sequence's tiles for the q heads of one kv head,
// wavefront w the slice's tiles w, w + 4, ...; a tile is 4 pages. The products are S^T = K Q^T and O^T = V^T P^T on
// the matrix cores (16 x 16 x 32, bf16 with f32 sums), the group's heads the 16 columns: lane (n = lane % 16, g =
// lane / 16) holds column n, so the softmax of a head is lane-local but for the four lanes n, n + 16, n + 32, n + 48.
// Codes become bf16 in one conversion, keys times their scale (exact); a value's scale goes into its weight (exact).
//  - Product m's row r = 4 g' + i is key 4 m + i of the tile's page g': its 16 outputs per lane are then the 16 keys of
//    page g, and with the value of dim 16 c + n at those keys as row n of product c (one 16-byte load: V is dim-major)
//    the weights are an operand as they lie, without a move between lanes.
//  - Dims of a product's k step j are 32 g + 8 j ..: a lane's keys come as two 16-byte loads.
//  - Weights enter as bf16 hi + lo (2^-17 of the weight): one bf16 would add as much error as the output's rounding.
// The running maximum and sum are f32. A slice's state (m, l, o) is joined by the last block of its (sequence, kv head)
// to count itself, slices in order; a sequence of one slice is written at once. Keys past the length, entries behind a
// list and pages that are not there weigh 0, their values are taken as 0.
__global__ void __launch_bounds__(64 * ATTEND_WAVES) kv8_attention_kernel(const Attend a) {
    __shared__ float wm[ATTEND_WAVES][MAX_GROUP], wl[ATTEND_WAVES][MAX_GROUP];
    __shared__ float wo[ATTEND_WAVES][MAX_GROUP][KV8_HEAD + 4];
    __shared__ uint32_t last;
    const uint32_t kh = blockIdx.x, y = blockIdx.y, s = blockIdx.z;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const uint32_t keys = kv8_keys(a.lens[s], a.t.seq_pages), pages = (keys + KV8_PAGE - 1) / KV8_PAGE;
    const uint32_t np = a.list ? min(a.budget, pages) : pages, tiles = (np + TILE_PAGES - 1) / TILE_PAGES;
    bf16_t* out = a.out + ((size_t)s * a.q_heads + kh * a.group) * KV8_HEAD;
    if (tiles == 0) {
        if (y == 0)
            for (uint32_t e = threadIdx.x; e < a.group * KV8_HEAD / 8; e += 256) reinterpret_cast<uint4*>(out)[e] = make_uint4(0, 0, 0, 0);
        return;
    }
    const uint32_t rounds = (tiles + ATTEND_WAVES - 1) / ATTEND_WAVES;
    const uint32_t per = ATTEND_WAVES * ((rounds + a.slices - 1) / a.slices), active = (tiles + per - 1) / per;
    if (y >= active) return;
    const uint32_t t_end = min(tiles, (y + 1) * per);

    // The page of the tile at index 4 t + j, with how many of its keys count.
    const uint32_t* list = a.list ? a.list + ((size_t)s * a.t.kv_heads + kh) * a.budget : nullptr;
    struct Place {
        uint32_t page, valid;
    };
    auto logical_of = [&](uint32_t t, uint32_t j) -> uint32_t {
        const uint32_t at = TILE_PAGES * t + j;
        return t >= t_end || at >= np ? KV8_NONE : list ? list[at] : at;
    };
    auto place = [&](uint32_t logical) -> Place {
        const uint32_t page = logical < pages ? a.t.page(s, logical) : KV8_NONE;
        return page == KV8_NONE ? Place{0u, 0u} : Place{page, (uint32_t)min(keys - logical * KV8_PAGE, KV8_PAGE)};
    };
    u32x4 k[4][2], v[8], ks, vs;
    auto load_k = [&](uint32_t page) {
        const uint8_t* p = a.codes + kv8_record(page, a.t.kv_heads, kh) + (n & 3) * KV8_HEAD + 32 * g;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            k[m][0] = *reinterpret_cast<const u32x4*>(p + m * 4 * KV8_HEAD);
            k[m][1] = *reinterpret_cast<const u32x4*>(p + m * 4 * KV8_HEAD + 16);
        }
        ks = *reinterpret_cast<const u32x4*>(a.scales + kv8_scale(page, a.t.kv_heads, kh));
    };
    auto load_v = [&](uint32_t page) {
        const uint8_t* p = a.codes + kv8_record(page, a.t.kv_heads, kh) + KV8_PART + n * KV8_PAGE;
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = *reinterpret_cast<const u32x4*>(p + c * 16 * KV8_PAGE);
        vs = *reinterpret_cast<const u32x4*>(a.scales + kv8_scale(page, a.t.kv_heads, kh) + KV8_PAGE);
    };
    const uint32_t t0 = y * per + wave, step = ATTEND_WAVES;
    Place pk = place(logical_of(t0, n >> 2)), pv = place(logical_of(t0, g));
    u32x4 qb[4];
    if (t0 < t_end) {
        load_k(pk.page);
        load_v(pv.page);
    }
    const bf16_t* qr = a.q + ((size_t)s * a.q_heads + kh * a.group + min(n, a.group - 1)) * KV8_HEAD + 32 * g;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        qb[j] = reinterpret_cast<const u32x4*>(qr)[j];
        if (n >= a.group) qb[j] = u32x4{0, 0, 0, 0};
    }
    Place pk1 = place(logical_of(t0 + step, n >> 2)), pv1 = place(logical_of(t0 + step, g));
    uint32_t lk2 = logical_of(t0 + 2 * step, n >> 2), lv2 = logical_of(t0 + 2 * step, g);

    float m_run = -INFINITY, lsum = 0.f;
    f32x4 o[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (uint32_t t = t0; t < t_end; t += step) {
        float sc[4][4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const float scale = __uint_as_float(((ks[m] >> (8 * (n & 3))) & 0xFFu) << 23);
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 4; ++j) acc = mfma(decode(k[m][j >> 1][2 * (j & 1)], k[m][j >> 1][2 * (j & 1) + 1], scale), qb[j], acc);
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[m][i] = acc[i] * a.scale2;
        }
        if (t + step < t_end) load_k(pk1.page);
        const bool whole = __all(pv.valid == KV8_PAGE);
        uint32_t keep[4];
        if (!whole) {
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const int left = (int)pv.valid - 4 * m;
                keep[m] = left >= 4 ? 0xFFFFFFFFu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i >= left) sc[m][i] = -INFINITY;
                vs[m] &= keep[m];
            }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sc[m][i]);
        mx = fmaxf(m_run, rows_max(mx));
        if (__any(mx > m_run)) {
            const float alpha = factor(m_run, mx);
            lsum *= alpha;
#pragma unroll
            for (int c = 0; c < 8; ++c) o[c] *= alpha;
            m_run = mx;
        }
        const float ref = m_run == -INFINITY ? 0.f : m_run;
        u32x4 hi[2], lo[2];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = __builtin_amdgcn_exp2f(sc[m][i] - ref);
                lsum += p;
                w[i] = p * __uint_as_float(((vs[m] >> (8 * i)) & 0xFFu) << 23);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t h = pack(w[2 * i], w[2 * i + 1]);
                hi[m >> 1][2 * (m & 1) + i] = h;
                lo[m >> 1][2 * (m & 1) + i] = pack(w[2 * i] - bf_lo(h), w[2 * i + 1] - bf_hi(h));
            }
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            if (!whole) v[c] &= u32x4{keep[0], keep[1], keep[2], keep[3]};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const u32x4 x = decode(v[c][2 * j], v[c][2 * j + 1], 1.f);
                o[c] = mfma(x, hi[j], o[c]);
                o[c] = mfma(x, lo[j], o[c]);
            }
        }
        pk = pk1;
        pv = pv1;
        pk1 = place(lk2);
        pv1 = place(lv2);
        lk2 = logical_of(t + 3 * step, n >> 2);
        lv2 = logical_of(t + 3 * step, g);
        if (t + step < t_end) load_v(pv.page);
    }
    lsum = rows_sum(lsum);

    // The block's four states.
    if (n < a.group) {
        if (g == 0) {
            wm[wave][n] = m_run;
            wl[wave][n] = lsum;
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) *reinterpret_cast<f32x4*>(&wo[wave][n][16 * c + 4 * g]) = o[c];
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < a.group * (KV8_HEAD / 4); e += 256) {
        const uint32_t h = e / (KV8_HEAD / 4), d = 4 * (e % (KV8_HEAD / 4));
        float top = wm[0][h], l = 0.f;
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (uint32_t w = 1; w < ATTEND_WAVES; ++w) top = fmaxf(top, wm[w][h]);
#pragma unroll
        for (uint32_t w = 0; w < ATTEND_WAVES; ++w) {
            const float f = factor(wm[w][h], top);
            l += f * wl[w][h];
            x += f * *reinterpret_cast<const f32x4*>(&wo[w][h][d]);
        }
        if (active == 1) {
            const float r = l == 0.f ? 0.f : 1.f / l;
            *reinterpret_cast<uint2*>(out + h * KV8_HEAD + d) = make_uint2(pack(x[0] * r, x[1] * r), pack(x[2] * r, x[3] * r));
        } else {
            float* st = a.state + (((size_t)s * a.q_heads + kh * a.group + h) * a.slices + y) * STATE;
            put2(st + 4 + d, x[0], x[1]);
            put2(st + 6 + d, x[2], x[3]);
            if (d == 0) put2(st, top, l);
        }
    }
    if (active == 1) return;
    // The states acknowledged, then the count: the block that completes it joins the slices.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    uint32_t* counter = a.counter + (size_t)s * a.t.kv_heads + kh;
    if (threadIdx.x == 0) last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == active - 1;
    __syncthreads();
    if (!last) return;
    for (uint32_t e = threadIdx.x; e < a.group * (KV8_HEAD / 4); e += 256) {
        const uint32_t h = e / (KV8_HEAD / 4), d = 4 * (e % (KV8_HEAD / 4));
        const float* st = a.state + ((size_t)s * a.q_heads + kh * a.group + h) * a.slices * STATE;
        float top = -INFINITY, l = 0.f;
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t z = 0; z < active; ++z) top = fmaxf(top, get2(st + z * STATE).x);
        for (uint32_t z = 0; z < active; ++z) {
            const float2 ml = get2(st + z * STATE), x0 = get2(st + z * STATE + 4 + d), x1 = get2(st + z * STATE + 6 + d);
            const float f = factor(ml.x, top);
            l += f * ml.y;
            x += f * f32x4{x0.x, x0.y, x1.x, x1.y};
        }
        const float r = l == 0.f ? 0.f : 1.f / l;
        *reinterpret_cast<uint2*>(out + h * KV8_HEAD + d) = make_uint2(pack(x[0] * r, x[1] * r), pack(x[2] * r, x[3] * r));
    }
    if (threadIdx.x == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next call
}

// The order of scores as whole numbers: larger scores larger, NaN above all.
__device__ __forceinline__ uint64_t score_key(double x) {
    if (x != x) return ~1ull;
    const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

// The pages of (sequence, kv head): scores in f64, then each page's rank by counting the better ones. The
// last page comes before all others; a page that is not there comes behind them.
__global__ void __launch_bounds__(256)
    kv8_select_kernel(Table t, const bf16_t* __restrict__ bounds, const bf16_t* __restrict__ q,
                      const uint32_t* __restrict__ lens, uint32_t budget, uint32_t* __restrict__ list,
                      uint64_t* __restrict__ keys_of, uint32_t q_heads) {
    __shared__ uint32_t flags[256];
    const uint32_t kh = blockIdx.x, s = blockIdx.y, i = threadIdx.x, group = q_heads / t.kv_heads;
    const uint32_t pages = (kv8_keys(lens[s], t.seq_pages) + KV8_PAGE - 1) / KV8_PAGE;
    uint64_t* key = keys_of + ((size_t)s * t.kv_heads + kh) * t.seq_pages;
    uint32_t* to = list + ((size_t)s * t.kv_heads + kh) * budget;
    for (uint32_t p = i; p < pages; p += 256) {
        const uint32_t page = t.page(s, p);
        uint64_t best = 0;
        if (page != KV8_NONE) {
            const bf16_t* b = bounds + kv8_bound(page, t.kv_heads, kh);
            for (uint32_t g = 0; g < group; ++g) {
                const bf16_t* qr = q + ((size_t)s * q_heads + kh * group + g) * KV8_HEAD;
                double sum = 0.0;
                for (uint32_t d = 0; d < KV8_HEAD; ++d) {
                    const float x = bf2f(qr[d]);
                    sum = fma((double)x, (double)bf2f(b[x < 0.f ? d : KV8_HEAD + d]), sum);
                }
                best = max(best, score_key(sum));
            }
        }
        key[p] = p == pages - 1 ? ~0ull : best;
    }
    __syncthreads();
    uint32_t taken = 0;
    for (uint32_t p0 = 0; p0 < pages; p0 += 256) {
        const uint32_t p = p0 + i;
        uint32_t rank = 0;
        if (p < pages)
            for (uint32_t o = 0; o < pages; ++o) rank += key[o] > key[p] || (key[o] == key[p] && o < p);
        flags[i] = p < pages && rank < budget;
        __syncthreads();
        uint32_t before = 0, all = 0;
        for (uint32_t j = 0; j < 256; ++j) {
            before += j < i ? flags[j] : 0;
            all += flags[j];
        }
        if (flags[i]) to[taken + before] = p;
        taken += all;
        __syncthreads();
    }
    for (uint32_t j = taken + i; j < budget; j += 256) to[j] = KV8_NONE;
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

x0ne_status check_cache(const char* what, const x0ne_kv8* c) {
    if (!c) return bad(what, "no cache");
    if (!c->codes || !c->scales || !c->page_table || c->codes % 16 || c->scales % 16 || c->page_table % 4)
        return bad(what, "codes and scales (16-byte aligned) and page_table are required");
    if (c->pool == 0 || c->kv_heads == 0 || c->kv_heads > 1024 || c->seqs > 65535 || c->seq_pages == 0 ||
        c->seq_pages >= (1u << 24))
        return bad(what, std::to_string(c->pool) + " pages of " + std::to_string(c->kv_heads) + " kv heads, " +
                             std::to_string(c->seqs) + " sequences of " + std::to_string(c->seq_pages) +
                             " pages (1 to 1024 kv heads, up to 65535 sequences, 1 to 2^24 - 1 pages)");
    return X0NE_OK;
}

x0ne_status check_heads(const char* what, const x0ne_kv8* c, uint32_t q_heads) {
    if (q_heads == 0 || q_heads % c->kv_heads != 0 || q_heads / c->kv_heads > 16)
        return bad(what, std::to_string(q_heads) + " q heads for " + std::to_string(c->kv_heads) +
                             " kv heads (1 to 16 per kv head)");
    return X0NE_OK;
}

Table table_of(const x0ne_kv8* c) {
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
    if (rows == 0 || c->seqs == 0) return X0NE_OK;
    const OnDevice on(g->device);
    const Table t = table_of(c);
    g->counts.launches += bounds ? 2 : 1;
    hipLaunchKernelGGL(kv8_write_kernel, dim3((uint32_t)rows, (q_heads + c->kv_heads + 3) / 4), dim3(256), 0, g->stream, t,
                       (uint8_t*)c->codes, (uint8_t*)c->scales, (const bf16_t*)qkv, (const bf16_t*)q_norm,
                       (const bf16_t*)k_norm, (const double*)rope_cs, (const uint32_t*)row_seq, (const uint32_t*)row_pos,
                       (bf16_t*)q_out, q_heads, positions, eps);
    X0NE_HIP(hipGetLastError(), what);
    if (!bounds) return X0NE_OK;
    hipLaunchKernelGGL(kv8_bounds_kernel, dim3((uint32_t)rows, (c->kv_heads + 3) / 4), dim3(256), 0, g->stream, t,
                       (const uint8_t*)c->codes, (const uint8_t*)c->scales, (const uint32_t*)row_seq,
                       (const uint32_t*)row_pos, positions, (bf16_t*)bounds);
    X0NE_HIP(hipGetLastError(), "kv8 bounds");
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
    hipLaunchKernelGGL(kv8_read_kernel, dim3(c->seq_pages, (c->kv_heads + 3) / 4, c->seqs), dim3(256), 0, g->stream,
                       table_of(c), (const uint8_t*)c->codes, (const uint8_t*)c->scales, (const uint32_t*)lens,
                       (bf16_t*)k, (bf16_t*)v, (const uint32_t*)out_table, out_pool);
    X0NE_HIP(hipGetLastError(), what);
    return X0NE_OK;
}

// Slices of a sequence's tiles: enough that the pairs of sequence and kv head fill 256 CUs with two blocks each.
static uint32_t slices_of(const x0ne_kv8* c) {
    const uint64_t pairs = std::max<uint64_t>(1, (uint64_t)c->seqs * c->kv_heads);
    return (uint32_t)std::min<uint64_t>(MAX_SLICES, std::max<uint64_t>(16, 512 / pairs));
}

// The workspace: a counter per (sequence, kv head), then the states of attention or the scores of selection.
static uint64_t counter_bytes(const x0ne_kv8* c) { return ((uint64_t)c->seqs * c->kv_heads * 4 + 255) / 256 * 256; }

extern "C" uint64_t x0ne_kv8_work_bytes(const x0ne_kv8* c, uint32_t q_heads) {
    if (check_cache("kv8 workspace", c) != X0NE_OK || check_heads("kv8 workspace", c, q_heads) != X0NE_OK) return 0;
    const uint64_t states = (uint64_t)c->seqs * q_heads * slices_of(c) * STATE * 4;
    const uint64_t scores = (uint64_t)c->seqs * c->kv_heads * c->seq_pages * 8;
    return std::max<uint64_t>(256, counter_bytes(c) + std::max(states, scores));
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
    g->counts.launches++;
    Attend a = {};
    a.t = table_of(c);
    a.codes = (const uint8_t*)c->codes;
    a.scales = (const uint8_t*)c->scales;
    a.q = (const bf16_t*)q;
    a.lens = (const uint32_t*)lens;
    a.list = (const uint32_t*)page_list;
    a.out = (bf16_t*)out;
    a.counter = (uint32_t*)work;
    a.state = (float*)(work + counter_bytes(c));
    a.budget = budget;
    a.q_heads = q_heads;
    a.group = q_heads / c->kv_heads;
    a.slices = slices_of(c);
    a.scale2 = scale * 1.44269504088896340736f;
    hipLaunchKernelGGL(kv8_attention_kernel, dim3(c->kv_heads, a.slices, c->seqs), dim3(64 * ATTEND_WAVES), 0, g->stream, a);
    X0NE_HIP(hipGetLastError(), what);
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
    if (!g) return fail(X0NE_ERR_GPU, "no device");
    if (c->seqs == 0) return X0NE_OK;
    const OnDevice on(g->device);
    g->counts.launches++;
    hipLaunchKernelGGL(kv8_select_kernel, dim3(c->kv_heads, c->seqs), dim3(256), 0, g->stream, table_of(c),
                       (const bf16_t*)bounds, (const bf16_t*)q, (const uint32_t*)lens, budget, (uint32_t*)page_list,
                       (uint64_t*)(work + counter_bytes(c)), q_heads);
    X0NE_HIP(hipGetLastError(), what);
    return X0NE_OK;
}
