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

// Decode attention, one wavefront per (sequence, q head): 64 keys at a time, a lane per key for the
// scores, then lane i dims i and i + 64 of the weighted values, with the running maximum and sum.
__global__ void __launch_bounds__(64)
    kv8_attention_kernel(Table t, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                         const bf16_t* __restrict__ q, const uint32_t* __restrict__ lens,
                         const uint32_t* __restrict__ list, uint32_t budget, bf16_t* __restrict__ out, uint32_t q_heads,
                         float scale) {
    __shared__ float qs[KV8_HEAD], ps[64], vscale[64];
    __shared__ size_t rec_of[64];
    const uint32_t h = blockIdx.x, s = blockIdx.y, i = threadIdx.x, kh = h / (q_heads / t.kv_heads);
    const uint32_t keys = kv8_keys(lens[s], t.seq_pages), pages = (keys + KV8_PAGE - 1) / KV8_PAGE;
    const uint32_t n = list ? min(budget, pages) : pages;
    const bf16_t* qr = q + ((size_t)s * q_heads + h) * KV8_HEAD;
    qs[i] = bf2f(qr[i]);
    qs[i + 64] = bf2f(qr[i + 64]);
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
    for (uint32_t p0 = 0; p0 < n; p0 += 4) {
        const uint32_t at = p0 + i / 16, slot = i % 16;
        const uint32_t logical = at >= n ? KV8_NONE : list ? list[((size_t)s * t.kv_heads + kh) * budget + at] : at;
        const uint32_t page = logical < pages ? t.page(s, logical) : KV8_NONE;
        const bool live = page != KV8_NONE && logical * KV8_PAGE + slot < keys;
        const size_t rec = kv8_record(live ? page : 0, t.kv_heads, kh);
        const size_t sc = kv8_scale(live ? page : 0, t.kv_heads, kh);
        float score = -INFINITY;
        __syncthreads();
        if (live) {
            float sum = 0.f;
            for (uint32_t d = 0; d < KV8_HEAD; ++d) sum = fmaf(kv8_value(codes[rec + slot * KV8_HEAD + d], scales[sc + slot]), qs[d], sum);
            score = sum * scale;
        }
        vscale[i] = live ? __uint_as_float((uint32_t)scales[sc + KV8_PAGE + slot] << 23) : 0.f;
        rec_of[i] = rec + KV8_PART + slot;
        float top = wave_max(score);
        top = fmaxf(m, top);
        const float ref = top == -INFINITY ? 0.f : top;
        const float p = expf(score - ref), alpha = expf(m - ref);
        m = top;
        l = l * alpha + wave_sum(p);
        ps[i] = live ? p : -1.f;
        __syncthreads();
        o0 *= alpha;
        o1 *= alpha;
        for (uint32_t k = 0; k < 64; ++k) {
            if (ps[k] < 0.f) continue;
            const float w = ps[k] * vscale[k];
            o0 = fmaf(w, kv8_value(codes[rec_of[k] + i * KV8_PAGE], 127), o0);
            o1 = fmaf(w, kv8_value(codes[rec_of[k] + (i + 64) * KV8_PAGE], 127), o1);
        }
    }
    bf16_t* d = out + ((size_t)s * q_heads + h) * KV8_HEAD;
    d[i] = f2bf(l == 0.f ? 0.f : o0 / l);
    d[i + 64] = f2bf(l == 0.f ? 0.f : o1 / l);
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

extern "C" uint64_t x0ne_kv8_work_bytes(const x0ne_kv8* c, uint32_t q_heads) {
    if (!c || check_cache("kv8 workspace", c) != X0NE_OK || check_heads("kv8 workspace", c, q_heads) != X0NE_OK) return 0;
    return std::max<uint64_t>(256, (uint64_t)c->seqs * c->kv_heads * c->seq_pages * 8);
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
    hipLaunchKernelGGL(kv8_attention_kernel, dim3(q_heads, c->seqs), dim3(64), 0, g->stream, table_of(c),
                       (const uint8_t*)c->codes, (const uint8_t*)c->scales, (const bf16_t*)q, (const uint32_t*)lens,
                       (const uint32_t*)page_list, budget, (bf16_t*)out, q_heads, scale);
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
                       (uint64_t*)work, q_heads);
    X0NE_HIP(hipGetLastError(), what);
    return X0NE_OK;
}
