// Log probabilities of rows of logits: those of given tokens, the entropy, and the top alternatives.
//
// With x = scale logit, m = max x, z = sum e^(x - m), t = sum (x - m) e^(x - m): log p = (x - m) - log z and the entropy
// is log z - t / z. One pass: a block holds SLICE logits of a row in registers, forms (m, z, t) of them and picks its
// top ones; the last block of a row to count itself joins the slices.
#include <algorithm>
#include <cmath>
#include <string>

#include "device.h"
#include "internal.h"

using namespace x0ne;

namespace {

constexpr uint32_t THREADS = 256, EACH = 16, SLICE = THREADS * EACH, WAVES = THREADS / 64;
constexpr uint32_t MOST_TOP = 64;
constexpr float LOG2E = 1.44269504088896340736f;
constexpr uint32_t NONE = 0xFFFFFFFFu;

struct Args {
    const void* logits;
    uint64_t stride;
    const uint32_t* tokens;
    float* token_lp;
    float* entropy;
    uint32_t* top_ids;
    float* top_lp;
    uint32_t* counter;  // one per row of the launch
    float4* state;      // [rows][slices]: m, z, t
    uint64_t* best;     // [rows][slices][top]
    uint32_t rows, vocab, slices, per_row, top;
    float scale;
};

// Logits in order, zeros alike, and lower ids first among equals; 0 stands for none (minus infinity is no alternative).
__device__ __forceinline__ uint64_t key_of(float x, uint32_t id) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    const uint32_t order = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    return x > -INFINITY ? (uint64_t)order << 32 | ~id : 0;
}
__device__ __forceinline__ float logit_of(uint64_t key) {
    const uint32_t order = (uint32_t)(key >> 32);
    return __uint_as_float(order ^ (order & 0x80000000u ? 0x80000000u : 0xFFFFFFFFu));
}

struct Shared {
    uint64_t key[SLICE];
    uint64_t floor[WAVES];
    uint64_t top[MOST_TOP];
    float4 state[WAVES];
    uint32_t count;
    uint32_t last;
};

// The `top` largest of the block's keys (key(i) of each thread for i < EACH, all different but for 0), in order, into
// sh.top, 0 behind the last. The top-th largest of a wavefront's lanes' largest keys is a floor that at least `top` keys
// reach; those that reach the highest of the wavefronts' floors, few more than `top`, are ranked by counting.
template <class Key>
__device__ __forceinline__ void pick(Key key, uint32_t top, Shared& sh) {
    const uint32_t wave = threadIdx.x >> 6;
    uint64_t mine = 0;
#pragma unroll
    for (uint32_t i = 0; i < EACH; ++i) mine = max(mine, key(i));
    uint32_t above = 0;
    for (uint32_t l = 0; l < 64; ++l) above += (uint64_t)__shfl((unsigned long long)mine, (int)l, 64) > mine;
    if (threadIdx.x == 0) sh.count = 0;
    if (threadIdx.x < WAVES) sh.floor[threadIdx.x] = 0;
    if (threadIdx.x < top) sh.top[threadIdx.x] = 0;
    __syncthreads();
    if (mine && above == top - 1) sh.floor[wave] = mine;
    __syncthreads();
    uint64_t floor = 1;
#pragma unroll
    for (uint32_t w = 0; w < WAVES; ++w) floor = max(floor, sh.floor[w]);
    if (mine >= floor) {
#pragma unroll
        for (uint32_t i = 0; i < EACH; ++i) {
            const uint64_t k = key(i);
            if (k >= floor) sh.key[atomicAdd(&sh.count, 1u)] = k;
        }
    }
    __syncthreads();
    const uint32_t count = sh.count;
    for (uint32_t c = threadIdx.x; c < count; c += THREADS) {
        const uint64_t k = sh.key[c];
        uint32_t rank = 0;
        for (uint32_t o = 0; o < count; ++o) rank += sh.key[o] > k;
        if (rank < top) sh.top[rank] = k;
    }
    __syncthreads();
}

// (m, z, t) of two sets. A set of nothing but -infinity has m = -infinity and z = t = 0, or NaN.
__device__ __forceinline__ float4 join(float4 a, float4 b) {
    const float m = fmaxf(a.x, b.x), da = a.x - m, db = b.x - m;
    float4 r = {m, 0.f, 0.f, 0.f};
    const float pa = __builtin_amdgcn_exp2f(da * LOG2E), pb = __builtin_amdgcn_exp2f(db * LOG2E);
    // A set at m as it is, and one so far below it that nothing is left without an infinity times zero.
    r.y = (a.x == m ? a.y : pa * a.y) + (b.x == m ? b.y : pb * b.y);
    r.z = (a.x == m ? a.z : pa > 0.f ? pa * (a.z + da * a.y) : pa * a.y) + (b.x == m ? b.z : pb > 0.f ? pb * (b.z + db * b.y) : pb * b.y);
    return r;
}

typedef float f32x4a __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4a __attribute__((ext_vector_type(4), aligned(2)));

template <bool BF16>
__device__ __forceinline__ float logit_at(const void* row, uint32_t i) {
    return BF16 ? bf2f(static_cast<const bf16_t*>(row)[i]) : static_cast<const float*>(row)[i];
}

template <bool BF16>
__global__ void __launch_bounds__(256) logprobs_kernel(Args a) {
    __shared__ Shared sh;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t r = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
    const void* row = static_cast<const uint8_t*>(a.logits) + r * a.stride * (BF16 ? 2 : 4);
    constexpr uint32_t PIECE = BF16 ? 8 : 4;  // logits of a 16-byte load
    float x[EACH];
    const uint32_t first = slice * SLICE + threadIdx.x * PIECE;
    // The id of x[i].
    auto id_of = [&](uint32_t i) { return first + i / PIECE * (THREADS * PIECE) + i % PIECE; };
#pragma unroll
    for (uint32_t v = 0; v < EACH / PIECE; ++v) {
        const uint32_t id = id_of(v * PIECE);
        if (id < a.vocab && a.vocab - id >= PIECE) {
            if (BF16) {
                const u32x4a w = *reinterpret_cast<const u32x4a*>(static_cast<const bf16_t*>(row) + id);
#pragma unroll
                for (uint32_t e = 0; e < PIECE; ++e) x[v * PIECE + e] = e & 1 ? bf_hi(w[e / 2 % 4]) : bf_lo(w[e / 2 % 4]);
            } else {
                const f32x4a w = *reinterpret_cast<const f32x4a*>(static_cast<const float*>(row) + id);
#pragma unroll
                for (uint32_t e = 0; e < PIECE; ++e) x[v * PIECE + e] = w[e % 4];
            }
        } else {
#pragma unroll
            for (uint32_t e = 0; e < PIECE; ++e) x[v * PIECE + e] = id + e < a.vocab ? logit_at<BF16>(row, id + e) : -INFINITY;
        }
    }
    float m = -INFINITY;
#pragma unroll
    for (uint32_t i = 0; i < EACH; ++i) m = fmaxf(m, x[i]);
    m = wave_max(m) * a.scale;
    const float base = m == -INFINITY ? 0.f : m;
    float z = 0.f, t = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < EACH; ++i) {
        const float d = x[i] * a.scale - base, p = __builtin_amdgcn_exp2f(d * LOG2E);
        z += p;
        t += p > 0.f ? p * d : p;
    }
    z = wave_sum(z);
    t = wave_sum(t);
    if (lane == 0) sh.state[wave] = float4{m, z, t, 0.f};
    if (a.top) pick([&](uint32_t i) { return key_of(x[i], id_of(i)); }, a.top, sh);
    __syncthreads();
    float4 all = sh.state[0];
#pragma unroll
    for (uint32_t w = 1; w < WAVES; ++w) all = join(all, sh.state[w]);
    if (a.slices > 1) {
        float* state = (float*)(a.state + (uint64_t)r * a.slices);
        uint64_t* best = a.best + (uint64_t)r * a.slices * a.top;
        if (threadIdx.x == 0) {
            __hip_atomic_store(state + 4 * slice, all.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(state + 4 * slice + 1, all.y, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(state + 4 * slice + 2, all.z, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        if (threadIdx.x < a.top)
            __hip_atomic_store(best + (uint64_t)slice * a.top + threadIdx.x, sh.top[threadIdx.x], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        // The stores acknowledged, then the count: the block that completes it joins the slices.
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0)
            sh.last = __hip_atomic_fetch_add(a.counter + r, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.slices - 1;
        __syncthreads();
        if (!sh.last) return;
        if (threadIdx.x == 0) __hip_atomic_store(a.counter + r, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next call
        all = float4{-INFINITY, 0.f, 0.f, 0.f};
        for (uint32_t s = threadIdx.x; s < a.slices; s += THREADS) {
            float v[3];
#pragma unroll
            for (int i = 0; i < 3; ++i) v[i] = __hip_atomic_load(state + 4 * s + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            all = join(all, float4{v[0], v[1], v[2], 0.f});
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1)
            all = join(all, float4{__shfl_xor(all.x, o, 64), __shfl_xor(all.y, o, 64), __shfl_xor(all.z, o, 64), 0.f});
        if (lane == 0) sh.state[wave] = all;
        if (a.top) {
            // SLICE keys at a time, the best so far among them.
            const uint32_t keys = a.slices * a.top;
            uint32_t done = 0, kept = 0;
            while (done < keys) {
                const uint32_t some = min(keys - done, SLICE - kept);
                uint64_t k[EACH];
#pragma unroll
                for (uint32_t i = 0; i < EACH; ++i) {
                    const uint32_t at = i * THREADS + threadIdx.x;
                    k[i] = 0;
                    if (at < kept)
                        k[i] = sh.top[at];
                    else if (at - kept < some)
                        k[i] = __hip_atomic_load(best + done + at - kept, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                __syncthreads();
                pick([&](uint32_t i) { return k[i]; }, a.top, sh);
                done += some;
                kept = a.top;
            }
        }
        __syncthreads();
        all = sh.state[0];
#pragma unroll
        for (uint32_t w = 1; w < WAVES; ++w) all = join(all, sh.state[w]);
    }
    // z is NaN with a NaN or an infinity among the logits, 0 where all are -infinity: no distribution.
    const bool none = !(all.y > 0.f);
    const float log_z = none ? NAN : logf(all.y);
    if (a.entropy && threadIdx.x == 0) a.entropy[r] = log_z - all.z / all.y;
    for (uint32_t i = threadIdx.x; i < a.per_row; i += THREADS) {
        const uint64_t at = (uint64_t)r * a.per_row + i;
        const uint32_t id = a.tokens[at];
        a.token_lp[at] = id < a.vocab ? logit_at<BF16>(row, id) * a.scale - all.x - log_z : NAN;
    }
    if (threadIdx.x < a.top) {
        const uint64_t k = sh.top[threadIdx.x], at = (uint64_t)r * a.top + threadIdx.x;
        a.top_ids[at] = none || !k ? NONE : ~(uint32_t)k;
        a.top_lp[at] = none ? NAN : k ? logit_of(k) * a.scale - all.x - log_z : -INFINITY;
    }
}

// ---- host ----

x0ne_status bad(const std::string& why) { return fail(X0NE_ERR_FORMAT, "logprobs: " + why); }

x0ne_status check_shape(const x0ne_logprobs* d) {
    if (!d) return bad("no descriptor");
    if (d->vocab == 0 || d->vocab > (1u << 24) || d->rows > (1u << 24) || d->top > MOST_TOP || d->per_row > (1u << 24) || d->bf16 > 1)
        return bad(std::to_string(d->rows) + " rows of " + std::to_string(d->vocab) + " logits, " + std::to_string(d->per_row) +
                   " tokens to a row, top " + std::to_string(d->top) + ", bf16 " + std::to_string(d->bf16) +
                   " (up to 2^24 rows, logits and tokens, top 64; bf16 0 or 1)");
    return X0NE_OK;
}

uint32_t slices_of(const x0ne_logprobs* d) { return (d->vocab + SLICE - 1) / SLICE; }

// The workspace: a counter per row, then the slices' states and top keys. The counters are as many for every call, as in
// the 8-bit cache's workspace, so that calls of all shapes may share one. More rows are further launches.
constexpr uint64_t COUNTERS = 65536, COUNTER_BYTES = 4 * COUNTERS;
uint64_t rows_at_once(const x0ne_logprobs* d) {
    // A launch has fewer than 2^32 threads.
    return std::min<uint64_t>(COUNTERS, ((1ull << 32) / THREADS - 1) / slices_of(d));
}

}  // namespace

extern "C" uint64_t x0ne_logprobs_work_bytes(const x0ne_logprobs* d) {
    if (check_shape(d) != X0NE_OK) return 0;
    const uint64_t slices = slices_of(d);
    return COUNTER_BYTES + (slices > 1 ? std::min<uint64_t>(d->rows, rows_at_once(d)) * slices * (sizeof(float4) + 8ull * d->top) : 0);
}

extern "C" x0ne_status x0ne_gpu_logprobs(x0ne_gpu* g, const x0ne_logprobs* d) {
    X0NE_TRY(check_shape(d));
    const uint64_t each = d->bf16 ? 2 : 4;
    if (!d->logits || d->logits % each || d->stride < d->vocab || d->stride >= (1ull << 32))
        return bad("logits (aligned to one), and a stride of at least a row's logits and below 2^32, are required");
    if (!(d->scale > 0.f) || !std::isfinite(d->scale)) return bad("a scale that is positive and finite is required");
    if (d->per_row && (!d->tokens || !d->token_lp || d->tokens % 4 || d->token_lp % 4))
        return bad("given tokens need tokens and token_lp (4-byte aligned)");
    if (d->top && (!d->top_ids || !d->top_lp || d->top_ids % 4 || d->top_lp % 4)) return bad("top alternatives need top_ids and top_lp (4-byte aligned)");
    if (d->entropy % 4) return bad("entropy is 4-byte aligned");
    if (!d->work || d->work % 256 || d->work_bytes < x0ne_logprobs_work_bytes(d))
        return bad("a workspace of x0ne_logprobs_work_bytes (256-byte aligned) is required");
    if (!g) return fail(X0NE_ERR_GPU, "no device");
    if (d->rows == 0) return X0NE_OK;
    const OnDevice on(g->device);
    const uint32_t slices = slices_of(d);
    for (uint64_t first = 0; first < d->rows; first += rows_at_once(d)) {
        Args a = {};
        a.rows = (uint32_t)std::min<uint64_t>(d->rows - first, rows_at_once(d));
        a.logits = (const uint8_t*)d->logits + first * d->stride * each;
        a.stride = d->stride;
        a.tokens = (const uint32_t*)d->tokens + first * d->per_row;
        a.token_lp = (float*)d->token_lp + first * d->per_row;
        a.entropy = d->entropy ? (float*)d->entropy + first : nullptr;
        a.top_ids = (uint32_t*)d->top_ids + first * d->top;
        a.top_lp = (float*)d->top_lp + first * d->top;
        a.counter = (uint32_t*)d->work;
        a.state = (float4*)(d->work + COUNTER_BYTES);
        a.best = (uint64_t*)(a.state + (uint64_t)a.rows * slices);
        a.vocab = d->vocab;
        a.slices = slices;
        a.per_row = d->per_row;
        a.top = d->top;
        a.scale = d->scale;
        g->counts.launches++;
        hipLaunchKernelGGL(d->bf16 ? logprobs_kernel<true> : logprobs_kernel<false>, dim3(a.rows * slices), dim3(THREADS), 0, g->stream, a);
        X0NE_HIP(hipGetLastError(), "logprobs");
    }
    return X0NE_OK;
}
