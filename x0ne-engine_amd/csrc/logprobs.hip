// Log probabilities of rows of logits: those of given tokens, the entropy, and the top alternatives.
//
// With l the logits, m = max l, z = sum e^(scale (l - m)), t = sum (l - m) e^(scale (l - m)): log p = scale (l - m) - log z
// and the entropy is log z - scale t / z. One pass over the logits: a block holds a row or a slice of one in registers, 16 or
// 32 logits to a thread, forms (m, z, t) of them and picks its top ones. A second, small kernel joins a row's slices: joined by
// the last block of the row to count itself, the code of that came from memory while the card waited (15 to 30 us).
#include <algorithm>
#include <string>

#include "device.h"
#include "internal.h"
#include "logprobs.h"

using namespace x0ne;

namespace {

constexpr uint32_t MOST_TOP = LOGPROBS_MOST_TOP;
constexpr uint32_t CANDIDATES = 512;
constexpr uint32_t RANKED = 128;  // so many keys are ranked without a floor
constexpr float LOG2E = 1.44269504088896340736f, LOWEST = -3.40282347e38f;
constexpr uint32_t NONE = 0xFFFFFFFFu;

struct Args {
    const void* logits;
    uint64_t stride;
    const uint32_t* tokens;
    float* token_lp;
    float* entropy;
    uint32_t* top_ids;
    float* top_lp;
    float4* state;   // [rows][slices]: m, z, t
    uint64_t* best;  // [rows][top][slices]
    uint32_t vocab, slices, length, per_row, top;  // logits of a slice
    float scale;
};

// Logits in order, zeros alike, and lower ids first among equals. No key of a logit above -infinity is 0.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t id) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (uint64_t)(b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u)) << 32 | (uint32_t)~id;
}
__device__ __forceinline__ float logit_of(uint64_t key) {
    const uint32_t order = (uint32_t)(key >> 32);
    return __uint_as_float(order ^ (order & 0x80000000u ? 0x80000000u : 0xFFFFFFFFu));
}

// A value joined with that of another lane of its row of 16 by DPP (0xB1, 0x4E: xor 1 and 2; 0x141, 0x140: lane 7 - i of each
// half row, lane 15 - i), and of other rows by the row swaps: after a step all lanes of 2, 4, 8, 16, 32, 64 have the same.
template <int CTRL>
__device__ __forceinline__ float moved(float x) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(x), CTRL, 0xF, 0xF, true));
}
template <int STEP, class Op>
__device__ __forceinline__ float fold(float x, Op op) {
    if (STEP == 0) return op(x, moved<0xB1>(x));
    if (STEP == 1) return op(x, moved<0x4E>(x));
    if (STEP == 2) return op(x, moved<0x141>(x));
    if (STEP == 3) return op(x, moved<0x140>(x));
    const auto a = STEP == 4 ? __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false)
                             : __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return op(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
template <class Op>
__device__ __forceinline__ float fold_all(float x, Op op) {
    return fold<5>(fold<4>(fold<3>(fold<2>(fold<1>(fold<0>(x, op), op), op), op), op), op);
}
struct Most {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Least {
    __device__ __forceinline__ float operator()(float a, float b) const { return fminf(a, b); }
};
struct Sum {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};

template <uint32_t THREADS>
struct Shared {
    uint64_t key[CANDIDATES + 16];
    uint64_t top[MOST_TOP];
    float4 state[THREADS / 64];
    float all[THREADS / 64], some[THREADS / 64], group[32];
    uint32_t count;
};

// The value of lane l ^ X.
template <int X>
__device__ __forceinline__ float other(float x) {
    if (X == 1) return moved<0xB1>(x);
    if (X == 2) return moved<0x4E>(x);
    if (X == 3) return moved<0x1B>(x);
    if (X == 4) return moved<0x1B>(moved<0x141>(x));
    if (X == 7) return moved<0x141>(x);
    if (X == 8) return moved<0x128>(x);
    if (X == 15) return moved<0x140>(x);
    if (X == 31) return other<16>(moved<0x140>(x));
    if (X == 63) return other<32>(other<16>(moved<0x140>(x)));
    const auto a = X == 16 ? __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false)
                           : __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(threadIdx.x & X ? a[0] : a[1]);
}
// A step of a bitonic sort of the wavefront's lanes, falling: the larger of lanes l and l ^ X to the one without BIT.
template <int X, int BIT>
__device__ __forceinline__ float sorted(float x) {
    const float o = other<X>(x);
    return threadIdx.x & BIT ? fminf(x, o) : fmaxf(x, o);
}

// A floor that at least `top` of the block's logits reach, by the largest of each thread's. -infinity is no alternative: the
// floor is above it. Few alternatives: the top-th of the largest of 16 or 32 groups of neighbouring threads, which few more
// reach (6 for 5, 31 for 20). More: each wavefront sorts its threads' largest, and the floor is the highest of the wavefronts'
// top-th ones or the lowest of the p-th ones, p top over the wavefronts rounded up (of 4096 logits 30 for 20, 80 for 64).
// 32 groups are for blocks of 512 and more, where the sort of 64 is dearer (61 rows of 32001, 20 alternatives: 9.7 us, 11.7
// by wavefronts; with 256 threads one row of 151936 11.4 and 10.7, as the join's keys lie in order).
// The floor supposes that the largest logits lie anywhere. Where they crowd into a few threads' pieces (rows that rise or fall
// with the id), many more reach it, in blocks of 512 and more than fit, so that the bisection takes over: with 5 alternatives
// one row of 151936 12.8 to 16.7 us instead of 9.6, 64 rows of 32001 in bf16 44 to 46 instead of 9.1, 4096 rows of 50257 in
// bf16 700 to 922 instead of 145.
template <uint32_t THREADS>
__device__ __forceinline__ float floor_of(float most, uint32_t top, Shared<THREADS>& sh) {
    constexpr uint32_t WAVES = THREADS / 64;
    const auto sorted16 = [](float x) {
        x = sorted<1, 1>(x);
        x = sorted<1, 1>(sorted<3, 2>(x));
        x = sorted<1, 1>(sorted<2, 2>(sorted<7, 4>(x)));
        return sorted<1, 1>(sorted<2, 2>(sorted<4, 4>(sorted<15, 8>(x))));
    };
    const auto nth = [](float x, uint32_t l) { return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), (int)l)); };
    const auto sorted32 = [&](float x) { return sorted<1, 1>(sorted<2, 2>(sorted<4, 4>(sorted<8, 8>(sorted<31, 16>(sorted16(x)))))); };
    if (top <= logprobs_in_groups(THREADS)) {
        const uint32_t lanes = THREADS / (top <= 12 ? 16 : 32);  // to a group: 16, 32 or 64
        float largest = fold<3>(fold<2>(fold<1>(fold<0>(most, Most()), Most()), Most()), Most());
        if (lanes >= 32) largest = fold<4>(largest, Most());
        if (lanes == 64) largest = fold<5>(largest, Most());
        if (threadIdx.x % lanes == 0) sh.group[threadIdx.x / lanes] = largest;
        __syncthreads();
        return fmaxf(top <= 12 ? nth(sorted16(sh.group[threadIdx.x & 15]), top - 1) : nth(sorted32(sh.group[threadIdx.x & 31]), top - 1), LOWEST);
    }
    float x = sorted32(most);
    x = sorted<1, 1>(sorted<2, 2>(sorted<4, 4>(sorted<8, 8>(sorted<16, 16>(sorted<63, 32>(x))))));
    sh.all[threadIdx.x >> 6] = nth(x, top - 1);
    sh.some[threadIdx.x >> 6] = nth(x, (top - 1) / WAVES);
    __syncthreads();
    const uint32_t w = threadIdx.x & (WAVES - 1);
    float one = sh.all[w], each = sh.some[w];
    one = fold<1>(fold<0>(one, Most()), Most());
    each = fold<1>(fold<0>(each, Least()), Least());
    if (WAVES >= 8) one = fold<2>(one, Most()), each = fold<2>(each, Least());
    if (WAVES == 16) one = fold<3>(one, Most()), each = fold<3>(each, Least());
    return fmaxf(fmaxf(one, each), LOWEST);
}

// Room for a thread's `own` keys among the block's candidates: where they go. All threads take part.
template <uint32_t THREADS>
__device__ __forceinline__ uint32_t room(uint32_t own, Shared<THREADS>& sh) {
    const uint32_t up_to = wave_up_to(own);
    uint32_t base = 0;
    if ((threadIdx.x & 63) == 63) base = __hip_atomic_fetch_add(&sh.count, up_to, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    return (uint32_t)__builtin_amdgcn_readlane((int)base, 63) + up_to - own;
}

// The `top` largest of the first `found` of sh.key, in order, into sh.top, by counting the larger ones of each.
template <uint32_t THREADS>
__device__ __forceinline__ void rank(uint32_t found, uint32_t top, Shared<THREADS>& sh) {
    if (threadIdx.x < 16) sh.key[found + threadIdx.x] = 0;
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < found; c += THREADS) {
        const uint64_t k = sh.key[c];
        uint32_t above = 0;
#pragma unroll 1
        for (uint32_t o = 0; o < found; o += 16) {
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) above += sh.key[o + i] > k;
        }
        if (k && above < top) sh.top[above] = k;
    }
    __syncthreads();
}

// x[i] of an i of the lane's own, by halving (bits, so that the compiler keeps x in registers).
template <uint32_t N, class T>
__device__ __forceinline__ T chosen(const T (&x)[N], uint32_t i) {
    if constexpr (N == 1)
        return x[0];
    else {
        T half[N / 2];
        const uint32_t odd = 0u - (i & 1);
#pragma unroll
        for (uint32_t k = 0; k < N / 2; ++k)
            half[k] = __builtin_bit_cast(T, (__builtin_bit_cast(uint32_t, x[2 * k + 1]) & odd) | (__builtin_bit_cast(uint32_t, x[2 * k]) & ~odd));
        return chosen(half, i >> 1);
    }
}

// The `top` largest of the block's logits x[i] of ids id(i), in order, as keys into sh.top, 0 behind the last; `most` is the
// largest of x. What reaches the floor is ranked by counting. Where that is too much (equal logits, parts that are masked
// throughout), the floor is raised by bisection over the keys: all differ, so some floor leaves from top to CANDIDATES.
template <uint32_t THREADS, uint32_t N, class Id>
__device__ __forceinline__ void pick(const float (&x)[N], float most, Id id, uint32_t top, Shared<THREADS>& sh) {
    if (threadIdx.x == 0) sh.count = 0;
    if (threadIdx.x < MOST_TOP) sh.top[threadIdx.x] = 0;
    const float floor = floor_of<THREADS>(most, top, sh);
    uint32_t reach = 0;  // bit i: x[i] does
#pragma unroll
    for (uint32_t i = N; i-- > 0;) reach += reach + (x[i] >= floor);
    uint32_t own = __popc(reach), at = room(own, sh);
    auto leave = [&] {
        for (; reach && at < CANDIDATES; reach &= reach - 1) {
            const uint32_t i = __ffs(reach) - 1;
            sh.key[at++] = key_of(chosen(x, i), id(i));
        }
    };
    leave();
    __syncthreads();
    if (sh.count > CANDIDATES) {
        const uint64_t from = key_of(floor, NONE);
        uint64_t low = (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(from >> 32)) << 32, high = ~0ull;
        for (bool found = false; !found;) {
            const uint64_t mid = low + (high - low) / 2;
            __syncthreads();
            if (threadIdx.x == 0) sh.count = 0;
            __syncthreads();
            // Keys of mid and more, by their logits and ids: none is that of -0, and above infinity's the edge is a NaN.
            const float edge = logit_of(mid);
            const uint32_t least = (uint32_t)(mid >> 32) == 0x7FFFFFFFu ? 0u : (uint32_t)mid;
            uint32_t zero = 0;
            asm volatile("" : "+v"(zero));  // the ids are formed here and not kept from turn to turn
            reach = 0;
#pragma unroll
            for (uint32_t i = N; i-- > 0;) reach += reach + (x[i] > edge || (x[i] == edge && ~(id(i) + zero) >= least));
            own = __popc(reach);
            at = room(own, sh);
            __syncthreads();
            const uint32_t count = __builtin_amdgcn_readfirstlane(sh.count);
            if (count >= top)
                low = mid;
            else
                high = mid;
            found = (count >= top && count <= CANDIDATES) || high - low < 2;
            if (found) leave();
        }
        __syncthreads();
    }
    rank<THREADS>(min(sh.count, CANDIDATES), top, sh);
}

// (m, z, t) of two sets: one at the larger m as it is, one so far below it that nothing is left without an infinity times
// zero. An exponential times its difference is at most 1 / (e scale) and comes first: a difference times z may be past f32.
// A set of nothing but -infinity has m = -infinity and z = t = 0, or NaN.
__device__ __forceinline__ float4 join(float4 a, float4 b, float scale2) {
    const float m = fmaxf(a.x, b.x), da = a.x - m, db = b.x - m;
    float4 r = {m, 0.f, 0.f, 0.f};
    const float pa = __builtin_amdgcn_exp2f(da * scale2), pb = __builtin_amdgcn_exp2f(db * scale2);
    r.y = (a.x == m ? a.y : pa * a.y) + (b.x == m ? b.y : pb * b.y);
    r.z = (a.x == m ? a.z : pa > 0.f ? fmaf(pa * da, a.y, pa * a.z) : 0.f) + (b.x == m ? b.z : pb > 0.f ? fmaf(pb * db, b.y, pb * b.z) : 0.f);
    return r;
}

// Joined over the first `lanes` lanes.
__device__ __forceinline__ float4 join_lanes(float4 all, int lanes, float scale2) {
#pragma unroll 1
    for (int o = 1; o < lanes; o <<= 1)
        all = join(all, float4{__shfl_xor(all.x, o, 64), __shfl_xor(all.y, o, 64), __shfl_xor(all.z, o, 64), 0.f}, scale2);
    return all;
}

typedef float f32x4a __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4a __attribute__((ext_vector_type(4), aligned(2)));

template <bool BF16>
__device__ __forceinline__ float logit_at(const void* row, uint32_t i) {
    return BF16 ? bf2f(static_cast<const bf16_t*>(row)[i]) : static_cast<const float*>(row)[i];
}

// What is asked of row r, whose (m, z, t) is `all` and whose top keys are in sh.top; `given` is the logit of the thread's
// first token.
template <bool BF16, uint32_t THREADS>
__device__ __forceinline__ void answer(const Args& a, const void* row, uint32_t r, float4 all, uint32_t token, float given, Shared<THREADS>& sh) {
    // z is NaN with a NaN or an infinity among the logits, 0 where all are -infinity: no distribution.
    const bool none = !(all.y > 0.f);
    const float log_z = none ? NAN : logf(all.y);
    auto log_p = [&](float l) { return (0.5f * l - 0.5f * all.x) * (2.f * a.scale) - log_z; };  // a difference may be past f32
    if (a.entropy && threadIdx.x == 0) a.entropy[r] = log_z - a.scale * (all.z / all.y);
    const uint64_t tokens = (uint64_t)r * a.per_row;
    if (threadIdx.x < a.per_row) a.token_lp[tokens + threadIdx.x] = token < a.vocab ? log_p(given) : NAN;
    for (uint32_t i = threadIdx.x + THREADS; i < a.per_row; i += THREADS) {
        const uint32_t id = a.tokens[tokens + i];
        a.token_lp[tokens + i] = id < a.vocab ? log_p(logit_at<BF16>(row, id)) : NAN;
    }
    if (threadIdx.x < a.top) {
        const uint64_t k = sh.top[threadIdx.x], at = (uint64_t)r * a.top + threadIdx.x;
        a.top_ids[at] = none || !k ? NONE : ~(uint32_t)k;
        a.top_lp[at] = none ? NAN : k ? log_p(logit_of(k)) : -INFINITY;
    }
}

template <bool BF16>
__device__ __forceinline__ const void* row_of(const Args& a, uint32_t r) {
    return static_cast<const uint8_t*>(a.logits) + r * a.stride * (BF16 ? 2 : 4);
}

// Measured on MI355X by a kernel trace: 46.8 us for 512 rows of 151936 f32 logits with one alternative (311 MB, 6.6 TB/s); 5.5
// for one row with 20, a launch, a trip to memory and the selection one after the other. Those 512 rows without alternatives
// and with 1, 5, 20 and 64, both kernels back to back in a captured graph, logits in turn past the Infinity Cache: 57, 57.7,
// 62.7, 66.1 and 73.5: the sort, the ranking and their barriers take the place of loads. So do they for bf16, whose logits come
// at twice the rate: 4096 rows of 50257 (412 MB) 111.5, 125.1, 144.7 and, with 64, 197.
// Wavefronts of a kernel to a SIMD: as many as its registers allow without a spill (512 rows of 151936 f32 logits, 20
// alternatives: 62 us with 6 of 32 logits to a thread, 79 with 7, 92 with 8).
constexpr int waves_of(uint32_t threads, uint32_t each) { return each == 16 ? 8 : threads == 1024 ? 4 : 6; }

template <bool BF16, uint32_t THREADS, uint32_t EACH>
__global__ void __launch_bounds__(THREADS, waves_of(THREADS, EACH)) logprobs_slices_kernel(Args a) {
    constexpr uint32_t WAVES = THREADS / 64;
    constexpr uint32_t PIECE = BF16 ? 8 : 4;  // logits of a 16-byte load
    // 56 registers of the 40 needed. 8 wavefronts to a SIMD are the most with either, but by the counters 24.2 to a CU are there on
    // average, 24.6 without it, and the fewer are faster (f32 logits that no cache has, one alternative: 512 rows of 151936 57.9
    // us, 58.7 without; 1024 rows 108.4 and 109.5; 2000 of 40000 62.5 and 63.2). Rows in one slice and few long rows take the
    // same with either.
    if constexpr (EACH == 16) asm volatile("" ::: "v55");
    __shared__ Shared<THREADS> sh;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t r = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
    const void* row = row_of<BF16>(a, r);
    const uint32_t start = slice * a.length, behind = min(start + a.length, a.vocab), first = start + threadIdx.x * PIECE;
    auto id_of = [&](uint32_t i) { return first + i / PIECE * (THREADS * PIECE) + i % PIECE; };  // of x[i]
    float x[EACH];
#pragma unroll
    for (uint32_t v = 0; v < EACH / PIECE; ++v) {
        const uint32_t id = id_of(v * PIECE);
        if (start + (v + 1) * THREADS * PIECE <= behind || id + PIECE <= behind) {  // all threads', or this one's
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
            for (uint32_t e = 0; e < PIECE; ++e) x[v * PIECE + e] = id + e < behind ? logit_at<BF16>(row, id + e) : -INFINITY;
        }
    }
    const float scale2 = a.scale * LOG2E;
    float most = x[0];
#pragma unroll
    for (uint32_t i = 1; i < EACH; ++i) most = fmaxf(most, x[i]);
    const float m = fmaxf(fold_all(most, Most()), -INFINITY), base = m == -INFINITY ? 0.f : m;
    float z = 0.f, t = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < EACH; ++i) {
        const float d = x[i] - base, p = __builtin_amdgcn_exp2f(d * scale2);
        z += p;
        t = fmaf(p, fmaxf(d, LOWEST), t);  // 0 for -infinity; what a NaN leaves here does not matter, as it is in z
    }
    z = fold_all(z, Sum());
    t = fold_all(t, Sum());
    if (lane == 0) sh.state[wave] = float4{m, z, t, 0.f};
    if (a.top == 1) {
        // The first of the largest of each wavefront, then of the block.
        if (threadIdx.x == 0) sh.top[0] = 0;
        __syncthreads();
        if (most == m && m > -INFINITY) {
            uint32_t id = 0;
#pragma unroll
            for (uint32_t i = EACH; i-- > 0;) id = x[i] == m ? id_of(i) : id;
            __hip_atomic_fetch_max(&sh.top[0], key_of(m, id), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
    } else if (a.top)
        pick<THREADS>(x, most, id_of, a.top, sh);
    __syncthreads();
    if (a.slices > 1 && wave > 0) return;
    float4 all = join_lanes(lane < WAVES ? sh.state[lane] : float4{-INFINITY, 0.f, 0.f, 0.f}, WAVES, scale2);
    if (a.slices > 1) {
        if (lane == 0) a.state[(uint64_t)r * a.slices + slice] = all;
        if (lane < a.top) a.best[((uint64_t)r * a.top + lane) * a.slices + slice] = sh.top[lane];
        return;
    }
    all = float4{__shfl(all.x, 0, 64), __shfl(all.y, 0, 64), __shfl(all.z, 0, 64), 0.f};
    const uint32_t token = threadIdx.x < a.per_row ? a.tokens[(uint64_t)r * a.per_row + threadIdx.x] : NONE;
    answer<BF16, THREADS>(a, row, r, all, token, token < a.vocab ? logit_at<BF16>(row, token) : 0.f, sh);
}

// A block joins the slices of a row, N keys to a thread at a time. One round after the other of a trip to memory and the
// selection: 5.3 to 5.6 us for 1 to 512 rows.
template <bool BF16, uint32_t N>
__global__ void __launch_bounds__(256) logprobs_join_kernel(Args a) {
    constexpr uint32_t THREADS = 256, WAVES = THREADS / 64;
    __shared__ Shared<THREADS> sh;
    __shared__ uint64_t kept[MOST_TOP];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = blockIdx.x;
    const void* row = row_of<BF16>(a, r);
    const float4* state = a.state + (uint64_t)r * a.slices;
    const uint64_t* best = a.best + (uint64_t)r * a.slices * a.top;
    const uint32_t keys = a.slices * a.top, token = threadIdx.x < a.per_row ? a.tokens[(uint64_t)r * a.per_row + threadIdx.x] : NONE;
    const float scale2 = a.scale * LOG2E;
    float4 all = {-INFINITY, 0.f, 0.f, 0.f};
    for (uint32_t s = threadIdx.x; s < a.slices; s += THREADS) all = join(all, state[s], scale2);
    const float given = token < a.vocab ? logit_at<BF16>(row, token) : 0.f;
    if (keys <= RANKED) {
        if (threadIdx.x < keys) sh.key[threadIdx.x] = best[threadIdx.x];
        if (threadIdx.x < MOST_TOP) sh.top[threadIdx.x] = 0;
        if (keys) rank<THREADS>(keys, a.top, sh);
    }
    // N keys to a thread at a time, the best so far among them. They lie by their place among a slice's, so that the wavefronts
    // that give a floor have high ones.
    for (uint32_t done = keys <= RANKED ? keys : 0, held = 0; done < keys; held = a.top) {
        const uint32_t some = min(keys - done, THREADS * N - held);
        float x[N], most = -INFINITY;
        uint32_t ids[N];
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) {
            const uint32_t at = i * THREADS + threadIdx.x;
            uint64_t k = 0;
            if (at < held)
                k = kept[at];
            else if (at - held < some)
                k = best[done + at - held];
            x[i] = k ? logit_of(k) : -INFINITY;
            ids[i] = ~(uint32_t)k;
        }
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) most = fmaxf(most, x[i]);
        pick<THREADS>(x, most, [&](uint32_t i) { return chosen(ids, i); }, a.top, sh);
        if (threadIdx.x < a.top) kept[threadIdx.x] = sh.top[threadIdx.x];
        done += some;
        if (done < keys) __syncthreads();
    }
    all = join_lanes(all, 64, scale2);
    if (lane == 0) sh.state[wave] = all;
    __syncthreads();
    all = join_lanes(lane < WAVES ? sh.state[lane] : float4{-INFINITY, 0.f, 0.f, 0.f}, WAVES, scale2);
    all = float4{__shfl(all.x, 0, 64), __shfl(all.y, 0, 64), __shfl(all.z, 0, 64), 0.f};
    answer<BF16, THREADS>(a, row, r, all, token, given, sh);
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

using Kernel = void (*)(Args);
template <bool BF16>
Kernel kernel_as(const LogprobsCut& s) {
    if (s.threads == 256) return s.each == 16 ? logprobs_slices_kernel<BF16, 256, 16> : logprobs_slices_kernel<BF16, 256, 32>;
    if (s.threads == 512) return s.each == 16 ? logprobs_slices_kernel<BF16, 512, 16> : logprobs_slices_kernel<BF16, 512, 32>;
    return logprobs_slices_kernel<BF16, 1024, 32>;
}
Kernel kernel_of(const LogprobsCut& s, bool bf16) { return bf16 ? kernel_as<true>(s) : kernel_as<false>(s); }

}  // namespace

// The workspace: the counters' part, which is left alone, the slices' states, then their top keys.
extern "C" uint64_t x0ne_logprobs_work_bytes(const x0ne_logprobs* d) {
    if (check_shape(d) != X0NE_OK) return 0;
    const uint64_t slices = logprobs_most_slices(d->rows, d->vocab, d->top, d->bf16);
    return WORK_COUNTER_BYTES + slices * (sizeof(float4) + 8ull * d->top);
}

extern "C" x0ne_status x0ne_gpu_logprobs(x0ne_gpu* g, const x0ne_logprobs* d) {
    X0NE_TRY(check_shape(d));
    const uint64_t each = d->bf16 ? 2 : 4;
    if (!d->logits || d->logits % each || d->stride < d->vocab || d->stride >= (1ull << 32))
        return bad("logits (aligned to one), and a stride of at least a row's logits and below 2^32, are required");
    if (!(d->scale >= 0x1p-100f && d->scale <= 0x1p100f)) return bad("a scale from 2^-100 to 2^100 is required");
    if (d->per_row && (!d->tokens || !d->token_lp || d->tokens % 4 || d->token_lp % 4))
        return bad("given tokens need tokens and token_lp (4-byte aligned)");
    if (d->top && (!d->top_ids || !d->top_lp || d->top_ids % 4 || d->top_lp % 4)) return bad("top alternatives need top_ids and top_lp (4-byte aligned)");
    if (d->entropy % 4) return bad("entropy is 4-byte aligned");
    if (!d->work || d->work % 256 || d->work_bytes < x0ne_logprobs_work_bytes(d))
        return bad("a workspace of x0ne_logprobs_work_bytes (256-byte aligned) is required");
    if (!g) return fail(X0NE_ERR_GPU, "no device");
    if (d->rows == 0) return X0NE_OK;
    const OnDevice on(g->device);
    const LogprobsCut cut = logprobs_cut(d->rows, d->vocab, d->top, d->bf16);
    const uint32_t slices = cut.count, threads = cut.threads;
    for (uint64_t first = 0; first < d->rows; first += cut.at_once) {
        const uint32_t rows = (uint32_t)std::min<uint64_t>(d->rows - first, cut.at_once);
        Args a = {};
        a.logits = (const uint8_t*)d->logits + first * d->stride * each;
        a.stride = d->stride;
        a.tokens = (const uint32_t*)d->tokens + first * d->per_row;
        a.token_lp = (float*)d->token_lp + first * d->per_row;
        a.entropy = d->entropy ? (float*)d->entropy + first : nullptr;
        a.top_ids = (uint32_t*)d->top_ids + first * d->top;
        a.top_lp = (float*)d->top_lp + first * d->top;
        a.state = (float4*)(d->work + WORK_COUNTER_BYTES);
        a.best = (uint64_t*)(a.state + (uint64_t)rows * slices);
        a.vocab = d->vocab;
        a.slices = slices;
        a.length = cut.length;
        a.per_row = d->per_row;
        a.top = d->top;
        a.scale = d->scale;
        g->counts.launches++;
        const auto kernel = kernel_of(cut, d->bf16);
        hipLaunchKernelGGL(kernel, dim3(rows * slices), dim3(threads), 0, g->stream, a);
        if (slices > 1) {
            g->counts.launches++;
            const auto joins = cut.join == 16 ? d->bf16 ? logprobs_join_kernel<true, 16> : logprobs_join_kernel<false, 16>
                                              : d->bf16 ? logprobs_join_kernel<true, 4> : logprobs_join_kernel<false, 4>;
            hipLaunchKernelGGL(joins, dim3(rows), dim3(256), 0, g->stream, a);
        }
        X0NE_HIP(hipGetLastError(), "logprobs");
    }
    return X0NE_OK;
}
