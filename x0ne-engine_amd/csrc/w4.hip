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

// A wavefront takes a tile. The four lanes of a row hold 8 columns of each 32: a group's largest magnitude is theirs.
template <int G>
__global__ void __launch_bounds__(256) w4_quantise_kernel(const bf16_t* __restrict__ from, Form f) {
    const uint32_t lane = threadIdx.x & 63, t = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= f.tiles) return;
    const uint32_t row = blockIdx.y * TILE_ROWS + (lane & 15), col = t * TILE_COLS + 8 * (lane >> 4);
    u32x4 w[4];
    uint32_t top[4];  // magnitudes as bits: infinities and NaN are above all others
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        w[s] = u32x4{0, 0, 0, 0};
        if (row < f.rows && col + 32 * s < f.cols) w[s] = *reinterpret_cast<const u32x4*>(from + (size_t)row * f.cols + col + 32 * s);
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

template <int G>
__global__ void __launch_bounds__(256) w4_read_kernel(Form f, bf16_t* __restrict__ to) {
    const uint32_t lane = threadIdx.x & 63, t = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= f.tiles) return;
    const uint32_t row = blockIdx.y * TILE_ROWS + (lane & 15), col = t * TILE_COLS + 8 * (lane >> 4);
    if (row >= f.rows) return;
    const size_t tile = (size_t)blockIdx.y * f.tiles + t;
    const u32x4 c = *reinterpret_cast<const u32x4*>(f.codes + tile * TILE_BYTES + 16 * lane);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        if (col + 32 * s >= f.cols) break;
        const float scale = scale_of<G>(f.scales, tile, lane & 15, s);
        const u32x4 v = __builtin_bit_cast(u32x4, decode8(c[s]));
        u32x4 out;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            out[i] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)(bf_lo(v[i]) * scale), (__bf16)(bf_hi(v[i]) * scale)});
        *reinterpret_cast<u32x4*>(to + (size_t)row * f.cols + col + 32 * s) = out;
    }
}

// Y = X W^T of 16 rows of X and 16 of W to a block (SwiGLU: 16 gate rows and the 16 up rows that go with them), the
// tiles of a panel to its wavefronts in turn. X is the A operand, W the B operand: a lane's four sums are four tokens of
// one row of W, whose scale of a group is one value.
template <int G, int OUT>
__global__ void __launch_bounds__(256) w4_gemv_kernel(Form f, const bf16_t* __restrict__ x, uint32_t n, void* __restrict__ y) {
    constexpr int PANELS = OUT == X0NE_W4_SWIGLU ? 2 : 1;
    __shared__ f32x4 part[4][PANELS][64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t token = blockIdx.y * 16 + (lane & 15), panels = (f.rows + 15) / 16;
    f32x4 sum[PANELS] = {};
    for (uint32_t t = wave; t < f.tiles; t += 4) {
        bf16x8 a[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const uint32_t col = t * TILE_COLS + 32 * s + 8 * (lane >> 4);
            u32x4 v = {0, 0, 0, 0};
            if (token < n && col < f.cols) v = *reinterpret_cast<const u32x4*>(x + (size_t)token * f.cols + col);
            a[s] = __builtin_bit_cast(bf16x8, v);
        }
#pragma unroll
        for (int p = 0; p < PANELS; ++p) {
            const size_t tile = (size_t)(blockIdx.x + p * (panels / 2)) * f.tiles + t;
            const u32x4 c = *reinterpret_cast<const u32x4*>(f.codes + tile * TILE_BYTES + 16 * lane);
            f32x4 acc = {};
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[s], decode8(c[s]), acc, 0, 0, 0);
                if ((s + 1) % (G / 32) == 0) {
                    const float scale = scale_of<G>(f.scales, tile, lane & 15, s);
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[p][i] = fmaf(acc[i], scale, sum[p][i]);
                    acc = f32x4{};
                }
            }
        }
    }
#pragma unroll
    for (int p = 0; p < PANELS; ++p) part[wave][p][lane] = sum[p];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int p = 0; p < PANELS; ++p)
#pragma unroll
        for (int v = 1; v < 4; ++v) sum[p] += part[v][p][lane];
    const uint32_t row = blockIdx.x * 16 + (lane & 15), out_rows = f.rows / PANELS;
    if (row >= out_rows) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t to = blockIdx.y * 16 + 4 * (lane >> 4) + i;
        if (to >= n) break;
        const size_t at = (size_t)to * out_rows + row;
        if (OUT == X0NE_W4_F32)
            static_cast<float*>(y)[at] = sum[0][i];
        else if (OUT == X0NE_W4_BF16)
            static_cast<bf16_t*>(y)[at] = f2bf(sum[0][i]);
        else
            static_cast<bf16_t*>(y)[at] = f2bf(sum[0][i] / (1.0f + expf(-sum[0][i])) * sum[PANELS - 1][i]);
    }
}

// ---- host ----

x0ne_status bad(const char* what, const std::string& why) { return fail(X0NE_ERR_FORMAT, std::string(what) + ": " + why); }

constexpr uint32_t MOST = 1u << 24;

x0ne_status check_shape(const char* what, const x0ne_w4* w) {
    if (!w) return bad(what, "no matrix");
    if (w->rows == 0 || w->rows > MOST || w->cols == 0 || w->cols > MOST || w->cols % 8 ||
        (w->group != 32 && w->group != 64 && w->group != 128))
        return bad(what, std::to_string(w->rows) + " rows of " + std::to_string(w->cols) + " columns in groups of " +
                             std::to_string(w->group) + " (1 to 2^24 rows and columns, columns a multiple of 8, groups of 32, 64 or 128)");
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
    const auto kernel = w->group == 32 ? w4_quantise_kernel<32> : w->group == 64 ? w4_quantise_kernel<64> : w4_quantise_kernel<128>;
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
    const auto kernel = w->group == 32 ? w4_read_kernel<32> : w->group == 64 ? w4_read_kernel<64> : w4_read_kernel<128>;
    return by_panels(g, what, w, [&](dim3 grid, const Form& f, size_t at) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, g->stream, f, (bf16_t*)to + at);
    });
}

template <int OUT>
static void launch_gemv(const x0ne_gpu* g, const x0ne_w4* w, const bf16_t* x, uint32_t n, void* y) {
    const auto kernel = w->group == 32 ? w4_gemv_kernel<32, OUT> : w->group == 64 ? w4_gemv_kernel<64, OUT> : w4_gemv_kernel<128, OUT>;
    const uint32_t panels = (w->rows + 15) / 16;
    hipLaunchKernelGGL(kernel, dim3(OUT == X0NE_W4_SWIGLU ? panels / 2 : panels, (n + 15) / 16), dim3(256), 0, g->stream, form_of(w), x,
                       n, y);
}

extern "C" x0ne_status x0ne_gpu_w4_gemv(x0ne_gpu* g, const x0ne_w4* w, uint64_t x, uint64_t n, uint64_t y, uint32_t out) {
    const char* what = "w4 gemv";
    X0NE_TRY(check_matrix(what, w));
    if (out > X0NE_W4_SWIGLU) return bad(what, "no output " + std::to_string(out));
    if (out == X0NE_W4_SWIGLU && w->rows % 32) return bad(what, std::to_string(w->rows) + " rows of gate and up (a multiple of 32)");
    if (n > 65535 * 16) return bad(what, std::to_string(n) + " rows of x (up to 65535 x 16)");
    if (n * w->cols * 2 >= (1ull << 32) - 16) return bad(what, std::to_string(n) + " rows of " + std::to_string(w->cols) + " columns of x (below 4 GiB)");
    if (!x || !y || x % 16 || y % 4) return bad(what, "x (16-byte aligned) and y (4-byte aligned) are required");
    if (!g) return fail(X0NE_ERR_GPU, "no device");
    if (n == 0) return X0NE_OK;
    const OnDevice on(g->device);
    g->counts.launches++;
    const auto launch = out == X0NE_W4_BF16 ? launch_gemv<X0NE_W4_BF16> : out == X0NE_W4_F32 ? launch_gemv<X0NE_W4_F32> : launch_gemv<X0NE_W4_SWIGLU>;
    launch(g, w, (const bf16_t*)x, (uint32_t)n, (void*)y);
    X0NE_HIP(hipGetLastError(), what);
    return X0NE_OK;
}
