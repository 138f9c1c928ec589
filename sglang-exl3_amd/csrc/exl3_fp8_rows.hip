// Row operators that produce the input of the block-scaled FP8 product
// (exl3_fp8_linear.hip): the quantization of 16-bit rows, of a root-mean-square
// norm with the residual's addition, and of a SwiGLU.  All three are bound by
// memory: each input is read once and each output written once.
#include "exl3_fp8.h"

namespace exl3 {
namespace {

constexpr int Q_THREADS = 256;
constexpr int Q_GROUPS = Q_THREADS / 16;  // groups a workgroup handles at once

// Group `id` of all rows: its row and column group.  magic and shift divide by the
// groups of a row (fast_div).
struct FastDiv {
    uint32_t d, magic, shift;
};
FastDiv fast_div(uint32_t d) {
    uint32_t s = 0;
    while ((1u << s) < d) ++s;
    return {d, (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << s) - d)) / d + 1), s};
}
__device__ __forceinline__ uint32_t divide(uint32_t v, const FastDiv& f) {  // v < 2^31
    return (__umulhi(v, f.magic) + v) >> f.shift;
}

// 16 lanes a group, one 16-byte load and one 8-byte store a lane; q and the scales are
// in the order of the groups.  2049 rows of 14336: 89 MB in 14.4 us, 6.2 TB/s.
template <bool BF16>
__global__ __launch_bounds__(Q_THREADS) void fp8_quant_kernel(const uint16_t* x, long long stride, uint8_t* q,
                                                              float* scale, uint32_t count, FastDiv div, int cols) {
    const uint32_t id = blockIdx.x * Q_GROUPS + (threadIdx.x >> 4);
    if (id >= count) return;
    const uint32_t row = divide(id, div), c0 = (id - row * div.d) * FP8_GROUP + (threadIdx.x & 15) * 8;
    const bool in = c0 < (uint32_t)cols;
    u32x4_t v = {0, 0, 0, 0};
    if (in) v = *reinterpret_cast<const EXL3_GLOBAL u32x4_t*>(gptr(x) + row * stride + c0);
    float s;
    const u32x2_t b = quantize8<BF16>(v, s);
    if (in) *reinterpret_cast<EXL3_GLOBAL u32x2_t*>(gptr(q) + (size_t)row * cols + c0) = b;
    if ((threadIdx.x & 15) == 0) gptr(scale)[id] = s;
}

struct NormArgs {
    const uint16_t *x, *residual, *weight;
    long long xs, rs;  // row strides
    uint16_t *sum, *rows;
    uint8_t* q;
    float* scale;
    float eps;
    int cols;
};

// v = h / sqrt(mean(h^2) + eps) * weight.  One row per workgroup; a thread holds CH
// chunks of 8 columns, blockDim apart, in fp32, so the row is read once, and its
// weights on the way with it.  The norm is of the fp32 sum, not of the rounded one
// that is stored: one rounding fewer.  2048 rows of 4096 with residual and both 16-bit
// outputs: 76 MB in 11.9 us, 6.4 TB/s; one row takes 2.7 us, 0.6 above an empty kernel.
template <bool BF16, int CH>
__global__ __launch_bounds__(1024) void fp8_norm_kernel(NormArgs p) {
    __shared__ float part[16];
    const int tid = threadIdx.x, wave = tid >> 6, waves = blockDim.x >> 6;
    const size_t row = blockIdx.x;
    float h[CH][8];
    float ss = 0.f;
    u32x4_t a[CH], b[CH], w[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * blockDim.x + tid) * 8;
        a[c] = b[c] = w[c] = u32x4_t{0, 0, 0, 0};
        if (col < p.cols) {
            a[c] = *reinterpret_cast<const EXL3_GLOBAL u32x4_t*>(gptr(p.x) + row * p.xs + col);
            if (p.residual) b[c] = *reinterpret_cast<const EXL3_GLOBAL u32x4_t*>(gptr(p.residual) + row * p.rs + col);
            w[c] = *reinterpret_cast<const EXL3_GLOBAL u32x4_t*>(gptr(p.weight) + col);
        }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * blockDim.x + tid) * 8;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = f2_of<BF16>(a[c][j]);
            const float2 g = f2_of<BF16>(b[c][j]);
            h[c][2 * j] = p.residual ? f.x + g.x : f.x;  // -0 stays -0 without a residual
            h[c][2 * j + 1] = p.residual ? f.y + g.y : f.y;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(h[c][j], h[c][j], ss);
        if (p.sum && col < p.cols) {
            u32x4_t o;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = bits_of<BF16>(h[c][2 * j], h[c][2 * j + 1]);
            *reinterpret_cast<EXL3_GLOBAL u32x4_t*>(gptr(p.sum) + row * p.cols + col) = o;
        }
    }
    ss += lane_xor<32>(ss);
    ss += lane_xor<16>(ss);
    ss += lane_xor<8>(ss);
    ss += lane_xor<4>(ss);
    ss += lane_xor<2>(ss);
    ss += lane_xor<1>(ss);
    if (waves > 1) {
        if ((tid & 63) == 0) part[wave] = ss;
        __syncthreads();
        ss = (tid & 15) < waves ? part[tid & 15] : 0.f;
        ss += lane_xor<8>(ss);
        ss += lane_xor<4>(ss);
        ss += lane_xor<2>(ss);
        ss += lane_xor<1>(ss);
    }
    const float inv = 1.0f / sqrtf(ss / (float)p.cols + p.eps);
    const int groups = fp8_groups(p.cols);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * blockDim.x + tid) * 8;
        float y[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 g = f2_of<BF16>(w[c][j]);
            y[2 * j] = h[c][2 * j] * inv * g.x;
            y[2 * j + 1] = h[c][2 * j + 1] * inv * g.y;
        }
        if (col >= p.cols)  // a row whose norm is not finite: no NaN into the last group
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = 0.f;
        float s;
        const u32x2_t b = quantize8_f32(y, s);
        if (col >= p.cols) continue;
        *reinterpret_cast<EXL3_GLOBAL u32x2_t*>(gptr(p.q) + row * p.cols + col) = b;
        if ((tid & 15) == 0) gptr(p.scale)[row * groups + (col >> 7)] = s;
        if (p.rows) {
            u32x4_t o;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = bits_of<BF16>(y[2 * j], y[2 * j + 1]);
            *reinterpret_cast<EXL3_GLOBAL u32x4_t*>(gptr(p.rows) + row * p.cols + col) = o;
        }
    }
}

// silu(g) = g / (1 + 2^(-g log2 e)).  The product with log2 e is kept to twice the
// precision: its rounding alone would be a relative error of 1e-6 at g = -20.
// The reciprocal is within one ulp.
__device__ __forceinline__ float silu_exact(float g) {
    const float t = g * -1.44269504088896341f;
    const float lo = fmaf(g, -1.44269504088896341f, -t) + g * -1.92596299e-8f;
    const float e = __builtin_amdgcn_exp2f(t);
    // at the ends lo is not finite, and does not count
    return g * __builtin_amdgcn_rcpf(1.0f + (e > 0.0f && e < 1e38f ? fmaf(e, lo * 0.693147181f, e) : e));
}

// Laid out like fp8_quant_kernel.  2048 rows of 14336: 148 MB in 25 us, 5.9 TB/s (with a
// division in place of the reciprocal, 32.2: bound by its instructions).
template <bool BF16>
__global__ __launch_bounds__(Q_THREADS) void fp8_swiglu_kernel(const uint16_t* x, long long stride, float limit,
                                                               uint8_t* q, float* scale, uint32_t count, FastDiv div,
                                                               int cols) {
    const uint32_t id = blockIdx.x * Q_GROUPS + (threadIdx.x >> 4);
    if (id >= count) return;
    const uint32_t row = divide(id, div), c0 = (id - row * div.d) * FP8_GROUP + (threadIdx.x & 15) * 8;
    const bool in = c0 < (uint32_t)cols;
    u32x4_t a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
    if (in) {
        const EXL3_GLOBAL uint16_t* r = gptr(x) + row * stride + c0;
        a = *reinterpret_cast<const EXL3_GLOBAL u32x4_t*>(r);
        b = *reinterpret_cast<const EXL3_GLOBAL u32x4_t*>(r + cols);
    }
    float y[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 f = f2_of<BF16>(a[j]), u = f2_of<BF16>(b[j]);
        float g[2] = {f.x, f.y}, v[2] = {u.x, u.y};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            // comparisons that a NaN fails, so that it stays one
            g[e] = g[e] > limit ? limit : g[e];
            v[e] = v[e] > limit ? limit : (v[e] < -limit ? -limit : v[e]);
            y[2 * j + e] = silu_exact(g[e]) * v[e];
        }
    }
    float s;
    const u32x2_t o = quantize8_f32(y, s);
    if (in) *reinterpret_cast<EXL3_GLOBAL u32x2_t*>(gptr(q) + (size_t)row * cols + c0) = o;
    if ((threadIdx.x & 15) == 0) gptr(scale)[id] = s;
}

// What every row operator asks of its rows: 16-byte loads of 8 numbers.
bool rows_ok(const void* x, long long stride, long long width) {
    return aligned(x, 16) && stride >= width && stride % 8 == 0;
}

}  // namespace

int fp8_quant_rows(const void* x, bool bf16, long long stride, uint8_t* q, float* scale, int rows, int cols,
                   hipStream_t st) {
    const uint32_t count = (uint32_t)rows * fp8_groups(cols), grid = (count + Q_GROUPS - 1) / Q_GROUPS;
    const FastDiv div = fast_div(fp8_groups(cols));
    const auto* p = static_cast<const uint16_t*>(x);
    if (bf16) fp8_quant_kernel<true><<<grid, Q_THREADS, 0, st>>>(p, stride, q, scale, count, div, cols);
    else fp8_quant_kernel<false><<<grid, Q_THREADS, 0, st>>>(p, stride, q, scale, count, div, cols);
    return launch_status("exl3_fp8_quant_rows launch");
}

}  // namespace exl3

using namespace exl3;

#define EXL3_FP8_ROWS(NAME)                                                                                        \
    clear_error();                                                                                                 \
    EXL3_REQUIRE(dtype == EXL3_DTYPE_F16 || dtype == EXL3_DTYPE_BF16, NAME ": dtype=%d (0 fp16, 1 bf16)", dtype);  \
    EXL3_REQUIRE(rows >= 0 && cols > 0 && cols % 16 == 0, NAME ": rows=%d cols=%d (cols must be a positive "       \
                 "multiple of 16)", rows, cols);                                                                   \
    EXL3_REQUIRE(cols <= FP8_MOST && (long long)rows * fp8_groups(cols) <= 0x7fffffffLL, NAME ": %d x %d is too large", rows, cols);   \
    if (rows == 0) return EXL3_OK;                                                                                 \
    EXL3_REQUIRE(x && q && scale, NAME ": null pointer");                                                          \
    EXL3_REQUIRE(aligned(q, 8) && aligned(scale, 4), NAME ": misaligned pointer")

extern "C" int exl3_fp8_quant_rows(const void* x, long long x_stride, uint8_t* q, float* scale, int dtype, int rows,
                                   int cols, void* stream) {
    EXL3_FP8_ROWS("exl3_fp8_quant_rows");
    EXL3_REQUIRE(rows_ok(x, x_stride, cols), "exl3_fp8_quant_rows: x must be 16-byte aligned, its row stride a "
                 "multiple of 8 and at least %d (got %lld)", cols, x_stride);
    return fp8_quant_rows(x, dtype == EXL3_DTYPE_BF16, x_stride, q, scale, rows, cols, as_stream(stream));
}

extern "C" int exl3_fp8_norm_quant(const void* x, long long x_stride, const void* residual, long long residual_stride,
                                   const void* weight, float eps, void* sum, void* rows_out, uint8_t* q, float* scale,
                                   int dtype, int rows, int cols, void* stream) {
    EXL3_FP8_ROWS("exl3_fp8_norm_quant");
    EXL3_REQUIRE(weight && (!sum || residual), "exl3_fp8_norm_quant: null pointer");
    EXL3_REQUIRE(cols <= 32768, "exl3_fp8_norm_quant: cols=%d above 32768", cols);
    EXL3_REQUIRE(eps >= 0.0f, "exl3_fp8_norm_quant: eps=%g is negative or NaN", eps);
    EXL3_REQUIRE(rows_ok(x, x_stride, cols) && (!residual || rows_ok(residual, residual_stride, cols)),
                 "exl3_fp8_norm_quant: x and residual must be 16-byte aligned, their row strides multiples of 8 and at "
                 "least %d (got %lld, %lld)", cols, x_stride, residual_stride);
    EXL3_REQUIRE(aligned(weight, 16) && aligned(sum, 16) && aligned(rows_out, 16), "exl3_fp8_norm_quant: misaligned "
                 "pointer");
    const NormArgs a = {static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(residual),
                        static_cast<const uint16_t*>(weight), x_stride, residual_stride, static_cast<uint16_t*>(sum),
                        static_cast<uint16_t*>(rows_out), q, scale, eps, cols};
    const int chunks = (cols + 7) / 8;
    const hipStream_t st = as_stream(stream);
    const bool bf16 = dtype == EXL3_DTYPE_BF16;
#define EXL3_NORM_GO(CH)                                                              \
    {                                                                                 \
        const int threads = ((chunks + CH - 1) / CH + 63) / 64 * 64;                  \
        if (bf16) fp8_norm_kernel<true, CH><<<rows, threads, 0, st>>>(a);             \
        else fp8_norm_kernel<false, CH><<<rows, threads, 0, st>>>(a);                 \
    }
    // two chunks a thread leave half the waves to meet: 4096 rows of 7168 36.5 -> 33.5 us,
    // 2048 of 8192 22.5 -> 21.1, of 4096 12.2 -> 11.9; of 2048 7.6 -> 7.9, one row of 4096
    // 2.7 -> 2.9.  Four only where two do not reach (2048 rows of 8192: 22.6).
    if (chunks < 512 || (chunks == 512 && rows <= 1024)) EXL3_NORM_GO(1)
    else if (chunks <= 2048) EXL3_NORM_GO(2)
    else EXL3_NORM_GO(4)
#undef EXL3_NORM_GO
    return launch_status("exl3_fp8_norm_quant launch");
}

extern "C" int exl3_fp8_swiglu_quant(const void* x, long long x_stride, float limit, uint8_t* q, float* scale,
                                     int dtype, int rows, int cols, void* stream) {
    EXL3_FP8_ROWS("exl3_fp8_swiglu_quant");
    EXL3_REQUIRE(limit >= 0.0f, "exl3_fp8_swiglu_quant: limit=%g (nonnegative; 0 or inf: no clamp)", limit);
    EXL3_REQUIRE(rows_ok(x, x_stride, 2LL * cols), "exl3_fp8_swiglu_quant: x must be 16-byte aligned, its row stride a "
                 "multiple of 8 and at least %lld (got %lld)", 2LL * cols, x_stride);
    const uint32_t count = (uint32_t)rows * fp8_groups(cols), grid = (count + Q_GROUPS - 1) / Q_GROUPS;
    const FastDiv div = fast_div(fp8_groups(cols));
    const float lim = limit > 0.0f ? limit : __builtin_huge_valf();
    const auto* p = static_cast<const uint16_t*>(x);
    const hipStream_t st = as_stream(stream);
    if (dtype == EXL3_DTYPE_BF16)
        fp8_swiglu_kernel<true><<<grid, Q_THREADS, 0, st>>>(p, x_stride, lim, q, scale, count, div, cols);
    else
        fp8_swiglu_kernel<false><<<grid, Q_THREADS, 0, st>>>(p, x_stride, lim, q, scale, count, div, cols);
    return launch_status("exl3_fp8_swiglu_quant launch");
}
