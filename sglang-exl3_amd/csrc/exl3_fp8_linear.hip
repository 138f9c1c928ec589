// Matrix product of e4m3 rows and an e4m3 weight, both with fp32 scales by block:
//   y[m][n] = sum_b xs[m][b] ws[n / 128][b] sum_{k in block b} x[m][k] w[n][k] + bias[n]
// b runs over blocks of 128 columns of k.  One v_mfma_f32_16x16x128_f8f6f4 is a
// block's inner sum for 16 x 16 outputs, in fp32 and from a zero accumulator; four
// FMAs a lane then add it, times the two scales, to the fp32 result.  (The unit
// itself adds e4m3 products in groups of 16, aligned to the group's largest and cut
// 13 bits below it, then in fp32: 1.5e-5 of the result for random operands, without
// a bias, a tenth of an fp16 output's rounding.  v_mfma_f32_16x16x32_fp8_fp8 gives the
// same bits at half the rate, 2220 against 4380 TFLOP/s.)  The weight is the first operand, so that a lane's four outputs are neighbours in a row of
// y and share the row's scale.
//
// 16-bit rows are quantized first (fp8_quant_rows), into the workspace.
#include "exl3_fp8.h"

namespace exl3 {
namespace {

struct LinearArgs {
    const uint8_t *x, *w;
    const float *xs, *ws;
    const uint16_t* bias;
    uint16_t* y;
    int m, k, n, groups;
};

__device__ __forceinline__ i32x8_t two16(u32x4_t a, u32x4_t b) {
    return i32x8_t{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}
__device__ __forceinline__ float4_t mfma_e4m3(i32x8_t a, i32x8_t b) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, float4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

// 16 columns of n per wave, 16 MB rows of m, operands straight from memory.  A lane
// reads 32 bytes of its row in each block, 16 of them from each half: the order of k
// within a block is free as long as both operands share it.
template <int MB, bool BF16>
__global__ __launch_bounds__(256, 2) void fp8_small_kernel(LinearArgs p) {
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int n0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 16, m0 = blockIdx.y * (16 * MB);
    if (n0 >= p.n) return;
    const EXL3_GLOBAL uint8_t* wr = gptr(p.w) + (size_t)min(n0 + i, p.n - 1) * p.k;
    const EXL3_GLOBAL uint8_t* xr[MB];
    const EXL3_GLOBAL float* sr[MB];
    float4_t acc[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) {
        const int row = min(m0 + 16 * b + i, p.m - 1);
        xr[b] = gptr(p.x) + (size_t)row * p.k;
        sr[b] = gptr(p.xs) + (size_t)row * p.groups;
        acc[b] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    const EXL3_GLOBAL float* ws = gptr(p.ws) + (size_t)(n0 >> 7) * p.groups;
    for (int kb = 0; kb < p.groups; ++kb) {
        const int c0 = kb * 128 + 16 * g, c1 = c0 + 64;  // a row ends at a multiple of 16
        const u32x4_t z = {0, 0, 0, 0};
        const i32x8_t a = two16(c0 < p.k ? *reinterpret_cast<const EXL3_GLOBAL u32x4_t*>(wr + c0) : z,
                                c1 < p.k ? *reinterpret_cast<const EXL3_GLOBAL u32x4_t*>(wr + c1) : z);
        const float s = ws[kb];
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            const i32x8_t v = two16(c0 < p.k ? *reinterpret_cast<const EXL3_GLOBAL u32x4_t*>(xr[b] + c0) : z,
                                    c1 < p.k ? *reinterpret_cast<const EXL3_GLOBAL u32x4_t*>(xr[b] + c1) : z);
            const float4_t t = mfma_e4m3(a, v);
            const float f = s * sr[b][kb];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[b][e] = fmaf(t[e], f, acc[b][e]);
        }
    }
#pragma unroll
    for (int b = 0; b < MB; ++b) {
        const int row = m0 + 16 * b + i;
        if (row >= p.m) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int col = n0 + 4 * g + e;
            if (col >= p.n) continue;
            float v = acc[b][e];
            if (p.bias) v += f2_of<BF16>(gptr(p.bias)[col]).x;
            gptr(p.y)[(size_t)row * p.n + col] = (uint16_t)bits_of<BF16>(v, 0.f);
        }
    }
}

// Workspace of 16-bit rows, after the shared regions: e4m3 rows, then their scales.
size_t rows_bytes(int m, int k) { return ((size_t)m * k + 255) / 256 * 256; }

}  // namespace
}  // namespace exl3

using namespace exl3;

extern "C" size_t exl3_fp8_linear_workspace_size(int x_dtype, int m, int k, int n) {
    if (m <= 0 || k <= 0 || n <= 0 || k % 16) return 0;
    if (x_dtype == EXL3_DTYPE_E4M3) return 0;
    return kWsScratchOffset + rows_bytes(m, k) + (size_t)m * fp8_groups(k) * sizeof(float);
}

extern "C" int exl3_fp8_linear(const void* x, int x_dtype, const float* x_scale, const uint8_t* w,
                               const float* w_scale, const void* bias, void* y, int y_dtype, int m, int k, int n,
                               void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    EXL3_REQUIRE(m >= 0 && k > 0 && k % 16 == 0 && n > 0, "exl3_fp8_linear: m=%d k=%d n=%d (k must be a positive "
                 "multiple of 16)", m, k, n);
    const bool rows = x_dtype == EXL3_DTYPE_F16 || x_dtype == EXL3_DTYPE_BF16;
    EXL3_REQUIRE(rows || x_dtype == EXL3_DTYPE_E4M3, "exl3_fp8_linear: x dtype=%d (0 fp16, 1 bf16, 3 e4m3)", x_dtype);
    EXL3_REQUIRE(y_dtype == EXL3_DTYPE_F16 || y_dtype == EXL3_DTYPE_BF16, "exl3_fp8_linear: y dtype=%d (0 fp16, "
                 "1 bf16)", y_dtype);
    const int groups = fp8_groups(k);
    EXL3_REQUIRE((long long)m * groups <= 0x7fffffffLL, "exl3_fp8_linear: %d x %d rows are too many", m, k);
    if (m == 0) return EXL3_OK;
    EXL3_REQUIRE(x && w && w_scale && y && (rows || x_scale), "exl3_fp8_linear: null pointer");
    EXL3_REQUIRE(aligned(x, 16) && aligned(w, 16) && aligned(x_scale, 4) && aligned(w_scale, 4) && aligned(bias, 2) &&
                 aligned(y, 2), "exl3_fp8_linear: misaligned pointer (x and w: 16 bytes)");
    const hipStream_t st = as_stream(stream);
    LinearArgs a = {static_cast<const uint8_t*>(x), w, x_scale, w_scale, static_cast<const uint16_t*>(bias),
                    static_cast<uint16_t*>(y), m, k, n, groups};
    if (rows) {
        const size_t need = exl3_fp8_linear_workspace_size(x_dtype, m, k, n);
        EXL3_REQUIRE_CODE(workspace && workspace_bytes >= need, EXL3_ERR_WORKSPACE, "exl3_fp8_linear: workspace of "
                          "%zu bytes, needs %zu", workspace_bytes, need);
        EXL3_REQUIRE(aligned(workspace, 256), "exl3_fp8_linear: misaligned workspace");
        uint8_t* q = static_cast<uint8_t*>(workspace) + kWsScratchOffset;
        float* s = reinterpret_cast<float*>(q + rows_bytes(m, k));
        const int rc = fp8_quant_rows(x, x_dtype == EXL3_DTYPE_BF16, k, q, s, m, k, st);
        if (rc) return rc;
        a.x = q;
        a.xs = s;
    }
    const bool bf16 = y_dtype == EXL3_DTYPE_BF16;
    const int mb = m <= 16 ? 1 : m <= 32 ? 2 : 4;
    const dim3 grid((n + 63) / 64, (m + 16 * mb - 1) / (16 * mb));
    EXL3_REQUIRE(grid.y <= 65535, "exl3_fp8_linear: m=%d is too large", m);
#define EXL3_FP8_SMALL(MB)                                                     \
    if (mb == MB) {                                                            \
        if (bf16) fp8_small_kernel<MB, true><<<grid, 256, 0, st>>>(a);         \
        else fp8_small_kernel<MB, false><<<grid, 256, 0, st>>>(a);             \
    }
    EXL3_FP8_SMALL(1)
    EXL3_FP8_SMALL(2)
    EXL3_FP8_SMALL(4)
#undef EXL3_FP8_SMALL
    return launch_status("exl3_fp8_linear launch");
}
