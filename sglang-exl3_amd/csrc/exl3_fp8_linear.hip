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
#include <type_traits>

#include "exl3_fp8.h"

namespace exl3 {
namespace {

struct LinearArgs {
    const uint8_t *x, *w;
    const float *xs, *ws;
    const uint16_t* bias;
    uint16_t* y;
    int m, k, n, groups;
    int vec;  // rows of y are 8-byte aligned
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

// Tiles for many rows.  A workgroup of 8 waves, 4 along n and 2 along m, owns 256
// columns of y and 32 FM rows.  Rows of x and of the weight go through LDS, copied
// there by the load unit (16 bytes a lane) one block of 128 columns ahead.
// LDS row r holds its 16-byte chunk c at slot c ^ (r & 7), by choice of the source
// address; a fragment's lanes read chunks g and g + 4 of rows i = lane & 15,
// g = lane >> 4, without bank conflicts (256 bytes a cycle; 2g and 2g + 1 at these
// slots, or the slots of a 64-column step, conflict and run at half of it).
constexpr int TILE_N = 256;
constexpr int FP8_MAX_K = 1 << 22;  // 256 rows within 31 bits

template <int FM>
constexpr int tile_m = 32 * FM;
template <int FM>  // rows of x, of the weight, the rows' scales, the weight's, and room for copies that nothing reads
constexpr int tile_buf = (tile_m<FM> + TILE_N) * 128 + (tile_m<FM> + 128) * 4;

// Buffer descriptor of `bytes` bytes at p.  A load at an offset past them (OUT) gives
// zeros, as long as the scalar part of its address lies inside.
typedef int i32x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4_t buffer_of(const void* p, uint32_t bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    return i32x4_t{__builtin_amdgcn_readfirstlane((int)a), __builtin_amdgcn_readfirstlane((int)(a >> 32)),
                   __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000};
}
constexpr uint32_t OUT = 0x80000000u;  // an offset past every buffer here

// 16 (or 4) bytes a lane from buffer offset off + step to LDS byte lds + 16 (4) lane.  The caller waits.
__device__ __forceinline__ void copy16(i32x4_t rsrc, uint32_t off, uint32_t step, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(off), "s"(rsrc),
                 "s"(step), "s"(lds)
                 : "memory", "m0");
}
__device__ __forceinline__ void copy4(i32x4_t rsrc, uint32_t off, uint32_t step, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dword %0, %1, %2 offen lds" ::"v"(off), "s"(rsrc),
                 "s"(step), "s"(lds)
                 : "memory", "m0");
}
template <int FM, bool BF16>
__global__ __launch_bounds__(512, 2) void fp8_tile_kernel(LinearArgs p, int tiles_m, int tiles) {
    static_assert(FM % 2 == 0, "fragments alternate between two register sets");
    constexpr int MT = tile_m<FM>, BUF = tile_buf<FM>, XC = MT / 64, WC = TILE_N / 64;  // copies of a wave in a step
    constexpr int WB = MT * 128, SB = WB + TILE_N * 128;                                // weight, scales in a buffer
    extern __shared__ __align__(16) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave & 3, wm = wave >> 2;
    // each XCD (workgroup % 8) gets a run of neighbouring tiles, rows fastest
    const int per = tiles >> 3, rest = tiles & 7, xcd = blockIdx.x & 7;
    const int id = xcd * per + min(xcd, rest) + (blockIdx.x >> 3);
    const int tn = __builtin_amdgcn_readfirstlane(id / tiles_m);
    const int tm = __builtin_amdgcn_readfirstlane(id - tn * tiles_m);
    const int m0 = tm * MT, n0 = tn * TILE_N;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;

    // rows past the end repeat the last one (never stored); columns past it read as zeros
    const int mr = min(MT, p.m - m0), nr = min(TILE_N, p.n - n0);
    const i32x4_t xbuf = buffer_of(p.x + (size_t)m0 * p.k, (uint32_t)mr * p.k);
    const i32x4_t wbuf = buffer_of(p.w + (size_t)n0 * p.k, (uint32_t)nr * p.k);
    const int chunk = 16 * ((lane & 7) ^ (lane >> 3)), lr = 8 * wave + (lane >> 3);
    uint32_t xoff[XC], woff[WC];
#pragma unroll
    for (int j = 0; j < XC; ++j) xoff[j] = (uint32_t)min(64 * j + lr, mr - 1) * p.k + chunk;
#pragma unroll
    for (int j = 0; j < WC; ++j) woff[j] = (uint32_t)min(64 * j + lr, nr - 1) * p.k + chunk;
    // scales: waves 0 .. MT / 64 - 1 those of 64 rows each, wave 7 the weight's (the others nothing that is read)
    const bool xs = wave < MT / 64;
    const int nb = (nr + 127) >> 7;
    const i32x4_t sbuf = xs ? buffer_of(p.xs + (size_t)m0 * p.groups, (uint32_t)mr * p.groups * 4)
                            : buffer_of(p.ws + (size_t)(n0 >> 7) * p.groups, (uint32_t)nb * p.groups * 4);
    const uint32_t soff = (uint32_t)(xs ? min(64 * wave + lane, mr - 1) : min(lane & 1, nb - 1)) * p.groups * 4;
    const uint32_t sdst = SB + (xs ? 256 * wave : 4 * MT + (wave == 7 ? 0 : 256));
    // copy j of step s: the weight's, then the rows', then the scales; `to` is the step's buffer
    auto copy = [&](int s, uint32_t to, int j) {
        int left = p.k - s * 128;  // columns
        asm("" : "+s"(left));      // the offsets below are made where they are used, not kept
        const uint32_t at = left > 0 ? s * 128 : 0;  // stays inside the buffer
        if (j < WC) copy16(wbuf, chunk < left ? woff[j] : OUT, at, lds0 + to + WB + (64 * j + 8 * wave) * 128);
        else if (j < WC + XC)
            copy16(xbuf, chunk < left ? xoff[j - WC] : OUT, at, lds0 + to + (64 * (j - WC) + 8 * wave) * 128);
        else if (j == WC + XC) copy4(sbuf, left > 0 ? soff : OUT, at >> 5, lds0 + to + sdst);
    };
    float4_t acc[4][FM];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < FM; ++b) acc[a][b] = float4_t{0.f, 0.f, 0.f, 0.f};
    const uint32_t slot = 16 * (g ^ (i & 7));
    const uint32_t xrd = (FM * wm * 16 + i) * 128 + slot, wrd = WB + (64 * wn + i) * 128 + slot;
    const uint32_t frd = SB + (FM * wm * 16 + i) * 4, srd = SB + (MT + (wn >> 1)) * 4;
    auto half = [&](i32x8_t& d, int h, uint32_t at) {
        const u32x4_t r = *reinterpret_cast<const u32x4_t*>(smem + (at ^ (64 * h)));
#pragma unroll
        for (int e = 0; e < 4; ++e) d[4 * h + e] = (int)r[e];
    };
    auto number = [&](uint32_t at) { return *reinterpret_cast<const float*>(smem + at); };

#pragma unroll
    for (int j = 0; j <= WC + XC; ++j) copy(0, 0, j);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    // w, x and f: the step's weight fragments, two fragments of rows and their
    // scales, read one ahead; t: products of the fragment before, added (scaled by
    // c) while the next ones run, so that no instruction waits for the matrix unit
    i32x8_t w[2][4], x[2];
    float4_t t[4] = {};
    float f[2], sb[2], c = 0.f;
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int h = 0; h < 2; ++h) half(w[0][a], h, wrd + a * 2048);
#pragma unroll
    for (int h = 0; h < 2; ++h) half(x[0], h, xrd);
    f[0] = number(frd);
    sb[0] = number(srd);
#pragma unroll
    for (int j = 0; j < 4; ++j) copy(1, BUF, j);
    // Step s with buffer `buf`, the other of which the next step has.  The barrier is
    // before the last fragment's products: those cover the next step's first reads.
    // Copies are spread out: at once, they would keep the load unit, and the waves
    // that wait for it, busy for half of the step.
    auto body = [&](int s, auto slot_c) {
        constexpr int S = decltype(slot_c)::value;
        constexpr uint32_t buf = S * BUF, other = (S ^ 1) * BUF;
#pragma unroll
        for (int b = 0; b < FM; ++b) {
            if (b == FM - 1) {
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const float4_t done = t[a];
                t[a] = mfma_e4m3(w[S][a], x[b & 1]);
                __builtin_amdgcn_sched_barrier(0);
                if (b < FM - 1) {
                    if (a < 2) half(x[(b + 1) & 1], a, xrd + buf + (b + 1) * 2048);
                    if (a == 2) f[(b + 1) & 1] = number(frd + buf + (b + 1) * 64);
                    const int j = 4 + 4 * b + a;
                    if (j <= WC + XC) copy(s + 1, other, j);
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (a == 1) half(x[0], h, xrd + other);
                        half(w[S ^ 1][a], h, wrd + other + a * 2048);
                    }
                    if (a == 2) {
                        f[0] = number(frd + other);
                        sb[S ^ 1] = number(srd + other);
                    }
                    copy(s + 2, buf, a);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    acc[a][(b + FM - 1) % FM][e] = fmaf(done[e], c, acc[a][(b + FM - 1) % FM][e]);
                __builtin_amdgcn_sched_barrier(0);
            }
            c = f[b & 1] * sb[S];
        }
    };
    for (int s = 0; s < p.groups; s += 2) {  // an odd number's last step adds zeros
        body(s, std::integral_constant<int, 0>{});
        body(s + 1, std::integral_constant<int, 1>{});
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // copies past the end land before the workgroup ends
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[a][FM - 1][e] = fmaf(t[a][e], c, acc[a][FM - 1][e]);
#pragma unroll
    for (int b = 0; b < FM; ++b) {
        const int row = m0 + (FM * wm + b) * 16 + i;
        if (row >= p.m) continue;
        EXL3_GLOBAL uint16_t* yr = gptr(p.y) + (size_t)row * p.n;
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const int col = n0 + 64 * wn + 16 * a + 4 * g;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = acc[a][b][e];
                if (p.bias && col + e < p.n) v[e] += f2_of<BF16>(gptr(p.bias)[col + e]).x;
            }
            const u32x2_t o = {bits_of<BF16>(v[0], v[1]), bits_of<BF16>(v[2], v[3])};
            if (p.vec && col + 4 <= p.n) {
                *reinterpret_cast<EXL3_GLOBAL u32x2_t*>(yr + col) = o;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (col + e < p.n) yr[col + e] = (uint16_t)(o[e >> 1] >> (16 * (e & 1)));
            }
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
    EXL3_REQUIRE(k <= FP8_MAX_K, "exl3_fp8_linear: k=%d above %d", k, FP8_MAX_K);
    if (m == 0) return EXL3_OK;
    EXL3_REQUIRE(x && w && w_scale && y && (rows || x_scale), "exl3_fp8_linear: null pointer");
    EXL3_REQUIRE(aligned(x, 16) && aligned(w, 16) && aligned(x_scale, 4) && aligned(w_scale, 4) && aligned(bias, 2) &&
                 aligned(y, 2), "exl3_fp8_linear: misaligned pointer (x and w: 16 bytes)");
    const hipStream_t st = as_stream(stream);
    LinearArgs a = {static_cast<const uint8_t*>(x), w, x_scale, w_scale, static_cast<const uint16_t*>(bias),
                    static_cast<uint16_t*>(y), m, k, n, groups, n % 4 == 0 && aligned(y, 8)};
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
    if (m > 64) {
        const bool tall = m > 128;
        const long long tm = tall ? (m + 255) / 256 : 1, tiles = tm * ((n + TILE_N - 1) / TILE_N);
        EXL3_REQUIRE(tiles <= 0x7fffffffLL, "exl3_fp8_linear: %d x %d outputs are too many", m, n);
#define EXL3_FP8_TILE(FM)                                                                                        \
    {                                                                                                            \
        const void* fn = bf16 ? reinterpret_cast<const void*>(&fp8_tile_kernel<FM, true>)                    \
                              : reinterpret_cast<const void*>(&fp8_tile_kernel<FM, false>);                  \
        const int rc = allow_dynamic_lds(fn, 2 * tile_buf<FM>, "exl3_fp8_linear");                              \
        if (rc) return rc;                                                                                       \
        if (bf16) fp8_tile_kernel<FM, true><<<(unsigned)tiles, 512, 2 * tile_buf<FM>, st>>>(a, (int)tm, (int)tiles); \
        else fp8_tile_kernel<FM, false><<<(unsigned)tiles, 512, 2 * tile_buf<FM>, st>>>(a, (int)tm, (int)tiles);     \
        return launch_status("exl3_fp8_linear launch");                                                          \
    }
        if (tall) EXL3_FP8_TILE(8)
        EXL3_FP8_TILE(4)
#undef EXL3_FP8_TILE
    }
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
