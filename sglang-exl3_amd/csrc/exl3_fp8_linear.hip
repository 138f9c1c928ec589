// Matrix product of e4m3 rows and an e4m3 weight, both with fp32 scales by block:
//   y[m][n] = sum_b xs[m][b] ws[n / 128][b] sum_{k in block b} x[m][k] w[n][k] + bias[n]
// b runs over blocks of 128 columns of k.  For a bf16 result one
// v_mfma_f32_16x16x128_f8f6f4 is a block's inner sum for 16 x 16 outputs, in fp32 and
// from a zero accumulator; four FMAs a lane then add it, times the two scales, to the
// fp32 result.  The weight is the first operand, so that a lane's four outputs are
// neighbours in a row of y and share the row's scale.
//
// That unit adds e4m3 products in groups of 16, aligned to the group's largest and cut
// 13 bits below it, then in fp32: 1.5e-5 of the result for random operands, without a
// bias, a hundredth of a bf16 output's rounding.  (v_mfma_f32_16x16x32_fp8_fp8 gives the
// same bits at half the rate, 2220 against 4380 TFLOP/s.)  It is a tenth of an fp16
// output's, and where that output is quantized again, a gate/up product in an MLP, it
// moves values over e4m3's ties: 2e-3 of the MLP's result where fp32 sums give 8e-4.  So
// for an fp16 result both operands are widened to fp16, which is exact, and four
// v_mfma_f32_16x16x32_f16 add them in fp32.  That costs up to a tenth where memory bounds
// (40 x 4096 x 28672: 25.3 -> 28.2 us) and the double where the matrix unit does (2048 x
// 4096 x 28672: 221 -> 436).
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
    int vec, vec16;  // rows of y are aligned to 8, 16 bytes
    int* counters;             // of tiles whose k is split: zero between calls
    void* part;                // their sums
};

__device__ __forceinline__ i32x8_t two16(u32x4_t a, u32x4_t b) {
    return i32x8_t{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}
__device__ __forceinline__ float4_t mfma_e4m3(i32x8_t a, i32x8_t b) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, float4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

// A fragment as the products take it: e4m3 for a bf16 result, fp16 for an fp16 one.
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
struct Wide {
    f16x8_t h[4];
};
__device__ __forceinline__ Wide widen(i32x8_t v) {
    Wide w;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const f16x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[j], 1.0f, false);
        const f16x2_t hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[j], 1.0f, true);
        w.h[j >> 1][4 * (j & 1)] = lo[0];
        w.h[j >> 1][4 * (j & 1) + 1] = lo[1];
        w.h[j >> 1][4 * (j & 1) + 2] = hi[0];
        w.h[j >> 1][4 * (j & 1) + 3] = hi[1];
    }
    return w;
}
template <bool BF16>
__device__ __forceinline__ auto fragment(i32x8_t v) {
    if constexpr (BF16) return v;
    else return widen(v);
}
__device__ __forceinline__ float4_t product(i32x8_t a, i32x8_t b) { return mfma_e4m3(a, b); }
__device__ __forceinline__ float4_t product(const Wide& a, const Wide& b) {
    float4_t c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h[j], b.h[j], c, 0, 0, 0);
    return c;
}

// Four neighbouring results of a row, with the bias: y[row][col ..], up to the row's end.
template <bool BF16>
__device__ __forceinline__ void store4(const LinearArgs& p, int row, int col, float4_t v) {
    EXL3_GLOBAL uint16_t* y = gptr(p.y) + (size_t)row * p.n + col;
    if (p.bias)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < p.n) v[e] += f2_of<BF16>(gptr(p.bias)[col + e]).x;
    const u32x2_t o = {bits_of<BF16>(v[0], v[1]), bits_of<BF16>(v[2], v[3])};
    if (p.vec && col + 4 <= p.n) {
        *reinterpret_cast<EXL3_GLOBAL u32x2_t*>(y) = o;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < p.n) y[e] = (uint16_t)(o[e >> 1] >> (16 * (e & 1)));
    }
}

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
__device__ __forceinline__ void copy16_once(i32x4_t rsrc, uint32_t off, uint32_t step, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen nt lds" ::"v"(off), "s"(rsrc),
                 "s"(step), "s"(lds)
                 : "memory", "m0");
}
__device__ __forceinline__ void copy4(i32x4_t rsrc, uint32_t off, uint32_t step, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dword %0, %1, %2 offen lds" ::"v"(off), "s"(rsrc),
                 "s"(step), "s"(lds)
                 : "memory", "m0");
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const void* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
}
constexpr int NT = 2;  // buffer loads: data that is read once (nontemporal)

// Few rows: the weight is streamed once, from memory to registers.  A workgroup owns
// 16 columns and 16 rows of y; its waves take turns in the blocks of k and meet in LDS
// at the end, in a fixed order.  A lane reads 32 bytes of its row in each block, 16 of
// them from each half: the order of k within a block is free as long as both operands
// share it.  U blocks of a wave are on their way at a time; blocks past the end read
// as zeros, so that no load waits for a branch.  (16 columns a workgroup were the best
// everywhere against 32 and 64, and 2 to 4 blocks of rows lost to the ring below.)
// Workgroups begin at different blocks: rows of a weight are often a multiple of 4 KB
// apart, and where all read the same columns at a time, a part of the memory's channels
// serves them (4096 x 28672, one row, fp8_ring_kernel: 26.9 -> 20.9 us; 40 rows: 29.0
// -> 25.8).
//
// ROWS: x is 16-bit and few enough for every workgroup to quantize it itself, into
// LDS, while its first weight requests are on their way.  One row, 4096 x 6144, weights
// from HBM: 25 MB in 9.7 us (graph replay, 2.1 of it an empty kernel's; 10.6 as two
// launches): latency of the first loads, then the memory's rate.  Larger weights are
// faster through the ring (4096 x 28672: 26.4 here, 22.6 there).
template <bool ROWS, bool XBF, bool BF16>
__global__ __launch_bounds__(512, 2) void fp8_stream_kernel(LinearArgs p) {
    constexpr int U = 4;
    extern __shared__ __align__(16) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x >> 6;
    const int n0 = blockIdx.x * 16, nr = min(16, p.n - n0);
    const int m0 = blockIdx.y * 16, mr = min(16, p.m - m0);
    const auto wbuf = rsrc_of(p.w + (size_t)n0 * p.k, (uint32_t)nr * p.k);
    const auto wsbuf = rsrc_of(p.ws + (size_t)(n0 >> 7) * p.groups, (uint32_t)p.groups * 4);
    const auto xbuf = rsrc_of(p.x + (size_t)m0 * p.k, (uint32_t)mr * p.k);
    const auto xsbuf = rsrc_of(p.xs + (size_t)m0 * p.groups, (uint32_t)mr * p.groups * 4);
    const uint32_t row = min(i, mr - 1);
    const uint32_t woff = (uint32_t)min(i, nr - 1) * p.k + 16 * g, xoff = row * p.k + 16 * g, xsoff = row * p.groups * 4;
    u32x4_t w[U][2], x[U][2];
    float s[U], xs[U];
    const int first = (int)blockIdx.x % p.groups;
    const auto block_of = [&](int turn) { return turn + first >= p.groups ? turn + first - p.groups : turn + first; };
    auto load_w = [&](int u, int turn) {
        const int kb = block_of(turn), left = turn < p.groups ? p.k - kb * 128 : 0, at = left > 0 ? kb : 0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            w[u][h] = __builtin_amdgcn_raw_buffer_load_b128(wbuf, 16 * g + 64 * h < left ? woff + 64 * h : OUT, at * 128, NT);
        s[u] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(wsbuf, left > 0 ? 0 : OUT, at * 4, 0));
    };
    const float* lsc = reinterpret_cast<const float*>(smem + (size_t)p.m * p.groups * 128);
    auto load_x = [&](int u, int turn) {
        const int kb = block_of(turn), left = turn < p.groups ? p.k - kb * 128 : 0, at = left > 0 ? kb : 0;
        const int group = row * p.groups + at;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if constexpr (ROWS)  // blocks past the end repeat the first: their weight is zero
                x[u][h] = *reinterpret_cast<const u32x4_t*>(smem + group * 128 + 16 * g + 64 * h);
            else
                x[u][h] = __builtin_amdgcn_raw_buffer_load_b128(xbuf, 16 * g + 64 * h < left ? xoff + 64 * h : OUT, at * 128, 0);
        }
        if constexpr (ROWS) xs[u] = lsc[group];
        else xs[u] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(xsbuf, left > 0 ? xsoff : OUT, at * 4, 0));
    };
#pragma unroll
    for (int u = 0; u < U; ++u) {
        load_w(u, wave + u * waves);
        if constexpr (!ROWS) load_x(u, wave + u * waves);
    }
    if constexpr (ROWS) {
        const EXL3_GLOBAL uint16_t* xp = reinterpret_cast<const EXL3_GLOBAL uint16_t*>(gptr(p.x));
        for (int id = tid >> 4; id < p.m * p.groups; id += waves * 4) {
            const int r = id / p.groups, c0 = (id - r * p.groups) * 128 + i * 8;
            u32x4_t v = {0, 0, 0, 0};
            if (c0 < p.k) v = *reinterpret_cast<const EXL3_GLOBAL u32x4_t*>(xp + (size_t)r * p.k + c0);
            float q;
            *reinterpret_cast<u32x2_t*>(smem + id * 128 + i * 8) = quantize8<XBF>(v, q);
            if (i == 0) const_cast<float*>(lsc)[id] = q;
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u) load_x(u, wave + u * waves);
    }
    float4_t acc = {0.f, 0.f, 0.f, 0.f};
    for (int turn = wave; turn < p.groups; turn += U * waves) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float4_t t = product(fragment<BF16>(two16(w[u][0], w[u][1])), fragment<BF16>(two16(x[u][0], x[u][1])));
            const float f = s[u] * xs[u];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = fmaf(t[e], f, acc[e]);
            load_w(u, turn + (u + U) * waves);
            load_x(u, turn + (u + U) * waves);
        }
    }
    // waves meet: [wave][lane] in LDS, summed in wave order
    if constexpr (ROWS) __syncthreads();
    float4_t* part = reinterpret_cast<float4_t*>(smem);
    part[wave * 64 + lane] = acc;
    __syncthreads();
    if (wave) return;
    float4_t v[8];
#pragma unroll
    for (int o = 0; o < 8; ++o) v[o] = part[(o < waves ? o : 0) * 64 + lane];  // all reads at once
#pragma unroll
    for (int o = 1; o < 8; ++o)
        if (o < waves) v[0] += v[o];
    if (i < mr) store4<BF16>(p, m0 + i, n0 + 4 * g, v[0]);
}

// One of `splits` ranges of k of a tile: hands this workgroup's sums v on, and returns
// whether it is the tile's last, which then has them all, added in the ranges' order.
// [tile][range][f][thread], 16 bytes each, through device-coherent stores and loads
// (sc1: past the XCD's own L2), so that the counter needs no write-back or invalidate.
constexpr int SC1 = 16;
template <int F, int THREADS>
__device__ __forceinline__ bool combine(const LinearArgs& p, int tile, int range, int splits, float4_t (&v)[F],
                                        unsigned char* smem) {
    constexpr int SIZE = F * THREADS * 16, R = F <= 4 ? 4 : 1;  // R ranges are read at once
    const int tid = threadIdx.x;
    const auto part = rsrc_of(reinterpret_cast<const char*>(p.part) + (size_t)tile * splits * SIZE, (uint32_t)splits * SIZE);
#pragma unroll
    for (int f = 0; f < F; ++f)
        __builtin_amdgcn_raw_buffer_store_b128(
            u32x4_t{__float_as_uint(v[f][0]), __float_as_uint(v[f][1]), __float_as_uint(v[f][2]), __float_as_uint(v[f][3])},
            part, tid * 16, range * SIZE + f * THREADS * 16, SC1);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    int* last = reinterpret_cast<int*>(smem);
    if (tid == 0) {
        const int old = __hip_atomic_fetch_add(p.counters + tile, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (old == splits - 1) __hip_atomic_store(p.counters + tile, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *last = old == splits - 1;
    }
    __syncthreads();
    if (!*last) return false;
    asm volatile("" ::: "memory");
#pragma unroll
    for (int f = 0; f < F; ++f) v[f] = float4_t{0.f, 0.f, 0.f, 0.f};
    for (int r = 0; r < splits; r += R) {
        u32x4_t u[R][F];
#pragma unroll
        for (int q = 0; q < R; ++q)
#pragma unroll
            for (int f = 0; f < F; ++f)  // ranges past the last repeat it, and are not added
                u[q][f] = __builtin_amdgcn_raw_buffer_load_b128(part, tid * 16, min(r + q, splits - 1) * SIZE + f * THREADS * 16, SC1);
#pragma unroll
        for (int q = 0; q < R; ++q)
            if (r + q < splits)
#pragma unroll
                for (int f = 0; f < F; ++f)
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[f][e] += __uint_as_float(u[q][f][e]);
    }
    return true;
}

// Tiles for a middling number of rows: 4 waves, 64 FN columns of y and 16 FM rows, and
// a range of k.  Wave v has columns 16 FN v ..; the rows of x are shared.  Both
// operands go through a ring of NB LDS buffers, a block of 128 columns each (slots as
// below), filled by the load unit NB - 1 blocks ahead: at two workgroups a CU
// that is 50 to 100 KB of weight on their way, which streaming it takes, without a
// register.  Bound by memory for few rows (40 rows, 4096 x 28672: 119 MB in 23.5 us,
// 5.1 TB/s; 24 rows, 14336 x 4096: 60 MB in 13.9 us, with k in four ranges and their
// hand-off), by the steps' latency for more.  ONCE: the weight is read by one block of rows, and past the caches'
// keeping (nontemporal): 4096 x 28672, one row, 24.7 -> 21.7 us; with several blocks
// of rows it would cost (200 rows, 4096 x 6144: 16.8 -> 18.1).
template <int FN, int FM>
constexpr int ring_buf = (64 * FN + 16 * FM) * 128 + 768;  // weight rows, rows of x, scales: 128 rows', 64 times the weight's

template <int FN, int FM, int NB, bool ONCE, bool BF16>
__global__ __launch_bounds__(256, 2) void fp8_ring_kernel(LinearArgs p, int tiles_m, int tiles, int splits) {
    constexpr int NT = 64 * FN, MT = 16 * FM, BUF = ring_buf<FN, FM>, XB = NT * 128, SB = XB + MT * 128;
    constexpr int WC = 2 * FN, XC = (2 * FM + 3) / 4, C = WC + XC + 1;  // copies of a wave in a step
    extern __shared__ __align__(16) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // each XCD (workgroup % 8) gets a run of neighbours: rows fastest, then ranges of k, then columns
    const int per = tiles >> 3, rest = tiles & 7, xcd = blockIdx.x & 7;
    const int id = __builtin_amdgcn_readfirstlane(xcd * per + min(xcd, rest) + (blockIdx.x >> 3));
    const int tm = id % tiles_m, range = id / tiles_m % splits, tn = id / tiles_m / splits;
    const int m0 = tm * MT, n0 = tn * NT;
    const int s0 = (int)((long long)p.groups * range / splits), s1 = (int)((long long)p.groups * (range + 1) / splits);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;

    // rows past the end repeat the last one (never stored); columns past it read as zeros
    const int mr = min(MT, p.m - m0), nr = min(NT, p.n - n0);
    const i32x4_t xbuf = buffer_of(p.x + (size_t)m0 * p.k, (uint32_t)mr * p.k);
    const i32x4_t wbuf = buffer_of(p.w + (size_t)n0 * p.k, (uint32_t)nr * p.k);
    const int chunk = 16 * ((lane & 7) ^ (lane >> 3));
    uint32_t xoff[XC], xdst[XC], woff[WC];
#pragma unroll
    for (int j = 0; j < XC; ++j) {
        const int c = (wave + 4 * j) % (2 * FM);  // more waves than copies: some are made twice
        xoff[j] = (uint32_t)min(8 * c + (lane >> 3), mr - 1) * p.k + chunk;
        xdst[j] = XB + c * 1024;
    }
#pragma unroll
    for (int j = 0; j < WC; ++j) woff[j] = (uint32_t)min((WC * wave + j) * 8 + (lane >> 3), nr - 1) * p.k + chunk;
    const bool xs = wave < 2;
    const i32x4_t sbuf = xs ? buffer_of(p.xs + (size_t)m0 * p.groups, (uint32_t)mr * p.groups * 4)
                            : buffer_of(p.ws + (size_t)(n0 >> 7) * p.groups, (uint32_t)p.groups * 4);
    const uint32_t soff = xs ? (uint32_t)min(64 * wave + lane, mr - 1) * p.groups * 4 : 0;
    const uint32_t sdst = SB + 256 * min(wave, 2);
    const int first = tn * 11 % (s1 - s0);  // see fp8_stream_kernel
    auto copy = [&](int s, uint32_t to) {
        int block = s + first;
        block -= block >= s1 ? s1 - s0 : 0;
        const int left = s < s1 ? p.k - block * 128 : 0;
        const uint32_t at = left > 0 ? block * 128 : 0;  // stays inside the buffer
#pragma unroll
        for (int j = 0; j < WC; ++j) {
            if (ONCE) copy16_once(wbuf, chunk < left ? woff[j] : OUT, at, to + (WC * wave + j) * 1024);
            else copy16(wbuf, chunk < left ? woff[j] : OUT, at, to + (WC * wave + j) * 1024);
        }
#pragma unroll
        for (int j = 0; j < XC; ++j) copy16(xbuf, chunk < left ? xoff[j] : OUT, at, to + xdst[j]);
        copy4(sbuf, left > 0 ? soff : OUT, at >> 5, to + sdst);
    };
    float4_t acc[FN][FM];
#pragma unroll
    for (int a = 0; a < FN; ++a)
#pragma unroll
        for (int b = 0; b < FM; ++b) acc[a][b] = float4_t{0.f, 0.f, 0.f, 0.f};
    const uint32_t slot = 16 * (g ^ (i & 7)), wrd = (16 * FN * wave + i) * 128 + slot, xrd = XB + i * 128 + slot;

#pragma unroll
    for (int j = 0; j < NB - 1; ++j) copy(s0 + j, lds0 + j * BUF);
    uint32_t buf = 0, free = (NB - 1) * BUF;
    for (int s = s0; s < s1; ++s) {
        // this step's copies are in, and every wave has read the buffer before
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NB - 2) * C) : "memory");
        __builtin_amdgcn_sched_barrier(0);
        const unsigned char* base = smem + buf;
        auto read = [&](uint32_t at) {
            return two16(*reinterpret_cast<const u32x4_t*>(base + at), *reinterpret_cast<const u32x4_t*>(base + (at ^ 64)));
        };
        decltype(fragment<BF16>(i32x8_t{})) w[FN];
#pragma unroll
        for (int a = 0; a < FN; ++a) w[a] = fragment<BF16>(read(wrd + a * 2048));
        const float sb = *reinterpret_cast<const float*>(base + SB + 512);
        copy(s + NB - 1, lds0 + free);
#pragma unroll
        for (int b = 0; b < FM; ++b) {
            const auto v = fragment<BF16>(read(xrd + b * 2048));
            const float f = *reinterpret_cast<const float*>(base + SB + (16 * b + i) * 4) * sb;
#pragma unroll
            for (int a = 0; a < FN; ++a) {
                const float4_t t = product(w[a], v);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[a][b][e] = fmaf(t[e], f, acc[a][b][e]);
            }
        }
        free = buf;
        buf = buf == (NB - 1) * BUF ? 0 : buf + BUF;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // copies past the end land before the workgroup ends
    if (splits > 1 && !combine<FN * FM, 256>(p, tn * tiles_m + tm, range, splits, *reinterpret_cast<float4_t(*)[FN * FM]>(acc), smem))
        return;
#pragma unroll
    for (int b = 0; b < FM; ++b) {
        const int row = m0 + 16 * b + i;
        if (row >= p.m) continue;
#pragma unroll
        for (int a = 0; a < FN; ++a) store4<BF16>(p, row, n0 + 16 * (FN * wave + a) + 4 * g, acc[a][b]);
    }
}

// Tiles for many rows.  A workgroup of WN x WM waves owns 64 WN columns of y and
// 16 FM WM rows, a wave 64 columns and 16 FM rows.  Rows of x and of the weight go
// through LDS, copied there by the load unit (16 bytes a lane) NB - 1 blocks of 128
// columns ahead.  LDS row r holds its 16-byte chunk c at slot c ^ (r & 7), by choice
// of the source address; a fragment's lanes read chunks g and g + 4 of rows
// i = lane & 15, g = lane >> 4, without bank conflicts (256 bytes a cycle; chunks 2g
// and 2g + 1 in these slots conflict and run at half of it).  2048 rows, 4096 x 28672:
// 227 us, 2120 TFLOP/s; 4096 rows, 8192 x 8192: 231 us, 2380.  Bound by the matrix unit
// with the FMAs beside it (on random operands in registers the same instructions reach
// 3063), and by first loads and last stores, 5 us for each round of tiles.
constexpr int FP8_MAX_K = 1 << 22;  // 256 rows within 31 bits

template <int WN, int WM, int FM>  // rows of x, of the weight, the rows' scales, the weight's, and room for copies that nothing reads
constexpr int tile_buf = (16 * FM * WM + 64 * WN) * 128 + (16 * FM * WM + 128) * 4;

template <int WN, int WM, int FM, int NB, bool BF16>
__device__ __forceinline__ void tile_body(const LinearArgs& p, unsigned char* smem, int m0, int n0, int s0, int len,
                                          int tile, int range, int splits) {
    static_assert(FM % 2 == 0, "fragments alternate between two register sets");
    constexpr int MT = 16 * FM * WM, NT = 64 * WN, BUF = tile_buf<WN, WM, FM>, WAVES = WN * WM;
    constexpr int XC = MT / 8 / WAVES, WC = NT / 8 / WAVES, C = WC + XC + 1;  // copies of a wave in a step
    static_assert(C <= 4 + 2 * (FM - 1) && MT / 64 < WAVES, "room for the copies in a step");
    constexpr int WB = MT * 128, SB = WB + NT * 128;  // weight, scales in a buffer
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave % WN, wm = wave / WN;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;

    // rows past the end repeat the last one (never stored); columns past it read as zeros
    const int mr = min(MT, p.m - m0), nr = min(NT, p.n - n0);
    const i32x4_t xbuf = buffer_of(p.x + (size_t)m0 * p.k, (uint32_t)mr * p.k);
    const i32x4_t wbuf = buffer_of(p.w + (size_t)n0 * p.k, (uint32_t)nr * p.k);
    const int chunk = 16 * ((lane & 7) ^ (lane >> 3)), lr = 8 * wave + (lane >> 3);
    uint32_t xoff[XC], woff[WC];
#pragma unroll
    for (int j = 0; j < XC; ++j) xoff[j] = (uint32_t)min(8 * WAVES * j + lr, mr - 1) * p.k + chunk;
#pragma unroll
    for (int j = 0; j < WC; ++j) woff[j] = (uint32_t)min(8 * WAVES * j + lr, nr - 1) * p.k + chunk;
    // scales: waves 0 .. MT / 64 - 1 those of 64 rows each, the last the weight's (the others nothing that is read)
    const bool xs = wave < MT / 64;
    const int nb = (nr + 127) >> 7;
    const i32x4_t sbuf = xs ? buffer_of(p.xs + (size_t)m0 * p.groups, (uint32_t)mr * p.groups * 4)
                            : buffer_of(p.ws + (size_t)(n0 >> 7) * p.groups, (uint32_t)nb * p.groups * 4);
    const uint32_t soff = (uint32_t)(xs ? min(64 * wave + lane, mr - 1) : min(lane & 1, nb - 1)) * p.groups * 4;
    const uint32_t sdst = SB + (xs ? 256 * wave : 4 * MT + (wave == WAVES - 1 ? 0 : 256));
    // XCDs begin at different blocks (see fp8_stream_kernel), and so do the tiles of one:
    // they share rows and columns in its L2, which holds what 8 blocks bring (1024 x
    // 8192 x 8192: 100 us with the same block, 90 with 4, 87 with 8, 86 with 16; 4096 x
    // 8192 x 8192: 238, 234, 231 and, with 32, 244)
    const int first = (int)(5 * (blockIdx.x & 7) + (blockIdx.x >> 3 & 7)) % len;
    // copy j of step s: the weight's, then the rows', then the scales; `to` is the step's buffer
    auto copy = [&](int s, uint32_t to, int j) {
        int block = s + first;
        block += s0 - (block >= len ? len : 0);
        int left = s < len ? p.k - block * 128 : 0;  // columns
        asm("" : "+s"(left));  // the offsets below are made where they are used, not kept
        const uint32_t at = left > 0 ? block * 128 : 0;  // stays inside the buffer
        if (j < WC) copy16(wbuf, chunk < left ? woff[j] : OUT, at,
                           lds0 + to + WB + 8 * (WAVES * j + wave) * 128);
        else if (j < WC + XC)
            copy16(xbuf, chunk < left ? xoff[j - WC] : OUT, at, lds0 + to + 8 * (WAVES * (j - WC) + wave) * 128);
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
    for (int s = 0; s < NB - 1; ++s)
#pragma unroll
        for (int j = 0; j < C; ++j) copy(s, s * BUF, j);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NB - 2) * C) : "memory");
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
    // the two waves of a SIMD in different phases: one waits while the other multiplies (8192 x 8192, 4096 rows:
    // 255 -> 236 us)
    if (wave >= WAVES / 2) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int j = 0; j < 4; ++j) copy(NB - 1, (NB - 1) * BUF, j);
    // Step s with buffer `buf`; `other` is the next step's, `free` the one before's.
    // The barrier is before the last fragment's products: those cover the next
    // step's first reads.  Copies are spread out: at once, they would keep the load
    // unit, and the waves that wait for it, busy for half of the step.
    uint32_t at_buf = 0, at_free = (NB - 1) * BUF;
    auto body = [&](int s, auto slot_c) {
        constexpr int S = decltype(slot_c)::value;
        const uint32_t buf = NB == 2 ? S * BUF : at_buf, free = NB == 2 ? (S ^ 1) * BUF : at_free;
        const uint32_t other = NB == 2 ? (S ^ 1) * BUF : buf == (NB - 1) * BUF ? 0 : buf + BUF;
#pragma unroll
        for (int b = 0; b < FM; ++b) {
            if (b == FM - 1) {
                // the next step's copies are in, and every wave has read this step's buffer
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NB - 2) * C) : "memory");
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const float4_t done = t[a];
                t[a] = product(fragment<BF16>(w[S][a]), fragment<BF16>(x[b & 1]));
                __builtin_amdgcn_sched_barrier(0);
                if (b < FM - 1) {
                    if (a < 2) half(x[(b + 1) & 1], a, xrd + buf + (b + 1) * 2048);
                    if (a == 2) f[(b + 1) & 1] = number(frd + buf + (b + 1) * 64);
                    if (a >= 2) copy(s + NB - 1, free, 4 + 2 * b + a - 2);
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
                    copy(s + NB, buf, a);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    acc[a][(b + FM - 1) % FM][e] = fmaf(done[e], c, acc[a][(b + FM - 1) % FM][e]);
                __builtin_amdgcn_sched_barrier(0);
            }
            c = f[b & 1] * sb[S];
        }
        at_free = buf;
        at_buf = other;
    };
    for (int s = 0; s < len; s += 2) {  // an odd number's last step adds zeros
        body(s, std::integral_constant<int, 0>{});
        body(s + 1, std::integral_constant<int, 1>{});
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // copies past the end land before the workgroup ends
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[a][FM - 1][e] = fmaf(t[a][e], c, acc[a][FM - 1][e]);
    if (splits > 1 && !combine<4 * FM, 64 * WAVES>(p, tile, range, splits, *reinterpret_cast<float4_t(*)[4 * FM]>(acc), smem))
        return;
    const int c0 = n0 + 64 * wn;
    if (!p.vec16 || c0 + 64 > p.n) {
#pragma unroll
        for (int b = 0; b < FM; ++b) {
            const int row = m0 + (FM * wm + b) * 16 + i;
            if (row >= p.m) continue;
#pragma unroll
            for (int a = 0; a < 4; ++a) store4<BF16>(p, row, c0 + 16 * a + 4 * g, acc[a][b]);
        }
        return;
    }
    // Through LDS, 128 bytes of a row at a time, so that whole lines are written.  A
    // wave uses its own 2 KB for each 16 rows, with chunk c of 16 bytes of row r at
    // c ^ (r & 7).
    float add[4][4];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) add[a][e] = p.bias ? f2_of<BF16>(gptr(p.bias)[c0 + 16 * a + 4 * g + e]).x : 0.f;
    __syncthreads();  // every wave has read its last fragments
    unsigned char* const own = smem + wave * (FM * 2048);
#pragma unroll
    for (int b = 0; b < FM; ++b)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const float4_t v = acc[a][b];
            *reinterpret_cast<u32x2_t*>(own + (16 * b + i) * 128 + 16 * ((2 * a + (g >> 1)) ^ (i & 7)) + 8 * (g & 1)) =
                u32x2_t{bits_of<BF16>(v[0] + add[a][0], v[1] + add[a][1]), bits_of<BF16>(v[2] + add[a][2], v[3] + add[a][3])};
        }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int j = 0; j < 2 * FM; ++j) {
        const int r = 8 * j + (lane >> 3), row = m0 + FM * wm * 16 + r;
        if (row < p.m)
            *reinterpret_cast<EXL3_GLOBAL u32x4_t*>(gptr(p.y) + (size_t)row * p.n + c0 + 8 * (lane & 7)) =
                *reinterpret_cast<const u32x4_t*>(own + r * 128 + 16 * ((lane & 7) ^ (r & 7)));
    }
}

// 256 x 256 tiles, and after them tiles of 128 rows: of the last rows where at most
// 128 are left, and the two halves of tiles that would run in a last round which is
// less than half full.  Three buffers where a tile of 128 rows has room for them (1100
// x 7168 x 4096: 61 us with two, 51 with three).
constexpr size_t TILE_LDS = 3 * tile_buf<4, 2, 4>;
static_assert(TILE_LDS >= 2 * tile_buf<4, 2, 8>, "both tiles' buffers");
struct Tiles {
    int tiles_m, whole, splits_at;  // tiles of 256 rows along m; whole ones; halves made of tiles, the others follow
    int halves;
};
__global__ __launch_bounds__(512, 2) void fp8_tile_kernel(LinearArgs p, Tiles t) {  // bf16 results
    extern __shared__ __align__(16) unsigned char smem[];
    int id = blockIdx.x;
    if (id < t.whole) {
        // each XCD (workgroup % 8) gets a run of neighbouring tiles, rows fastest
        const int per = t.whole >> 3, rest = t.whole & 7, xcd = id & 7;
        id = xcd * per + min(xcd, rest) + (id >> 3);
        const int tn = __builtin_amdgcn_readfirstlane(id / t.tiles_m);
        tile_body<4, 2, 8, 2, true>(p, smem, __builtin_amdgcn_readfirstlane(id - tn * t.tiles_m) * 256, tn * 256, 0,
                                   p.groups, 0, 0, 1);
        return;
    }
    id -= t.whole;
    int tn, m0;
    if (id < t.splits_at) {
        const int w = t.whole + (id >> 1);
        tn = w / t.tiles_m;
        m0 = (w - tn * t.tiles_m) * 256 + (id & 1) * 128;
    } else {
        tn = id - t.splits_at;
        m0 = t.tiles_m * 256;
    }
    tn = __builtin_amdgcn_readfirstlane(tn);
    m0 = __builtin_amdgcn_readfirstlane(m0);
    if (m0 < p.m) tile_body<4, 2, 4, 3, true>(p, smem, m0, tn * 256, 0, p.groups, 0, 0, 1);
}

// 128 x 128 tiles of 4 waves, where 256 x 256 ones are too few, k split where these
// are too few as well (512 rows, 14336 x 4096: 84 us unsplit, 54 in two): with NB = 2
// two workgroups share a CU; NB = 4 where there is one for each (4 ranges of 256 rows,
// 14336 x 4096: 37.6 against 33.3 us).
template <int NB, bool BF16>
__global__ __launch_bounds__(256, NB == 2 ? 2 : 1) void fp8_quad_kernel(LinearArgs p, int tiles_m, int wgs, int splits) {
    extern __shared__ __align__(16) unsigned char smem[];
    const int per = wgs >> 3, rest = wgs & 7, xcd = blockIdx.x & 7;
    const int id = __builtin_amdgcn_readfirstlane(xcd * per + min(xcd, rest) + (blockIdx.x >> 3));
    const int tm = id % tiles_m, range = id / tiles_m % splits, tn = id / tiles_m / splits;
    const int s0 = (int)((long long)p.groups * range / splits), s1 = (int)((long long)p.groups * (range + 1) / splits);
    tile_body<2, 2, 4, NB, BF16>(p, smem, tm * 128, tn * 128, s0, s1 - s0, tn * tiles_m + tm, range, splits);
}

// ------------------------------------------------------------------- host side

struct Plan {
    enum Kind { STREAM, RING, TILE, QUAD } kind;
    bool fused;  // STREAM quantizes 16-bit rows itself
    int fn, fm, kw, splits, deep;
    long long tiles_m, tiles;
    Tiles t;
    size_t part_bytes;
    double us;
};

constexpr int CUS = 256;  // of the one device this is built for

long long up(long long a, long long b) { return (a + b - 1) / b; }

// The kernel and its tile by estimated time (us), fitted to sweeps of 150 shapes from
// 1 x 2048 x 1536 to 4096 x 8192 x 8192: within 7 % of the best of each but for a few
// (15 %).  What the terms stand for: a launch and its first requests; a step's (block
// of k's) time with one workgroup a CU and with more; the split's hand-off; the weight
// from HBM, which overlaps the steps, and takes a workgroup on every CU.  Both sides of
// some borders, in us: 1 x 4096 x 6144 of 16-bit rows streamed 9.7, in a ring 10.7, 1 x
// 4096 x 28672 26.4 and 22.6; 80 x 4096 x 28672 in a ring 37.8, in 128 x 128 tiles 31.0;
// 1024 x 8192 x 8192 in those 88.7, in 256 x 256 tiles 87.1, 900 x 8192 x 10240 140 and
// 104; 384 x 14336 x 4096 in 128 x 128 tiles unsplit 84, in two ranges 50.2, in four 51.6.
Plan choose(bool rows, int m, int k, int n) {
    const int groups = fp8_groups(k);
    Plan best = {};
    best.us = 1e30;
    const double memory = ((double)n * k + (double)m * k + 2.0 * m * n) / 6e6, quantize = rows ? 1.8 : 0;
    const auto overlap = [](double t, double mem) { return t > mem ? t + 0.1 * mem : mem + 0.1 * t; };
    const auto take = [&](const Plan& p) {
        if (p.us < best.us) best = p;
    };
    const bool fused = rows && m <= 4 && (size_t)m * groups * 132 <= 96 * 1024;
    const long long wgs = up(n, 16) * up(m, 16);
    if (m <= 4 || wgs <= 1280)
        for (int kw = 2; kw <= 8; kw *= 2) {
            Plan p = {Plan::STREAM, fused, 1, 1, kw, 1};
            // what a workgroup's loads take (longer with distinct rows of x), its waves' turns, all loads together
            const int r = m < 16 ? m : 16;
            const double own = groups * (0.09 + 0.0034 * r), turns = up(groups, kw) * 0.35;
            const double all = (double)(wgs > CUS ? up(wgs, CUS) * CUS : wgs) * k * (16 + 0.4 * r) / 5.4e6, most = own > turns ? (own > all ? own : all) : (turns > all ? turns : all);
            p.us = 1.5 + 0.2 * kw + most + 0.25 * (own + turns + all - most) + (fused ? k * (6e-4 * m / kw + 5e-5 * (m - 1)) : quantize);
            take(p);
        }
    if (m <= 1024) {
        const double one[5][2] = {{.24, .31}, {.27, .43}, {.33, .48}, {.38, .55}, {.63, .97}};
        const double two[5][2] = {{.35, .64}, {.50, .81}, {.64, 1.03}, {.75, 1.11}, {1.2, 1.42}};
        const int fms[5] = {1, 2, 3, 4, 8};
        for (int f = 0; f < 5; ++f) {
            const int fm = fms[f];
            if ((f > 0 && 16 * fms[f - 1] >= m) || m > 16 * fm * 8) continue;
            for (int fn = 1; fn <= 2; ++fn) {
                const long long tm = up(m, 16 * fm), tiles = tm * up(n, 64 * fn);
                for (int sp = 1; sp <= 16; sp += sp < 4 ? 1 : sp < 8 ? 2 : 4) {
                    if (sp > 1 && (tiles * sp > 2 * CUS || 2 * sp > groups || tiles > (long long)kWsMaxCounters)) break;
                    const double w = (double)(tiles * sp) / CUS;
                    // above one a CU, the CUs that have two decide
                    const double step = w <= 1 ? one[f][fn - 1] : two[f][fn - 1] * (w <= 2 ? 0.7 + 0.15 * w : w / 2);
                    // blocks of rows share the weight in L2, but not all of it; one CU's requests bring 28 KB a us
                    const double cu = (double)up(tiles * sp, CUS) * 64 * fn * ((double)k / sp) / 28e3;
                    const double mem = tm > 1 ? (memory + 0.3 * (tm - 1) * ((double)n * k / 6e6)) / (w < 0.87 ? 0.35 + 0.75 * w : 1)
                                              : memory > cu ? memory : cu;
                    Plan p = {Plan::RING, false, fn, fm, 0, sp};
                    p.tiles_m = tm;
                    p.tiles = tiles;
                    p.us = (fm <= 2 ? 2.5 : 3) + overlap(up(groups, sp) * step, mem) + quantize +
                           (sp > 1 ? 1.2 + 0.17 * fm * fn + sp * (0.3 + 0.1 * fm * fn) : 0);
                    if (sp > 1) p.part_bytes = (size_t)tiles * sp * fn * fm * 4096;
                    take(p);
                }
            }
        }
    }
    if (m > 64) {
        Plan p;
        for (int sp = 1; sp <= 8; sp += sp < 4 ? 1 : 2) {
            p = {Plan::QUAD, false, 0, 0, 0, sp};
            p.tiles_m = up(m, 128);
            p.tiles = p.tiles_m * up(n, 128);
            if (sp > 1 && (p.tiles * sp > 2 * CUS || 8 * sp > groups)) break;
            const double w = (double)(p.tiles * sp) / CUS;
            const long long steps = up(groups, sp);
            p.deep = w <= 1 && steps > 16;
            // rounds of two a CU, and the last one's
            const double pairs = (double)((p.tiles * sp) / (2 * CUS)), last = w - 2 * pairs;
            const double step = p.deep ? 0.62 + 0.12 * w : 1.38 * pairs + (last > 1 ? 0.83 + 0.28 * last : last > 0 ? 0.93 : 0);
            p.us = 4.5 + quantize + overlap(steps * step, memory) + (sp == 1 ? 0 : p.deep ? 3.5 + sp : 5 + 1.7 * sp);
            if (sp > 1) p.part_bytes = (size_t)p.tiles * sp * 65536;
            take(p);
        }
        p = {Plan::TILE, false, 0, 0, 0, 1};
        const long long tn = up(n, 256), full = (m % 256 == 0 || m % 256 > 128) ? up(m, 256) : m / 256;
        const long long last = full * 256 < m ? tn : 0, whole = tn * full, over = whole % CUS;
        const long long split = over && 2 * over + last <= CUS ? over : 0, halves = 2 * split + last;
        const double full_rounds = (double)((whole - split) / CUS), rest = (double)((whole - split) % CUS) / CUS;
        p.tiles = whole + split + last;
        if (p.tiles <= 0x7fffffff) {
            p.t = {(int)full, (int)(whole - split), (int)(2 * split), (int)halves};
            const double part = rest > 0 ? 1.1 + 0.55 * rest : 0, half = halves ? 0.8 + 0.5 * (double)halves / CUS : 0;
            const bool beside = (whole - split) % CUS + halves <= CUS;  // in the same round
            p.us = 8 + quantize + 5 * full_rounds +
                   overlap(groups * (1.62 * full_rounds + (!beside ? part + half : part > half ? part : half)), memory);
            take(p);
        }
    }
    return best;
}

// choose(), kept for the shapes that this thread has asked for: a call needs it twice.
const Plan& plan_of(bool rows, int m, int k, int n) {
    struct Entry {
        int rows, m, k, n;
        Plan plan;
    };
    static thread_local Entry table[64];
    const uint32_t h = ((uint32_t)m * 0x9E3779B1u) ^ ((uint32_t)k * 0x85EBCA77u) ^ ((uint32_t)n * 0xC2B2AE3Du) ^ (uint32_t)rows;
    Entry& e = table[(h ^ (h >> 15)) >> 3 & 63];
    if (e.rows != rows + 1 || e.m != m || e.k != k || e.n != n) e = {rows + 1, m, k, n, choose(rows, m, k, n)};
    return e.plan;
}

// Scratch: sums of split tiles, then e4m3 rows, then their scales.
size_t rows_bytes(int m, int k) { return ((size_t)m * k + 255) / 256 * 256; }

}  // namespace
}  // namespace exl3

using namespace exl3;

extern "C" size_t exl3_fp8_linear_workspace_size(int x_dtype, int m, int k, int n) {
    if (m <= 0 || k <= 0 || n <= 0 || k % 16) return 0;
    const bool rows = x_dtype != EXL3_DTYPE_E4M3;
    const Plan pl = plan_of(rows, m, k, n);
    const size_t q = rows && !pl.fused ? rows_bytes(m, k) + (size_t)m * fp8_groups(k) * sizeof(float) : 0;
    return pl.part_bytes || q ? kWsScratchOffset + pl.part_bytes + q : 0;
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
    EXL3_REQUIRE(m <= FP8_MOST && n <= FP8_MOST, "exl3_fp8_linear: m=%d n=%d above %d", m, n, FP8_MOST);
    EXL3_REQUIRE((long long)m * groups <= 0x7fffffffLL, "exl3_fp8_linear: %d x %d rows are too many", m, k);
    EXL3_REQUIRE(k <= FP8_MAX_K, "exl3_fp8_linear: k=%d above %d", k, FP8_MAX_K);
    if (m == 0) return EXL3_OK;
    EXL3_REQUIRE(x && w && w_scale && y && (rows || x_scale), "exl3_fp8_linear: null pointer");
    EXL3_REQUIRE(aligned(x, 16) && aligned(w, 16) && aligned(x_scale, 4) && aligned(w_scale, 4) && aligned(bias, 2) &&
                 aligned(y, 2), "exl3_fp8_linear: misaligned pointer (x and w: 16 bytes)");
    Plan pl = plan_of(rows, m, k, n);
    const size_t q_bytes = rows && !pl.fused ? rows_bytes(m, k) + (size_t)m * groups * sizeof(float) : 0;
    // a workspace without room for the split's sums (it was sized for other rows) runs unsplit
    if (pl.part_bytes && (!workspace || workspace_bytes < kWsScratchOffset + pl.part_bytes + q_bytes)) {
        pl.splits = 1;
        pl.part_bytes = 0;
    }
    if (pl.kind == Plan::TILE && y_dtype == EXL3_DTYPE_F16) {  // 256 x 256 tiles have no registers for wide fragments
        pl.kind = Plan::QUAD;
        pl.deep = 0;
        pl.tiles_m = up(m, 128);
        pl.tiles = pl.tiles_m * up(n, 128);
    }
    EXL3_REQUIRE(pl.tiles * pl.splits <= 0x7fffffffLL, "exl3_fp8_linear: %d x %d outputs are too many", m, n);
    const hipStream_t st = as_stream(stream);
    LinearArgs a = {static_cast<const uint8_t*>(x), w, x_scale, w_scale, static_cast<const uint16_t*>(bias),
                    static_cast<uint16_t*>(y), m, k, n, groups, n % 4 == 0 && aligned(y, 8),
                    n % 8 == 0 && aligned(y, 16), nullptr, nullptr};
    uint8_t* scratch = static_cast<uint8_t*>(workspace) + kWsScratchOffset;
    if (q_bytes || pl.part_bytes) {
        const size_t need = kWsScratchOffset + pl.part_bytes + q_bytes;
        EXL3_REQUIRE_CODE(workspace && workspace_bytes >= need, EXL3_ERR_WORKSPACE, "exl3_fp8_linear: workspace of "
                          "%zu bytes, needs %zu", workspace_bytes, need);
        EXL3_REQUIRE(aligned(workspace, 256), "exl3_fp8_linear: misaligned workspace");
        a.counters = static_cast<int*>(workspace);
        a.part = scratch;
    }
    if (q_bytes) {
        uint8_t* q = scratch + pl.part_bytes;
        float* s = reinterpret_cast<float*>(q + rows_bytes(m, k));
        const int rc = fp8_quant_rows(x, x_dtype == EXL3_DTYPE_BF16, k, q, s, m, k, st);
        if (rc) return rc;
        a.x = q;
        a.xs = s;
    }
    const bool bf16 = y_dtype == EXL3_DTYPE_BF16, xbf = x_dtype == EXL3_DTYPE_BF16;
#define EXL3_FP8_LAUNCH(GRID, THREADS, LDS, ARGS, ...)  /* a kernel up to its last argument, BF16 */  \
    {                                                                                                 \
        const void* fn = bf16 ? reinterpret_cast<const void*>(&__VA_ARGS__ true>)                     \
                              : reinterpret_cast<const void*>(&__VA_ARGS__ false>);                   \
        const int rc = allow_dynamic_lds(fn, LDS, "exl3_fp8_linear");                                 \
        if (rc) return rc;                                                                            \
        if (bf16) __VA_ARGS__ true><<<GRID, THREADS, LDS, st>>> ARGS;                                 \
        else __VA_ARGS__ false><<<GRID, THREADS, LDS, st>>> ARGS;                                     \
        return launch_status("exl3_fp8_linear launch");                                               \
    }
    const int wgs = (int)(pl.tiles * pl.splits), tm = (int)pl.tiles_m;
    if (pl.kind == Plan::TILE) {
        const int rc = allow_dynamic_lds(reinterpret_cast<const void*>(&fp8_tile_kernel), TILE_LDS, "exl3_fp8_linear");
        if (rc) return rc;
        fp8_tile_kernel<<<(unsigned)(pl.t.whole + pl.t.halves), 512, TILE_LDS, st>>>(a, pl.t);
        return launch_status("exl3_fp8_linear launch");
    }
    if (pl.kind == Plan::QUAD) {
        if (pl.deep)
            EXL3_FP8_LAUNCH(wgs, 256, (4 * tile_buf<2, 2, 4>), (a, tm, wgs, pl.splits), fp8_quad_kernel<4,)
        EXL3_FP8_LAUNCH(wgs, 256, (2 * tile_buf<2, 2, 4>), (a, tm, wgs, pl.splits), fp8_quad_kernel<2,)
    }
    if (pl.kind == Plan::RING) {
#define EXL3_FP8_RING(FN, FM, NB)                                                                                     \
    if (pl.fn == FN && pl.fm == FM) {                                                                                 \
        if (FM < 8 && tm == 1)                                                                                        \
            EXL3_FP8_LAUNCH(wgs, 256, (NB * ring_buf<FN, FM>), (a, tm, wgs, pl.splits), fp8_ring_kernel<FN, FM, NB, FM != 8,)  \
        EXL3_FP8_LAUNCH(wgs, 256, (NB * ring_buf<FN, FM>), (a, tm, wgs, pl.splits), fp8_ring_kernel<FN, FM, NB, false,)        \
    }
        EXL3_FP8_RING(1, 1, 7) EXL3_FP8_RING(1, 2, 6) EXL3_FP8_RING(1, 3, 5) EXL3_FP8_RING(1, 4, 4) EXL3_FP8_RING(1, 8, 3)
        EXL3_FP8_RING(2, 1, 4) EXL3_FP8_RING(2, 2, 3) EXL3_FP8_RING(2, 3, 3) EXL3_FP8_RING(2, 4, 3) EXL3_FP8_RING(2, 8, 2)
#undef EXL3_FP8_RING
    }
    size_t lds = (size_t)pl.kw * 1024;
    if (pl.fused && (size_t)m * groups * 132 > lds) lds = (size_t)m * groups * 132;
    const dim3 grid((n + 15) / 16, (m + 15) / 16);
    if (!pl.fused) EXL3_FP8_LAUNCH(grid, 64 * pl.kw, lds, (a), fp8_stream_kernel<false, false,)
    if (xbf) EXL3_FP8_LAUNCH(grid, 64 * pl.kw, lds, (a), fp8_stream_kernel<true, true,)
    EXL3_FP8_LAUNCH(grid, 64 * pl.kw, lds, (a), fp8_stream_kernel<true, false,)
#undef EXL3_FP8_LAUNCH
}
