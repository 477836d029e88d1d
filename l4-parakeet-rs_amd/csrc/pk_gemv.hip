// Matrix-vector products with INT4-g128 weights for 1 to 16 rows:
//   y[m, n] = (sum_g s[n, g] * sum_{k in g} x[m, k] * (q[n, k] - z[n, g])) * xs[m] + b[n]
// The weights are the traffic (n * k / 2 bytes and n * k / 32 of scales and zeros, each read
// once); the rows ride along on the MFMA's second operand, so a few rows cost little more than
// one.  A workgroup owns 16, 32 or 64 weight rows and its waves split the 128-k groups; a lane
// (weight row l % 16, quarter g = l / 16) reads the 16 contiguous bytes that hold
// k = 32g .. 32g + 31 of a group, so a load instruction covers one group of 16 rows.  Word i of
// the lane is the MFMA's k-slots of step i, and x is read in the same order: the products' order
// within a group is free.  Group sums (exact in int32 for INT8 rows, fp32 for fp16 rows) are
// scaled in fp32, and how they are joined depends on n and k alone: a row's result is the same
// whatever rows stand beside it.
// Measured: 1030 x 640 2.4 us (a launch's latency); 16384 x 8192 (71.6 MB) one row 17.3 us with
// INT8 and 18.2 with fp16 rows, 4.1 and 3.9 TB/s, against 11.7 us for reading that much alone;
// what is missing is each CU's first and last loads, for every workgroup starts and ends at once.
#include <type_traits>

#include "pk_kernels.hpp"

namespace pk {

// One word of eight levels -> fp16 q - z in k order (exact: |q - z| <= 15).
// 0x64xx is 1024 + xx in fp16; zz holds 1024 + z twice.
__device__ __forceinline__ v8h levels_f16(uint32_t w, v2h zz) {
    const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu, k64 = 0x64646464u;
    const uint32_t p[4] = {__builtin_amdgcn_perm(k64, lo, 0x04010400u), __builtin_amdgcn_perm(k64, lo, 0x04030402u),
                           __builtin_amdgcn_perm(k64, hi, 0x04010400u), __builtin_amdgcn_perm(k64, hi, 0x04030402u)};
    v8h r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const v2h d = __builtin_bit_cast(v2h, p[i]) - zz;
        r[2 * i] = d[0];
        r[2 * i + 1] = d[1];
    }
    return r;
}

// The same as int8 q - z: no borrow leaves a byte of (q | 0x80) - z.
__device__ __forceinline__ void levels_i8(uint32_t w, uint32_t zzzz, int& lo, int& hi) {
    lo = (int)((((w & 0x0f0f0f0fu) | 0x80808080u) - zzzz) ^ 0x80808080u);
    hi = (int)(((((w >> 4) & 0x0f0f0f0fu) | 0x80808080u) - zzzz) ^ 0x80808080u);
}

// acc += scale * (levels . rows) for one group of 16 weight rows: w are the lane's 32 levels of
// row l % 16, whose zero is the fp16 `zero`; s the fp16 scales of rows 4 (l / 16) + r.
template <bool kInt8>
__device__ __forceinline__ void add_group(const uint4& w, uint32_t zero, const uint4& s, const uint4 (&x)[kInt8 ? 2 : 4], v4f& acc) {
    const uint32_t words[4] = {w.x, w.y, w.z, w.w}, scale[4] = {s.x, s.y, s.z, s.w};
    const float z = h2f((uint16_t)zero);
    if constexpr (kInt8) {
        const uint32_t zzzz = (uint32_t)(int)z * 0x01010101u;
        v4i sum{};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            int a[4];
            levels_i8(words[2 * j], zzzz, a[0], a[1]);
            levels_i8(words[2 * j + 1], zzzz, a[2], a[3]);
            sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(v4i{a[0], a[1], a[2], a[3]}, __builtin_bit_cast(v4i, x[j]), sum, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r] = __builtin_fmaf((float)sum[r], h2f((uint16_t)scale[r]), acc[r]);
    } else {
        const _Float16 zh = (_Float16)(1024.0f + z);
        v4f sum{};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(levels_f16(words[j], v2h{zh, zh}), __builtin_bit_cast(v8h, x[j]), sum, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r] = __builtin_fmaf(sum[r], h2f((uint16_t)scale[r]), acc[r]);
    }
}

constexpr int kGemvRows = 16;  // weight rows of a row tile
constexpr int kWaves = 8;
constexpr int kGemvWorkgroups = 256;  // one for each CU

// The waves' parts of the sums, joined in their order.
template <bool kInt8, int kTiles>
__device__ __forceinline__ void store_sums(float (*part)[kGemvRows * kTiles][17], const v4f (&acc)[kTiles], const float* xs, const float* bias,
                                           void* out, int out_f32, int m, int n, int n0) {
    constexpr int kRows = kGemvRows * kTiles;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, g4 = lane >> 4;
    // lane (column m = l16) holds weight rows 4 g4 + r of each tile
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) part[wave][16 * t + 4 * g4 + r][l16] = acc[t][r];
    __syncthreads();
    for (int i = threadIdx.x; i < kRows * m; i += 64 * kWaves) {
        const int col = i % kRows, mr = i / kRows;
        if (n0 + col >= n) continue;
        float v = 0.0f;
#pragma unroll
        for (int w2 = 0; w2 < kWaves; ++w2) v += part[w2][col][mr];
        if constexpr (kInt8) v *= xs[mr];
        if (bias) v += bias[n0 + col];
        const size_t at = (size_t)mr * n + n0 + col;
        if (out_f32) ((float*)out)[at] = v;
        else ((uint16_t*)out)[at] = f2h(v);
    }
}

// A workgroup owns kTiles row tiles; a wave takes kRun consecutive groups at once, and its next
// run's weights are on their way while it works on one.  A lane loads one scale and zero of the
// 16 kTiles kRun that a run needs; they are handed round in a table of the wave's own.
template <bool kInt8, int kTiles, int kRun>
__global__ __launch_bounds__(64 * kWaves) void gemv_g128_kernel(const void* __restrict__ x, const float* __restrict__ xs,
                                                                       const uint32_t* __restrict__ q, const uint16_t* __restrict__ scales,
                                                                       const uint16_t* __restrict__ zeros, const float* __restrict__ bias,
                                                                       void* __restrict__ out, int out_f32, int m, int n, int k) {
    constexpr int kRows = kGemvRows * kTiles, kLoads = kInt8 ? 2 : 4, kBytes = kInt8 ? 1 : 2;
    static_assert(kRows * kRun <= 64);
    __shared__ uint32_t table[kWaves][kRun][kRows];
    __shared__ float part[kWaves][kRows][17];
    const int groups = k >> 7, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * kRows, l16 = lane & 15, g4 = lane >> 4;
    const uint4* wp[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
        const int row = n0 + 16 * t + l16 < n ? n0 + 16 * t + l16 : n - 1;
        wp[t] = (const uint4*)(q + (size_t)row * (k >> 3)) + g4;
    }
    const int srow = n0 + lane / kRun % kRows < n ? n0 + lane / kRun % kRows : n - 1;
    const size_t sbase = (size_t)srow * groups;
    uint4 w[kTiles][kRun];
    uint32_t entry = 0;
    const auto load = [&](int g0) {
        const int mine = g0 + lane % kRun < groups ? g0 + lane % kRun : groups - 1;
        entry = (uint32_t)scales[sbase + mine] | ((uint32_t)zeros[sbase + mine] << 16);
#pragma unroll
        for (int i = 0; i < kRun; ++i)
#pragma unroll
            for (int t = 0; t < kTiles; ++t) w[t][i] = wp[t][(size_t)(g0 + i < groups ? g0 + i : groups - 1) * 4];
    };
    int g0 = wave * kRun;
    if (g0 < groups) load(g0);
    v4f acc[kTiles] = {};
    const uint8_t* xp = (const uint8_t*)x + ((size_t)l16 * k + g4 * 32) * kBytes;
    for (; g0 < groups; g0 += kWaves * kRun) {
        if (lane < kRows * kRun) table[wave][lane % kRun][lane / kRun] = entry;
        uint4 now[kTiles][kRun];
#pragma unroll
        for (int i = 0; i < kRun; ++i)
#pragma unroll
            for (int t = 0; t < kTiles; ++t) now[t][i] = w[t][i];
        uint4 xr[kRun][kLoads];
#pragma unroll
        for (int i = 0; i < kRun; ++i)
#pragma unroll
            for (int j = 0; j < kLoads; ++j)
                xr[i][j] = l16 < m && g0 + i < groups ? *(const uint4*)(xp + (size_t)(g0 + i) * 128 * kBytes + 16 * j) : uint4{0, 0, 0, 0};
        if (g0 + kWaves * kRun < groups) load(g0 + kWaves * kRun);
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            if (g0 + i >= groups) break;
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                const uint32_t* e = &table[wave][i][16 * t];
                const uint4 s4 = *(const uint4*)(e + 4 * g4);
                add_group<kInt8>(now[t][i], e[l16] >> 16, s4, xr[i], acc[t]);
            }
        }
    }
    store_sums<kInt8, kTiles>(part, acc, xs, bias, out, out_f32, m, n, n0);
}

template <bool kInt8, int kTiles, int kRun>
static void launch_gemv(const void* x, const float* xs, const uint32_t* q, const uint16_t* scales, const uint16_t* zeros, const float* bias,
                          void* out, int out_f32, int m, int n, int k, hipStream_t s) {
    constexpr int kRows = kGemvRows * kTiles;
    gemv_g128_kernel<kInt8, kTiles, kRun><<<(unsigned)((n + kRows - 1) / kRows), 64 * kWaves, 0, s>>>(
        x, xs, q, scales, zeros, bias, out, out_f32, m, n, k);
}

template <bool kInt8>
static void launch_gemv_type(const void* x, const float* xs, const uint32_t* q, const uint16_t* scales, const uint16_t* zeros,
                             const float* bias, void* out, int out_f32, int m, int n, int k, hipStream_t s) {
    const auto launch = [&](auto tiles, auto run) {
        launch_gemv<kInt8, tiles, run>(x, xs, q, scales, zeros, bias, out, out_f32, m, n, k, s);
    };
    // Wide workgroups fetch a row of x and a wave's start once for more weights, but fewer of them
    // exist: 64 rows each where that still gives every CU one, 32 where those do.  With k = 8192,
    // one INT8 row: n = 16384 takes 17.3 us with 64 rows, 17.5 with 32 and 19.0 with 16 (16 fp16
    // rows: 22.6, 29.3, 46.6); n = 8192, k = 4096 the other way round 9.4 and 7.0, 6.9 (16 rows:
    // 10.1, 7.5, 8.9).  Between the two, with k = 8192, 64 rows would already be ahead: one INT8 row
    // 16.3 us against 16.6 at n = 10000, 16.7 and 16.9 at 14000, 16 fp16 rows 21.9 and 28.5, 22.7
    // and 28.9; n = 8192 takes 16.1 and 11.8, 21.5 and 16.7.
    if (n >= 64 * kGemvWorkgroups) launch(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
    else if (n >= 32 * kGemvWorkgroups) launch(std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{});
    // Few weight rows: the waves' number of turns counts.  One row, 1024 x 4096: 5.2 us with one
    // group a turn, 4.5 with two, 4.1 with four; 4096 x 1024 (8 groups for 8 waves) 2.8, 2.8, 3.4.
    else if (k <= 8 * 128) launch(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
    else if (k <= 16 * 128) launch(std::integral_constant<int, 1>{}, std::integral_constant<int, 2>{});
    else launch(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
}

void launch_gemv_g128(const void* x, const float* xs, const uint32_t* q, const uint16_t* scales, const uint16_t* zeros, const float* bias,
                      void* out, int out_f32, int m, int n, int k, hipStream_t s) {
    if (xs) launch_gemv_type<true>(x, xs, q, scales, zeros, bias, out, out_f32, m, n, k, s);
    else launch_gemv_type<false>(x, xs, q, scales, zeros, bias, out, out_f32, m, n, k, s);
}

}  // namespace pk
