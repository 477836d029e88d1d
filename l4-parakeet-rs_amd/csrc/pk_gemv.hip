// Matrix-vector products with INT4-g128 weights for 1 to 16 rows:
//   y[m, n] = (sum_g s[n, g] * sum_{k in g} x[m, k] * (q[n, k] - z[n, g])) * xs[m] + b[n]
// The weights are the traffic (n * k / 2 bytes, read once); the rows ride along on
// the MFMA's second operand, so one row costs what sixteen do.  A workgroup owns 16
// weight rows, its waves split the 128-k groups; a lane (weight row l % 16, quarter
// g = l / 16) reads the 16 contiguous bytes that hold k = 32g .. 32g + 31 of a group,
// so a load instruction covers one group of the 16 rows.  Word i of the lane is the
// MFMA's k-slots of step i, and x is read in the same order: the products' order
// within a group is free.  Group sums (exact in int32 for INT8 rows, fp32 for fp16
// rows) are scaled in fp32.
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

constexpr int kGemvRows = 16;

template <bool kInt8, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void gemv_g128_kernel(const void* __restrict__ x, const float* __restrict__ xs,
                                                                const uint32_t* __restrict__ q, const uint16_t* __restrict__ scales,
                                                                const uint16_t* __restrict__ zeros, const float* __restrict__ bias,
                                                                void* __restrict__ out, int out_f32, int m, int n, int k) {
    extern __shared__ uint32_t table[];  // [16 x groups] scale | zero << 16 of the workgroup's rows
    __shared__ float part[kWaves][16][17];
    const int groups = k >> 7, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n0 = blockIdx.x * kGemvRows, l16 = lane & 15, g4 = lane >> 4;
    for (int i = threadIdx.x; i < kGemvRows * groups; i += 64 * kWaves) {
        const size_t at = (size_t)n0 * groups + i;
        const bool in = at < (size_t)n * groups;
        table[i] = in ? (uint32_t)scales[at] | ((uint32_t)zeros[at] << 16) : 0u;
    }
    __syncthreads();

    const int row = n0 + l16 < n ? n0 + l16 : n - 1;
    const uint4* wp = (const uint4*)(q + (size_t)row * (k >> 3)) + g4;
    v4f acc{};
    for (int g = wave; g < groups; g += kWaves) {
        const uint4 w = wp[(size_t)g * 4];
        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
        const float z = h2f((uint16_t)(table[l16 * groups + g] >> 16));
        if constexpr (kInt8) {
            v4i xv[2] = {};
            if (l16 < m) {
                const v4i* xp = (const v4i*)((const int8_t*)x + (size_t)l16 * k + g * 128 + g4 * 32);
                xv[0] = xp[0];
                xv[1] = xp[1];
            }
            const uint32_t zzzz = (uint32_t)(int)z * 0x01010101u;
            v4i sum{};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                int a[4];
                levels_i8(words[2 * i], zzzz, a[0], a[1]);
                levels_i8(words[2 * i + 1], zzzz, a[2], a[3]);
                sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(v4i{a[0], a[1], a[2], a[3]}, xv[i], sum, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
                acc[r] = __builtin_fmaf((float)sum[r], h2f((uint16_t)(table[(4 * g4 + r) * groups + g] & 0xffffu)), acc[r]);
        } else {
            v8h xv[4] = {};
            if (l16 < m) {
                const v8h* xp = (const v8h*)((const uint16_t*)x + (size_t)l16 * k + g * 128 + g4 * 32);
#pragma unroll
                for (int i = 0; i < 4; ++i) xv[i] = xp[i];
            }
            const _Float16 zh = (_Float16)(1024.0f + z);
            v4f sum{};
#pragma unroll
            for (int i = 0; i < 4; ++i) sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(levels_f16(words[i], v2h{zh, zh}), xv[i], sum, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                acc[r] = __builtin_fmaf(sum[r], h2f((uint16_t)(table[(4 * g4 + r) * groups + g] & 0xffffu)), acc[r]);
        }
    }
    // lane (column m = l16) holds weight rows 4 g4 + r
#pragma unroll
    for (int r = 0; r < 4; ++r) part[wave][l16][4 * g4 + r] = acc[r];
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += 64 * kWaves) {
        const int col = i & 15, mr = i >> 4;
        if (mr >= m || n0 + col >= n) continue;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) v += part[w][mr][col];
        if constexpr (kInt8) v *= xs[mr];
        if (bias) v += bias[n0 + col];
        const size_t at = (size_t)mr * n + n0 + col;
        if (out_f32) ((float*)out)[at] = v;
        else ((uint16_t*)out)[at] = f2h(v);
    }
}

void launch_gemv_g128(const void* x, const float* xs, const uint32_t* q, const uint16_t* scales, const uint16_t* zeros, const float* bias,
                      void* out, int out_f32, int m, int n, int k, hipStream_t s) {
    const unsigned grid = (unsigned)((n + kGemvRows - 1) / kGemvRows);
    const size_t lds = (size_t)kGemvRows * (k >> 7) * 4;
    if (xs) gemv_g128_kernel<true, 4><<<grid, 256, lds, s>>>(x, xs, q, scales, zeros, bias, out, out_f32, m, n, k);
    else gemv_g128_kernel<false, 4><<<grid, 256, lds, s>>>(x, xs, q, scales, zeros, bias, out, out_f32, m, n, k);
}

}  // namespace pk
