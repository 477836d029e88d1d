// Residual addition, root-mean-square norm and per-row 8-bit quantization in
// one pass over the row:
//   h = x + r,  residual_out = fp16(h),  y = h / sqrt(mean(h^2) + eps) * w,
//   scale = max|y| / 448 (INT8: / 127),  q = e4m3(y / scale) (INT8: rne).
// h, the sum of squares and y stay in fp32: the only roundings are the stored
// residual stream's and the codes'.  A row is read once and held in registers
// between its two reductions.  Bound by HBM: 45000 x 1024 with a residual in and
// out, e4m3 (323 MB), 59 us, 5.5 TB/s; one row 2.7 us, about a launch.
#include "pk_kernels.hpp"

namespace pk {

// Maximum of the bits of non-negative floats: NaN > inf > every finite value,
// so one comparison afterwards tells a row that cannot be scaled.
__device__ __forceinline__ uint32_t umax_level(uint32_t v, int off) {
    uint32_t a = v, b;
    if (off <= 8) {
        b = (uint32_t)partner((int)v, off);
    } else {
        int x, y;
        pair_of((int)v, off, x, y);
        a = (uint32_t)x;
        b = (uint32_t)y;
    }
    return a > b ? a : b;
}

// kLanes lanes a row (64: a wave, 256: the workgroup), kChunks 8-feature chunks
// a lane: width <= 8 * kLanes * kChunks.
template <bool kInt8, int kLanes, int kChunks>
__global__ __launch_bounds__(256) void rms_norm_quantize_kernel(const uint16_t* in, const uint16_t* residual,
                                                                const uint16_t* __restrict__ weight, uint16_t* residual_out,
                                                                uint8_t* __restrict__ out, float* __restrict__ scales, int rows,
                                                                int width, float epsilon) {
    constexpr int kRows = 256 / kLanes;
    __shared__ float part_sum[4];
    __shared__ uint32_t part_max[4];
    const int lane = threadIdx.x % kLanes;
    const int row = blockIdx.x * kRows + threadIdx.x / kLanes;
    if (kLanes == 64 && row >= rows) return;  // whole waves; the 256-lane form has one row a workgroup
    const size_t base = (size_t)row * width;

    float h[kChunks][8];
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int f = (c * kLanes + lane) * 8;
        uint4 x{}, r{};
        if (f < width) {
            x = *(const uint4*)(in + base + f);
            if (residual) r = *(const uint4*)(residual + base + f);
        }
        const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, rw[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            h[c][j] = h2f((uint16_t)(xw[j >> 1] >> (16 * (j & 1)))) + h2f((uint16_t)(rw[j >> 1] >> (16 * (j & 1))));
            sum = __builtin_fmaf(h[c][j], h[c][j], sum);
        }
        if (residual_out && f < width) {
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = (uint32_t)f2h(h[c][2 * j]) | ((uint32_t)f2h(h[c][2 * j + 1]) << 16);
            *(uint4*)(residual_out + base + f) = uint4{o[0], o[1], o[2], o[3]};
        }
    }
    sum = sum_desc<64>(sum);
    if constexpr (kLanes == 256) {
        if ((threadIdx.x & 63) == 0) part_sum[threadIdx.x >> 6] = sum;
        __syncthreads();
        sum = (part_sum[0] + part_sum[1]) + (part_sum[2] + part_sum[3]);
    }
    const float mean = sum / (float)width + epsilon;
    const float rstd = mean > 0.0f ? 1.0f / sqrtf(mean) : (mean == 0.0f ? 0.0f : mean);  // NaN stays NaN; all zero with eps 0: zeros

    uint32_t most = 0;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int f = (c * kLanes + lane) * 8;
        uint4 g{};
        if (f < width) g = *(const uint4*)(weight + f);
        const uint32_t gw[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            h[c][j] = (h[c][j] * rstd) * h2f((uint16_t)(gw[j >> 1] >> (16 * (j & 1))));
            const uint32_t bits = __float_as_uint(h[c][j]) & 0x7fffffffu;
            if (f < width) most = bits > most ? bits : most;
        }
    }
#pragma unroll
    for (int off = 1; off <= 32; off <<= 1) most = umax_level(most, off);
    if constexpr (kLanes == 256) {
        if ((threadIdx.x & 63) == 0) part_max[threadIdx.x >> 6] = most;
        __syncthreads();
        const uint32_t a = part_max[0] > part_max[1] ? part_max[0] : part_max[1];
        const uint32_t b = part_max[2] > part_max[3] ? part_max[2] : part_max[3];
        most = a > b ? a : b;
    }
    const bool bad = most >= 0x7f800000u;
    const float scale = bad ? __builtin_nanf("") : (most == 0 ? 1.0f : __uint_as_float(most) / (kInt8 ? 127.0f : 448.0f));
    const float inv = 1.0f / scale;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int f = (c * kLanes + lane) * 8;
        if (f >= width) break;
        uint32_t o[2] = {0, 0};
        if constexpr (kInt8) {
            if (!bad) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    o[j >> 2] |= (uint32_t)(rne_clamp(div_rn(h[c][j], scale, inv), -127, 127) & 0xff) << (8 * (j & 3));
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                o[j >> 1] |= (bad ? 0x7f7fu : e4m3x2(div_rn(h[c][2 * j], scale, inv), div_rn(h[c][2 * j + 1], scale, inv))) << (16 * (j & 1));
        }
        *(uint2*)(out + base + f) = uint2{o[0], o[1]};
    }
    if (lane == 0) scales[row] = scale;
}

// A launch has fewer than 2^32 threads in a dimension (a larger grid wraps, without an
// error): more rows than this, of 64 or 256 threads, go in several launches.
constexpr int kMostRows = 1 << 23;

template <bool kInt8>
static void launch_rms(const uint16_t* in, const uint16_t* residual, const uint16_t* w, uint16_t* r_out, uint8_t* out, float* scales,
                       int rows, int width, float eps, hipStream_t s) {
    const unsigned waves = (unsigned)((rows + 3) / 4);
    // A wave a row up to 1024 features: 45000 rows take 60 us, with a workgroup each 85 (one row
    // 3.0 and 2.7).  Above, a workgroup: 12000 x 2048 35 us against 38 for waves, x 4096 64 and 76,
    // one row of 4096 3.3 and 6.5.
#define PK_RMS(lanes, chunks, grid) \
    rms_norm_quantize_kernel<kInt8, lanes, chunks><<<grid, 256, 0, s>>>(in, residual, w, r_out, out, scales, rows, width, eps)
    if (width <= 512) PK_RMS(64, 1, waves);
    else if (width <= 1024) PK_RMS(64, 2, waves);
    else if (width <= 2048) PK_RMS(256, 1, (unsigned)rows);
    else if (width <= 4096) PK_RMS(256, 2, (unsigned)rows);
    else if (width <= 8192) PK_RMS(256, 4, (unsigned)rows);
    else PK_RMS(256, 8, (unsigned)rows);
#undef PK_RMS
}

void launch_rms_norm_quantize(int kind, const uint16_t* in, const uint16_t* residual, const uint16_t* w, uint16_t* r_out, void* out,
                              float* scales, int rows, int width, float eps, hipStream_t s) {
    for (int done = 0; rows > 0; done = kMostRows) {
        const size_t skip = (size_t)done * width;
        in += skip;
        if (residual) residual += skip;
        if (r_out) r_out += skip;
        out = (uint8_t*)out + skip;
        scales += done;
        const int part = rows < kMostRows ? rows : kMostRows;
        if (kind == 1) launch_rms<true>(in, residual, w, r_out, (uint8_t*)out, scales, part, width, eps, s);
        else launch_rms<false>(in, residual, w, r_out, (uint8_t*)out, scales, part, width, eps, s);
        rows -= part;
    }
}

}  // namespace pk
