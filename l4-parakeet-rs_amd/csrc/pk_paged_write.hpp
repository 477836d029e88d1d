// How new keys and values reach their slots of the paged cache, for the kernels that write it.
#pragma once

#include "pk_kernels.hpp"

namespace pk {

// A 16-byte chunk of eight fp16 values as the cache holds them (fp16: 4 words, e4m3: 2).
template <bool kF8> __device__ __forceinline__ void encode(const uint4& raw, float inverse, uint32_t (&out)[kF8 ? 2 : 4]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (kF8) {
            const uint32_t pair = e4m3x2(h2f((uint16_t)w[j]) * inverse, h2f((uint16_t)(w[j] >> 16)) * inverse);
            if (j & 1) out[j >> 1] |= pair << 16;
            else out[j >> 1] = pair;
        } else {
            out[j] = w[j];
        }
    }
}

struct WriteArgs {
    const uint16_t* key;
    const uint16_t* value;
    const int* slots;
    uint8_t* key_cache;
    uint8_t* value_cache;
    long long key_stride, value_stride, slot_count;
    int tokens, kv_heads, shift;
    float k_inv, v_inv;
};

// First byte of a kv head's keys (or values) in a slot's page.
template <int kD, bool kF8> __device__ __forceinline__ size_t page_base(const WriteArgs& a, int slot, int head) {
    return (((size_t)(slot >> a.shift) * a.kv_heads + head) * kD << a.shift) * (kF8 ? 1 : 2);
}

// Prompts: a workgroup takes 64 tokens of one kv head and turns their values around in
// LDS, so that eight tokens in consecutive slots leave as one store a feature and the
// features' rows of a page leave together.  Workgroups meet where a slot is a multiple of
// 64 (two that wrote parts of a line would do so from two L2s), so a workgroup has up to
// 127 tokens, in turns of 64; groups of eight begin where the first token's slot asks for
// it, and tokens that do not follow each other there are stored one by one.
constexpr int kWriteTokens = 64;

// Without kKeys the values alone: the keys are another kernel's.
template <int kD, bool kF8, bool kKeys> __device__ __forceinline__ void write_tile(const WriteArgs& a, int head, int index) {
    constexpr int kBytes = kF8 ? 1 : 2, kChunks = kD / 8, kWords = kF8 ? 2 : 4, kEach = kWriteTokens * kChunks / 256;
    constexpr int kRow = kD * kBytes / 4 + 1;  // words: the odd one spreads a feature's tokens over the banks
    __shared__ uint32_t tile[kWriteTokens * kRow];
    __shared__ int slot_of[kWriteTokens + 8];
    const int in_page = (1 << a.shift) - 1;
    const auto border = [&](int i) {  // first token of workgroup i
        const int t = i * kWriteTokens;
        if (i == 0 || t >= a.tokens) return i == 0 ? 0 : a.tokens;
        const int s = a.slots[t], b = t + (s < 0 ? 0 : -s & (kWriteTokens - 1));
        return b < a.tokens ? b : a.tokens;
    };
    const int end = border(index + 1);
    for (int t0 = border(index); t0 < end; t0 += kWriteTokens) {
        const int count = end - t0 < kWriteTokens ? end - t0 : kWriteTokens;
        uint4 kraw[kEach] = {}, vraw[kEach] = {};
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = threadIdx.x + 256 * e, t = i / kChunks, f = i % kChunks * 8;
            if (t < count) {
                if constexpr (kKeys) kraw[e] = *(const uint4*)(a.key + (size_t)(t0 + t) * a.key_stride + (size_t)head * kD + f);
                vraw[e] = *(const uint4*)(a.value + (size_t)(t0 + t) * a.value_stride + (size_t)head * kD + f);
            }
        }
        if (threadIdx.x < kWriteTokens + 8) {
            const int s = (int)threadIdx.x < count ? a.slots[t0 + threadIdx.x] : -1;
            slot_of[threadIdx.x] = s < 0 || s >= a.slot_count ? -1 : s;
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = threadIdx.x + 256 * e, t = i / kChunks, f = i % kChunks * 8, slot = slot_of[t];
            uint32_t k[kWords], v[kWords];
            if constexpr (kKeys) encode<kF8>(kraw[e], a.k_inv, k);
            encode<kF8>(vraw[e], a.v_inv, v);
            if (kKeys && slot >= 0) {
                uint8_t* kp = a.key_cache + page_base<kD, kF8>(a, slot, head) + (size_t)((slot & in_page) * kD + f) * kBytes;
                if constexpr (kF8) *(uint2*)kp = uint2{k[0], k[1]};
                else *(uint4*)kp = uint4{k[0], k[1], k[2], k[3]};
            }
#pragma unroll
            for (int w = 0; w < kWords; ++w) tile[t * kRow + f * kBytes / 4 + w] = v[w];
        }
        const auto value_at = [&](int t, int d) {
            if constexpr (kF8) return (uint32_t)((const uint8_t*)(tile + t * kRow))[d];
            else return (uint32_t)((const uint16_t*)(tile + t * kRow))[d];
        };
        const int ahead = slot_of[0] < 0 ? 0 : -slot_of[0] & 7;  // tokens before the first group
        // this thread's group of eight; each wave has all eight groups
        const int first = ahead + (threadIdx.x & 7) * 8, slot = first < kWriteTokens ? slot_of[first] : -1;
        bool together = slot >= 0 && (slot & 7) == 0;
#pragma unroll
        for (int j = 1; j < 8; ++j) together = together && slot_of[first + j] == slot + j;  // (slots behind the tile's are -1)
        const uint32_t groups = (uint32_t)__ballot(together) & 0xffu;
        __syncthreads();
        if (together) {
            uint8_t* vp = a.value_cache + page_base<kD, kF8>(a, slot, head) + (size_t)(slot & in_page) * kBytes;
#pragma unroll
            for (int d = threadIdx.x >> 3; d < kD; d += 32) {
                uint32_t w[kWords] = {};
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j * kBytes / 4] |= value_at(first + j, d) << (8 * kBytes * (j % (4 / kBytes)));
                uint8_t* row = vp + ((size_t)(d * kBytes) << a.shift);
                if constexpr (kF8) *(uint2*)row = uint2{w[0], w[1]};
                else *(uint4*)row = uint4{w[0], w[1], w[2], w[3]};
            }
        }
        if (groups != 0xffu) {
            constexpr int kSide = 256 / kD;  // tokens at once
            const int d = threadIdx.x % kD;
            for (int t = threadIdx.x / kD; t < count; t += kSide) {
                if (t >= ahead && groups >> ((t - ahead) >> 3) & 1u) continue;
                const int one = slot_of[t];
                if (one < 0) continue;
                uint8_t* vp = a.value_cache + page_base<kD, kF8>(a, one, head) + (((size_t)d << a.shift) + (one & in_page)) * kBytes;
                if constexpr (kF8) *vp = (uint8_t)value_at(t, d);
                else *(uint16_t*)vp = (uint16_t)value_at(t, d);
            }
        }
        __syncthreads();  // the tile is read
    }
}

}  // namespace pk
