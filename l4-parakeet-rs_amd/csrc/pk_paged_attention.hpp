// Device pieces that the paged attention's kernels share: which keys a row sees, cache
// values as matrix operands, and infinities and NaN in values that some rows do not see.
#pragma once

#include "pk_kernels.hpp"

namespace pk {

constexpr float kNegInf = -__builtin_inff();

// Eight cache values of an operand -> fp16 (e4m3 values are exact in fp16).
template <bool kF8> __device__ __forceinline__ v8h operand(const uint4& raw, int half) {
    if constexpr (kF8) {
        const uint32_t w[2] = {half ? raw.z : raw.x, half ? raw.w : raw.y};
        v8h r;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const v2h a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.0f, false);
            const v2h b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.0f, true);
            r[4 * i] = a[0];
            r[4 * i + 1] = a[1];
            r[4 * i + 2] = b[0];
            r[4 * i + 3] = b[1];
        }
        return r;
    } else {
        return __builtin_bit_cast(v8h, raw);
    }
}

// Nonzero where 16 bytes of cache values hold an infinity or a NaN: all ones under the sign
// (e4m3: exponent and mantissa, its only NaN; fp16: the exponent), so that adding one
// there carries into the sign bit, and nowhere else.
template <bool kF8> __device__ __forceinline__ uint32_t not_finite(const uint4& w) {
    const uint32_t e = kF8 ? 0x7f7f7f7fu : 0x7c007c00u, one = kF8 ? 0x01010101u : 0x04000400u;
    return (((w.x & e) + one) | ((w.y & e) + one) | ((w.z & e) + one) | ((w.w & e) + one)) & (kF8 ? 0x80808080u : 0x80008000u);
}

// Which values of a word are NaN (0), +inf (1) or -inf (2): the cache's 1.0 where so.
template <bool kF8> __device__ __forceinline__ uint32_t odd_ones(uint32_t w, int which) {
    if constexpr (kF8) {
        return (((w & 0x7f7f7f7fu) + 0x01010101u) >> 7 & 0x01010101u) * 0x38u;
    } else {
        const uint32_t odd = (((w & 0x7c007c00u) + 0x04000400u) >> 15) & 0x00010001u;
        const uint32_t nan = odd & (((w & 0x03ff03ffu) + 0x03ff03ffu) >> 10);
        const uint32_t sign = (w >> 15) & 0x00010001u, inf = odd & ~nan;
        return (which == 0 ? nan : (which == 1 ? inf & ~sign : inf & sign)) * 0x3c00u;
    }
}
template <bool kF8> __device__ __forceinline__ uint32_t odd_cleared(uint32_t w) {
    if constexpr (kF8) return w & ~((((w & 0x7f7f7f7fu) + 0x01010101u) >> 7 & 0x01010101u) * 0xffu);
    else return w & ~(((((w & 0x7c007c00u) + 0x04000400u) >> 15) & 0x00010001u) * 0xffffu);
}

// Infinities and NaN in values, where a product with the zero of a masked key would
// spoil rows that do not see that key: each kind is counted over the keys that a row
// sees (bits of `seen`), added to the rows that see one, and cleared from the operand.
// Rare; in place and one kind after the other, so that it needs few registers.
template <bool kF8> __device__ __forceinline__ void add_not_finite(uint4& raw, uint32_t seen, v4f& o) {
#pragma unroll
    for (int kind = 0; kind < (kF8 ? 1 : 3); ++kind) {
        asm volatile("" : "+v"(seen));  // operands are made anew: not kept in registers
        const uint4 ones{odd_ones<kF8>(raw.x, kind), odd_ones<kF8>(raw.y, kind), odd_ones<kF8>(raw.z, kind), odd_ones<kF8>(raw.w, kind)};
        v4f count{};
#pragma unroll
        for (int u = 0; u < (kF8 ? 2 : 1); ++u) {
            uint32_t vis[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) vis[i] = ((seen >> (8 * u + 2 * i) & 1u) | (seen >> (8 * u + 2 * i + 1) & 1u) << 16) * 0x3c00u;
            count = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand<kF8>(ones, u), __builtin_bit_cast(v8h, uint4{vis[0], vis[1], vis[2], vis[3]}), count,
                                                           0, 0, 0);
        }
        const float add = kind == 0 ? __builtin_nanf("") : (kind == 1 ? __builtin_inff() : -__builtin_inff());
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (count[r] > 0.0f) o[r] += add;
        __builtin_amdgcn_sched_barrier(0);
    }
    raw = uint4{odd_cleared<kF8>(raw.x), odd_cleared<kF8>(raw.y), odd_cleared<kF8>(raw.z), odd_cleared<kF8>(raw.w)};
}

// One sequence's view for a tile of 16 query rows.
struct RowTile {
    int start, rows, length, first_pos;  // first_pos: position of the sequence's first new token
};

__device__ __forceinline__ RowTile sequence_of(const PagedArgs& a, int seq) {
    int s = a.starts[seq], e = a.starts[seq + 1], len = a.lengths[seq];
    s = s < 0 ? 0 : (s > a.tokens ? a.tokens : s);
    e = e < s ? s : (e > a.tokens ? a.tokens : e);
    const int most = a.max_pages << a.shift;
    len = len < 0 ? 0 : (len > most ? most : len);
    return {s, (e - s) * a.group, len, len - (e - s)};
}

// The same for a sequence that the whole wave works on, in scalar registers.
__device__ __forceinline__ RowTile wave_sequence(const PagedArgs& a, int seq) {
    const RowTile t = sequence_of(a, seq);
    return {__builtin_amdgcn_readfirstlane(t.start), __builtin_amdgcn_readfirstlane(t.rows), __builtin_amdgcn_readfirstlane(t.length),
            __builtin_amdgcn_readfirstlane(t.first_pos)};
}

// Keys [lo, hi) that a query at `pos` sees.
__device__ __forceinline__ void window(const PagedArgs& a, int pos, int length, int& lo, int& hi) {
    lo = a.left < 0 || pos < a.left ? 0 : pos - a.left;
    hi = a.right < 0 || length - pos <= a.right ? length : pos + a.right + 1;
    if (hi < 0) hi = 0;
}

__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

__device__ __forceinline__ long long uniform(long long v) {
    return (long long)((unsigned long long)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

template <int kN>
__device__ __forceinline__ void store_row(const PagedArgs& a, const RowTile& t, int kvh, int row, int dim, int d0, float total, const float (&v)[kN]) {
    const float inv = total == 0.0f ? 0.0f : a.value_scale / total;
    uint16_t* op = a.out + (size_t)(t.start + row / a.group) * a.out_stride + (size_t)(kvh * a.group + row % a.group) * dim + d0;
    uint32_t w[kN / 2];
#pragma unroll
    for (int j = 0; j < kN / 2; ++j) w[j] = (uint32_t)f2h(v[2 * j] * inv) | ((uint32_t)f2h(v[2 * j + 1] * inv) << 16);
    if constexpr (kN == 8) *(uint4*)op = uint4{w[0], w[1], w[2], w[3]};
    else *(uint2*)op = uint2{w[0], w[1]};
}

// The work of all sequences in a row, in blocks of keys, dealt to `shares` workgroups in
// equal contiguous shares: every workgroup sums the blocks of all sequences (256 threads)
// and finds the sequence that its share begins in.
struct Share {
    long long from, to, size;  // its blocks, and the blocks of a full share
    long long offset;          // blocks of `seq` before `from`
    int seq;
};

template <class Blocks> __device__ __forceinline__ bool deal(const PagedArgs& a, int shares, int least, int index, Blocks blocks_of, Share& out) {
    __shared__ long long wave_total[4], found_offset;
    __shared__ int found_seq;
    const int per = (a.sequences + 255) / 256, s0 = threadIdx.x * per;
    long long mine = 0;
    for (int s = s0; s < s0 + per && s < a.sequences; ++s) mine += blocks_of(sequence_of(a, s));
    long long end = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const long long up = __shfl_up(end, off, 64);
        if ((threadIdx.x & 63) >= off) end += up;
    }
    if ((threadIdx.x & 63) == 63) wave_total[threadIdx.x >> 6] = end;
    __syncthreads();
    for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) end += wave_total[w];
    const long long all = uniform((wave_total[0] + wave_total[1]) + (wave_total[2] + wave_total[3]));
    out.size = (all + shares - 1) / shares;
    if (out.size < least) out.size = least;
    out.from = index * out.size;
    out.to = out.from + out.size < all ? out.from + out.size : all;
    if (out.from >= all) return false;
    if (end - mine <= out.from && out.from < end) {
        long long at = end - mine;
        for (int s = s0;; ++s) {
            const long long n = blocks_of(sequence_of(a, s));
            if (out.from < at + n) {
                found_seq = s;
                found_offset = out.from - at;
                break;
            }
            at += n;
        }
    }
    __syncthreads();
    out.seq = __builtin_amdgcn_readfirstlane(found_seq);
    out.offset = uniform(found_offset);
    return true;
}

// A share boundary leaves an item (rows of a sequence and kv head) in parts: what a
// workgroup has of kRows rows, before the division by the sum.  At most two a workgroup:
// slot 0 for the item that its share begins in, slot 1 for the one that it ends in.
template <int kD, int kRows> struct Part {
    float acc[kRows][kD];
    float top[kRows], total[kRows];
};
struct Join {  // of the workgroup in whose share a divided item begins; count 0: none
    int start, rows, kvh, row0, count, first_slot;
    int pad[2];
};

size_t paged_chunks_workspace(int head_dim);
void launch_paged_chunks(int kind, const PagedArgs& args, int head_dim, bool direct, int max_queries, void* workspace, hipStream_t s);

}  // namespace pk
