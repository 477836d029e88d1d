// Device pieces that the paged attention's kernels share: which keys a row sees, cache
// values as matrix operands, and infinities and NaN in values that some rows do not see.
#pragma once

#include "pk_kernels.hpp"
#include "pk_paged_deal.hpp"

namespace pk {

constexpr float kNegInf = -__builtin_inff();

// The weight of sums whose maximum is `below` (factors of two) under the new one: not zero, which
// would make NaN of an infinity among them; sums of 2^61 at most vanish all the same.
__device__ __forceinline__ float weight_of(float below) { return __builtin_fmaxf(__builtin_amdgcn_exp2f(below), 0x1p-126f); }

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

template <bool kF8> __device__ __forceinline__ uint32_t odd_cleared(uint32_t w) {
    if constexpr (kF8) return w & ~((((w & 0x7f7f7f7fu) + 0x01010101u) >> 7 & 0x01010101u) * 0xffu);
    else return w & ~(((((w & 0x7c007c00u) + 0x04000400u) >> 15) & 0x00010001u) * 0xffffu);
}
// All ones in the halves of a word of fp16 values that are infinities.
__device__ __forceinline__ uint32_t infinite(uint32_t w) {
    return ((w & 0x7fffu) == 0x7c00u ? 0xffffu : 0u) | ((w & 0x7fff0000u) == 0x7c000000u ? 0xffff0000u : 0u);
}

// Infinities and NaN in values: a product with the zero of a masked key would spoil rows
// that do not see that key.  At the edges of the rows' keys they are therefore taken out
// of the operands, and which outputs they belong to (those of the rows that do see the
// key) is noted in LDS, for the end; so are infinities where a probability is one that fp16
// rounds to zero, of which they would make NaN.  Rare, and kept out of the way of everything else.
template <int kD, int kRows> struct Odd {
    static constexpr int kWords = (kRows + 31) / 32;
    uint32_t any;
    uint32_t marks[3][kD][kWords];  // NaN, +inf, -inf: bit of the row

    __device__ __forceinline__ void clear(int threads) {
        for (int i = threadIdx.x; i < 3 * kD * kWords; i += threads) (&marks[0][0][0])[i] = 0;
        if (threadIdx.x == 0) any = 0;
    }
    // 16 bytes of values of feature d from key `key` on, a lane; window(r, lo, hi): the keys that row r of this lane sees.
    // inside: all rows see these keys, and a NaN may stay (so may all of e4m3, which has no infinity).
    template <bool kF8, class Window> __device__ __forceinline__ void take(uint4& raw, int d, int key, bool inside, Window window) {
        if (kF8 && inside) return;
        const int lane = threadIdx.x & 63;
        unsigned long long todo = __ballot(not_finite<kF8>(raw) != 0);
        if (inside && todo) todo = __ballot((infinite(raw.x) | infinite(raw.y) | infinite(raw.z) | infinite(raw.w)) != 0);
        while (__builtin_expect(todo != 0, 0)) {
            const int from = __builtin_ctzll(todo);
            todo &= todo - 1;
            const uint32_t w[4] = {(uint32_t)__builtin_amdgcn_readlane((int)raw.x, from), (uint32_t)__builtin_amdgcn_readlane((int)raw.y, from),
                                   (uint32_t)__builtin_amdgcn_readlane((int)raw.z, from), (uint32_t)__builtin_amdgcn_readlane((int)raw.w, from)};
            const int feature = __builtin_amdgcn_readlane(d, from), first = __builtin_amdgcn_readlane(key, from);
#pragma unroll 1
            for (int j = 0; j < (kF8 ? 16 : 8); ++j) {
                const int at = kF8 ? j >> 2 : j >> 1;
                const uint32_t word = at == 0 ? w[0] : (at == 1 ? w[1] : (at == 2 ? w[2] : w[3]));
                const uint32_t v = kF8 ? word >> (8 * (j & 3)) & 0xffu : word >> (16 * (j & 1)) & 0xffffu;
                if (kF8 ? (v & 0x7fu) != 0x7fu : (v & 0x7c00u) != 0x7c00u) continue;
                const int kind = kF8 || v & 0x3ffu ? 0 : (v >> 15 ? 2 : 1);
                if (inside && kind == 0) continue;
                for (int r = lane; r < kRows; r += 64) {
                    int lo, hi;
                    window(r, lo, hi);
                    if (first + j >= lo && first + j < hi) atomicOr(&marks[kind][feature][r >> 5], 1u << (r & 31));
                }
                if (lane == 0) any = 1;
            }
        }
        if (inside) raw = uint4{raw.x & ~infinite(raw.x), raw.y & ~infinite(raw.y), raw.z & ~infinite(raw.z), raw.w & ~infinite(raw.w)};
        else raw = uint4{odd_cleared<kF8>(raw.x), odd_cleared<kF8>(raw.y), odd_cleared<kF8>(raw.z), odd_cleared<kF8>(raw.w)};
    }
    // What row r's sum of feature d becomes.
    __device__ __forceinline__ float put(float v, int r, int d) const {
        if (marks[1][d][r >> 5] >> (r & 31) & 1u) v += __builtin_inff();
        if (marks[2][d][r >> 5] >> (r & 31) & 1u) v -= __builtin_inff();
        return marks[0][d][r >> 5] >> (r & 31) & 1u ? __builtin_nanf("") : v;
    }
};

__device__ __forceinline__ RowTile sequence_of(const PagedArgs& a, int s, int e, int len) {
    s = s < 0 ? 0 : (s > a.tokens ? a.tokens : s);
    e = e < s ? s : (e > a.tokens ? a.tokens : e);
    const int most = a.max_pages << a.shift;
    len = len < 0 ? 0 : (len > most ? most : len);
    return {s, (e - s) * a.group, len, len - (e - s)};
}
__device__ __forceinline__ RowTile sequence_of(const PagedArgs& a, int seq) { return sequence_of(a, a.starts[seq], a.starts[seq + 1], a.lengths[seq]); }

// What a launch does not write is read through the scalar cache where a whole wave needs it:
// such loads do not wait behind the cache's, which return in order.
typedef const __attribute__((address_space(4))) int* ScalarInts;
__device__ __forceinline__ int scalar_at(const int* p, int index) {  // 0 <= index < 2^30: the byte offset is one register
    typedef const __attribute__((address_space(4))) uint8_t* ScalarBytes;
    return *(ScalarInts)((ScalarBytes)(uintptr_t)p + (uint32_t)(__builtin_amdgcn_readfirstlane(index) << 2));
}

// The same for a sequence that the whole wave works on, in scalar registers.
__device__ __forceinline__ RowTile wave_sequence(const PagedArgs& a, int seq) {
    return sequence_of(a, scalar_at(a.starts, seq), scalar_at(a.starts, seq + 1), scalar_at(a.lengths, seq));
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

// A workgroup's share of the work: every workgroup (kThreads threads) sums the blocks of all
// sequences and finds the sequences that its share begins and ends in.
struct Share {
    long long from, to, all;  // its blocks, and the blocks of all shares
    long long offset;          // blocks of `seq` before `from`
    long long last_offset;     // and of `last_seq` before `to` - 1
    int seq, last_seq;
};

__device__ __forceinline__ long long lane_value(long long v, int lane) {
    return (long long)((unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
                       (uint32_t)__builtin_amdgcn_readlane((int)v, lane));
}

// Up to 64 sequences: one a lane, each wave for itself (one sequence of 1900 e4m3 keys 12.4 us
// against 12.8 through LDS, 16 of them 19.7 and 20.2).
template <int kShares, int kLeast, class Blocks> __device__ __forceinline__ bool deal_wave(const PagedArgs& a, int index, Blocks blocks_of, Share& out) {
    const int lane = threadIdx.x & 63;
    const long long mine = lane < a.sequences ? blocks_of(sequence_of(a, lane)) : 0;
    long long end = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const long long up = __shfl_up(end, off, 64);
        if (lane >= off) end += up;
    }
    const long long all = lane_value(end, 63);
    out.all = all;
    out.from = uniform(share_begin<kShares, kLeast>(all, index));
    out.to = uniform(share_begin<kShares, kLeast>(all, index + 1));
    if (out.from >= out.to) return false;
    const long long at = end - mine, last = out.to - 1;
    out.seq = __builtin_ctzll(__ballot(at <= out.from && out.from < end));
    out.last_seq = __builtin_ctzll(__ballot(at <= last && last < end));
    out.offset = out.from - lane_value(at, out.seq);
    out.last_offset = last - lane_value(at, out.last_seq);
    return true;
}

// (No barrier with up to 64 sequences.)
template <int kThreads, int kShares, int kLeast, class Blocks> __device__ __forceinline__ bool deal(const PagedArgs& a, int index, Blocks blocks_of, Share& out) {
    if (a.sequences <= 64) return deal_wave<kShares, kLeast>(a, index, blocks_of, out);
    __shared__ long long wave_total[kThreads / 64], found_offset[2];
    __shared__ int found_seq[2];
    const int per = (a.sequences + kThreads - 1) / kThreads, s0 = threadIdx.x * per;
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
    long long all = 0;
    for (int w = 0; w < kThreads / 64; ++w) all += wave_total[w];
    out.all = all = uniform(all);
    out.from = uniform(share_begin<kShares, kLeast>(all, index));
    out.to = uniform(share_begin<kShares, kLeast>(all, index + 1));
    if (out.from >= out.to) return false;
    const long long last = out.to - 1;
    if (end - mine <= last && out.from < end) {  // this thread's sequences hold blocks of the share
        long long at = end - mine;
        for (int s = s0; s < s0 + per && s < a.sequences; ++s) {
            const long long n = blocks_of(sequence_of(a, s));
            if (at <= out.from && out.from < at + n) {
                found_seq[0] = s;
                found_offset[0] = out.from - at;
            }
            if (at <= last && last < at + n) {
                found_seq[1] = s;
                found_offset[1] = last - at;
            }
            at += n;
        }
    }
    __syncthreads();
    out.seq = __builtin_amdgcn_readfirstlane(found_seq[0]);
    out.offset = uniform(found_offset[0]);
    out.last_seq = __builtin_amdgcn_readfirstlane(found_seq[1]);
    out.last_offset = uniform(found_offset[1]);
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
