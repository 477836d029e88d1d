// The paged cache around the attention: planning a step's pages, block tables and
// slots from the requests' lengths, and writing new keys and values into their
// slots.
//
// Cache layout, per page and kv head: keys [page_size x head_dim], values
// [head_dim x page_size].  Values are transposed because the attention's second
// product contracts over keys: a lane then loads the 8 (fp16) or 16 (e4m3)
// consecutive keys of a feature that one matrix operand wants as 16 bytes.
#include "pk_kernels.hpp"

namespace pk {

// Inclusive scans of two values a thread over the workgroup (256 threads).
__device__ __forceinline__ void block_scan(long long& v, long long& u, long long (*wave_total)[2]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const long long v_up = __shfl_up(v, off, 64), u_up = __shfl_up(u, off, 64);
        if (lane >= off) {
            v += v_up;
            u += u_up;
        }
    }
    if (lane == 63) {
        wave_total[wave][0] = v;
        wave_total[wave][1] = u;
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
        v += wave_total[w][0];
        u += wave_total[w][1];
    }
}

// First index whose inclusive end is above i.
__device__ __forceinline__ int owner_of(const int* ends, int count, int i) {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid] > i) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// Every workgroup scans all requests (they are few next to the slots; a thread has up to
// kPer) and keeps the ends of their tokens and new pages in LDS; slots and table entries
// are then found by bisection, spread over the whole grid, so that one launch does it
// without an exchange between workgroups.  Bound by latency: 8 requests 3.0 us, about a
// launch; 2000 requests and 65536 slots 8.4 us: the lengths' loads, a scan, the
// bisection's eleven dependent LDS reads, a table entry and the store, one after another.
template <int kPer>
__global__ __launch_bounds__(256) void page_plan_kernel(const int* __restrict__ held, const int* __restrict__ added,
                                                        const int* __restrict__ free_pages, const int* __restrict__ free_range,
                                                        int free_capacity, int* table, int* __restrict__ starts, int* __restrict__ lengths,
                                                        int* __restrict__ slots, int* __restrict__ positions, int* __restrict__ info,
                                                        int requests, int max_pages, int shift, int capacity) {
    extern __shared__ int ends[];  // [requests] tokens, [requests] new pages
    __shared__ long long wave_total[4][2];
    __shared__ int flags;
    int* page_ends = ends + requests;
    const int per = (requests + 255) / 256, first = threadIdx.x * per;
    const int round = (1 << shift) - 1;
    if (threadIdx.x == 0) flags = 0;
    // a thread's lengths, all asked for at once
    const int begin = free_range[0], end = free_range[1] < free_capacity ? free_range[1] : free_capacity;
    int mine_held[kPer], mine_added[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const bool there = j < per && first + j < requests;
        mine_held[j] = there ? held[first + j] : 0;
        mine_added[j] = there ? added[first + j] : 0;
    }
    long long tokens = 0, pages = 0;
    int bad = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        if (j >= per) break;
        const long long h = mine_held[j], a = mine_added[j];
        if (h < 0 || a < 0) bad |= 8;
        const long long want = (h + a + round) >> shift;
        if (want > max_pages) bad |= 2;
        tokens += a;
        pages += want - ((h + round) >> shift);
    }
    long long token_end = tokens, page_end = pages;
    block_scan(token_end, page_end, wave_total);
    if (bad) atomicOr(&flags, bad);  // behind the scan's barrier, which flags = 0 stands before
    const long long all_tokens = wave_total[0][0] + wave_total[1][0] + wave_total[2][0] + wave_total[3][0];
    const long long all_pages = wave_total[0][1] + wave_total[1][1] + wave_total[2][1] + wave_total[3][1];
    __syncthreads();
    int status = flags;
    if (begin < 0) status |= 8;
    if (all_tokens > capacity) status |= 4;
    if (all_pages > (long long)end - begin) status |= 1;
    const int n_tokens = status ? 0 : (int)all_tokens, n_pages = status ? 0 : (int)all_pages;
    if (!status) {
        int t = (int)(token_end - tokens), p = (int)(page_end - pages);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if (j >= per || first + j >= requests) break;
            const int h = mine_held[j], a = mine_added[j];
            t += a;
            p += (int)((((long long)h + a + round) >> shift) - (((long long)h + round) >> shift));
            ends[first + j] = t;
            page_ends[first + j] = p;
        }
    }
    __syncthreads();

    // unsigned: behind the last of 2^31 - 1 slots the next index is still one that ends the loop
    const uint32_t at = blockIdx.x * 256 + threadIdx.x, step = gridDim.x * 256;
    for (uint32_t i = at; i < (uint32_t)requests; i += step) {
        starts[i + 1] = status ? 0 : ends[i];
        lengths[i] = status ? held[i] : held[i] + added[i];
    }
    if (at == 0) {
        starts[0] = 0;
        info[0] = n_tokens;
        info[1] = n_pages;
        info[2] = status;
        info[3] = 0;
    }
    for (uint32_t i = at; i < (uint32_t)n_pages; i += step) {
        const int r = owner_of(page_ends, requests, (int)i);
        const int have = (held[r] + round) >> shift;
        table[(size_t)r * max_pages + have + (int)i - (r ? page_ends[r - 1] : 0)] = free_pages[begin + (int)i];
    }
    for (uint32_t t = at; t < (uint32_t)capacity; t += step) {
        int slot = -1, pos = 0;
        if (t < (uint32_t)n_tokens) {
            const int r = owner_of(ends, requests, (int)t);
            const int h = held[r], have = (int)(((long long)h + round) >> shift);
            pos = h + (int)t - (r ? ends[r - 1] : 0);
            const int page = pos >> shift;
            // a page of this step is read from the free list: the table entry is another workgroup's to write
            const int id = page < have ? table[(size_t)r * max_pages + page] : free_pages[begin + (r ? page_ends[r - 1] : 0) + page - have];
            const long long wide = ((long long)id << shift) | (pos & round);
            slot = id < 0 || wide > 0x7fffffffll ? -1 : (int)wide;
        }
        slots[t] = slot;
        if (positions) positions[t] = pos;
    }
}

void launch_page_plan(const int* held, const int* added, const int* free_pages, const int* free_range, int free_capacity, int* table,
                      int* starts, int* lengths, int* slots, int* positions, int* info, int requests, int max_pages, int page_shift,
                      int capacity, hipStream_t s) {
    const int work = capacity > requests ? capacity : requests;
    const int grid = work > 65536 - 256 ? 256 : (work > 256 ? (work + 255) / 256 : 1);
    const auto launch = [&](auto kernel) {
        kernel<<<grid, 256, (size_t)requests * 8, s>>>(held, added, free_pages, free_range, free_capacity, table, starts, lengths, slots, positions,
                                                       info, requests, max_pages, page_shift, capacity);
    };
    // One request a thread without the others' sixteen-fold loops: 8 requests 3.0 us against 4.0.
    if (requests <= 256) launch(page_plan_kernel<1>);
    else launch(page_plan_kernel<kMostPlanRequests / 256>);
}

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

// Single tokens of many sequences: a thread takes 8 features of a token's key and value.
// Their values lie in as many rows of a page as they are features.
template <int kD, bool kF8> __global__ __launch_bounds__(256) void paged_cache_write_kernel(WriteArgs a) {
    constexpr int kBytes = kF8 ? 1 : 2, kChunks = kD / 8;
    const int chunks = a.kv_heads * kChunks;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const int t = (int)(i / chunks), c = (int)(i % chunks);
    if (t >= a.tokens) return;
    const int slot = a.slots[t];
    if (slot < 0 || slot >= a.slot_count) return;
    const int f = c % kChunks * 8, off = slot & ((1 << a.shift) - 1);
    const size_t base = page_base<kD, kF8>(a, slot, c / kChunks);
    uint32_t k[kF8 ? 2 : 4], v[kF8 ? 2 : 4];
    encode<kF8>(*(const uint4*)(a.key + (size_t)t * a.key_stride + (size_t)c * 8), a.k_inv, k);
    encode<kF8>(*(const uint4*)(a.value + (size_t)t * a.value_stride + (size_t)c * 8), a.v_inv, v);
    uint8_t* kp = a.key_cache + base + (size_t)(off * kD + f) * kBytes;
    uint8_t* vp = a.value_cache + base + (((size_t)f << a.shift) + off) * kBytes;
    if constexpr (kF8) *(uint2*)kp = uint2{k[0], k[1]};
    else *(uint4*)kp = uint4{k[0], k[1], k[2], k[3]};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if constexpr (kF8) vp[(size_t)j << a.shift] = (uint8_t)(v[j >> 2] >> (8 * (j & 3)));
        else ((uint16_t*)vp)[(size_t)j << a.shift] = (uint16_t)(v[j >> 1] >> (16 * (j & 1)));
    }
}

// Prompts: a workgroup takes 64 tokens of one kv head and turns their values around in
// LDS, so that eight tokens in consecutive slots leave as one store a feature and the
// features' rows of a page leave together.  Workgroups meet where a slot is a multiple of
// 64 (two that wrote parts of a line would do so from two L2s), so a workgroup has up to
// 127 tokens, in turns of 64; groups of eight begin where the first token's slot asks for
// it, and tokens that do not follow each other there are stored one by one.
constexpr int kWriteTokens = 64;

template <int kD, bool kF8> __global__ __launch_bounds__(256) void paged_cache_write_tile_kernel(WriteArgs a) {
    constexpr int kBytes = kF8 ? 1 : 2, kChunks = kD / 8, kWords = kF8 ? 2 : 4, kEach = kWriteTokens * kChunks / 256;
    constexpr int kRow = kD * kBytes / 4 + 1;  // words: the odd one spreads a feature's tokens over the banks
    __shared__ uint32_t tile[kWriteTokens * kRow];
    __shared__ int slot_of[kWriteTokens + 8];
    const int head = blockIdx.x, in_page = (1 << a.shift) - 1;
    const auto border = [&](int i) {  // first token of workgroup i
        const int t = i * kWriteTokens;
        if (i == 0 || t >= a.tokens) return i == 0 ? 0 : a.tokens;
        const int s = a.slots[t], b = t + (s < 0 ? 0 : -s & (kWriteTokens - 1));
        return b < a.tokens ? b : a.tokens;
    };
    const int end = border(blockIdx.y + 1);
    for (int t0 = border(blockIdx.y); t0 < end; t0 += kWriteTokens) {
        const int count = end - t0 < kWriteTokens ? end - t0 : kWriteTokens;
        uint4 kraw[kEach] = {}, vraw[kEach] = {};
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = threadIdx.x + 256 * e, t = i / kChunks, f = i % kChunks * 8;
            if (t < count) {
                kraw[e] = *(const uint4*)(a.key + (size_t)(t0 + t) * a.key_stride + (size_t)head * kD + f);
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
            encode<kF8>(kraw[e], a.k_inv, k);
            encode<kF8>(vraw[e], a.v_inv, v);
            if (slot >= 0) {
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

// Fewer tokens than this are mostly single ones, and too few tiles to fill the GPU (8 heads of
// 128, one prompt, e4m3 / fp16: 1024 tokens 8.3 / 9.7 us against 9.7 / 8.2 for tiles, 2048 15.3 /
// 15.8 against 11.2 / 10.2, 16000 117 / 130 against 28 / 38, 3.5 TB/s).  What tiles are short of
// a copy's rate is a chain: a border's slot, then the rows, then the stores, in workgroups that
// the GPU holds hardly more than once over, so that reading and writing barely overlap.
constexpr int kTileTokens = 1536;

template <int kD, bool kF8> static void launch_write(const WriteArgs& a, hipStream_t s) {
    if (a.tokens < kTileTokens) {
        const unsigned grid = (unsigned)(((long long)a.tokens * a.kv_heads * (kD / 8) + 255) / 256);
        paged_cache_write_kernel<kD, kF8><<<grid, 256, 0, s>>>(a);
    } else {
        const dim3 grid((unsigned)a.kv_heads, (unsigned)((a.tokens + kWriteTokens - 1) / kWriteTokens));
        paged_cache_write_tile_kernel<kD, kF8><<<grid, 256, 0, s>>>(a);
    }
}

void launch_paged_cache_write(int kind, const uint16_t* key, const uint16_t* value, long long key_stride, long long value_stride,
                              const int* slots, void* key_cache, void* value_cache, int tokens, int kv_heads, int head_dim, int page_shift,
                              int pages, float k_inv, float v_inv, hipStream_t s) {
    const WriteArgs a{key, value, slots, (uint8_t*)key_cache, (uint8_t*)value_cache, key_stride, value_stride, (long long)pages << page_shift,
                      tokens, kv_heads, page_shift, k_inv, v_inv};
    if (head_dim == 128) {
        if (kind == 1) launch_write<128, true>(a, s);
        else launch_write<128, false>(a, s);
    } else {
        if (kind == 1) launch_write<64, true>(a, s);
        else launch_write<64, false>(a, s);
    }
}

}  // namespace pk
