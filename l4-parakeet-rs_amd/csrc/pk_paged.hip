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

// Inclusive scan of one value a thread over the workgroup (256 threads).
__device__ __forceinline__ long long block_scan(long long v, long long* wave_total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const long long up = __shfl_up(v, off, 64);
        if (lane >= off) v += up;
    }
    if (lane == 63) wave_total[wave] = v;
    __syncthreads();
    for (int w = 0; w < wave; ++w) v += wave_total[w];
    __syncthreads();
    return v;
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

// Every workgroup scans all requests (they are few next to the slots) and keeps
// the ends of their tokens and new pages in LDS; slots and table entries are then
// found by bisection, spread over the whole grid, so that one launch does it
// without an exchange between workgroups.
__global__ __launch_bounds__(256) void page_plan_kernel(const int* __restrict__ held, const int* __restrict__ added,
                                                        const int* __restrict__ free_pages, const int* __restrict__ free_range,
                                                        int free_capacity, int* table, int* __restrict__ starts, int* __restrict__ lengths,
                                                        int* __restrict__ slots, int* __restrict__ positions, int* __restrict__ info,
                                                        int requests, int max_pages, int shift, int capacity) {
    extern __shared__ int ends[];  // [requests] tokens, [requests] new pages
    __shared__ long long wave_total[4];
    __shared__ int flags;
    int* page_ends = ends + requests;
    const int per = (requests + 255) / 256, first = threadIdx.x * per;
    const int round = (1 << shift) - 1;
    if (threadIdx.x == 0) flags = 0;
    __syncthreads();

    long long tokens = 0, pages = 0;
    int bad = 0;
    for (int i = first; i < first + per && i < requests; ++i) {
        const long long h = held[i], a = added[i];
        if (h < 0 || a < 0) bad |= 8;
        const long long want = (h + a + round) >> shift;
        if (want > max_pages) bad |= 2;
        tokens += a;
        pages += want - ((h + round) >> shift);
    }
    if (bad) atomicOr(&flags, bad);
    const long long token_end = block_scan(tokens, wave_total), page_end = block_scan(pages, wave_total);
    __shared__ long long totals[2];
    if (threadIdx.x == 255) {
        totals[0] = token_end;
        totals[1] = page_end;
    }
    const int begin = free_range[0], end = free_range[1] < free_capacity ? free_range[1] : free_capacity;
    __syncthreads();
    int status = flags;
    if (begin < 0) status |= 8;
    if (totals[0] > capacity) status |= 4;
    if (totals[1] > (long long)end - begin) status |= 1;
    const int n_tokens = status ? 0 : (int)totals[0], n_pages = status ? 0 : (int)totals[1];
    if (!status) {
        int t = (int)(token_end - tokens), p = (int)(page_end - pages);
        for (int i = first; i < first + per && i < requests; ++i) {
            const int h = held[i], a = added[i];
            t += a;
            p += (int)((((long long)h + a + round) >> shift) - (((long long)h + round) >> shift));
            ends[i] = t;
            page_ends[i] = p;
        }
    }
    __syncthreads();

    const int at = blockIdx.x * 256 + threadIdx.x, step = gridDim.x * 256;
    for (int i = at; i < requests; i += step) {
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
    for (int i = at; i < n_pages; i += step) {
        const int r = owner_of(page_ends, requests, i);
        const int have = (held[r] + round) >> shift;
        table[(size_t)r * max_pages + have + i - (r ? page_ends[r - 1] : 0)] = free_pages[begin + i];
    }
    for (int t = at; t < capacity; t += step) {
        int slot = -1, pos = 0;
        if (t < n_tokens) {
            const int r = owner_of(ends, requests, t);
            const int h = held[r], have = (int)(((long long)h + round) >> shift);
            pos = h + t - (r ? ends[r - 1] : 0);
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
    const int grid = work <= 256 ? 1 : (work + 255) / 256 < 256 ? (work + 255) / 256 : 256;
    page_plan_kernel<<<grid, 256, (size_t)requests * 8, s>>>(held, added, free_pages, free_range, free_capacity, table, starts, lengths, slots,
                                                             positions, info, requests, max_pages, page_shift, capacity);
}

// One 8-feature chunk of a token's key and value a thread.
template <bool kF8>
__global__ __launch_bounds__(256) void paged_cache_write_kernel(const uint16_t* __restrict__ key, const uint16_t* __restrict__ value,
                                                                long long key_stride, long long value_stride,
                                                                const int* __restrict__ slots, uint8_t* __restrict__ key_cache,
                                                                uint8_t* __restrict__ value_cache, int tokens, int chunks, int d_chunks,
                                                                int shift, long long slot_count, float k_inv, float v_inv) {
    constexpr int kBytes = kF8 ? 1 : 2;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const int t = (int)(i / chunks), c = (int)(i % chunks);
    if (t >= tokens) return;
    const int slot = slots[t];
    if (slot < 0 || slot >= slot_count) return;
    const int head = c / d_chunks, f = (c % d_chunks) * 8, d = d_chunks * 8, kv_heads = chunks / d_chunks;
    const int off = slot & ((1 << shift) - 1);
    const size_t page = ((size_t)(slot >> shift) * kv_heads + head) * ((size_t)d << shift);  // elements
    const uint4 k = *(const uint4*)(key + (size_t)t * key_stride + (size_t)c * 8);
    const uint4 v = *(const uint4*)(value + (size_t)t * value_stride + (size_t)c * 8);
    const uint32_t kw[4] = {k.x, k.y, k.z, k.w}, vw[4] = {v.x, v.y, v.z, v.w};
    uint8_t* kp = key_cache + (page + (size_t)off * d + f) * kBytes;
    uint8_t* vp = value_cache + (page + ((size_t)f << shift) + off) * kBytes;
    if constexpr (kF8) {
        uint32_t o[4], u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o[j] = e4m3x2(h2f((uint16_t)kw[j]) * k_inv, h2f((uint16_t)(kw[j] >> 16)) * k_inv);
            u[j] = e4m3x2(h2f((uint16_t)vw[j]) * v_inv, h2f((uint16_t)(vw[j] >> 16)) * v_inv);
        }
        *(uint2*)kp = uint2{o[0] | (o[1] << 16), o[2] | (o[3] << 16)};
#pragma unroll
        for (int j = 0; j < 8; ++j) vp[(size_t)j << shift] = (uint8_t)(u[j >> 1] >> (8 * (j & 1)));
    } else {
        *(uint4*)kp = k;
#pragma unroll
        for (int j = 0; j < 8; ++j) ((uint16_t*)vp)[(size_t)j << shift] = (uint16_t)(vw[j >> 1] >> (16 * (j & 1)));
    }
}

void launch_paged_cache_write(int kind, const uint16_t* key, const uint16_t* value, long long key_stride, long long value_stride,
                              const int* slots, void* key_cache, void* value_cache, int tokens, int kv_heads, int head_dim, int page_shift,
                              int pages, float k_inv, float v_inv, hipStream_t s) {
    const int chunks = kv_heads * head_dim / 8;
    const unsigned grid = (unsigned)(((long long)tokens * chunks + 255) / 256);
    const long long slot_count = (long long)pages << page_shift;
    if (kind == 1)
        paged_cache_write_kernel<true><<<grid, 256, 0, s>>>(key, value, key_stride, value_stride, slots, (uint8_t*)key_cache, (uint8_t*)value_cache,
                                                            tokens, chunks, head_dim / 8, page_shift, slot_count, k_inv, v_inv);
    else
        paged_cache_write_kernel<false><<<grid, 256, 0, s>>>(key, value, key_stride, value_stride, slots, (uint8_t*)key_cache, (uint8_t*)value_cache,
                                                             tokens, chunks, head_dim / 8, page_shift, slot_count, k_inv, v_inv);
}

}  // namespace pk
