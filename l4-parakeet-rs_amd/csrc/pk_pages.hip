// Pages that follow their beams: new block tables from the rows' parents, pages that no row
// lists any more, the pages that have to be copied, and the copies.
//
// A row's full pages are shared by all its children.  A partly filled page gets new tokens,
// so it goes to the first child (the lowest row) alone, and each other child gets a page of
// its own from the free list and a pair (page, new page) to be copied.
//
// A page goes back if a row without children listed it and no row with children does: marks
// are bytes that any number of rows set to 1, so their order does not matter, and the pages
// that go back are listed in ascending order.
#include "pk_kernels.hpp"

namespace pk {

struct RowPlan {
    int parent;    // the row whose pages it takes; -1: none
    int last;      // the page in the last column if it is not the parent's; -1
    int has_child; // of the row as an old one
};
constexpr int kPageSegment = 4096;  // pages a workgroup of the last two launches

__device__ __forceinline__ int pages_of(int length, int shift) { return (int)(((long long)length + (1 << shift) - 1) >> shift); }

// Inclusive scan over 1024 threads.
__device__ __forceinline__ int scan_1024(int v, int* wave_total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int up = __shfl_up(v, off, 64);
        if (lane >= off) v += up;
    }
    if (lane == 63) wave_total[wave] = v;
    __syncthreads();
    for (int w = 0; w < wave; ++w) v += wave_total[w];
    return v;
}

// Workgroup 0: children, copies and lengths; the others clear the marks.
__global__ __launch_bounds__(1024) void fork_plan_kernel(ForkArgs a, RowPlan* __restrict__ plan, uint32_t* __restrict__ marks, long long mark_words) {
    if (blockIdx.x > 0) {
        for (long long i = (long long)(blockIdx.x - 1) * 1024 + threadIdx.x; i < mark_words; i += (long long)(gridDim.x - 1) * 1024) marks[i] = 0;
        return;
    }
    __shared__ int eldest[kMostForkRows];
    __shared__ int wave_total[16];
    __shared__ int flags;
    constexpr int kPer = kMostForkRows / 1024;
    const int per = (a.rows + 1023) / 1024, first = threadIdx.x * per, page = 1 << a.shift;
    if (threadIdx.x == 0) flags = 0;
    for (int i = threadIdx.x; i < a.rows; i += 1024) eldest[i] = a.rows;
    __syncthreads();
    int parent[kPer], length[kPer], source[kPer];
    int bad = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        parent[j] = -1;
        length[j] = 0;
        if (j >= per || first + j >= a.rows) continue;
        const int p = a.parents[first + j], own = a.lengths[first + j];
        if (p < -1 || p >= a.rows || own < 0 || ((long long)own + page - 1) >> a.shift > a.max_pages) bad = 8;
        else if (p >= 0) {
            parent[j] = p;
            atomicMin(&eldest[p], first + j);
        }
    }
    if (bad) atomicOr(&flags, bad);
    __syncthreads();
    int status = flags;
    const int begin = a.free_range[0], end = a.free_range[1] < a.free_capacity ? a.free_range[1] : a.free_capacity;
    if (begin < 0) status |= 8;
    int wanted = 0, rows = 0;
    if (!status) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            source[j] = -1;
            if (parent[j] < 0) continue;
            ++rows;
            length[j] = a.lengths[parent[j]];
            if (length[j] & (page - 1) && eldest[parent[j]] != first + j) {
                const int id = a.table[(size_t)parent[j] * a.max_pages + (length[j] >> a.shift)];
                if (id >= 0 && id < a.pages) {
                    source[j] = id;
                    ++wanted;
                }
            }
        }
    }
    // both counts in one scan: neither passes 4096
    const int scanned = scan_1024(wanted | (rows << 16), wave_total);
    int all = 0;
    for (int w = 0; w < 16; ++w) all += wave_total[w];
    const int taken = all & 0xffff, forked = all >> 16;
    if (!status && taken > 0 && taken > (long long)end - begin) status = 1;
    int at = begin + (scanned & 0xffff) - wanted;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int r = first + j;
        if (j >= per || r >= a.rows) break;
        RowPlan one{status ? r : parent[j], -1, status || eldest[r] < a.rows};
        int from = -1, to = -1;
        if (!status && source[j] >= 0) {
            from = source[j];
            to = one.last = a.free_pages[at++];
        }
        plan[r] = one;
        a.copies[2 * r] = from;
        a.copies[2 * r + 1] = to;
        a.new_lengths[r] = status ? a.lengths[r] : length[j];
    }
    if (threadIdx.x == 0) {
        a.info[0] = status ? 0 : forked;
        a.info[1] = status ? 0 : taken;
        a.info[2] = status;
        a.info[3] = 0;
    }
}

// A wave a row: as a new one its pages, as an old one its marks.
__global__ __launch_bounds__(256) void fork_table_kernel(ForkArgs a, const RowPlan* __restrict__ plan, uint8_t* __restrict__ kept, uint8_t* __restrict__ gone) {
    const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (r >= a.rows) return;
    const RowPlan one = plan[r];
    if (one.parent >= 0) {
        const int count = min(pages_of(a.lengths[one.parent], a.shift), a.max_pages);
        const int* from = a.table + (size_t)one.parent * a.max_pages;
        int* to = a.new_table + (size_t)r * a.max_pages;
        for (int c = lane; c < count; c += 64) to[c] = c == count - 1 && one.last >= 0 ? one.last : from[c];
    }
    if (a.info[2]) return;  // nothing goes back
    const int count = min(pages_of(a.lengths[r], a.shift), a.max_pages);
    const int* mine = a.table + (size_t)r * a.max_pages;
    uint8_t* mark = one.has_child ? kept : gone;
    for (int c = lane; c < count; c += 64) {
        const int id = mine[c];
        if (id >= 0 && id < a.pages) mark[id] = 1;
    }
}

// Sixteen pages' marks as bits: those that go back.
__device__ __forceinline__ uint32_t going(const ForkArgs& a, const uint8_t* kept, const uint8_t* gone, int page0) {
    if (page0 >= a.pages) return 0;
    uint32_t bits = 0;
    for (int i = 0; i < 16 && page0 + i < a.pages; ++i)
        if (gone[page0 + i] && !kept[page0 + i] && !(a.held && a.held[page0 + i])) bits |= 1u << i;
    return bits;
}

__global__ __launch_bounds__(256) void fork_count_kernel(ForkArgs a, const uint8_t* __restrict__ kept, const uint8_t* __restrict__ gone, int* __restrict__ counts) {
    __shared__ int sum;
    if (threadIdx.x == 0) sum = 0;
    __syncthreads();
    const int n = __popc(going(a, kept, gone, (int)((blockIdx.x * 256 + threadIdx.x) * 16)));
    if (n) atomicAdd(&sum, n);
    __syncthreads();
    if (threadIdx.x == 0) counts[blockIdx.x] = sum;
}

__global__ __launch_bounds__(256) void fork_list_kernel(ForkArgs a, const uint8_t* __restrict__ kept, const uint8_t* __restrict__ gone, const int* __restrict__ counts) {
    __shared__ int before, wave_total[4];
    if (threadIdx.x == 0) before = 0;
    __syncthreads();
    int n = 0;
    for (int i = threadIdx.x; i < (int)blockIdx.x; i += 256) n += counts[i];
    if (n) atomicAdd(&before, n);
    const int page0 = (int)((blockIdx.x * 256 + threadIdx.x) * 16), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t bits = going(a, kept, gone, page0);
    const int mine = __popc(bits);
    int v = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int up = __shfl_up(v, off, 64);
        if (lane >= off) v += up;
    }
    if (lane == 63) wave_total[wave] = v;
    __syncthreads();
    int at = before + v - mine;
    for (int w = 0; w < wave; ++w) at += wave_total[w];
    while (bits) {
        const int i = __ffs(bits) - 1;
        bits &= bits - 1;
        a.freed[at++] = page0 + i;
    }
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0)
        a.info[3] = before + wave_total[0] + wave_total[1] + wave_total[2] + wave_total[3];
}

static long long mark_bytes(int pages) { return ((long long)pages + 15) / 16 * 16; }  // of one of the two
static int segments(int pages) { return (int)(((long long)pages + kPageSegment - 1) / kPageSegment); }

size_t fork_workspace(int rows, int pages) {
    return (size_t)mark_bytes(pages) * 2 + (size_t)rows * sizeof(RowPlan) + (size_t)segments(pages) * 4;
}

void launch_page_fork(const ForkArgs& a, hipStream_t s) {
    uint8_t* kept = (uint8_t*)a.workspace;
    uint8_t* gone = kept + mark_bytes(a.pages);
    RowPlan* plan = (RowPlan*)(gone + mark_bytes(a.pages));
    int* counts = (int*)(plan + a.rows);
    const long long words = mark_bytes(a.pages) / 2;
    const unsigned clear = (unsigned)((words + 4095) / 4096 > 255 ? 255 : (words + 4095) / 4096);
    fork_plan_kernel<<<1 + clear, 1024, 0, s>>>(a, plan, (uint32_t*)kept, words);
    fork_table_kernel<<<(unsigned)(a.rows + 3) / 4, 256, 0, s>>>(a, plan, kept, gone);
    fork_count_kernel<<<(unsigned)segments(a.pages), 256, 0, s>>>(a, kept, gone, counts);
    fork_list_kernel<<<(unsigned)segments(a.pages), 256, 0, s>>>(a, kept, gone, counts);
}

// The free list behind a plan or a fork that is kept: pages taken leave its front, pages that
// went back stand there.
__global__ __launch_bounds__(256) void page_keep_kernel(const int* __restrict__ info, const int* __restrict__ freed, int* __restrict__ free_pages,
                                                        int* free_range, int free_capacity) {
    if (info[2]) return;
    const int begin = free_range[0] + info[1];
    if (begin < 0) return;
    int back = freed ? info[3] : 0;
    back = back < begin ? back : begin;  // a list that gave out what the tables hold has room for all
    __syncthreads();
    for (int i = threadIdx.x; i < back; i += 256)
        if (begin - back + i < free_capacity) free_pages[begin - back + i] = freed[i];
    if (threadIdx.x == 0) free_range[0] = begin - back;
}

void launch_page_keep(const int* info, const int* freed, int* free_pages, int* free_range, int free_capacity, hipStream_t s) {
    page_keep_kernel<<<1, 256, 0, s>>>(info, freed, free_pages, free_range, free_capacity);
}

// Pairs (source, destination) of pages in all layers' keys and values.
__global__ __launch_bounds__(256) void paged_cache_copy_kernel(const int* __restrict__ copies, uint4* key_cache, uint4* value_cache, long long units,
                                                               int pages, int layers) {
    const int from = copies[2 * blockIdx.y], to = copies[2 * blockIdx.y + 1];
    if (from < 0 || from >= pages || to < 0 || to >= pages || from == to) return;
    const int layer = blockIdx.z % layers;
    uint4* cache = (int)blockIdx.z < layers ? key_cache : value_cache;
    const uint4* src = cache + ((long long)layer * pages + from) * units;
    uint4* dst = cache + ((long long)layer * pages + to) * units;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < units; i += (long long)gridDim.x * 256) dst[i] = src[i];
}

void launch_paged_cache_copy(const int* copies, int count, void* key_cache, void* value_cache, long long page_bytes, int pages, int layers, hipStream_t s) {
    const long long units = page_bytes / 16;
    const dim3 grid((unsigned)((units + 255) / 256 > 64 ? 64 : (units + 255) / 256), (unsigned)count, (unsigned)(2 * layers));
    paged_cache_copy_kernel<<<grid, 256, 0, s>>>(copies, (uint4*)key_cache, (uint4*)value_cache, units, pages, layers);
}

}  // namespace pk
