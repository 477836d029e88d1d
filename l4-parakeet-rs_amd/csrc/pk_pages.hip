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

// Small tables are one workgroup's, with the marks as bits in LDS.  Large ones take four launches:
// children, copies and lengths (and the marks cleared); tables and marks; how many pages of each
// 4096 go back; their list.  Bound by latency: each launch is a chain of a few dependent loads.
struct RowPlan {
    int parent;     // the row whose pages it takes; -1: none
    int last;       // the page in the last column if it is not the parent's; -1
    int has_child;  // of the row as an old one
};

__device__ __forceinline__ int pages_of(const ForkArgs& a, int length) {
    const int n = (int)(((long long)length + (1 << a.shift) - 1) >> a.shift);
    return n < a.max_pages ? n : a.max_pages;  // (a length that is refused)
}

// Inclusive scan over 1024 threads; `all` is the total.
__device__ __forceinline__ int scan_1024(int v, int* wave_total, int& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int up = __shfl_up(v, off, 64);
        if (lane >= off) v += up;
    }
    if (lane == 63) wave_total[wave] = v;
    __syncthreads();
    all = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        const int t = wave_total[w];
        v += w < wave ? t : 0;
        all += t;
    }
    return v;
}

// Children, copies, lengths and info by 1024 threads, up to kPer rows each (1024 apart, so that
// neighbours' loads and stores lie together); returns the status.  wave_total: 16 * kPer.  Loads are made
// without branches, at a place that exists where none is wanted, so that none waits for another.
template <int kPer> __device__ __forceinline__ int plan_rows(const ForkArgs& a, int* eldest, int* wave_total, int* flags, RowPlan* plan) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, page = 1 << a.shift;
    const int begin = a.free_range[0], end = a.free_range[1] < a.free_capacity ? a.free_range[1] : a.free_capacity;
    int parent[kPer], own[kPer], length[kPer], source[kPer];
    const auto there = [&](int j) { return j * 1024 + tid < a.rows; };
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int r = there(j) ? j * 1024 + tid : 0;
        parent[j] = a.parents[r];
        own[j] = a.lengths[r];
    }
    for (int i = tid; i < a.rows; i += 1024) eldest[i] = a.rows;
    if (tid == 0) *flags = 0;
    __syncthreads();
    int bad = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        parent[j] = there(j) ? parent[j] : -1;
        own[j] = there(j) ? own[j] : 0;
        const bool odd = parent[j] < -1 || parent[j] >= a.rows || own[j] < 0 || ((long long)own[j] + page - 1) >> a.shift > a.max_pages;
        bad |= odd ? 8 : 0;
        parent[j] = odd ? -1 : parent[j];
        length[j] = a.lengths[parent[j] >= 0 ? parent[j] : 0];
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        if (parent[j] >= 0) atomicMin(&eldest[parent[j]], j * 1024 + tid);
        length[j] = parent[j] >= 0 ? length[j] : 0;
        source[j] = -1;
    }
    if (bad) atomicOr(flags, bad);
    __syncthreads();
    int status = *flags | (begin < 0 ? 8 : 0);
    if (!status) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int c = length[j] >> a.shift;  // (of lengths that are all right)
            source[j] = a.table[(size_t)(parent[j] >= 0 ? parent[j] : 0) * a.max_pages + (c < a.max_pages ? c : 0)];
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const bool copied = parent[j] >= 0 && length[j] & (page - 1) && eldest[parent[j] >= 0 ? parent[j] : 0] != j * 1024 + tid;
            source[j] = copied && source[j] >= 0 && source[j] < a.pages ? source[j] : -1;
        }
    }
    // rows before this one that take a page: in its wave, and in the waves of lower rows; both counts are at most 4096
    int before[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const unsigned long long takes = __builtin_amdgcn_ballot_w64(source[j] >= 0), real = __builtin_amdgcn_ballot_w64(parent[j] >= 0);
        before[j] = __popcll(takes & ((1ull << lane) - 1));
        if (lane == 0) wave_total[j * 16 + wave] = __popcll(takes) | (__popcll(real) << 16);
    }
    __syncthreads();
    static_assert(kPer <= 4);  // a lane a wave's total
    const int mine = lane < 16 * kPer ? wave_total[lane] : 0;
    int sums = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int up = __shfl_up(sums, off, 64);
        if (lane >= off) sums += up;
    }
    const int all = __builtin_amdgcn_readlane(sums, 63);
#pragma unroll
    for (int j = 0; j < kPer; ++j) before[j] += __builtin_amdgcn_readlane(sums - mine, __builtin_amdgcn_readfirstlane(j * 16 + wave)) & 0xffff;
    const int taken = all & 0xffff, forked = all >> 16;
    if (!status && taken > 0 && taken > (long long)end - begin) status = 1;
    const int failed = status ? -1 : 0;
    int to[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) to[j] = -1;
    if (!status && taken > 0) {  // so that there is a free page
#pragma unroll
        for (int j = 0; j < kPer; ++j) to[j] = a.free_pages[begin + (source[j] >= 0 ? before[j] : 0)];
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int r = j * 1024 + tid;
        if (there(j)) {
            const bool copied = !status && source[j] >= 0;
            plan[r].parent = status ? r : parent[j];
            plan[r].last = copied ? to[j] : -1;
            plan[r].has_child = status || eldest[r] < a.rows;
            a.copies[2 * r] = copied ? source[j] : -1;
            a.copies[2 * r + 1] = copied ? to[j] : -1;
            a.new_lengths[r] = (own[j] & failed) | (length[j] & ~failed);
        }
    }
    if (tid == 0) {
        a.info[0] = status ? 0 : forked;
        a.info[1] = status ? 0 : taken;
        a.info[2] = status;
        a.info[3] = 0;
    }
    return status;
}

// A row's entries by a wave; of long rows eight a lane at once, all asked for before the first is used
// (`other`: a second row that is read beside it up to `others`).
template <typename Use> __device__ __forceinline__ void each_entry(const int* row, const int* other, int others, int count, int lane, Use use) {
    if (count <= 256) {
        for (int c = lane; c < count; c += 64) {
            const int id = row[c];
            use(c, id, c < others ? other[c] : -1);
        }
        return;
    }
    for (int first = lane; first < count; first += 512) {
        int id[8], beside[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const int c = first + 64 * n < count ? first + 64 * n : first;
            id[n] = row[c];
            beside[n] = c < others ? other[c] : -1;
        }
#pragma unroll
        for (int n = 0; n < 8; ++n)
            if (first + 64 * n < count) use(first + 64 * n, id[n], beside[n]);
    }
}

// A row as a new one, by a wave: its parent's pages.
__device__ __forceinline__ void new_row(const ForkArgs& a, int r, const RowPlan& one, int length, int lane) {
    if (one.parent < 0) return;
    const int count = pages_of(a, length);
    int* to = a.new_table + (size_t)r * a.max_pages;
    each_entry(a.table + (size_t)one.parent * a.max_pages, nullptr, 0, count, lane,
               [&](int c, int id, int) { to[c] = c == count - 1 && one.last >= 0 ? one.last : id; });
}

constexpr int kSmallRows = 1024, kSmallEntries = 1 << 14, kSmallPages = 1 << 17;

__global__ __launch_bounds__(1024) void fork_small_kernel(ForkArgs a) {
    extern __shared__ uint32_t marks[];  // a bit a page: kept, then gone
    __shared__ int eldest[kSmallRows];
    __shared__ RowPlan plan[kSmallRows];
    __shared__ int wave_total[16], flags;
    const int words = (a.pages + 31) / 32, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    uint32_t *kept = marks, *gone = marks + words;
    for (int i = threadIdx.x; i < 2 * words; i += 1024) marks[i] = 0;
    const int status = plan_rows<1>(a, eldest, wave_total, &flags, plan);
    __syncthreads();
    for (int r = wave; r < a.rows; r += 16) {
        const RowPlan one = plan[r];
        const int own = a.lengths[r];
        new_row(a, r, one, a.lengths[one.parent >= 0 ? one.parent : r], lane);
        if (status) continue;  // nothing goes back
        uint32_t* mark = one.has_child ? kept : gone;
        each_entry(a.table + (size_t)r * a.max_pages, nullptr, 0, pages_of(a, own), lane, [&](int, int id, int) {
            if (id >= 0 && id < a.pages) atomicOr(&mark[id >> 5], 1u << (id & 31));
        });
    }
    __syncthreads();
    // up to four words a thread, in order
    const int per = (words + 1023) / 1024, first = threadIdx.x * per;
    int mine = 0;
    for (int i = first; i < first + per && i < words; ++i) {
        uint32_t bits = gone[i] & ~kept[i];
        if (bits && a.held)
            for (uint32_t left = bits; left; left &= left - 1) {
                const int b = __ffs(left) - 1;
                if (a.held[i * 32 + b]) bits &= ~(1u << b);
            }
        gone[i] = bits;
        mine += __popc(bits);
    }
    int all;
    int at = scan_1024(mine, wave_total, all) - mine;
    for (int i = first; i < first + per && i < words; ++i)
        for (uint32_t left = gone[i]; left; left &= left - 1) a.freed[at++] = i * 32 + __ffs(left) - 1;
    if (threadIdx.x == 0) a.info[3] = all;
}

// Workgroup 0 plans the rows; the others clear the marks.
__global__ __launch_bounds__(1024) void fork_plan_kernel(ForkArgs a, RowPlan* __restrict__ plan, uint4* __restrict__ marks, long long mark_units) {
    __shared__ int eldest[kMostForkRows];
    __shared__ int wave_total[kMostForkRows / 64], flags;
    if (blockIdx.x == 0) {
        plan_rows<kMostForkRows / 1024>(a, eldest, wave_total, &flags, plan);
    } else {
        for (long long i = (long long)(blockIdx.x - 1) * 1024 + threadIdx.x; i < mark_units; i += (long long)(gridDim.x - 1) * 1024) marks[i] = uint4{};
    }
}

// A wave a row and task: as a new one its pages, as an old one its marks, but for those that the row
// before it (often another beam of the same request) sets.
__global__ __launch_bounds__(256) void fork_table_kernel(ForkArgs a, const RowPlan* __restrict__ plan, uint8_t* __restrict__ kept, uint8_t* __restrict__ gone) {
    // neighbouring rows, which list the same pages, on one XCD: workgroups go to the eight in turn
    const int r = (int)(blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8) * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (r >= a.rows) return;
    const RowPlan one = plan[r];
    if (blockIdx.y == 0) {
        new_row(a, r, one, a.new_lengths[r], lane);
        return;
    }
    const int own = a.lengths[r], above = r > 0 ? a.lengths[r - 1] : 0, failed = a.info[2];
    if (failed) return;  // nothing goes back
    const int before = r > 0 && plan[r - 1].has_child == one.has_child ? pages_of(a, above) : 0;
    const int* mine = a.table + (size_t)r * a.max_pages;
    uint8_t* mark = one.has_child ? kept : gone;
    each_entry(mine, mine - a.max_pages, before, pages_of(a, own), lane, [&](int, int id, int beside) {
        if (id >= 0 && id < a.pages && id != beside) mark[id] = 1;
    });
}

constexpr int kPageSegment = 4096;  // pages a workgroup of the last two launches, 16 a thread

// A thread's 16 pages as bytes: 1 for those that go back.  (Marks reach to a multiple of 16 pages.)
__device__ __forceinline__ uint4 going(const ForkArgs& a, const uint8_t* kept, const uint8_t* gone, long long page0) {
    if (page0 >= a.pages) return uint4{};
    const uint4 k = *(const uint4*)(kept + page0), g = *(const uint4*)(gone + page0);
    uint32_t w[4] = {g.x & ~k.x, g.y & ~k.y, g.z & ~k.z, g.w & ~k.w};
    if (a.held && (w[0] | w[1] | w[2] | w[3]))
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (w[i >> 2] >> (8 * (i & 3)) & 1u && a.held[page0 + i]) w[i >> 2] &= ~(1u << (8 * (i & 3)));
    return uint4{w[0], w[1], w[2], w[3]};
}
__device__ __forceinline__ int count_of(const uint4& w) { return __popc(w.x) + __popc(w.y) + __popc(w.z) + __popc(w.w); }

__global__ __launch_bounds__(256) void fork_count_kernel(ForkArgs a, const uint8_t* __restrict__ kept, const uint8_t* __restrict__ gone, int* __restrict__ counts) {
    __shared__ int sum;
    if (threadIdx.x == 0) sum = 0;
    __syncthreads();
    const int n = count_of(going(a, kept, gone, ((long long)blockIdx.x * 256 + threadIdx.x) * 16));
    if (n) atomicAdd(&sum, n);
    __syncthreads();
    if (threadIdx.x == 0) counts[blockIdx.x] = sum;
}

__global__ __launch_bounds__(256) void fork_list_kernel(ForkArgs a, const uint8_t* __restrict__ kept, const uint8_t* __restrict__ gone, const int* __restrict__ counts) {
    __shared__ int before, wave_total[4];
    const long long page0 = ((long long)blockIdx.x * 256 + threadIdx.x) * 16;
    const uint4 back = going(a, kept, gone, page0);
    if (threadIdx.x == 0) before = 0;
    __syncthreads();
    int n = 0;
    for (int i = threadIdx.x; i < (int)blockIdx.x; i += 256) n += counts[i];
    if (n) atomicAdd(&before, n);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, mine = count_of(back);
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
    const uint32_t words[4] = {back.x, back.y, back.z, back.w};
#pragma unroll
    for (int w = 0; w < 4; ++w)
        for (uint32_t left = words[w]; left; left &= left - 1) a.freed[at++] = (int)page0 + 4 * w + (__ffs(left) - 1) / 8;
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) a.info[3] = before + wave_total[0] + wave_total[1] + wave_total[2] + wave_total[3];
}

static long long mark_bytes(int pages) { return ((long long)pages + 15) / 16 * 16; }  // of one of the two
static int segments(int pages) { return (int)(((long long)pages + kPageSegment - 1) / kPageSegment); }

size_t fork_workspace(int rows, int pages) {
    return (size_t)mark_bytes(pages) * 2 + (size_t)rows * sizeof(RowPlan) + (size_t)segments(pages) * 4;
}

void launch_page_fork(const ForkArgs& a, hipStream_t s) {
    if (a.rows <= kSmallRows && (long long)a.rows * a.max_pages <= kSmallEntries && a.pages <= kSmallPages) {
        fork_small_kernel<<<1, 1024, (size_t)(a.pages + 31) / 32 * 8, s>>>(a);
        return;
    }
    uint8_t* kept = (uint8_t*)a.workspace;
    uint8_t* gone = kept + mark_bytes(a.pages);
    RowPlan* plan = (RowPlan*)(gone + mark_bytes(a.pages));
    int* counts = (int*)(plan + a.rows);
    const long long units = mark_bytes(a.pages) / 8, blocks = (units + 1023) / 1024;
    fork_plan_kernel<<<1 + (unsigned)(blocks < 255 ? blocks : 255), 1024, 0, s>>>(a, plan, (uint4*)kept, units);
    fork_table_kernel<<<dim3((unsigned)(a.rows + 31) / 32 * 8, 2), 256, 0, s>>>(a, plan, kept, gone);
    fork_count_kernel<<<(unsigned)segments(a.pages), 256, 0, s>>>(a, kept, gone, counts);
    fork_list_kernel<<<(unsigned)segments(a.pages), 256, 0, s>>>(a, kept, gone, counts);
}

// The free list behind a plan or a fork that is kept: pages taken leave its front, pages that
// went back stand there.
__global__ __launch_bounds__(256) void page_keep_kernel(const int* __restrict__ info, const int* __restrict__ freed, int* __restrict__ free_pages,
                                                        int* free_range, int free_capacity, int pages) {
    if (info[2]) return;
    const int begin = free_range[0] + info[1];
    if (begin < 0) return;
    int back = freed ? info[3] : 0;
    back = back < 0 ? 0 : back < pages ? back : pages;
    back = back < begin ? back : begin;  // a list that gave out what the tables hold has room for all
    __syncthreads();
    for (int i = threadIdx.x; i < back; i += 256)
        if (begin - back + i < free_capacity) free_pages[begin - back + i] = freed[i];
    if (threadIdx.x == 0) free_range[0] = begin - back;
}

void launch_page_keep(const int* info, const int* freed, int* free_pages, int* free_range, int free_capacity, int pages, hipStream_t s) {
    page_keep_kernel<<<1, 256, 0, s>>>(info, freed, free_pages, free_range, free_capacity, pages);
}

// Pairs (source, destination) of pages in all layers' keys and values.  Bound by HBM: 1434 pages of
// 16 KB in 12 layers' keys and values (1.13 GB read and written) 214 us, 5.3 TB/s, with stores past the
// caches; 223 without.
template <bool kPast>
__global__ __launch_bounds__(256) void paged_cache_copy_kernel(const int* __restrict__ copies, v4i* key_cache, v4i* value_cache, long long units,
                                                               int pages, int layers) {
    const int from = copies[2 * blockIdx.y], to = copies[2 * blockIdx.y + 1];
    if (from < 0 || from >= pages || to < 0 || to >= pages || from == to) return;
    const int layer = blockIdx.z % layers;
    v4i* cache = (int)blockIdx.z < layers ? key_cache : value_cache;
    const v4i* src = cache + ((long long)layer * pages + from) * units;
    v4i* dst = cache + ((long long)layer * pages + to) * units;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < units; i += (long long)gridDim.x * 256) {
        const v4i v = src[i];
        if constexpr (kPast) __builtin_nontemporal_store(v, dst + i);
        else dst[i] = v;
    }
}

void launch_paged_cache_copy(const int* copies, int count, void* key_cache, void* value_cache, long long page_bytes, int pages, int layers, hipStream_t s) {
    const long long units = page_bytes / 16;
    const dim3 grid((unsigned)((units + 255) / 256 > 64 ? 64 : (units + 255) / 256), (unsigned)count, (unsigned)(2 * layers));
    const auto launch = [&](auto kernel) { kernel<<<grid, 256, 0, s>>>(copies, (v4i*)key_cache, (v4i*)value_cache, units, pages, layers); };
    if (2 * page_bytes * layers * count > kCached) launch(paged_cache_copy_kernel<true>);
    else launch(paged_cache_copy_kernel<false>);
}

}  // namespace pk
