// Pages that follow their beams: new block tables from the rows' parents, pages that no row
// lists any more, the pages that have to be copied, and the copies.
//
// A row's full pages are shared by all its children.  A partly filled page gets new tokens,
// so it goes to the first child (the lowest row) alone, and each other child gets a page of
// its own from the free list and a pair (page, new page) to be copied.
//
// A page goes back if a row without children listed it and no row with children does: marks
// are bits that any number of rows set, and then any number clear, so their order does not
// matter, and the pages that go back are listed in ascending order.
#include <type_traits>

#include "pk_kernels.hpp"

namespace pk {

// Small tables are one workgroup's, with the marks in LDS.  Large ones take four launches: marks cleared;
// children, copies and lengths, and marks of what rows without children list; tables, and marks cleared of
// what rows with children list; the list.  Bound by latency: each launch is a chain of a few dependent loads
// (4096 rows of 501 entries over 1.29 M pages 2.1 + 8.8 + 5.5 + 4.8 us).
struct RowPlan {
    int parent;     // the row whose pages it takes; -1: none
    int last;       // the page in the last column if it is not the parent's; -1
    int has_child;  // of the row as an old one
};

__device__ __forceinline__ int pages_of(const ForkArgs& a, int length) {
    const int n = (int)(((long long)length + (1 << a.shift) - 1) >> a.shift);
    return n < a.max_pages ? n : a.max_pages;  // (a length that is refused)
}

// Inclusive sum over a wave's lanes.
__device__ __forceinline__ int wave_scan(int v) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int up = __shfl_up(v, off, 64);
        if ((int)(threadIdx.x & 63) >= off) v += up;
    }
    return v;
}

// Inclusive scan over 1024 threads; `all` is the total.
__device__ __forceinline__ int scan_1024(int v, int* wave_total, int& all) {
    const int wave = threadIdx.x >> 6;
    v = wave_scan(v);
    if ((threadIdx.x & 63) == 63) wave_total[wave] = v;
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
    bool copied[kPer];
    if (!status) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            copied[j] = parent[j] >= 0 && length[j] & (page - 1) && eldest[parent[j] >= 0 ? parent[j] : 0] != j * 1024 + tid;
            source[j] = a.table[copied[j] ? (size_t)parent[j] * a.max_pages + (length[j] >> a.shift) : 0];  // (lengths are all right)
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j) source[j] = copied[j] && source[j] >= 0 && source[j] < a.pages ? source[j] : -1;
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
    const int sums = wave_scan(mine);
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
            const bool new_page = !status && source[j] >= 0;
            plan[r].parent = status ? r : parent[j];
            plan[r].last = new_page ? to[j] : -1;
            plan[r].has_child = status || eldest[r] < a.rows;
            a.copies[2 * r] = new_page ? source[j] : -1;
            a.copies[2 * r + 1] = new_page ? to[j] : -1;
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

// A row's entries by a wave; of long rows eight a lane at once, all asked for before the first is used, beside
// those of two other rows up to their counts (else -1).
struct Beside {
    const int* row;
    int count;
};
template <typename Use> __device__ __forceinline__ void each_entry(const int* row, int count, Beside x, Beside y, int lane, Use use) {
    const auto some = [&](int first, auto per) {
        constexpr int kPer = decltype(per)::value;
        int id[kPer], ix[kPer], iy[kPer];
#pragma unroll
        for (int n = 0; n < kPer; ++n) {
            const int c = first + 64 * n < count ? first + 64 * n : first;
            id[n] = row[c];
            ix[n] = c < x.count ? x.row[c] : -1;
            iy[n] = c < y.count ? y.row[c] : -1;
        }
#pragma unroll
        for (int n = 0; n < kPer; ++n)
            if (first + 64 * n < count) use(first + 64 * n, id[n], ix[n], iy[n]);
    };
    if (count <= 256) {
        for (int c = lane; c < count; c += 64) some(c, std::integral_constant<int, 1>{});
    } else {
        for (int c = lane; c < count; c += 512) some(c, std::integral_constant<int, 8>{});
    }
}

// A row as a new one, by a wave: its parent's pages.
__device__ __forceinline__ void new_row(const ForkArgs& a, int r, const RowPlan& one, int length, int lane) {
    if (one.parent < 0) return;
    const int count = pages_of(a, length);
    int* to = a.new_table + (size_t)r * a.max_pages;
    each_entry(a.table + (size_t)one.parent * a.max_pages, count, Beside{}, Beside{}, lane,
               [&](int c, int id, int, int) { to[c] = c == count - 1 && one.last >= 0 ? one.last : id; });
}

// Up to here one workgroup: its 16 waves take rows in turn, so rows tell most (rows of 60 entries, calls of a captured graph:
// 32 of them 5.8 us and 10.4 in four launches, 64 7.2 and 10.6, 128 10.1 and 10.4, 160 11.6 and 10.4, 256 16.0 and 10.6;
// 1024 of 16 48.4 and 10.8), then a row's length (64 rows of 256 entries 9.1 and 11.0, of 512 10.1 and 11.7, 96 of 256
// 11.4 and 11.0, 128 of 512 15.7 and 12.6), then the words of marks that are cleared and counted (32 rows of 30 in 673
// pages 5.4 and 9.9, in 2^17 6.9 and 10.3).
constexpr int kSmallRows = 128, kSmallEntries = 1 << 14, kSmallPages = 1 << 17;

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
        each_entry(a.table + (size_t)r * a.max_pages, pages_of(a, own), Beside{}, Beside{}, lane, [&](int, int id, int, int) {
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

__global__ __launch_bounds__(256) void fork_clear_kernel(v4i* gone, int units) {
    const int i = (int)blockIdx.x * 256 + threadIdx.x;
    if (i < units) gone[i] = v4i{};
}

// Workgroup 0 plans the rows; the others mark what rows without children list, a wave a row.  Most of that
// is also in the next row with children, of another beam of the same request, above or below it: those
// entries are passed over (marked, they would be cleared again).  The rest, pages of a beam of its own, are
// 3 of the 9 us of 4096 rows of 501 entries: an atomic each, as the bits of a word are many rows'.
__global__ __launch_bounds__(1024) void fork_plan_kernel(ForkArgs a, RowPlan* __restrict__ plan, uint32_t* __restrict__ gone) {
    __shared__ int eldest[kMostForkRows];
    __shared__ int wave_total[kMostForkRows / 64], flags;
    if (blockIdx.x == 0) {
        plan_rows<kMostForkRows / 1024>(a, eldest, wave_total, &flags, plan);
        return;
    }
    uint8_t* has_child = (uint8_t*)eldest;
    const int r = __builtin_amdgcn_readfirstlane((int)(blockIdx.x - 1) * 16 + (int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
    int parent[kMostForkRows / 1024];
#pragma unroll
    for (int j = 0; j < kMostForkRows / 1024; ++j) {
        const int i = j * 1024 + threadIdx.x;
        parent[j] = i < a.rows ? a.parents[i] : -1;
        eldest[j * 256 + (threadIdx.x >> 2)] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kMostForkRows / 1024; ++j)
        if (parent[j] >= 0 && parent[j] < a.rows) has_child[parent[j]] = 1;
    __syncthreads();
    if (r >= a.rows || has_child[r]) return;
    const int near = r - 32 + lane;
    const unsigned long long with = __builtin_amdgcn_ballot_w64(near >= 0 && near < a.rows && has_child[near >= 0 && near < a.rows ? near : 0]);
    const uint32_t lower = (uint32_t)with, upper = (uint32_t)(with >> 32);
    const int above = lower ? r - 1 - __clz(lower) : r, below = upper ? r - 1 + __ffs(upper) : r;
    const auto beside = [&](int other) { return Beside{a.table + (size_t)other * a.max_pages, other == r ? 0 : pages_of(a, a.lengths[other])}; };
    each_entry(a.table + (size_t)r * a.max_pages, pages_of(a, a.lengths[r]), beside(above), beside(below), lane, [&](int, int id, int x, int y) {
        if (id >= 0 && id < a.pages && id != x && id != y && !(a.held && a.held[id])) atomicOr(&gone[id >> 5], 1u << (id & 31));
    });
}

// A wave a row and task: as a new one its pages, as an old one with children their marks cleared, but for
// those that the row above clears.
__global__ __launch_bounds__(256) void fork_table_kernel(ForkArgs a, const RowPlan* __restrict__ plan, uint32_t* gone) {
    // neighbouring rows, which list the same pages, on one XCD: workgroups go to the eight in turn
    const int r = (int)(blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8) * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (r >= a.rows) return;
    const RowPlan one = plan[r];
    if (blockIdx.y == 0) {
        new_row(a, r, one, a.new_lengths[r], lane);
        return;
    }
    if (!one.has_child) return;
    const int own = a.lengths[r], up = r > 0 ? r - 1 : 0, up_length = a.lengths[up];
    const Beside above{a.table + (size_t)up * a.max_pages, r > 0 && plan[up].has_child ? pages_of(a, up_length) : 0};
    each_entry(a.table + (size_t)r * a.max_pages, pages_of(a, own), above, Beside{}, lane, [&](int, int id, int x, int) {
        if (id >= 0 && id < a.pages && id != x && gone[id >> 5] >> (id & 31) & 1) atomicAnd(&gone[id >> 5], ~(1u << (id & 31)));
    });
}

constexpr int kListWords = 1024;  // a workgroup of the list: a word of 32 pages a thread
// Up to this many workgroups each counts what goes back before its words by itself, else a launch counts first
// (1.3 M pages 4.8 us by themselves and 2.3 + 4.0 with a launch, 2.9 M 5.5 and 3.9 + 4.1, 4.5 M 7.2 and 4.6 + 4.0).
constexpr int kMostCounting = 128;

__global__ __launch_bounds__(kListWords) void fork_count_kernel(const uint32_t* __restrict__ gone, int words, int* __restrict__ counts) {
    __shared__ int wave_total[16];
    const int i = (int)blockIdx.x * kListWords + threadIdx.x;
    int all;
    scan_1024(i < words ? __popc(gone[i]) : 0, wave_total, all);
    if (threadIdx.x == 0) counts[blockIdx.x] = all;
}

__global__ __launch_bounds__(kListWords) void fork_list_kernel(ForkArgs a, const uint32_t* __restrict__ gone, int words, const int* __restrict__ counts) {
    __shared__ int wave_total[16], wave_before[16];
    const int i = (int)blockIdx.x * kListWords + threadIdx.x;
    uint32_t back = i < words ? gone[i] : 0;
    const int failed = a.info[2];  // nothing goes back
    int n = 0;
    if (counts) {
        for (int k = threadIdx.x; k < (int)blockIdx.x; k += kListWords) n += counts[k];
    } else {
        const int units = (int)blockIdx.x * (kListWords / 4);
#pragma unroll 4
        for (int k = threadIdx.x; k < units; k += kListWords) {
            const uint4 x = ((const uint4*)gone)[k];
            n += __popc(x.x) + __popc(x.y) + __popc(x.z) + __popc(x.w);
        }
    }
    if (failed) return;
    n = wave_scan(n);
    if ((threadIdx.x & 63) == 63) wave_before[threadIdx.x >> 6] = n;
    const int mine = __popc(back);
    int all, before = 0;
    int at = scan_1024(mine, wave_total, all) - mine;  // (its barrier is also wave_before's)
#pragma unroll
    for (int w = 0; w < 16; ++w) before += wave_before[w];
    for (at += before; back; back &= back - 1) a.freed[at++] = i * 32 + __ffs(back) - 1;
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) a.info[3] = before + all;
}

static int mark_words(int pages) { return (int)(((long long)pages + 127) / 128 * 4); }
static int segments(int pages) { return (mark_words(pages) + kListWords - 1) / kListWords; }

size_t fork_workspace(int rows, int pages) {
    return (size_t)mark_words(pages) * 4 + (size_t)rows * sizeof(RowPlan) + (size_t)segments(pages) * 4;
}

void launch_page_fork(const ForkArgs& a, hipStream_t s) {
    if (a.rows <= kSmallRows && (long long)a.rows * a.max_pages <= kSmallEntries && a.pages <= kSmallPages) {
        fork_small_kernel<<<1, 1024, (size_t)(a.pages + 31) / 32 * 8, s>>>(a);
        return;
    }
    const int words = mark_words(a.pages), blocks = segments(a.pages);
    uint32_t* gone = (uint32_t*)a.workspace;
    RowPlan* plan = (RowPlan*)(gone + words);
    int* counts = (int*)(plan + a.rows);
    fork_clear_kernel<<<(unsigned)(words / 4 + 255) / 256, 256, 0, s>>>((v4i*)gone, words / 4);
    fork_plan_kernel<<<1 + (unsigned)(a.rows + 15) / 16, 1024, 0, s>>>(a, plan, gone);
    fork_table_kernel<<<dim3((unsigned)(a.rows + 31) / 32 * 8, 2), 256, 0, s>>>(a, plan, gone);
    if (blocks > kMostCounting) fork_count_kernel<<<blocks, kListWords, 0, s>>>(gone, words, counts);
    else counts = nullptr;
    fork_list_kernel<<<blocks, kListWords, 0, s>>>(a, gone, words, counts);
}

// The free list behind a plan or a fork that is kept: pages taken leave its front, pages that
// went back stand there.  One workgroup, as the list's front is read before it is moved: bound by the latency of a load and
// a store a lane at a time (100 pages 1.3 us, 1000 1.7, 10000 6.8, 100000 55, 111755 behind a fork of 4096 rows 114).
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
