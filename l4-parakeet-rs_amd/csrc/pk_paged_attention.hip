// Attention of new tokens over a paged cache.  Query i of a sequence with n new
// tokens and L keys stands at position p = L - n + i and sees the keys
// j in [p - left, p + right], 0 <= j < L:
//   o = sum_j softmax_j(scale * q . k_j) * v_j
// in one pass over the keys with a running maximum and sum (fp32).
//
// The query heads that share a kv head are rows of one matrix tile (row = token *
// group + head of the group), so the cache is read once for all of them.  Both
// products run with the cache as the MFMA's first operand: S^T = K Q^T leaves a lane
// with the scores of one query row (column l % 16), and the key rows are dealt to
// the MFMA's rows so that those are 8 consecutive keys: exactly the lane's operand
// of O^T = V^T P^T.  Probabilities therefore never leave their registers, and keys
// and (transposed) values are loaded from the cache straight into operand layout, 16
// bytes a lane.
#include "pk_paged_attention.hpp"

namespace pk {

// One wave's pass over key tiles for 16 query rows.  Loads are issued a stage ahead: a
// tile's values while its scores are computed, the next tile's keys before the softmax,
// and page ids two tiles ahead, since loads return in order.
template <int kD, bool kF8> struct RowPass {
    static constexpr int kSteps = kD / 32, kBlocks = kD / 16;  // MFMA steps of S over features, feature blocks of O
    static constexpr int kU = kF8 ? 2 : 1, kKeys = 32 * kU;    // 16 bytes of a value row hold 8 * kU keys; keys a wave tile
    static constexpr int kBytes = kF8 ? 1 : 2;
    static constexpr int kLoads = kSteps / kU;                 // 16-byte loads of a key row
    static constexpr int kSpan = 4 * kKeys;                    // keys that the four waves take at once

    const PagedArgs& a;
    const int lane, l16, g, kvh;
    RowTile t;
    const int* table;
    int last_page;
    int row0, last;              // first row of the tile, index of its last row in it
    int lo, hi;                  // keys this lane's row sees
    int tile_lo, tile_hi;        // keys that any row sees
    int full_lo, full_hi;        // keys that all rows see
    v8h qf[kSteps];
    v4f acc[kBlocks];
    float top, total;

    __device__ __forceinline__ RowPass(const PagedArgs& args, int kv_head) : a(args), lane(threadIdx.x & 63), l16(lane & 15), g(lane >> 4), kvh(kv_head) {}

    __device__ __forceinline__ void start(int seq, const RowTile& rows, int first_row) {
        t = rows;
        row0 = first_row;
        table = a.table + (size_t)seq * a.max_pages;
        last_page = t.length > 0 ? (t.length - 1) >> a.shift : 0;
        last = t.rows - row0 < 16 ? t.rows - row0 - 1 : 15;
        const int row = row0 + (l16 < last ? l16 : last);  // rows behind the last repeat it and are not stored
        const int tok = row / a.group, head = kvh * a.group + row % a.group;
        window(a, t.first_pos + tok, t.length, lo, hi);
        window(a, t.first_pos + row0 / a.group, t.length, tile_lo, full_hi);           // the first row's bounds are the lowest
        window(a, t.first_pos + (row0 + last) / a.group, t.length, full_lo, tile_hi);  // the last row's the highest
        const uint16_t* qp = a.query + (size_t)(t.start + tok) * a.query_stride + (size_t)head * kD;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) qf[s] = *(const v8h*)(qp + (kF8 ? (s >> 1) * 64 + 16 * g + 8 * (s & 1) : 32 * s + 8 * g));
#pragma unroll
        for (int c = 0; c < kBlocks; ++c) acc[c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        top = kNegInf;
        total = 0.0f;
    }

    // This lane reads keys (as rows of S) and values (as columns of O) from one page each.
    struct Ids {
        int key, value;
    };
    __device__ __forceinline__ Ids ids(int k0) const {
        int kc = (k0 + 8 * kU * (l16 >> 2)) >> a.shift, vc = (k0 + 8 * kU * g) >> a.shift;
        kc = kc > last_page ? last_page : kc;
        vc = vc > last_page ? last_page : vc;
        return {table[kc], table[vc]};
    }
    __device__ __forceinline__ size_t page_of(int id) const {
        id = (unsigned)id < (unsigned)a.pages ? id : 0;
        return ((size_t)id * a.kv_heads + kvh) * ((size_t)kD * kBytes << a.shift);
    }
    __device__ __forceinline__ void load_keys(int k0, int id, uint4 (&raw)[kU][2][kLoads]) const {
        const int key = k0 + 8 * kU * (l16 >> 2) + (l16 & 3);
        const uint8_t* p = a.key + page_of(id) + (size_t)(key & ((1 << a.shift) - 1)) * (kD * kBytes) + 16 * g;
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int s = 0; s < kLoads; ++s) raw[u][b][s] = *(const uint4*)(p + (8 * u + 4 * b) * kD * kBytes + 64 * s);
    }
    __device__ __forceinline__ void load_values(int k0, int id, uint4 (&raw)[kBlocks]) const {
        const int key = k0 + 8 * kU * g;
        const uint8_t* p = a.value + page_of(id) + (((size_t)l16 << a.shift) + (key & ((1 << a.shift) - 1))) * kBytes;
#pragma unroll
        for (int c = 0; c < kBlocks; ++c) raw[c] = *(const uint4*)(p + (((size_t)c * 16) << a.shift) * kBytes);
    }

    // Tiles k0, k0 + kSpan, ... below `end` (and inside the rows' range).
    __device__ __forceinline__ void run(int k0, int end, Odd<kD, 16>& odd) {
        while (k0 + kKeys <= tile_lo) k0 += kSpan;
        if (end > tile_hi) end = tile_hi;
        if (k0 >= end) return;
        Ids id = ids(k0), next = ids(k0 + kSpan);
        uint4 kraw[kU][2][kLoads], vraw[kBlocks];
        load_keys(k0, id.key, kraw);
        for (; k0 < end; k0 += kSpan) {
            load_values(k0, id.value, vraw);
            __builtin_amdgcn_sched_barrier(0);  // out before the wait for this tile's keys
            const int mine = k0 + 8 * kU * g;
            const bool ok = (unsigned)id.value < (unsigned)a.pages;
            const int there = ok ? t.length - mine : 0;  // keys from `mine` on that exist
            float p[8 * kU];
#pragma unroll
            for (int u = 0; u < kU; ++u)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    v4f sc{};
#pragma unroll
                    for (int s = 0; s < kSteps; ++s)
                        sc = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand<kF8>(kraw[u][b][s / kU], s % kU), qf[s], sc, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 4; ++r) p[8 * u + 4 * b + r] = sc[r] * a.scale_log2;
                }
            if (k0 + kSpan < end) load_keys(k0 + kSpan, next.key, kraw);
            const Ids later = ids(k0 + 2 * kSpan);
            __builtin_amdgcn_sched_barrier(0);
            const bool whole = k0 >= full_lo && k0 + kKeys <= full_hi && __all(ok);
            if (!whole) {
#pragma unroll
                for (int j = 0; j < 8 * kU; ++j)
                    if (mine + j < lo || mine + j >= hi || j >= there) p[j] = kNegInf;
            }
            float m = p[0];
#pragma unroll
            for (int j = 1; j < 8 * kU; ++j) m = __builtin_fmaxf(m, p[j]);
            m = max_level(max_level(m, 16), 32);
            const float new_top = __builtin_fmaxf(top, m);
            const float base = new_top == kNegInf ? 0.0f : new_top;
            const float keep = __builtin_amdgcn_exp2f(top - base);
            top = new_top;
            float sum = 0.0f;
            v8h pf[kU];
#pragma unroll
            for (int j = 0; j < 8 * kU; ++j) {
                p[j] = __builtin_amdgcn_exp2f(p[j] - base);
                sum += p[j];
                pf[j >> 3][j & 7] = (_Float16)p[j];
            }
            total = total * keep + sum;
#pragma unroll
            for (int c = 0; c < kBlocks; ++c) acc[c] = acc[c] * keep;
            if (!whole) {
                // keys that do not exist hold anything: their values are taken as zero
                constexpr int kPerWord = 4 / kBytes;
                uint32_t there_mask[4];
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const int n = there - w * kPerWord;  // keys of this word that exist
                    there_mask[w] = n >= kPerWord ? 0xffffffffu : (n <= 0 ? 0u : (1u << (8 * kBytes * n)) - 1u);
                }
#pragma unroll
                for (int c = 0; c < kBlocks; ++c) {
                    vraw[c].x &= there_mask[0];
                    vraw[c].y &= there_mask[1];
                    vraw[c].z &= there_mask[2];
                    vraw[c].w &= there_mask[3];
                    odd.template take<kF8>(vraw[c], 16 * c + l16, mine, [&](int r, int& from, int& to) {
                        from = lo;  // lane r < 16 has row r
                        to = r <= last ? hi : lo;
                    });
                }
            }
#pragma unroll
            for (int c = 0; c < kBlocks; ++c)
#pragma unroll
                for (int u = 0; u < kU; ++u) acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand<kF8>(vraw[c], u), pf[u], acc[c], 0, 0, 0);
            id = next;
            next = later;
        }
    }
};

// What the four waves hold of 16 rows, side by side in LDS.
template <int kD> struct Parts {
    float acc[4][16][kD + 4];
    float top[4][16], total[4][16];
};

template <int kD, bool kF8> __device__ __forceinline__ void to_lds(RowPass<kD, kF8>& pass, Parts<kD>& parts) {
    const int wave = threadIdx.x >> 6;
    const float total = add_level(add_level(pass.total, 16), 32);
#pragma unroll
    for (int c = 0; c < kD / 16; ++c) *(v4f*)&parts.acc[wave][pass.l16][16 * c + 4 * pass.g] = pass.acc[c];
    if (pass.g == 0) {
        parts.top[wave][pass.l16] = pass.top;
        parts.total[wave][pass.l16] = total;
    }
}

// Row r of the joined waves: its maximum and sum, and kD / 16 features from d0 on.
template <int kD> __device__ __forceinline__ void join(const Parts<kD>& parts, int r, int d0, float& best, float& total, float (&v)[kD / 16]) {
    best = parts.top[0][r];
#pragma unroll
    for (int w = 1; w < 4; ++w) best = __builtin_fmaxf(best, parts.top[w][r]);
    const float base = best == kNegInf ? 0.0f : best;
    total = 0.0f;
#pragma unroll
    for (int j = 0; j < kD / 16; ++j) v[j] = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float f = __builtin_amdgcn_exp2f(parts.top[w][r] - base);
        total += parts.total[w][r] * f;
#pragma unroll
        for (int j = 0; j < kD / 16; ++j) v[j] += parts.acc[w][r][d0 + j] * f;
    }
}

template <int kD> __device__ __forceinline__ bool put_odd(const Odd<kD, 16>& odd, int r, int d0, float (&v)[kD / 16]) {
    const bool any = __builtin_amdgcn_readfirstlane((int)odd.any) != 0;
    if (__builtin_expect(any, 0)) {
#pragma unroll
        for (int j = 0; j < kD / 16; ++j) v[j] = odd.put(v[j], r, d0 + j);
    }
    return any;
}

// Short contexts: one workgroup for the keys of a (sequence, kv head, 16 rows).
template <int kD, bool kF8> __global__ __launch_bounds__(256, 2) void paged_attention_rows_kernel(PagedArgs a) {
    __shared__ Parts<kD> parts;
    __shared__ Odd<kD, 16> odd;
    odd.clear(256);
    __syncthreads();
    const int kvh = blockIdx.x, seq = blockIdx.z, row0 = blockIdx.y * 16;
    const RowTile t = wave_sequence(a, seq);
    if (row0 >= t.rows) return;
    RowPass<kD, kF8> pass(a, kvh);
    pass.start(seq, t, row0);
    pass.run((pass.tile_lo & ~(pass.kKeys - 1)) + wave_index() * pass.kKeys, pass.tile_hi, odd);
    to_lds<kD, kF8>(pass, parts);
    __syncthreads();
    const int r = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * (kD / 16);
    if (r > pass.last) return;
    float best, total, v[kD / 16];
    join<kD>(parts, r, d0, best, total, v);
    put_odd<kD>(odd, r, d0, v);
    store_row<kD / 16>(a, t, kvh, row0 + r, kD, d0, total, v);
}

// ---- long contexts: the work of all sequences in equal shares --------------------------
//
// An item is a (sequence, kv head, 16 rows); its keys are a run of blocks of kSpan keys,
// and the items' blocks in a row are dealt to kShares workgroups in equal contiguous
// shares, so that one long sequence among short ones, or a single one, keeps the whole
// GPU busy.  A share boundary inside an item leaves it in parts: at most two a workgroup
// (the item its share begins in and the one it ends in), which a second launch joins.
constexpr int kShares = 512;  // two workgroups on each of 256 CUs
constexpr int kLeastShare = 2;

// Blocks of one item of a sequence (0: the sequence has no rows) and its first block.
template <int kSpan> __device__ __forceinline__ int item_blocks(const PagedArgs& a, const RowTile& t, int& first) {
    first = 0;
    if (t.rows == 0) return 0;
    int lo, hi, none;
    window(a, t.first_pos, t.length, lo, none);
    window(a, t.first_pos + (t.rows - 1) / a.group, t.length, none, hi);
    first = lo / kSpan;
    const int blocks = (hi + kSpan - 1) / kSpan - first;
    return blocks > 0 ? blocks : 1;  // rows that see nothing are still written
}
__device__ __forceinline__ int items_of(const PagedArgs& a, const RowTile& t) { return ((t.rows + 15) >> 4) * a.kv_heads; }

template <int kD, bool kF8>
__global__ __launch_bounds__(256, 2) void paged_attention_shares_kernel(PagedArgs a, Part<kD, 16>* slots, Join* joins) {
    constexpr int kSpan = RowPass<kD, kF8>::kSpan;
    __shared__ Parts<kD> parts;
    __shared__ Odd<kD, 16> odd;
    odd.clear(256);
    if (threadIdx.x == 0) joins[blockIdx.x].count = 0;
    Share share;
    const auto blocks_of = [&](const RowTile& t) {
        int first;
        return (long long)item_blocks<kSpan>(a, t, first) * items_of(a, t);
    };
    if (!deal<256>(a, kShares, kLeastShare, blockIdx.x, blocks_of, share)) return;

    int seq = share.seq;
    long long at = share.from, offset = share.offset;
    const int r = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * (kD / 16);
    while (at < share.to) {
        const RowTile t = wave_sequence(a, seq);
        int first;
        const int blocks = item_blocks<kSpan>(a, t, first), items = items_of(a, t);
        for (int item = blocks ? (int)(offset / blocks) : 0; blocks && item < items && at < share.to; ++item) {
            const int b0 = (int)(offset - (long long)item * blocks);
            const int n = share.to - at < blocks - b0 ? (int)(share.to - at) : blocks - b0;
            const int kvh = item % a.kv_heads, row0 = item / a.kv_heads * 16;
            RowPass<kD, kF8> pass(a, kvh);
            pass.start(seq, t, row0);
            pass.run((first + b0) * kSpan + wave_index() * pass.kKeys, (first + b0 + n) * kSpan, odd);
            __syncthreads();  // the previous item's parts are read
            to_lds<kD, kF8>(pass, parts);
            __syncthreads();
            float best, total, v[kD / 16];
            join<kD>(parts, r, d0, best, total, v);
            const bool any_odd = put_odd<kD>(odd, r, d0, v);
            if (n == blocks) {
                if (r <= pass.last) store_row<kD / 16>(a, t, kvh, row0 + r, kD, d0, total, v);
            } else {
                Part<kD, 16>& slot = slots[2 * blockIdx.x + (at == share.from ? 0 : 1)];
#pragma unroll
                for (int j = 0; j < kD / 16; j += 4) *(v4f*)&slot.acc[r][d0 + j] = v4f{v[j], v[j + 1], v[j + 2], v[j + 3]};
                if (d0 == 0) {
                    slot.top[r] = best;
                    slot.total[r] = total;
                }
                if (b0 == 0 && threadIdx.x == 0)
                    joins[blockIdx.x] = {t.start, t.rows, kvh, row0, (int)((at + blocks - 1) / share.size - blockIdx.x) + 1, at == share.from ? 0 : 1, {}};
            }
            if (any_odd) {
                __syncthreads();
                odd.clear(256);
                __syncthreads();
            }
            at += n;
            offset += n;
        }
        ++seq;
        offset = 0;
    }
}

// The parts of a divided item: the slot its first workgroup ended in, and the first slot
// of each of the following workgroups.  A workgroup joins one row; kJoinGroups groups of
// lanes take every kJoinGroups-th part each, because a single long sequence is divided
// into as many parts as there are shares (grouped: 9 us for 469 parts; a thread that
// takes all parts of its features in turn: 130 us).
constexpr int kJoinGroups = 16;

template <int kD> __global__ __launch_bounds__(kJoinGroups * kD / 4) void paged_attention_join_kernel(PagedArgs a, const Part<kD, 16>* slots, const Join* joins) {
    constexpr int kLanes = kD / 4;  // 4 features each
    __shared__ float part_acc[kJoinGroups][kD], part_top[kJoinGroups], part_total[kJoinGroups];
    const Join job = joins[blockIdx.x];
    const int r = blockIdx.y;
    if (job.count == 0) return;
    if (job.row0 + r >= job.rows) return;
    const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
    const Part<kD, 16>* first = slots + 2 * blockIdx.x;
    float top = kNegInf, total = 0.0f;
    v4f v{};
#pragma unroll 4
    for (int i = group; i < job.count; i += kJoinGroups) {
        const Part<kD, 16>& slot = first[2 * i + (i == 0 ? job.first_slot : 0)];
        const float new_top = __builtin_fmaxf(top, slot.top[r]);
        const float base = new_top == kNegInf ? 0.0f : new_top;
        const float f = __builtin_amdgcn_exp2f(slot.top[r] - base), keep = __builtin_amdgcn_exp2f(top - base);
        total = total * keep + slot.total[r] * f;
        v = v * keep + *(const v4f*)&slot.acc[r][4 * lane] * f;
        top = new_top;
    }
    *(v4f*)&part_acc[group][4 * lane] = v;
    if (lane == 0) {
        part_top[group] = top;
        part_total[group] = total;
    }
    __syncthreads();
    if (group != 0) return;
    float best = kNegInf;
#pragma unroll
    for (int w = 0; w < kJoinGroups; ++w) best = __builtin_fmaxf(best, part_top[w]);
    const float base = best == kNegInf ? 0.0f : best;
    total = 0.0f;
    v = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kJoinGroups; ++w) {
        const float f = __builtin_amdgcn_exp2f(part_top[w] - base);
        total += part_total[w] * f;
        v = v + *(const v4f*)&part_acc[w][4 * lane] * f;
    }
    const float o[4] = {v[0], v[1], v[2], v[3]};
    store_row<4>(a, {job.start, job.rows, 0, 0}, job.kvh, job.row0 + r, kD, 4 * lane, total, o);
}

// Whether one workgroup an item does: at most kDirectKeys keys each, by the table's width.
constexpr int kDirectKeys = 512;

// From this many query rows a sequence on, chunks of 128 rows share their loads.
constexpr int kChunksFrom = 17;

size_t paged_attention_workspace(int head_dim, int page_shift, int max_pages, int max_rows) {
    if ((long long)max_pages << page_shift <= kDirectKeys) return 0;
    if (max_rows >= kChunksFrom) return paged_chunks_workspace(head_dim);
    return 2 * kShares * (head_dim == 128 ? sizeof(Part<128, 16>) : sizeof(Part<64, 16>)) + kShares * sizeof(Join);
}

template <int kD, bool kF8> static void launch_rows(const PagedArgs& a, bool direct, int max_queries, void* workspace, hipStream_t s) {
    const unsigned rows = (unsigned)(max_queries * a.group);
    if (direct) {
        const dim3 grid((unsigned)a.kv_heads, (rows + 15) / 16, (unsigned)a.sequences);
        paged_attention_rows_kernel<kD, kF8><<<grid, 256, 0, s>>>(a);
        return;
    }
    auto* slots = (Part<kD, 16>*)workspace;
    Join* joins = (Join*)(slots + 2 * kShares);
    paged_attention_shares_kernel<kD, kF8><<<kShares, 256, 0, s>>>(a, slots, joins);
    paged_attention_join_kernel<kD><<<dim3(kShares, rows < 16 ? rows : 16), kJoinGroups * kD / 4, 0, s>>>(a, slots, joins);
}

void launch_paged_attention(int kind, const PagedArgs& a, int head_dim, int max_queries, void* workspace, hipStream_t s) {
    const bool direct = (long long)a.max_pages << a.shift <= kDirectKeys;
    if (max_queries * a.group >= kChunksFrom) {
        launch_paged_chunks(kind, a, head_dim, direct, max_queries, workspace, s);
        return;
    }
    if (head_dim == 128) {
        if (kind == 1) launch_rows<128, true>(a, direct, max_queries, workspace, s);
        else launch_rows<128, false>(a, direct, max_queries, workspace, s);
    } else {
        if (kind == 1) launch_rows<64, true>(a, direct, max_queries, workspace, s);
        else launch_rows<64, false>(a, direct, max_queries, workspace, s);
    }
}

}  // namespace pk
