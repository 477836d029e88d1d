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

// 16 query rows of a sequence and kv head, in scalar registers.
struct Rows {
    RowTile t;
    int seq, kvh, row0;
    __device__ __forceinline__ int last() const { return t.rows - row0 < 16 ? t.rows - row0 - 1 : 15; }  // index of the last row in the tile
};

// One wave's pass over key tiles for 16 query rows.  Loads are issued a stage ahead: the
// next tile's keys before the softmax, its values behind the products, and page ids two
// tiles ahead.
constexpr int kRowWaves = 4;  // of a workgroup; a CU holds two of them
// The largest probability is 2^kLift, not 1 (the division by the sum takes it out again): fp16
// then holds those down to 2^-29 of it to full precision and down to 2^-39 at all, where 2^-14
// and 2^-24 left out small ones that the sum counts and that are many in a long context.
// 2^15 times a value of 65504 and 2^30 keys stays far inside fp32.
constexpr float kLift = 15.0f;

template <int kD, bool kF8> struct RowPass {
    static constexpr int kSteps = kD / 32, kBlocks = kD / 16;  // MFMA steps of S over features, feature blocks of O
    static constexpr int kU = kF8 ? 2 : 1, kKeys = 32 * kU;    // 16 bytes of a value row hold 8 * kU keys; keys a wave tile
    static constexpr int kBytes = kF8 ? 1 : 2;
    static constexpr int kLoads = kSteps / kU;                 // 16-byte loads of a key row
    static constexpr int kSpan = kRowWaves * kKeys;            // keys that the waves take at once

    // The pages of a tile, by 16 keys, in scalar registers: their loads go through the scalar
    // cache, out of the way of the cache's, which return in order.
    struct Ids {
        int page0, page1, page2, page3;  // the last two with 64 keys only
        // The page of the 16 keys `part`, which differs from lane to lane.
        __device__ __forceinline__ int of(int part) const {
            const int p0 = page0, p1 = page1, p2 = page2, p3 = page3;
            int r = part & 1 ? p1 : p0;
            if constexpr (kKeys == 64) {
                const int up = part & 1 ? p3 : p2;
                r = part & 2 ? up : r;
            }
            return r;
        }
    };

    const PagedArgs& a;
    const int lane, l16, g;
    v8h qf[kSteps];
    uint4 kraw[kU][2][kLoads], vraw[kBlocks];
    Ids id, next;  // pages of the tile in kraw and vraw, and of the tile behind it
    v4f acc[kBlocks];
    float top, total;

    __device__ __forceinline__ explicit RowPass(const PagedArgs& args) : a(args), lane(threadIdx.x & 63), l16(lane & 15), g(lane >> 4) {}

    // Keys that any of the rows sees.
    __device__ __forceinline__ void reach(const Rows& w, int& lo, int& hi) const {
        int none;
        window(a, w.t.first_pos + w.row0 / a.group, w.t.length, lo, none);               // the first row's bounds are the lowest
        window(a, w.t.first_pos + (w.row0 + w.last()) / a.group, w.t.length, none, hi);  // the last row's the highest
    }
    // The wave's tiles k0, k0 + kSpan, ... < end among the keys [from, to) (from < to); with none of
    // them seen by a row, its first one there.
    __device__ __forceinline__ void tiles(const Rows& w, int from, int to, int& k0, int& end) const {
        int lo, hi;
        reach(w, lo, hi);
        const int first = from + wave_index() * kKeys;
        k0 = first;
        while (k0 + kKeys <= lo) k0 += kSpan;
        end = to < hi ? to : hi;
        if (k0 >= end) {
            k0 = first;
            end = first + 1;
        }
        k0 = __builtin_amdgcn_readfirstlane(k0);
        end = __builtin_amdgcn_readfirstlane(end);
    }
    __device__ __forceinline__ int row_of(const Rows& w) const { return w.row0 + (l16 < w.last() ? l16 : w.last()); }  // rows behind the last repeat it and are not stored

    __device__ __forceinline__ void load_query(const Rows& w) {
        const int row = row_of(w), tok = row / a.group, head = w.kvh * a.group + row % a.group;
        const uint16_t* qp = a.query + (size_t)(w.t.start + tok) * a.query_stride + (size_t)head * kD;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) qf[s] = *(const v8h*)(qp + (kF8 ? (s >> 1) * 64 + 16 * g + 8 * (s & 1) : 32 * s + 8 * g));
    }
    __device__ __forceinline__ Ids ids(const Rows& w, int k0) const {
        const int* table = a.table + (size_t)w.seq * a.max_pages;
        const int last_page = w.t.length > 0 ? (w.t.length - 1) >> a.shift : 0;
        const auto page = [&](int part) {
            const int c = (k0 + 16 * part) >> a.shift;
            return scalar_at(table, c > last_page ? last_page : c);
        };
        Ids r = {page(0), page(1), 0, 0};
        if constexpr (kKeys == 64) {
            r.page2 = page(2);
            r.page3 = page(3);
        }
        return r;
    }
    __device__ __forceinline__ size_t page_of(const Rows& w, int page) const {
        page = (unsigned)page < (unsigned)a.pages ? page : 0;
        return ((size_t)page * a.kv_heads + w.kvh) * ((size_t)kD * kBytes << a.shift);
    }
    __device__ __forceinline__ void load_keys(const Rows& w, int k0, const Ids& pages) {
        const int key = k0 + 8 * kU * (l16 >> 2) + (l16 & 3);
        const uint8_t* p = a.key + page_of(w, pages.of(kU * (l16 >> 2) >> 1)) + (size_t)(key & ((1 << a.shift) - 1)) * (kD * kBytes) + 16 * g;
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int s = 0; s < kLoads; ++s) kraw[u][b][s] = *(const uint4*)(p + (8 * u + 4 * b) * kD * kBytes + 64 * s);
    }
    __device__ __forceinline__ void load_values(const Rows& w, int k0, const Ids& pages) {
        const int key = k0 + 8 * kU * g;
        const uint8_t* p = a.value + page_of(w, pages.of(kU * g >> 1)) + (((size_t)l16 << a.shift) + (key & ((1 << a.shift) - 1))) * kBytes;
#pragma unroll
        for (int c = 0; c < kBlocks; ++c) vraw[c] = *(const uint4*)(p + (((size_t)c * 16) << a.shift) * kBytes);
    }

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int c = 0; c < kBlocks; ++c) acc[c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        top = kNegInf;
        total = 0.0f;
    }

    // The first tile's loads.
    __device__ __forceinline__ void open(const Rows& w, int k0) {
        id = ids(w, k0);
        next = ids(w, k0 + kSpan);
        load_query(w);
        load_keys(w, k0, id);
        load_values(w, k0, id);
    }

    // The tiles k0, k0 + kSpan, ... < end (at least one), the first of which is on its way
    // already.  With `chain`, the tile k1 of the rows w1, in the pages id1, and their query are
    // asked for behind the last.
    __device__ __forceinline__ void run(const Rows& w, int k0, int end, Odd<kD, 16>& odd, bool chain, const Rows& w1, int k1, Ids id1) {
        int lo, hi, all_lo, all_hi, none;  // the keys that this lane's row sees, and those that all rows see
        window(a, w.t.first_pos + row_of(w) / a.group, w.t.length, lo, hi);
        window(a, w.t.first_pos + w.row0 / a.group, w.t.length, none, all_hi);
        window(a, w.t.first_pos + (w.row0 + w.last()) / a.group, w.t.length, all_lo, none);
        for (bool more = true; more; k0 += kSpan) {
            more = k0 + kSpan < end;
            const int mine = k0 + 8 * kU * g;
            const bool ok = (unsigned)id.of(kU * g >> 1) < (unsigned)a.pages;
            const int there = ok ? w.t.length - mine : 0;  // keys from `mine` on that exist
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
            const Rows up = more ? w : w1;
            const Ids up_id = more ? next : id1;
            const int up_k0 = more ? k0 + kSpan : k1;
            Ids later = next;
            if (more || chain) {
                if (!more) load_query(w1);
                load_keys(up, up_k0, up_id);
                later = ids(up, up_k0 + kSpan);
            }
            __builtin_amdgcn_sched_barrier(0);
            const bool whole = k0 >= all_lo && k0 + kKeys <= all_hi && __all(ok);
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
            const float keep = weight_of(top - base);
            top = new_top;
            float sum = 0.0f;
            v8h pf[kU];
#pragma unroll
            for (int j = 0; j < 8 * kU; ++j) {
                p[j] = __builtin_amdgcn_exp2f((p[j] - base) + kLift);  // in this order: base - kLift would be rounded
                sum += p[j];
                pf[j >> 3][j & 7] = (_Float16)p[j];
            }
            total = total * keep + sum;
#pragma unroll
            for (int c = 0; c < kBlocks; ++c) acc[c] = acc[c] * keep;
            // a probability that is zero in fp16, while all rows see all keys
            bool faint = false;
            if constexpr (!kF8) {
                float least = p[0];
#pragma unroll
                for (int j = 1; j < 8; ++j) least = __builtin_fminf(least, p[j]);
                faint = __any(least <= 0x1p-25f);
            }
            if (!whole || faint) {
                // keys that do not exist hold anything: their values are taken as zero
                constexpr int kPerWord = 4 / kBytes;
                uint32_t there_mask[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int n = there - i * kPerWord;  // keys of this word that exist
                    there_mask[i] = n >= kPerWord ? 0xffffffffu : (n <= 0 ? 0u : (1u << (8 * kBytes * n)) - 1u);
                }
                uint32_t any = 0;  // (one look for all of them: the code for each stays out of the way)
#pragma unroll
                for (int c = 0; c < kBlocks; ++c) {
                    vraw[c].x &= there_mask[0];
                    vraw[c].y &= there_mask[1];
                    vraw[c].z &= there_mask[2];
                    vraw[c].w &= there_mask[3];
                    any |= not_finite<kF8>(vraw[c]);
                }
                if (__builtin_expect(__any(any != 0), 0)) {
#pragma unroll
                    for (int c = 0; c < kBlocks; ++c)
                        odd.template take<kF8>(vraw[c], 16 * c + l16, mine, whole, [&](int r, int& from, int& to) {
                            from = lo;  // lane r < 16 has row r
                            to = r <= w.last() ? hi : lo;
                        });
                }
            }
#pragma unroll
            for (int c = 0; c < kBlocks; ++c)
#pragma unroll
                for (int u = 0; u < kU; ++u) acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand<kF8>(vraw[c], u), pf[u], acc[c], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
            if (more || chain) load_values(up, up_k0, up_id);
            id = up_id;
            next = later;
            __builtin_amdgcn_sched_barrier(0);  // out before the wait for the next tile's keys
        }
    }
};

// What the waves hold of 16 rows, side by side in LDS.
template <int kD> struct Parts {
    float acc[kRowWaves][16][kD + 4];
    float top[kRowWaves][16], total[kRowWaves][16];
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

// Row r of the joined waves: its maximum and sum, and kN features from d0 on.
template <int kD, int kN> __device__ __forceinline__ void join(const Parts<kD>& parts, int r, int d0, float& best, float& total, float (&v)[kN]) {
    best = parts.top[0][r];
#pragma unroll
    for (int w = 1; w < kRowWaves; ++w) best = __builtin_fmaxf(best, parts.top[w][r]);
    const float base = best == kNegInf ? 0.0f : best;
    total = 0.0f;
#pragma unroll
    for (int j = 0; j < kN; ++j) v[j] = 0.0f;
#pragma unroll
    for (int w = 0; w < kRowWaves; ++w) {
        const float f = weight_of(parts.top[w][r] - base);
        total += parts.total[w][r] * f;
#pragma unroll
        for (int j = 0; j < kN; ++j) v[j] += parts.acc[w][r][d0 + j] * f;
    }
}

template <int kD, int kN> __device__ __forceinline__ void put_odd(const Odd<kD, 16>& odd, bool any, int r, int d0, float (&v)[kN]) {
    if (__builtin_expect(any, 0)) {
#pragma unroll
        for (int j = 0; j < kN; ++j) v[j] = odd.put(v[j], r, d0 + j);
    }
}

// Short contexts: one workgroup for the keys of a (sequence, kv head, 16 rows).
// A single token's 93 keys, 8 heads, fp16: 4.7 us, of which a launch is 2.5 and the rest the
// chain length -> page id -> keys -> scores -> values -> the waves' join.
template <int kD, bool kF8> __global__ __launch_bounds__(64 * kRowWaves, 2) void paged_attention_rows_kernel(PagedArgs a) {
    constexpr int kN = kD / (4 * kRowWaves);
    using Pass = RowPass<kD, kF8>;
    __shared__ Parts<kD> parts;
    __shared__ Odd<kD, 16> odd;
    odd.clear(64 * kRowWaves);
    __syncthreads();
    const Rows w = {wave_sequence(a, blockIdx.z), (int)blockIdx.z, (int)blockIdx.x, (int)blockIdx.y * 16};
    if (w.row0 >= w.t.rows) return;
    Pass pass(a);
    int lo, hi, k0, end;
    pass.reach(w, lo, hi);
    lo &= ~(Pass::kSpan - 1);  // a wave's tiles are the same keys whichever row comes first
    pass.tiles(w, lo, hi > lo ? hi : lo + 1, k0, end);
    pass.clear();
    pass.open(w, k0);
    pass.run(w, k0, end, odd, false, w, 0, {});
    to_lds(pass, parts);
    __syncthreads();
    const int r = threadIdx.x / (4 * kRowWaves), d0 = threadIdx.x % (4 * kRowWaves) * kN;
    if (r > w.last()) return;
    float best, total, v[kN];
    join(parts, r, d0, best, total, v);
    put_odd(odd, odd.any != 0, r, d0, v);
    store_row<kN>(a, w.t, w.kvh, w.row0 + r, kD, d0, total, v);
}

// ---- long contexts: the work of all sequences in equal shares --------------------------
//
// An item is a (sequence, kv head, 16 rows); its keys are a run of blocks of kSpan keys,
// and the items' blocks in a row are dealt to kShares workgroups in equal contiguous
// shares, so that one long sequence among short ones, or a single one, keeps the whole
// GPU busy.  A share boundary inside an item leaves it in parts: at most two a workgroup
// (the item its share begins in and the one it ends in), which a second launch joins.
//
// The cache's bytes are what bounds it: 64 sequences of 4096 e4m3 keys, 8 kv heads of 128 (538
// MB), take 95 us, 5.6 TB/s (the same loads alone 92 us); of 1 to 8111 keys (532 to 568 MB) 112,
// where the workgroups' ends lie 70 to 110 us after the start, for the memory does not serve
// them alike.  More, smaller shares even that out but pay more beginnings and parts: 1024 take
// 102 and 116 us, 2048 110 and 123.  One sequence of 131072 fp16 keys, 2 kv heads (134 MB): 31
// us, of which 5 are the way to the first keys.
constexpr int kShares = 512;  // two workgroups on each of 256 CUs
constexpr int kLeastShare = 2;  // one sequence of 1900 e4m3 keys 11.9 us; with 1 13.5, with 4 14.3

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

// A share's part of one item: its blocks [b0, b0 + n) of `blocks`, the first of the item's being `first`.
struct ShareRun {
    Rows w;
    long long left;  // blocks of the share from here on
    int item, first, blocks, b0, n;
    __device__ __forceinline__ void cut(const PagedArgs& a) {
        w.kvh = __builtin_amdgcn_readfirstlane(item % a.kv_heads);
        w.row0 = __builtin_amdgcn_readfirstlane(item / a.kv_heads * 16);
        n = __builtin_amdgcn_readfirstlane(left < blocks - b0 ? (int)left : blocks - b0);
    }
    // The one behind it; false: the share ends.
    template <int kSpan> __device__ __forceinline__ bool advance(const PagedArgs& a) {
        left -= n;
        if (left <= 0) return false;
        b0 = 0;
        if (++item >= items_of(a, w.t)) {
            item = 0;
            do {
                w.t = wave_sequence(a, ++w.seq);
                blocks = __builtin_amdgcn_readfirstlane(item_blocks<kSpan>(a, w.t, first));
            } while (blocks == 0);  // ends: blocks are left
        }
        cut(a);
        return true;
    }
};

template <int kD, bool kF8>
__global__ __launch_bounds__(64 * kRowWaves, 2) void paged_attention_shares_kernel(PagedArgs a, Part<kD, 16>* slots, Join* joins) {
    constexpr int kN = kD / (4 * kRowWaves);
    using Pass = RowPass<kD, kF8>;
    constexpr int kSpan = Pass::kSpan;
    __shared__ Parts<kD> parts;
    __shared__ Odd<kD, 16> odd;
    odd.clear(64 * kRowWaves);
    if (threadIdx.x == 0) joins[blockIdx.x].count = 0;
    Share share;
    const auto blocks_of = [&](const RowTile& t) {
        int first;
        return (long long)item_blocks<kSpan>(a, t, first) * items_of(a, t);
    };
    if (!deal<64 * kRowWaves, kShares, kLeastShare>(a, blockIdx.x, blocks_of, share)) return;
    __syncthreads();  // `odd` is clear

    Pass pass(a);
    // The run behind the current one: its first tile's pages are asked for at the current one's
    // start, its query and that tile at the current one's end, before the parts are joined.
    ShareRun next;
    next.w.seq = share.seq;
    next.w.t = wave_sequence(a, share.seq);
    next.left = share.to - share.from;
    next.blocks = __builtin_amdgcn_readfirstlane(item_blocks<kSpan>(a, next.w.t, next.first));
    next.item = __builtin_amdgcn_readfirstlane((int)(share.offset / next.blocks));
    next.b0 = (int)(share.offset - (long long)next.item * next.blocks);
    next.cut(a);
    int k0, end;
    const auto tiles = [&] { pass.tiles(next.w, (next.first + next.b0) * kSpan, (next.first + next.b0 + next.n) * kSpan, k0, end); };
    tiles();
    pass.open(next.w, k0);

    const int r = threadIdx.x / (4 * kRowWaves), d0 = threadIdx.x % (4 * kRowWaves) * kN;
    for (bool more = true; more;) {
        const ShareRun now = next;
        const int now_k0 = k0, now_end = end;
        more = next.advance<kSpan>(a);
        typename Pass::Ids id = {};
        if (more) {
            tiles();
            id = pass.ids(next.w, k0);
        }
        pass.clear();
        pass.run(now.w, now_k0, now_end, odd, more, next.w, k0, id);
        __syncthreads();  // the previous item's parts are read, and what this one's values hold is noted
        // Between the barriers no wave is in a run: all waves find the same here, and take the
        // same way to the next run, whose values are noted only after that.
        const bool any_odd = __builtin_amdgcn_readfirstlane((int)odd.any) != 0;
        to_lds(pass, parts);
        __syncthreads();
        float best, total, v[kN];
        join(parts, r, d0, best, total, v);
        put_odd(odd, any_odd, r, d0, v);
        if (now.n == now.blocks) {
            if (r <= now.w.last()) store_row<kN>(a, now.w.t, now.w.kvh, now.w.row0 + r, kD, d0, total, v);
        } else {
            const long long at = share.to - now.left;
            Part<kD, 16>& slot = slots[2 * blockIdx.x + (at == share.from ? 0 : 1)];
#pragma unroll
            for (int j = 0; j < kN; j += 4) *(v4f*)&slot.acc[r][d0 + j] = v4f{v[j], v[j + 1], v[j + 2], v[j + 3]};
            if (d0 == 0) {
                slot.top[r] = best;
                slot.total[r] = total;
            }
            if (now.b0 == 0 && threadIdx.x == 0)
                joins[blockIdx.x] = {now.w.t.start, now.w.t.rows, now.w.kvh, now.w.row0, share_of<kShares, kLeastShare>(share.all, at + now.blocks - 1) - (int)blockIdx.x + 1,
                                     at == share.from ? 0 : 1, {}};
        }
        if (any_odd) {
            __syncthreads();
            odd.clear(64 * kRowWaves);
            __syncthreads();
        }
    }
}

// The parts of a divided item are the slot that its first workgroup ended in, and the first
// slots of the following workgroups.  A workgroup joins row blockIdx.y of the items that
// begin in kJoinGroups shares: each of its groups of lanes takes one of them that has few
// parts, and all groups together those that have many (a single long sequence is divided
// into as many parts as there are shares: 6 us for 469 of them, 8 rows; 4 us where items have
// two or three).
constexpr int kJoinGroups = 16;
constexpr int kFewParts = 4;

// Parts i, i + step, ... of row r, four features a lane; kDeep of them are asked for at once.
template <int kD, int kDeep>
__device__ __forceinline__ void join_parts(const Part<kD, 16>* first, const Join& job, int i, int step, int r, int lane, float& top, float& total, v4f& v) {
    top = kNegInf;
    total = 0.0f;
    v = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    for (; i < job.count; i += kDeep * step) {
        float tops[kDeep], totals[kDeep];
        v4f accs[kDeep];
#pragma unroll
        for (int j = 0; j < kDeep; ++j) {
            const int at = i + j * step < job.count ? i + j * step : i;
            const Part<kD, 16>& slot = first[2 * at + (at == 0 ? job.first_slot : 0)];
            tops[j] = i + j * step < job.count ? slot.top[r] : kNegInf;
            totals[j] = slot.total[r];
            accs[j] = *(const v4f*)&slot.acc[r][4 * lane];
        }
        float new_top = top;
#pragma unroll
        for (int j = 0; j < kDeep; ++j) new_top = __builtin_fmaxf(new_top, tops[j]);
        const float base = new_top == kNegInf ? 0.0f : new_top, keep = weight_of(top - base);
        top = new_top;
        total *= keep;
        v = v * keep;
#pragma unroll
        for (int j = 0; j < kDeep; ++j) {
            const float f = weight_of(tops[j] - base);
            if (i + j * step >= job.count) continue;  // no part twice, not even with weight 0: it may hold a NaN
            total += totals[j] * f;
            v = v + accs[j] * f;
        }
    }
}

template <int kD> __global__ __launch_bounds__(kJoinGroups * kD / 4) void paged_attention_join_kernel(PagedArgs a, const Part<kD, 16>* slots, const Join* joins) {
    constexpr int kLanes = kD / 4;
    __shared__ float part_acc[kJoinGroups][kD], part_top[kJoinGroups], part_total[kJoinGroups];
    __shared__ int many[kJoinGroups];
    const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes, r = blockIdx.y, share0 = blockIdx.x * kJoinGroups;
    const Join mine = joins[share0 + group];
    const bool here = mine.count && mine.row0 + r < mine.rows;
    float top, total;
    v4f v;
    const auto store = [&](const Join& job) {
        const float o[4] = {v[0], v[1], v[2], v[3]};
        store_row<4>(a, {job.start, job.rows, 0, 0}, job.kvh, job.row0 + r, kD, 4 * lane, total, o);
    };
    if (lane == 0) many[group] = here && mine.count > kFewParts;
    if (here && mine.count <= kFewParts) {
        join_parts<kD, kFewParts>(slots + 2 * (share0 + group), mine, 0, 1, r, lane, top, total, v);
        store(mine);
    }
    __syncthreads();
    for (int j = 0; j < kJoinGroups; ++j) {
        if (!many[j]) continue;
        const Join job = joins[share0 + j];
        join_parts<kD, 8>(slots + 2 * (share0 + j), job, group, kJoinGroups, r, lane, top, total, v);
        *(v4f*)&part_acc[group][4 * lane] = v;
        if (lane == 0) {
            part_top[group] = top;
            part_total[group] = total;
        }
        __syncthreads();
        if (group == 0) {
            float best = kNegInf;
#pragma unroll
            for (int w = 0; w < kJoinGroups; ++w) best = __builtin_fmaxf(best, part_top[w]);
            const float base = best == kNegInf ? 0.0f : best;
            total = 0.0f;
            v = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < kJoinGroups; ++w) {
                const float f = weight_of(part_top[w] - base);
                total += part_total[w] * f;
                v = v + *(const v4f*)&part_acc[w][4 * lane] * f;
            }
            store(job);
        }
        __syncthreads();
    }
}

// One launch, a workgroup an item, where a full table's keys and values of a kv head are few
// bytes: a CU reads about 33 bytes a ns, while shares take 12 us however little there is
// (one sequence, 8 kv heads of 128, e4m3: 900 keys 9.2 us against 11.8, 1900 14.2 and 12.0;
// fp16: 448 keys 9.1 and 11.5, 900 16.3 and 11.7).  With kManyItems it is ahead further up, since
// workgroups that end early make room: 16 sequences of 1900 e4m3 keys 15.5 us against 19.5, 64 of
// them 49 and 54, 200 146 and 157, 64 of 900 fp16 keys 48 and 53.  Four times as far (200 of
// 4000) it is still 297 and 305 us, but a lone long sequence among idle ones waits for one CU.
// The table's width decides, not the lengths, which the host does not know: a short sequence in
// a wide table takes shares (93 keys 12.3 us).
constexpr long long kDirectBytes = 384 << 10, kDirectBytesMany = 512 << 10;
constexpr long long kManyItems = 128;
// So do up to 32 rows of a kv head, in two tiles that read the same keys: one sequence of 24
// rows, 448 keys, 9.9 us against 14.7 for a chunk's kernel, 64 of them of 1900 keys 62 and 92.
// With four tiles the reading overtakes the gain (64 sequences of 48 rows, 1900 fp16 keys: 180
// and 117).  Long tables (8 sequences of 24 rows, 12000 keys) take 115 in shares, 78 in chunks.
constexpr int kDirectRows = 32;
// A chunk's kernel divides even short tables: one sequence of 80 rows, 1900 keys, 37 us in
// shares, 51 directly.
constexpr int kChunkDirectKeys = 512;

static bool rows_directly(int head_dim, int key_bytes, long long keys, long long rows, long long items) {
    return keys * head_dim * key_bytes * 2 <= (items >= kManyItems ? kDirectBytesMany : kDirectBytes) && rows <= kDirectRows;
}

// Enough for either kind of cache and for any smaller call: fewer sequences, queries or pages.
size_t paged_attention_workspace(int head_dim, int page_shift, int max_pages, int max_rows) {
    const long long keys = (long long)max_pages << page_shift;
    if (rows_directly(head_dim, 2, keys, max_rows, 0)) return 0;
    if (max_rows > 16) return keys <= kChunkDirectKeys ? 0 : paged_chunks_workspace(head_dim);
    return 2 * kShares * (head_dim == 128 ? sizeof(Part<128, 16>) : sizeof(Part<64, 16>)) + kShares * sizeof(Join);
}

template <int kD, bool kF8> static void launch_rows(const PagedArgs& a, bool direct, int max_queries, void* workspace, hipStream_t s) {
    const unsigned rows = (unsigned)(max_queries * a.group);
    if (direct) {
        const dim3 grid((unsigned)a.kv_heads, (rows + 15) / 16, (unsigned)a.sequences);
        paged_attention_rows_kernel<kD, kF8><<<grid, 64 * kRowWaves, 0, s>>>(a);
        return;
    }
    auto* slots = (Part<kD, 16>*)workspace;
    Join* joins = (Join*)(slots + 2 * kShares);
    paged_attention_shares_kernel<kD, kF8><<<kShares, 64 * kRowWaves, 0, s>>>(a, slots, joins);
    paged_attention_join_kernel<kD><<<dim3(kShares / kJoinGroups, rows < 16 ? rows : 16), kJoinGroups * kD / 4, 0, s>>>(a, slots, joins);
}

void launch_paged_attention(int kind, const PagedArgs& a, int head_dim, int max_queries, void* workspace, hipStream_t s) {
    const long long keys = (long long)a.max_pages << a.shift, rows = (long long)max_queries * a.group;
    const bool direct = rows_directly(head_dim, kind == 1 ? 1 : 2, keys, rows, (long long)a.sequences * a.kv_heads);
    if (rows > 16 && !direct) {
        launch_paged_chunks(kind, a, head_dim, keys <= kChunkDirectKeys, max_queries, workspace, s);
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
