// Which keys a row of the paged attention sees, and how the work of a batch is cut into
// blocks and dealt to workgroups.  constexpr, so that the same functions run in a host test.
// Args: the call's sizes (PagedArgs): left, right (-1: unlimited), group, kv_heads.
#pragma once

namespace pk {

// One sequence's view for a tile of query rows.
struct RowTile {
    int start, rows, length, first_pos;  // first_pos: position of the sequence's first new token
};

// Keys [lo, hi) that a query at `pos` sees.
template <class Args> constexpr void window(const Args& a, int pos, int length, int& lo, int& hi) {
    lo = a.left < 0 || pos < a.left ? 0 : pos - a.left;
    hi = a.right < 0 || length - pos <= a.right ? length : pos + a.right + 1;
    if (hi < 0) hi = 0;
}

// The work of all sequences in a row, in blocks of keys, is dealt to kShares workgroups in
// contiguous shares that differ by one block at most, or of kLeast blocks where there are
// too few.
template <int kShares, int kLeast> constexpr long long share_begin(long long all, int index) {
    if (all >= kShares * kLeast) return index * all / kShares;
    return index * kLeast < all ? index * kLeast : all;
}
// The share that holds a block: the last one that begins at or before it.
template <int kShares, int kLeast> constexpr int share_of(long long all, long long block) {
    return (int)(all >= kShares * kLeast ? ((block + 1) * kShares - 1) / all : block / kLeast);
}

// ---- chunks: row tiles of 256 rows, tiles of 64 keys -------------------------------------

constexpr int kChunkRows = 256, kTileKeys = 64;

// Blocks (tiles of keys) that the rows of one row tile see, from block `first` on.
template <class Args> constexpr int chunk_blocks(const Args& a, const RowTile& t, int tile, int& first) {
    const int r0 = tile * kChunkRows, r1 = r0 + kChunkRows < t.rows ? r0 + kChunkRows - 1 : t.rows - 1;
    int lo = 0, hi = 0, none = 0;
    window(a, t.first_pos + r0 / a.group, t.length, lo, none);
    window(a, t.first_pos + r1 / a.group, t.length, none, hi);
    first = lo / kTileKeys;
    const int n = (hi + kTileKeys - 1) / kTileKeys - first;
    return n > 0 ? n : 1;
}

// With a causal mask the row tiles of a sequence differ in length; tile j and tile n - 1 -
// j together hardly do (their keys are concave in j, and the blocks of a tile less than two
// more than its keys), so they are dealt as one item of `pair` blocks, at least what any pair
// has; the middle tile of an odd number is an item by itself.  Keys are not concave where the
// first rows stand before key 0 and see nothing (more new tokens than keys): a pair then has
// room for two tiles of all keys.
struct Pairs {
    int tiles, pair, middle;
    long long per_head;
};
template <class Args> constexpr Pairs pairs_of(const Args& a, const RowTile& t) {
    Pairs p{};
    p.tiles = (t.rows + kChunkRows - 1) / kChunkRows;
    if (p.tiles == 0) return p;
    int first = 0;
    const int mid = chunk_blocks(a, t, p.tiles / 2, first);
    if (p.tiles & 1) p.middle = mid;
    const int all = (t.length + kTileKeys - 1) / kTileKeys;
    if (p.tiles > 1 && a.right >= 0 && t.first_pos + a.right + 1 < 0) p.pair = 2 * (all > 1 ? all : 1);
    else if (p.tiles > 1) p.pair = mid + chunk_blocks(a, t, (p.tiles - 1) / 2, first) + 3;
    p.per_head = (long long)(p.tiles / 2) * p.pair + p.middle;
    return p;
}

// A row tile's blocks among its sequence's: `tile` < 0 where a pair has blocks too many.
struct Span {
    int kvh, tile, first;      // first: the block of keys that the tile begins with
    int at, blocks;            // the place in the span, and the span's length
};
// (A kv head may have more than 2^31 blocks: 2^23 rows over 2^22 keys.)
template <class Args> constexpr Span span_at(const Args& a, const RowTile& t, const Pairs& p, long long offset) {
    Span s{};
    s.kvh = (int)(offset / p.per_head);
    const long long in_head = offset - s.kvh * p.per_head;
    const int pair = p.pair ? (int)(in_head / p.pair) : 0;
    const bool middle = pair == p.tiles / 2;
    s.tile = pair;
    s.at = (int)(in_head - (long long)pair * p.pair);
    s.blocks = chunk_blocks(a, t, s.tile, s.first);
    if (!middle && s.at >= s.blocks) {
        s.at -= s.blocks;
        const int rest = p.pair - s.blocks;
        s.tile = p.tiles - 1 - pair;
        s.blocks = chunk_blocks(a, t, s.tile, s.first);
        if (s.at >= s.blocks) {
            s.at -= s.blocks;
            s.blocks = rest - s.blocks;
            s.tile = -1;
        }
    }
    return s;
}

}  // namespace pk
