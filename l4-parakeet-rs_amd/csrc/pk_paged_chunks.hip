// The paged attention for chunks of new tokens: 256 query rows a workgroup, 32 a wave.
//
// The same two products as for few rows (S^T = K Q^T, O^T = V^T P^T, probabilities in
// registers), on 32 x 32 x 16 MFMAs.  The eight waves share 64-key tiles of keys and
// values in LDS, which the loads fill directly, three tiles ahead of the one that is
// multiplied (four buffers, two barriers a tile).  Tile rows are whole key or value rows
// whose 16-byte chunks are XOR-swizzled at the source, since such loads write LDS in lane
// order.
//
// Probabilities are fp16, which the matrix instructions multiply; fp32 ones run at a
// sixteenth of the rate.
//
// Bound by the vector instructions next to the MFMAs: 32 scores a lane and tile, each a
// maximum, a fused scale and subtraction, an exponential, a sum and half a conversion, about
// 130 of some 230; the others are addresses and bookkeeping.  The running output is only
// rescaled on tiles that raise some row's maximum.  4 sequences of up to 777 new tokens over
// up to 12007 fp16 keys, 32 / 8 heads of 128: 770 to 920 TFLOP/s with the joins, by the
// lengths (135 to 342 GFLOP; equal lengths 960; a library product of fp16 8192^3 1431).  Of
// about 3470 cycles a tile (of two waves a SIMD) the products take 1290, the softmax with the
// next loads 1500 to 1650, and 820 are waits at the two barriers; the clock is at 1.9 GHz then.
// A run of tiles begins and ends with 9 us of loads and stores that nothing covers.  The same
// with e4m3 keys 970 TFLOP/s, with heads of 64 740 (half the products for the same softmax;
// e4m3 700), and with a window of 145 keys 59 us for 7.4 GFLOP: most tiles lie at an edge.
#include "pk_paged_attention.hpp"

typedef float v16f __attribute__((ext_vector_type(16)));

namespace pk {

constexpr int kChunkWaves = 8, kChunkThreads = 64 * kChunkWaves, kBuffers = 4;
static_assert(kChunkRows == 32 * kChunkWaves);
constexpr int kChunkShares = 256;  // a workgroup on each of 256 CUs
// Fewer blocks a share than this are more parts to join than work: 100 tokens over 3000 keys, 8 kv
// heads of 4: 47 us, with one block at least 117, with twelve 52; 24 rows over 1900 keys 25, 41, 34.
constexpr int kLeastChunkShare = 4;

template <int kD, bool kF8> struct ChunkPass {
    static constexpr int kBytes = kF8 ? 1 : 2;
    static constexpr int kSteps = kD / 16, kBlocks = kD / 32;          // MFMA steps of S over features, feature blocks of O
    static constexpr int kKeyBytes = kD * kBytes, kValueBytes = kTileKeys * kBytes;  // tile rows
    static constexpr int kKeyTile = kTileKeys * kKeyBytes, kValueTile = kD * kValueBytes;
    static constexpr int kBuffer = kKeyTile + kValueTile;
    static constexpr int kKeyChunks = kKeyBytes / 16, kValueChunks = kValueBytes / 16;
    static constexpr uint32_t kAllPages = (1u << kValueChunks) - 1u;
    // a load of a wave fills 1 KB: the keys' units go to the waves in runs, the values' in
    // turn; where there are fewer units than waves, the keys' go to the first waves and the
    // values' to the others, so that every wave has kLoads a tile
    static constexpr int kKeyUnits = kKeyTile / 1024, kValueUnits = kValueTile / 1024;
    static constexpr bool kSplit = kKeyUnits < kChunkWaves;
    static constexpr int kKeyLoads = kSplit ? 1 : kKeyUnits / kChunkWaves, kValueLoads = kSplit ? 1 : kValueUnits / kChunkWaves;
    static constexpr int kLoads = kSplit ? 1 : kKeyLoads + kValueLoads;
    static_assert(!kSplit || kKeyUnits + kValueUnits == kChunkWaves);
    static constexpr int kKeyRun = 16 / (kSplit ? 1 : 2);  // keys that a wave loads

    const PagedArgs& a;
    uint8_t* lds;
    const int lane, wave, l32, h, kvh;
    RowTile t;
    const int* table;
    int last_page, ring;      // ring: tile b lies in buffer (b + ring) mod kBuffers
    int row0, last, row;      // this wave's first row, its last row's index (< 0: none), this lane's row
    int lo, hi, full_lo, full_hi, wave_lo, wave_hi;
    uint32_t key_off[kKeyLoads], value_off[kValueLoads];
    int tile_full_lo, tile_full_hi;  // keys that all of the workgroup's rows see
    float scale, sign;
    v8h qf[kSteps];
    v16f acc[kBlocks];
    float top, total;         // in raw scores; total of this lane's keys

    __device__ __forceinline__ ChunkPass(const PagedArgs& args, uint8_t* buffers, int kv_head)
        : a(args), lds(buffers), lane(threadIdx.x & 63), wave(wave_index()), l32(lane & 31), h(lane >> 5), kvh(kv_head) {
        // a negative scale turns the queries' signs, so that the largest score has the largest
        // product; 0 becomes tiny, so that -inf stays -inf
        sign = a.scale_log2 < 0.0f ? -1.0f : 1.0f;
        scale = __builtin_fmaxf(__builtin_fabsf(a.scale_log2), 1e-30f);
        place_loads();
    }

    __device__ __forceinline__ void start(int seq, const RowTile& rows, int tile) {
        t = rows;
        table = a.table + (size_t)seq * a.max_pages;
        last_page = t.length > 0 ? (t.length - 1) >> a.shift : 0;
        row0 = tile * kChunkRows + wave * 32;
        last = t.rows - row0 < 32 ? t.rows - row0 - 1 : 31;
        const int at = row0 + (l32 < last ? l32 : last);
        row = at < 0 ? 0 : (at < t.rows ? at : t.rows - 1);
        const int tok = row / a.group, head = kvh * a.group + row % a.group;
        window(a, t.first_pos + tok, t.length, lo, hi);
        if (last >= 0) {
            window(a, t.first_pos + row0 / a.group, t.length, wave_lo, full_hi);
            window(a, t.first_pos + (row0 + last) / a.group, t.length, full_lo, wave_hi);
        } else {
            wave_lo = wave_hi = full_lo = full_hi = 0;
        }
        int none;
        const int tile_last = (tile + 1) * kChunkRows < t.rows ? (tile + 1) * kChunkRows - 1 : t.rows - 1;
        window(a, t.first_pos + tile * kChunkRows / a.group, t.length, none, tile_full_hi);
        window(a, t.first_pos + tile_last / a.group, t.length, tile_full_lo, none);
        const uint16_t* qp = a.query + (size_t)(t.start + tok) * a.query_stride + (size_t)head * kD;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            qf[s] = *(const v8h*)(qp + (kF8 ? 32 * (s >> 1) + 16 * h + 8 * (s & 1) : 16 * s + 8 * h));
            if (sign < 0.0f) qf[s] = -qf[s];
        }
#pragma unroll
        for (int c = 0; c < kBlocks; ++c) acc[c] = v16f{};
        top = kNegInf;
        total = 0.0f;
    }

    // ---- tiles ----

    // Pages of the tile's four groups of 16 keys.  The table is read through the scalar
    // cache: a vector load among the tiles' would have to wait for all of them.
    struct Ids {
        int page[4];
    };
    __device__ __forceinline__ int page_at(int key) const {
        const int c = key >> a.shift;
        return scalar_at(table, c > last_page ? last_page : c);
    }
    __device__ __forceinline__ Ids tile_ids(int block) const {
        const int k0 = block * kTileKeys;
        // also where a tile lies in one page: copies would be waited for right here
        return {{page_at(k0), page_at(k0 + 16), page_at(k0 + 32), page_at(k0 + 48)}};
    }
    // Of one of the groups, chosen by the wave or by a lane.
    __device__ __forceinline__ static int pick(const Ids& id, int group) {
        const int a = id.page[0], b = id.page[1], c = id.page[2], d = id.page[3];
        const int low = group & 1 ? b : a, high = group & 1 ? d : c;
        return group & 2 ? high : low;
    }
    // Bit c: the page of value chunk c of the tile exists.
    __device__ __forceinline__ uint32_t pages_ok(const Ids& id) const {
        uint32_t ok = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if ((unsigned)id.page[i] < (unsigned)a.pages) ok |= kF8 ? 1u << i : 3u << (2 * i);
        return ok;
    }
    // Keys that 16 lanes of a fragment read differ in bits 0-3 (fp16) or 0-2 and 4 (e4m3).
    __device__ __forceinline__ static int key_swizzle(int key) {
        if constexpr (kKeyBytes == 256) return key & 15;
        else if constexpr (kKeyBytes == 128) return (key >> 1 & 3) | ((key >> 3 ^ key >> 4) & 1) << 2;
        else return (key >> 2 & 1) | ((key >> 3 ^ key >> 4) & 1) << 1;
    }
    __device__ __forceinline__ static int value_swizzle(int d) {
        if constexpr (kValueBytes == 128) return d >> 1 & 7;
        else return d >> 2 & 3;
    }
    __device__ __forceinline__ int value_unit(int i) const { return kSplit ? wave - kKeyUnits : wave + kChunkWaves * i; }
    // Of this lane's loads, whose rows differ by multiples of what the swizzle sees.
    __device__ __forceinline__ int value_chunk() const {
        return (lane & (kValueChunks - 1)) ^ value_swizzle(value_unit(0) * (64 / kValueChunks) + lane / kValueChunks);
    }
    __device__ __forceinline__ size_t page_of(int id) const {
        id = (unsigned)id < (unsigned)a.pages ? id : 0;
        return ((size_t)id * a.kv_heads + kvh) << (a.shift + (kD == 128 ? 7 : 6) + (kF8 ? 0 : 1));
    }
    __device__ __forceinline__ int buffer_of(int block) const { return (block + ring) & (kBuffers - 1); }
    __device__ __forceinline__ uint32_t lds_of(int block) const {
        return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + buffer_of(block) * kBuffer;
    }
    // Where the lane's loads lie, from the wave's first key (one page) or the first value of
    // its place in a page on: the same for every tile.
    __device__ __forceinline__ void place_loads() {
#pragma unroll
        for (int i = 0; i < kKeyLoads; ++i) {
            const int slot = (wave * kKeyLoads + i) * 64 + lane, key = slot / kKeyChunks;
            key_off[i] = (uint32_t)((key & (kKeyRun - 1)) * kKeyBytes + ((slot & (kKeyChunks - 1)) ^ key_swizzle(key)) * 16);
        }
#pragma unroll
        for (int i = 0; i < kValueLoads; ++i) {
            const int d = value_unit(i) * (64 / kValueChunks) + lane / kValueChunks;
            value_off[i] = (uint32_t)(((d * kBytes) << a.shift) + (value_chunk() * 16 & ((kBytes << a.shift) - 1)));
        }
    }
    // The wave's loads of a step, one by one: the keys of a tile, then the values of another.
    struct Step {
        bool keys, values;
        const uint8_t *key, *value;  // value: the lane's where its place decides the page, else the wave's
        uint32_t key_lds, value_lds;
    };
    __device__ __forceinline__ Step step_of(int key_block, const Ids& key_ids, int value_block, const Ids& value_ids, int to) const {
        Step s;
        s.keys = key_block < to && !(kSplit && wave >= kKeyUnits);
        s.values = value_block < to && !(kSplit && wave < kKeyUnits);
        const int run = kKeyRun * wave, in_page = (1 << a.shift) - 1;
        s.key = a.key + page_of(pick(key_ids, run / 16)) + ((key_block * kTileKeys + run) & in_page) * kKeyBytes;
        s.value = a.value + (a.shift >= 6 ? page_of(value_ids.page[0]) + ((value_block * kTileKeys) & in_page) * kBytes
                                          : page_of(pick(value_ids, value_chunk() * 4 / kValueChunks)));
        s.key_lds = lds_of(key_block) + wave * kKeyLoads * 1024;
        s.value_lds = lds_of(value_block) + kKeyTile + value_unit(0) * 1024;
        return s;
    }
    __device__ __forceinline__ void load_keys(const Step& s, int i) const {
        if (s.keys) dma16(s.key, key_off[i], s.key_lds + i * 1024);
    }
    __device__ __forceinline__ void load_values(const Step& s, int i) const {
        if (s.values) dma16(s.value + value_off[i], s.value_lds + i * kChunkWaves * 1024);
    }
    __device__ __forceinline__ void load_all(const Step& s) const {
#pragma unroll
        for (int i = 0; i < kKeyLoads; ++i) load_keys(s, i);
#pragma unroll
        for (int i = 0; i < kValueLoads; ++i) load_values(s, i);
    }

    // First of the 8 consecutive keys of step s (of 4) that this lane holds scores of.
    __device__ __forceinline__ int step_key(int s) const { return kF8 ? 32 * (s >> 1) + 16 * h + 8 * (s & 1) : 16 * s + 8 * h; }

    // The value itself, computed from anew at this place: what only edge tiles need is not
    // kept in registers over the loop.
    __device__ __forceinline__ static int here(int v) {
        asm volatile("" : "+v"(v));
        return v;
    }
    // Bit j: this lane's row sees key j of step s.
    __device__ __forceinline__ uint32_t sees(int k0, int s, uint32_t ok) const {
        if (!(ok >> (step_key(s) * kBytes / 16) & 1u)) return 0;
        const int k = k0 + step_key(s), from = here(lo) - k, to = here(hi) - k;
        if (to <= 0 || from >= 8) return 0;
        return (to >= 8 ? 0xffu : (1u << to) - 1u) & (from <= 0 ? 0xffu : 0xffu << from);
    }

    // The values that this wave loaded of a tile at an edge of some row's keys: those of keys
    // that do not exist hold anything and are cleared, infinities and NaN are taken out.
    // kInside: of a tile that all rows see, infinities only.
    template <bool kInside> __device__ __forceinline__ void tidy_values(int block, uint32_t ok, Odd<kD, kChunkRows>& odd) const {
        if (kSplit && wave < kKeyUnits) return;
        uint8_t* vt = lds + buffer_of(block) * kBuffer + kKeyTile + here(lane) * 16;
        const int chunk = here(value_chunk()), key = block * kTileKeys + chunk * (16 / kBytes), there = ok >> chunk & 1u ? t.length - key : 0;
        const int tile_row0 = row0 - 32 * wave;
        const auto seen = [&](int r, int& from, int& to) {
            from = to = 0;
            if (tile_row0 + r < t.rows) window(a, t.first_pos + (tile_row0 + r) / a.group, t.length, from, to);
        };
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < kValueLoads; ++i) {
            uint4* p = (uint4*)(vt + value_unit(i) * 1024);
            const uint4 old = *p;
            uint32_t w[4] = {old.x, old.y, old.z, old.w};
            constexpr int kPerWord = 4 / kBytes;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int n = there - j * kPerWord;  // keys of this word that exist
                w[j] &= n >= kPerWord ? 0xffffffffu : (n <= 0 ? 0u : (1u << (8 * kBytes * n)) - 1u);
            }
            *p = uint4{w[0], w[1], w[2], w[3]};
            any |= not_finite<kF8>(*p);
        }
        if (__builtin_expect(__any(any != 0), 0)) {
#pragma unroll
            for (int i = 0; i < kValueLoads; ++i) {
                uint4* p = (uint4*)(vt + value_unit(i) * 1024);
                uint4 now = *p;
                odd.template take<kF8>(now, value_unit(i) * (64 / kValueChunks) + here(lane) / kValueChunks, key, kInside, seen);
                *p = now;
            }
        }
    }

    __device__ __forceinline__ void mask(int block, uint32_t ok, v16f (&sc)[2]) const {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const uint32_t seen = sees(block * kTileKeys, s, ok);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (!(seen >> j & 1u)) sc[s >> 1][8 * (s & 1) + j] = kNegInf;
        }
    }
    // The largest of the scores and m, three at once: the compiler's own form of it first
    // passes products of the MFMA through another maximum each, for signalling NaN (a NaN among
    // the scores comes through the exponentials), and between asms of one it places a wait.
    __device__ __forceinline__ static float max3(float m, const v16f& x, const v16f& y) {
        asm("v_max3_f32 %0, %0, %1, %9\n\tv_max3_f32 %0, %0, %2, %10\n\tv_max3_f32 %0, %0, %3, %11\n\tv_max3_f32 %0, %0, %4, %12\n\t"
            "v_max3_f32 %0, %0, %5, %13\n\tv_max3_f32 %0, %0, %6, %14\n\tv_max3_f32 %0, %0, %7, %15\n\tv_max3_f32 %0, %0, %8, %16"
            : "+v"(m)
            : "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(x[4]), "v"(x[5]), "v"(x[6]), "v"(x[7]), "v"(y[0]), "v"(y[1]), "v"(y[2]), "v"(y[3]),
              "v"(y[4]), "v"(y[5]), "v"(y[6]), "v"(y[7]));
        asm("v_max3_f32 %0, %0, %1, %9\n\tv_max3_f32 %0, %0, %2, %10\n\tv_max3_f32 %0, %0, %3, %11\n\tv_max3_f32 %0, %0, %4, %12\n\t"
            "v_max3_f32 %0, %0, %5, %13\n\tv_max3_f32 %0, %0, %6, %14\n\tv_max3_f32 %0, %0, %7, %15\n\tv_max3_f32 %0, %0, %8, %16"
            : "+v"(m)
            : "v"(x[8]), "v"(x[9]), "v"(x[10]), "v"(x[11]), "v"(x[12]), "v"(x[13]), "v"(x[14]), "v"(x[15]), "v"(y[8]), "v"(y[9]), "v"(y[10]),
              "v"(y[11]), "v"(y[12]), "v"(y[13]), "v"(y[14]), "v"(y[15]));
        return m;
    }
    // Scores are taken relative to a running maximum that is only raised where a row's
    // falls kSlack short (factors of two), so that the output so far is rarely rescaled.
    // Probabilities are 2^kLift at that maximum and at most 2^15: fp16 then holds those down to
    // 2^-21 of it to full precision and down to 2^-31 at all, so that the sum counts no small
    // ones that the output leaves out.
    static constexpr float kSlack = 8.0f, kLift = 15.0f - kSlack, kHuge = 1 << 20;
    // Scores -> probabilities as operands; the sums so far are scaled to the new maximum.
    // Scaling and subtraction are one step, in which the rounding of the scaled maximum, half a
    // step of its own, becomes a factor of all probabilities: harmless up to 2^20, far outside
    // fp16 from 2^28 on.  With kCareful the subtraction, exact near the maximum, comes first there.
    template <bool kCareful> __device__ __forceinline__ void soften(const v16f (&sc)[2], v8h (&pf)[4]) {
        const float m = max_level(max3(kNegInf, sc[0], sc[1]), 32);
        const bool far = (m - top) * scale > kSlack;  // also from -inf; false while nothing is seen
        if (__any(far)) {
            const float keep = far ? __builtin_amdgcn_exp2f((top - m) * scale) : 1.0f;
            top = far ? m : top;
            total *= keep;
#pragma unroll
            for (int c = 0; c < kBlocks; ++c) acc[c] = acc[c] * keep;
        }
        const float from = top == kNegInf ? 0.0f : top, base = from * scale - kLift;
        const bool huge = kCareful && !(__builtin_fabsf(base) < kHuge);
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float score = sc[s >> 1][8 * (s & 1) + j];
                const float p = __builtin_amdgcn_exp2f(huge ? (score - from) * scale + kLift : __builtin_fmaf(score, scale, -base));
                total += p;
                pf[s][j] = (_Float16)p;
            }
    }
    // The scores of tile `block` and (or) the output of the tile before it, LDS reads
    // kAhead operands ahead of the products: one at a time, each is waited for in full (the
    // order is pinned because the compiler brings them together again).
    static constexpr int kAhead = 4;
    template <bool kScores, bool kOutput> __device__ __forceinline__ void products(int block, v16f (&sc)[2], const v8h (&pf)[4]) {
        constexpr int kPer = kF8 ? 2 : 1;  // products an operand's 16 bytes feed
        constexpr int kScoreReads = kScores ? 2 * kSteps / kPer : 0, kReads = kScoreReads + (kOutput ? 4 * kBlocks / kPer : 0);
        const uint8_t* kt = lds + buffer_of(block) * kBuffer;
        const uint8_t* vt = lds + buffer_of(block - 1) * kBuffer + kKeyTile;
        // row m of the MFMA is the key whose score lands in place: see step_key
        const int quad = (l32 >> 3) & 3, half = (l32 >> 2) & 1;
        const int key0 = (kF8 ? 16 * half + 8 * (quad >> 1) : 16 * (quad >> 1) + 8 * half) + 4 * (quad & 1) + (l32 & 3);
        const auto read = [&](int i) {
            if (i < kScoreReads) {
                const int key = key0 + 32 * (i / (kSteps / kPer)), s = i % (kSteps / kPer);
                return *(const uint4*)(kt + key * kKeyBytes + ((2 * s + h) ^ key_swizzle(key)) * 16);
            }
            const int j = i - kScoreReads, d = l32 + 32 * (j / (4 / kPer)), s = j % (4 / kPer);
            return *(const uint4*)(vt + d * kValueBytes + ((2 * s + h) ^ value_swizzle(d)) * 16);
        };
        __builtin_amdgcn_s_setprio(1);  // over the other wave's softmax
        if constexpr (kScores) sc[0] = sc[1] = v16f{};
        uint4 raw[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) raw[i] = read(i);
#pragma unroll
        for (int i = 0; i < kReads; ++i) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                const v8h first = operand<kF8>(raw[i % kAhead], e);
                if (i < kScoreReads) {
                    const int blk = i / (kSteps / kPer);
                    sc[blk] = __builtin_amdgcn_mfma_f32_32x32x16_f16(first, qf[i % (kSteps / kPer) * kPer + e], sc[blk], 0, 0, 0);
                } else {
                    const int j = i - kScoreReads, c = j / (4 / kPer);
                    acc[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(first, pf[j % (4 / kPer) * kPer + e], acc[c], 0, 0, 0);
                }
            }
            if (i + kAhead < kReads) raw[i % kAhead] = read(i + kAhead);
        }
        __builtin_amdgcn_s_setprio(0);
        // the scores are next read by max3, before which the compiler places no wait for the MFMA
        if constexpr (kScores && !kOutput) asm volatile("s_nop 15\n\ts_nop 7" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    }

    // Loads go out in steps: K(t + 3) and V(t + 2) with tile t's softmax.  Waits until
    // all but the last `steps` steps (of kLoads a wave) have arrived, which they do in order.
    template <int steps> __device__ __forceinline__ static void wait_steps(bool more) {
        if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(steps * kLoads) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    __device__ __forceinline__ static void meet() {
        __builtin_amdgcn_sched_barrier(0);
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
    }

    // Tiles [from, to); `tick`: of the first, a number that counts the workgroup's tiles and
    // gives each its buffer.
    //
    // Two waves share a SIMD (w and w + 4); the second four run half a period behind, so
    // that one's products (the scores of a tile and the output of the one before) run under
    // the other's softmax and loads.  Buffers: K(t + 3) replaces K(t - 1) and V(t + 2)
    // replaces V(t - 2) at tile t's softmax, when the other waves are at the products of
    // that tile, which read K(t) and V(t - 1), or of the next.  The waves that are behind
    // are at their last products when the others go on to the next tiles' first loads,
    // which go to other buffers than V(to - 1).
    template <bool kCareful> __device__ __forceinline__ void run(int from, int to, int& tick, Odd<kD, kChunkRows>& odd) {
        ring = (tick - from) & (kBuffers - 1);
        const bool behind = wave >= 4;
        uint32_t ok[3];  // pages of tiles b, b + 1, b + 2
        Ids ids = tile_ids(from + 2), next = tile_ids(from + 3);  // of tiles b + 2 and b + 3
        {
            const Ids first = tile_ids(from), second = tile_ids(from + 1);
            ok[0] = pages_ok(first);
            ok[1] = pages_ok(second);
            Step s = step_of(from, first, to, first, to);
            load_all(s);
            load_all(step_of(from + 1, second, from, first, to));
            load_all(step_of(from + 2, ids, from + 1, second, to));
        }
        wait_steps<2>(from + 2 < to);
        meet();
        if (behind) meet();
        const bool active = last >= 0;
        v16f sc[2];
        v8h pf[4];
        Step step = step_of(from + 3, next, from + 2, ids, to);
        if (active) products<true, false>(from, sc, pf);
        for (int b = from; b < to; ++b) {
            wait_steps<1>(b + 2 < to);
            const bool edge = b * kTileKeys < tile_full_lo || (b + 1) * kTileKeys > tile_full_hi || ok[0] != kAllPages;
            if (edge) tidy_values<false>(b, ok[0], odd);
            else if constexpr (kCareful && !kF8) tidy_values<true>(b, ok[0], odd);
            meet();
            load_all(step);
            ok[2] = pages_ok(ids);
            ids = next;
            next = tile_ids(b + 4);
            if (active) {
                // a tile that none of the wave's rows sees has probabilities of zero and tidy values
                if (edge && (b * kTileKeys < full_lo || (b + 1) * kTileKeys > full_hi || ok[0] != kAllPages)) mask(b, ok[0], sc);
                soften<kCareful>(sc, pf);
            }
            step = step_of(b + 4, next, b + 3, ids, to);
            meet();
            ok[0] = ok[1];
            ok[1] = ok[2];
            if (b + 1 < to && active) products<true, true>(b + 1, sc, pf);
        }
        if (active) products<false, true>(to, sc, pf);
        tick += to - from;
        if (!behind) meet();
    }

    // Whether a row of this wave may have come out wrong in a run without care: its maximum is
    // large, or its sums are not finite (a value was infinite, or early probabilities were too
    // large for fp16).
    __device__ __forceinline__ bool doubtful() const {
        v16f sums = acc[0];
#pragma unroll
        for (int c = 1; c < kBlocks; ++c) sums += acc[c];
#pragma unroll
        for (int n = 8; n > 0; n >>= 1)
#pragma unroll
            for (int j = 0; j < n; ++j) sums[j] += sums[j + n];
        const bool far = top != kNegInf && !(__builtin_fabsf(top * scale - kLift) < kHuge);
        return last >= 0 && __any(far || !(__builtin_fabsf(sums[0] + total) < __builtin_inff()));
    }
    // A row tile's tiles [from, to), all of them read by all waves at the end.  Where a wave has
    // doubts all start again, with care: it costs a second pass, and only these calls.
    __device__ __forceinline__ void attend(int seq, const RowTile& rows, int tile, int from, int to, int& tick, Odd<kD, kChunkRows>& odd, int& again) {
        start(seq, rows, tile);
        run<false>(from, to, tick, odd);
        if (doubtful()) again = 1;
        __syncthreads();
        if (__builtin_expect(__builtin_amdgcn_readfirstlane(again) != 0, 0)) {
            start(seq, rows, tile);
            run<true>(from, to, tick, odd);  // (its first barrier stands behind all reads of `again`)
            if (threadIdx.x == 0) again = 0;
            __syncthreads();
        }
    }

    // The lane's row (unless it repeats the last) of the output, or of a part.
    __device__ __forceinline__ void finish(bool whole, Part<kD, kChunkRows>* slot, const Odd<kD, kChunkRows>& odd, bool any_odd) {
        int sum_a, sum_b;
        pair_of(__float_as_int(total), 32, sum_a, sum_b);
        const float sum = __int_as_float(sum_a) + __int_as_float(sum_b);
        if (l32 > last) return;
        const int r = wave * 32 + l32;
        const float inv = sum == 0.0f ? 0.0f : a.value_scale / sum;
        uint16_t* op = a.out + (size_t)(t.start + row / a.group) * a.out_stride + (size_t)(kvh * a.group + row % a.group) * kD;
#pragma unroll
        for (int c = 0; c < kBlocks; ++c)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int d = 32 * c + 8 * q + 4 * h;
                v4f v{acc[c][4 * q], acc[c][4 * q + 1], acc[c][4 * q + 2], acc[c][4 * q + 3]};
                if (__builtin_expect(any_odd, 0)) v = v4f{odd.put(v[0], r, d), odd.put(v[1], r, d + 1), odd.put(v[2], r, d + 2), odd.put(v[3], r, d + 3)};
                if (whole)
                    *(uint2*)(op + d) = uint2{(uint32_t)f2h(v[0] * inv) | ((uint32_t)f2h(v[1] * inv) << 16),
                                              (uint32_t)f2h(v[2] * inv) | ((uint32_t)f2h(v[3] * inv) << 16)};
                else
                    *(v4f*)&slot->acc[r][d] = v;
            }
        if (!whole && h == 0) {
            slot->top[r] = top == kNegInf ? kNegInf : top * scale;
            slot->total[r] = sum;
        }
    }
};

// Short contexts: a workgroup for all keys of a (sequence, kv head, 256 rows).
template <int kD, bool kF8> __global__ __launch_bounds__(kChunkThreads, 2) void paged_chunks_direct_kernel(PagedArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[kBuffers * ChunkPass<kD, kF8>::kBuffer];
    __shared__ Odd<kD, kChunkRows> odd;
    __shared__ int again;
    odd.clear(kChunkThreads);
    if (threadIdx.x == 0) again = 0;
    const int kvh = blockIdx.x, seq = blockIdx.z, tile = blockIdx.y;
    const RowTile t = wave_sequence(a, seq);
    if (tile * kChunkRows >= t.rows) return;
    int first, tick = 0;
    const int blocks = chunk_blocks(a, t, tile, first);
    ChunkPass<kD, kF8> pass(a, lds, kvh);
    pass.attend(seq, t, tile, first, first + blocks, tick, odd, again);
    pass.finish(true, nullptr, odd, odd.any != 0);
}

template <int kD, bool kF8>
__global__ __launch_bounds__(kChunkThreads, 2) void paged_chunks_shares_kernel(PagedArgs a, Part<kD, kChunkRows>* slots, Join* joins) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[kBuffers * ChunkPass<kD, kF8>::kBuffer];
    __shared__ Odd<kD, kChunkRows> odd;
    __shared__ int again;
    odd.clear(kChunkThreads);
    if (threadIdx.x == 0) again = 0;
    // neighbouring shares read the same keys: they go to one XCD's L2
    const int index = (blockIdx.x & 7) * (kChunkShares / 8) + (blockIdx.x >> 3);
    if (threadIdx.x == 0) joins[index].count = 0;
    Share share;
    const auto blocks_of = [&](const RowTile& t) { return pairs_of(a, t).per_head * a.kv_heads; };
    if (!deal<kChunkThreads, kChunkShares, kLeastChunkShare>(a, index, blocks_of, share)) return;

    // The beginning of the row tile that the share ends in comes first, then the rest in
    // order: as shares are equal, the workgroups then stand at about the same keys at the
    // same time, and find them in their L2.
    int seq = share.last_seq, tick = 0;
    RowTile t = wave_sequence(a, seq);
    Pairs p = pairs_of(a, t);
    const Span tail = span_at(a, t, p, share.last_offset);
    const long long head = share.to - 1 - tail.at;  // where that row tile begins
    const bool first_out = tail.at + 1 < tail.blocks && head > share.from;
    long long at = first_out ? head : share.from, offset = first_out ? share.last_offset - tail.at : share.offset, to = share.to;
    if (!first_out && seq != share.seq) {
        seq = share.seq;
        t = wave_sequence(a, seq);
        p = pairs_of(a, t);
    }
    for (;;) {
        const Span s = span_at(a, t, p, offset);
        const int n = to - at < s.blocks - s.at ? (int)(to - at) : s.blocks - s.at;
        if (s.tile >= 0) {
            ChunkPass<kD, kF8> pass(a, lds, s.kvh);
            pass.attend(seq, t, s.tile, s.first + s.at, s.first + s.at + n, tick, odd, again);
            const int which = at == share.from ? 0 : 1;
            const bool any_odd = __builtin_amdgcn_readfirstlane((int)odd.any) != 0;
            pass.finish(n == s.blocks, slots + 2 * index + which, odd, any_odd);
            if (any_odd) {
                __syncthreads();
                odd.clear(kChunkThreads);
            }
            if (n != s.blocks && s.at == 0 && threadIdx.x == 0)
                joins[index] = {t.start, t.rows, s.kvh, s.tile * kChunkRows, share_of<kChunkShares, kLeastChunkShare>(share.all, at + s.blocks - 1) - index + 1, which, {}};
        }
        at += n;
        offset += n;
        if (at == share.to && to == share.to && first_out) {  // the beginning is done: the rest
            to = head;
            at = share.from;
            offset = share.offset;
            if (seq == share.seq) continue;
            seq = share.seq;
        } else if (at >= to) {
            break;
        } else if (offset < p.per_head * a.kv_heads) {
            continue;
        } else {
            offset = 0;
            do {
                t = wave_sequence(a, ++seq);
                p = pairs_of(a, t);
            } while (p.per_head == 0);
            continue;
        }
        t = wave_sequence(a, seq);
        p = pairs_of(a, t);
    }
}

// Joins the parts of the divided row tiles, 16 rows a workgroup: a row a group of lanes
// where the parts are few, else a row at a time with the groups taking parts in turn.
template <int kD> __global__ __launch_bounds__(16 * kD / 4) void paged_chunks_join_kernel(PagedArgs a, const Part<kD, kChunkRows>* slots, const Join* joins) {
    constexpr int kLanes = kD / 4;
    __shared__ float part_acc[16][kD], part_top[16], part_total[16];
    const Join job = joins[blockIdx.x];
    const int r0 = blockIdx.y * 16;
    if (job.count == 0 || job.row0 + r0 >= job.rows) return;
    const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
    const Part<kD, kChunkRows>* first = slots + 2 * blockIdx.x;
    const bool few = job.count <= 16;
    for (int row = few ? group : 0; row < 16; row += few ? 16 : 1) {
        const int r = r0 + row;
        if (job.row0 + r >= job.rows) break;
        float top = kNegInf, total = 0.0f;
        v4f v{};
#pragma unroll 4
        for (int i = few ? 0 : group; i < job.count; i += few ? 1 : 16) {
            const Part<kD, kChunkRows>& slot = first[2 * i + (i == 0 ? job.first_slot : 0)];
            const float new_top = __builtin_fmaxf(top, slot.top[r]);
            const float base = new_top == kNegInf ? 0.0f : new_top;
            const float f = weight_of(slot.top[r] - base), keep = weight_of(top - base);
            total = total * keep + slot.total[r] * f;
            v = v * keep + *(const v4f*)&slot.acc[r][4 * lane] * f;
            top = new_top;
        }
        if (!few) {
            __syncthreads();  // the row before is read
            *(v4f*)&part_acc[group][4 * lane] = v;
            if (lane == 0) {
                part_top[group] = top;
                part_total[group] = total;
            }
            __syncthreads();
            if (group != 0) continue;
            float best = kNegInf;
#pragma unroll
            for (int w = 0; w < 16; ++w) best = __builtin_fmaxf(best, part_top[w]);
            const float base = best == kNegInf ? 0.0f : best;
            total = 0.0f;
            v = v4f{};
#pragma unroll
            for (int w = 0; w < 16; ++w) {
                const float f = weight_of(part_top[w] - base);
                total += part_total[w] * f;
                v = v + *(const v4f*)&part_acc[w][4 * lane] * f;
            }
        }
        const float o[4] = {v[0], v[1], v[2], v[3]};
        store_row<4>(a, {job.start, job.rows, 0, 0}, job.kvh, job.row0 + r, kD, 4 * lane, total, o);
    }
}

size_t paged_chunks_workspace(int head_dim) {
    return 2 * kChunkShares * (head_dim == 128 ? sizeof(Part<128, kChunkRows>) : sizeof(Part<64, kChunkRows>)) + kChunkShares * sizeof(Join);
}

template <int kD, bool kF8> static void launch_chunks(const PagedArgs& a, bool direct, int max_queries, void* workspace, hipStream_t s) {
    const int rows = max_queries * a.group;
    if (direct) {
        const dim3 grid((unsigned)a.kv_heads, (unsigned)((rows + kChunkRows - 1) / kChunkRows), (unsigned)a.sequences);
        paged_chunks_direct_kernel<kD, kF8><<<grid, kChunkThreads, 0, s>>>(a);
        return;
    }
    auto* slots = (Part<kD, kChunkRows>*)workspace;
    Join* joins = (Join*)(slots + 2 * kChunkShares);
    paged_chunks_shares_kernel<kD, kF8><<<kChunkShares, kChunkThreads, 0, s>>>(a, slots, joins);
    const int part_rows = rows < kChunkRows ? rows : kChunkRows;
    paged_chunks_join_kernel<kD><<<dim3(kChunkShares, (unsigned)((part_rows + 15) / 16)), 16 * kD / 4, 0, s>>>(a, slots, joins);
}

void launch_paged_chunks(int kind, const PagedArgs& a, int head_dim, bool direct, int max_queries, void* workspace, hipStream_t s) {
    if (head_dim == 128) {
        if (kind == 1) launch_chunks<128, true>(a, direct, max_queries, workspace, s);
        else launch_chunks<128, false>(a, direct, max_queries, workspace, s);
    } else {
        if (kind == 1) launch_chunks<64, true>(a, direct, max_queries, workspace, s);
        else launch_chunks<64, false>(a, direct, max_queries, workspace, s);
    }
}

}  // namespace pk
