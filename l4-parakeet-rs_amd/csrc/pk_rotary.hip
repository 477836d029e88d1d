// Norm of each query and key head and its rotation by the token's position, in one pass:
//   y = x / sqrt(mean(x^2) + eps) * w   over the features of a head (no weight: y = x),
//   (u, v) -> a (u cos t - v sin t, v cos t + u sin t),  t = position * frequency,
// for the pairs (y_i, y_{i + R/2}) or (y_2i, y_2i+1) of the first R features; and the same
// with keys and values written into the paged cache.
//
// Angles: a frequency is held as turns a position in units of 2^-64, so that position *
// frequency modulo 2^64 is the phase, exact however far the position.  Its upper 32 bits
// are taken to the nearest quarter turn, and sine and cosine of the rest (within pi / 4)
// are the Taylor sums to x^9 and x^8, off by less than x^10 / 10! = 2.5e-8.
//
// A lane holds twice 8 features of a head, in either layout both members of 8 pairs; head_dim / 16
// lanes make a head.  Everything between the loads and the one rounding at the store is fp32.
//
// Bound by HBM: 16000 tokens, 32 / 8 heads of 128, rows to rows (328 MB) 60 us, 5.5 TB/s; with keys
// and values into an fp16 cache (393 MB) 76 us, 5.2 TB/s, into an e4m3 one (360 MB) 74 us, 4.9 TB/s.
// One token 2.7 us, about a launch; 61 into an e4m3 cache 4.6 us: a load, the angles, and values that
// lie in as many rows of a page as they are.
#include <math.h>

#include "pk_paged_write.hpp"

namespace pk {

// amplitude * (cos, sin) of a phase in 2^-64 turns
__device__ __forceinline__ float2 turned_by(unsigned long long phase, float amplitude) {
    const uint32_t u = (uint32_t)(phase >> 32), quarter = (u + 0x20000000u) >> 30;
    const float x = (float)(int)(u - (quarter << 30)) * 1.46291807926715968e-9f;  // 2 pi / 2^32
    const float z = x * x;
    const float s = x * __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), 1.0f);
    const float c = __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, 1.0f / 40320, -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const float a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;
    return float2{(quarter + 1) & 2 ? -a * amplitude : a * amplitude, quarter & 2 ? -b * amplitude : b * amplitude};
}

typedef float v2f __attribute__((ext_vector_type(2)));

// A lane's 16 features: u and v of 8 pairs.
struct Pairs {
    v4i u, v;
};

// Neighbours (u0 v0 u1 v1 ..) to (u0 u1 ..), (v0 v1 ..).
__device__ __forceinline__ void apart(Pairs& x) {
    const uint32_t w[8] = {(uint32_t)x.u[0], (uint32_t)x.u[1], (uint32_t)x.u[2], (uint32_t)x.u[3],
                           (uint32_t)x.v[0], (uint32_t)x.v[1], (uint32_t)x.v[2], (uint32_t)x.v[3]};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        x.u[j] = (int)__builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x05040100u);
        x.v[j] = (int)__builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x07060302u);
    }
}
// And back.
__device__ __forceinline__ void together(Pairs& x) {
    const v4i u = x.u, v = x.v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t a = __builtin_amdgcn_perm((uint32_t)v[j], (uint32_t)u[j], 0x05040100u),
                       b = __builtin_amdgcn_perm((uint32_t)v[j], (uint32_t)u[j], 0x07060302u);
        (j < 2 ? x.u : x.v)[2 * (j & 1)] = (int)a;
        (j < 2 ? x.u : x.v)[2 * (j & 1) + 1] = (int)b;
    }
}

__device__ __forceinline__ void unpack(const v4i& raw, float (&y)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = h2f((uint16_t)((uint32_t)raw[j >> 1] >> (16 * (j & 1))));
}
__device__ __forceinline__ v4i pack(const float (&y)[8]) {
    v4i w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = __builtin_bit_cast(int, __builtin_convertvector(v2f{y[2 * j], y[2 * j + 1]}, v2h));  // to nearest even, both at once
    return w;
}

// kPast: past the caches, for results larger than they are (16000 tokens of 32 / 8 heads of 128 60 us; kept in them 4 us more).
template <bool kPast, typename T> __device__ __forceinline__ void store(void* to, T v) {
    if constexpr (kPast) __builtin_nontemporal_store(v, (T*)to);
    else *(T*)to = v;
}
__device__ __forceinline__ v2i e4m3x8(const float (&y)[8], float inverse) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = e4m3x2(y[2 * j] * inverse, y[2 * j + 1] * inverse);
    return v2i{(int)(w[0] | (w[1] << 16)), (int)(w[2] | (w[3] << 16))};
}

// kLanes lanes a head (a power of two of at least head_dim / 16), 64 / kLanes heads a set: query sets,
// then key sets, then (few tokens into a cache) value sets.  kCache: -1 rows out, 0 an fp16 cache, 1 an
// e4m3 one.  A wave takes `sets` sets of a token, the next one's loads in flight.
template <int kLanes, int kCache, bool kPast>
__global__ __launch_bounds__(256) void head_norm_rotary_kernel(RotaryArgs a, int parts, int sets, int value_blocks) {
    constexpr int kSlots = 64 / kLanes;
    constexpr bool kF8 = kCache == 1;
    __shared__ float2 angles[4][128];
    if constexpr (kCache >= 0) {
        if ((int)blockIdx.x < value_blocks) {  // prompts: the values, turned around in tiles
            const WriteArgs w{nullptr, a.value, a.slots, nullptr, (uint8_t*)a.value_cache, 0, a.value_stride, a.slot_count, a.tokens, a.kv_heads,
                              a.shift, 1.0f, a.v_inv};
            if (a.head_dim == 128) write_tile<128, kF8, false>(w, blockIdx.x % a.kv_heads, blockIdx.x / a.kv_heads);
            else write_tile<64, kF8, false>(w, blockIdx.x % a.kv_heads, blockIdx.x / a.kv_heads);
            return;
        }
    }
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, p = lane % kLanes, place = lane / kLanes;
    const int unit = (int)(blockIdx.x - value_blocks) * 4 + wave, t = unit / parts;  // (at most 2^21 tokens, or kMostSetWaves)
    const int query_sets = (a.heads + kSlots - 1) / kSlots, kv_sets = (a.kv_heads + kSlots - 1) / kSlots;
    const int all = query_sets + kv_sets + (kCache >= 0 && value_blocks == 0 ? kv_sets : 0);
    const int first = unit % parts * sets, stop = first + sets < all ? first + sets : all;
    const bool there = t < a.tokens && first < stop, rotates = there && a.rotary_dim && first < query_sets + kv_sets;
    const bool inside = p * 16 < a.head_dim, turning = p * 16 < a.rotary_dim && !a.interleaved;
    // 8 features each, those of neighbouring lanes behind one another (where lanes held 16 in a row, stores past
    // the caches were halves of lines: 16000 tokens of 32 / 8 heads of 128, neighbours, 82 us instead of 60)
    const int f0 = 8 * p + (turning || a.interleaved ? 0 : a.rotary_dim / 2), f1 = 8 * p + (turning ? a.rotary_dim : a.head_dim) / 2;
    const bool turn0 = a.interleaved ? f0 < a.rotary_dim : turning, turn1 = a.interleaved ? f1 < a.rotary_dim : turning;
    // lanes without a feature or a head read those of the first
    const int r0 = inside ? f0 : 0, r1 = inside ? f1 : 0;
    const auto ask = [&](int set) {
        const bool query = set < query_sets, value = set >= query_sets + kv_sets;
        const int h = (query ? set : value ? set - query_sets - kv_sets : set - query_sets) * kSlots + place, n = query ? a.heads : a.kv_heads;
        const uint16_t* row = (query ? a.query + (size_t)t * a.query_stride : value ? a.value + (size_t)t * a.value_stride : a.key + (size_t)t * a.key_stride) +
                              (h < n ? h : 0) * a.head_dim;
        return Pairs{*(const v4i*)(row + r0), *(const v4i*)(row + r1)};
    };
    // all that can be asked for at once: a chain of one load, the angles and the store is left
    Pairs now{};
    if (there) now = ask(first);
    int slot = 0;
    if constexpr (kCache >= 0) slot = there ? a.slots[t] : -1;
    const long long position = rotates ? a.positions[t] : 0;  // (no rotation: there may be no positions)
    const uint16_t* weight = nullptr;
    Pairs weights{};
    const auto ask_weight = [&](int set) {
        weight = set < query_sets ? a.query_weight : a.key_weight;
        if (weight) weights = Pairs{*(const v4i*)(weight + r0), *(const v4i*)(weight + r1)};
        if (a.interleaved) apart(weights);
    };
    if (there) ask_weight(first);
    if (rotates)
        for (int i = lane; i < a.rotary_dim / 2; i += 64) angles[wave][i] = turned_by((unsigned long long)position * a.frequencies[i], a.amplitude);
    __syncthreads();
    if (!there || slot < 0 || (kCache >= 0 && slot >= a.slot_count)) return;
    float2 angle[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        angle[j] = turn0 ? angles[wave][(a.interleaved ? f0 / 2 : 8 * p) + j] : float2{};
        angle[4 + j] = turn1 ? angles[wave][(a.interleaved ? f1 / 2 : 8 * p + 4) + j] : float2{};
    }
    const int off = slot & ((1 << a.shift) - 1);
    const float per_feature = 1.0f / (float)a.head_dim;
    float w0[8], w1[8];
    unpack(weights.u, w0);
    unpack(weights.v, w1);
    for (int set = first; set < stop; ++set) {
        const bool query = set < query_sets, value = set >= query_sets + kv_sets;
        const int h = (query ? set : value ? set - query_sets - kv_sets : set - query_sets) * kSlots + place;
        const bool mine = inside && h < (query ? a.heads : a.kv_heads);
        if (a.interleaved && !value) apart(now);
        float u[8], v[8];
        unpack(now.u, u);
        unpack(now.v, v);
        if (set + 1 < stop) now = ask(set + 1);
        if constexpr (kCache >= 0) {
            if (value) {  // features lie a page's tokens apart
                if (mine) {
                    const size_t base = ((size_t)(slot >> a.shift) * a.kv_heads + h) * a.head_dim;
                    const size_t at0 = ((base + f0) << a.shift) + off, at1 = ((base + f1) << a.shift) + off;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if constexpr (kF8) {
                            ((uint8_t*)a.value_cache)[at0 + ((size_t)j << a.shift)] = e4m3(u[j] * a.v_inv);
                            ((uint8_t*)a.value_cache)[at1 + ((size_t)j << a.shift)] = e4m3(v[j] * a.v_inv);
                        } else {
                            ((uint16_t*)a.value_cache)[at0 + ((size_t)j << a.shift)] = f2h(u[j]);
                            ((uint16_t*)a.value_cache)[at1 + ((size_t)j << a.shift)] = f2h(v[j]);
                        }
                    }
                }
                continue;
            }
        }
        if (set == query_sets && set > first) {
            ask_weight(set);
            unpack(weights.u, w0);
            unpack(weights.v, w1);
        }
        if (weight) {
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = __builtin_fmaf(v[j], v[j], __builtin_fmaf(u[j], u[j], sum));
            sum = inside ? sum : 0.0f;
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1) sum = add_level(sum, o);
            const float mean = __builtin_fmaf(sum, per_feature, a.epsilon);
            // the instruction's reciprocal root (1 ulp) for normal numbers; NaN stays NaN; all zero with eps 0: zeros
            float rstd = __builtin_amdgcn_rsqf(mean);
            if (!(mean >= 1.17549435e-38f)) rstd = mean > 0.0f ? 1.0f / sqrtf(mean) : (mean == 0.0f ? 0.0f : mean);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                u[j] = u[j] * rstd * w0[j];
                v[j] = v[j] * rstd * w1[j];
            }
        }
        const auto turn = [&](int j) {
            const float x = u[j];
            u[j] = __builtin_fmaf(x, angle[j].x, -(v[j] * angle[j].y));
            v[j] = __builtin_fmaf(v[j], angle[j].x, x * angle[j].y);
        };
        if (turn0)
#pragma unroll
            for (int j = 0; j < 4; ++j) turn(j);
        if (turn1)
#pragma unroll
            for (int j = 4; j < 8; ++j) turn(j);
        if (!mine) continue;
        if (kF8 && !query) {  // neighbours: the unrounded features in their order
            float x[8], y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = a.interleaved ? (j & 1 ? v : u)[j >> 1] : u[j];
                y[j] = a.interleaved ? (j & 1 ? v : u)[4 + (j >> 1)] : v[j];
            }
            uint8_t* to = (uint8_t*)a.key_cache + ((((size_t)(slot >> a.shift) * a.kv_heads + h) << a.shift) + off) * a.head_dim;
            store<kPast>(to + f0, e4m3x8(x, a.k_inv));
            store<kPast>(to + f1, e4m3x8(y, a.k_inv));
        } else {
            Pairs out{pack(u), pack(v)};
            if (a.interleaved) together(out);
            uint16_t* to = query        ? a.query_out + (size_t)t * a.query_out_stride + h * a.head_dim
                           : kCache < 0 ? a.key_out + (size_t)t * a.key_out_stride + h * a.head_dim
                                        : (uint16_t*)a.key_cache + ((((size_t)(slot >> a.shift) * a.kv_heads + h) << a.shift) + off) * a.head_dim;
            store<kPast>(to + f0, out.u);
            store<kPast>(to + f1, out.v);
        }
    }
}

// From this many tokens on, and this many rows of values (tokens times kv heads), the values go in tiles: a tile's chain is
// as long for one head as for many, and a lane's scattered stores are hidden while they are few (one prompt, fp16, heads of
// 128, us without and with tiles: 8 kv heads 400 tokens 7.7 and 9.9, 800 13.2 and 11.1; 4 800 7.5 and 9.1, 2000 14.2 and
// 9.3; 2 2000 9.3 and 9.9, 4000 14.6 and 10.9; 1 2000 7.8 and 9.8, 8000 17.5 and 13.6; as many single tokens, 8 kv heads,
// 400 10.0 and 16.5, 800 16.1 and 18.1, 4000 206 and 212; e4m3 like these).
constexpr int kTileTokens = 768, kTileRows = 6144;
// Up to this many waves a wave takes one set of heads, else all of its token's (rows of fp16: 1000 tokens
// 7.2 us in 5000 waves and 7.6 in 1000, 1500 9.2 and 9.1, 3000 15.0 and 12.0).
constexpr int kMostSetWaves = 8192;

template <int kCache, bool kPast> static void launch_rotary(const RotaryArgs& a, hipStream_t s) {
    const bool tiles = kCache >= 0 && a.tokens >= kTileTokens && a.tokens * a.kv_heads >= kTileRows;  // (at most 2^29)
    const int value_blocks = tiles ? a.kv_heads * ((a.tokens + kWriteTokens - 1) / kWriteTokens) : 0;
    const auto launch = [&](auto kernel, int lanes) {
        const int each = 64 / lanes, kv_sets = (a.kv_heads + each - 1) / each;
        const int all = (a.heads + each - 1) / each + kv_sets + (kCache >= 0 && !tiles ? kv_sets : 0);
        const int parts = (long long)a.tokens * all <= kMostSetWaves ? all : 1, sets = (all + parts - 1) / parts;
        const unsigned grid = (unsigned)(((long long)a.tokens * parts + 3) / 4 + value_blocks);
        kernel<<<grid, 256, 0, s>>>(a, parts, sets, value_blocks);
    };
    if (a.head_dim <= 64) launch(head_norm_rotary_kernel<4, kCache, kPast>, 4);
    else if (a.head_dim <= 128) launch(head_norm_rotary_kernel<8, kCache, kPast>, 8);
    else if constexpr (kCache < 0) launch(head_norm_rotary_kernel<16, kCache, kPast>, 16);  // (a cache holds heads of 64 or 128)
}

// Bytes that neighbouring lanes store behind one another at the least; of less than 64 the caches put lines
// together (16000 tokens of 32 / 8 heads of 128 of which 32 turn by halves 65 us, past the caches 76; 64 both 64.5).
constexpr int kShortPiece = 64;

template <int kCache> static void rotary(const RotaryArgs& a, hipStream_t s) {
    const int rest = a.head_dim - a.rotary_dim, piece = a.interleaved || !rest || rest == a.head_dim ? a.head_dim : (rest < a.rotary_dim ? rest : a.rotary_dim);
    if ((long long)a.tokens * (a.heads + a.kv_heads) * a.head_dim * 2 > kCached && piece >= kShortPiece) launch_rotary<kCache, true>(a, s);
    else launch_rotary<kCache, false>(a, s);
}

void launch_head_norm_rotary(const RotaryArgs& a, hipStream_t s) { rotary<-1>(a, s); }

void launch_head_norm_rotary_write(int kind, const RotaryArgs& a, hipStream_t s) {
    if (kind == 1) rotary<1>(a, s);
    else rotary<0>(a, s);
}

// Radians a position, i of `pairs` (frequencies fall from 1 by a constant factor).
void rotary_frequencies(int scaling, int pairs, double base, double factor, double low, double high, int original, uint64_t* out) {
    const double pi2 = 6.283185307179586476925286766559, dim = 2.0 * pairs;
    if (scaling == 0) factor = 1.0;  // not looked at, and 0 or a NaN would be left of (1 - kept) / factor
    if (scaling == 2) base *= pow(factor, dim / (dim - 2.0));
    const auto border = [&](double turns) { return dim * log(original / (pi2 * turns)) / (2.0 * log(base)); };
    double first = 0.0, last = 0.0;
    if (scaling == 4) {
        first = fmax(floor(border(high)), 0.0);
        last = fmin(ceil(border(low)), dim - 1.0);
    }
    for (int i = 0; i < pairs; ++i) {
        const double f = pow(base, -2.0 * i / dim);
        double kept = 1.0;
        if (scaling == 1) kept = 0.0;
        else if (scaling == 3) kept = fmin(fmax((original * f / pi2 - low) / (high - low), 0.0), 1.0);
        else if (scaling == 4) kept = 1.0 - fmin(fmax((i - first) / fmax(last - first, 0.001), 0.0), 1.0);
        out[i] = (uint64_t)llround(ldexp(f * (kept + (1.0 - kept) / factor) / pi2, 64));  // below 2^62
    }
}

}  // namespace pk
