// A step of beam search: the best candidates over the beams of a sequence and the
// vocabulary, and rows of states put in their beams' new order.
//
//   score(b, t) = scores[b] + (x[b, t] - log sum_t exp x[b, t])
//
// The logits are read once, in parts of a row that a workgroup holds in registers: the part's
// maximum, its sum of exponentials, and its best `choices` logits, in order.  A second launch puts
// a sequence's parts together; short rows of few beams are one launch, whose workgroup does both
// (8 sequences of 4 beams, 1025 fp32 logits: 7.5 us against 8.9 in two launches; 512 of 16 beams 19 against
// 37; 8 of 16 beams of 2048 11.9 and 11.3).
//
// The best of a part: a bound is the choices-th largest of the lanes' maxima of any one
// wave (as many logits at least reach it) or, for many choices, of all threads' maxima, found by
// bisection over the upper bits of the value with ballots; the few logits that reach it are listed
// in LDS and ranked by counting.  Keys are unique (value, then index), so the order of the list does
// not matter.
//
// The sum's terms are fp32, their sum and the scores 64 bits: beams are compared by
// differences of sums, and a rounding of 2^-24 of a score of -30 would change places of
// candidates that 64 bits tell apart.
//
// Wide rows are bound by vector instructions (some 660 a wave for 64 logits a lane, which keep the SIMDs
// busy for four fifths of the time) at 4.5 TB/s; so are short rows of many sequences, a wave a row (850 a wave for 600
// fp16 logits, of which the wave has places for 4096: 4096 sequences of 8 beams 56 us, SIMDs busy 95 % of the time); a
// call of few is a chain: loads, a maximum and a bisection over lanes, exponentials, the list, the join.
#include "pk_kernels.hpp"

namespace pk {

constexpr float kLog2e = 1.44269504f;
constexpr int kMostLoads = 8;  // of 16 bytes a thread
// Scalar registers: with more a SIMD holds fewer than 8 waves, and a CU one workgroup of 16 waves instead of two (a
// call of thousands of them 47 us instead of 34).
constexpr int kSgprs = 80;
// Up to as many choices a bound of one wave is near enough, in one launch (and in parts of one load a thread) and in two
// (64 sequences of 16 beams, 1025 logits: 15.7 us with it and 18.6 with the other for 24 choices, 17.9 and 19.3 for 32,
// 23.2 and 21.8 for 40; 1000 of 20 beams, 300 fp32 logits: 68 and 84 for 20, 76 and 91 for 32; of parts of two loads 8 of
// 16 beams, 20000 logits: 18.8 and 18.4 for 20, 23.2 and 20.3 for 32; of eight 64 of 8 beams, 131071 fp16 logits: 40.5 and
// 39.6 for 16, 47 and 40.5 for 24, and 897 and 50 for 64, where it is the lowest of its lanes).
constexpr int kFewWhole = 32, kFewChoices = 16;

// Of a part: its largest logit m and sum exp2(x log2e - c), c = fp32(m log2e) (fp16 logits), or
// sum exp2((x - m) log2e) (fp32 ones, whose m log2e may pass fp32's range).
struct PartSum {
    double sum;
    float most;
    int pad;
};

// Larger floats have larger bits (NaN aside); the two zeros have the same.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ unsigned long long ordered(double v) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
    return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ double unordered(unsigned long long o) {
    return __longlong_as_double((long long)(o >> 63 ? o & ~(1ull << 63) : ~o));
}

// The `count`-th largest of a wave's 64 values, 0 where count is more; bits below `last` are left 0.
__device__ __forceinline__ uint32_t wave_bound(uint32_t v, int count, int last) {
    uint32_t bound = 0;
    for (int bit = 31; bit >= last; --bit) {
        const uint32_t tried = bound | (1u << bit);
        if (__popcll(__builtin_amdgcn_ballot_w64(v >= tried)) >= count) bound = tried;
    }
    return bound;
}
// The same of the first `waves` times 64 values in LDS; each wave finds it by itself, lane l by values l, l + 64, ..
template <int kWaves> __device__ __forceinline__ uint32_t bound_of(const uint32_t* values, int waves, int lane, int count, int last) {
    uint32_t v[kWaves], bound = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v[w] = w < waves ? values[w * 64 + lane] : 0;
    for (int bit = 31; bit >= last; --bit) {
        const uint32_t tried = bound | (1u << bit);
        int reach = 0;
#pragma unroll
        for (int first = 0; first < kWaves; first += 4)
            if (first < waves)
#pragma unroll
                for (int w = first; w < first + 4 && w < kWaves; ++w) reach += __popcll(__builtin_amdgcn_ballot_w64(v[w] >= tried));
        if (reach >= count) bound = tried;
        if (reach == count) break;
    }
    return bound;
}

// Sums over a wave.
__device__ __forceinline__ long long wave_sum(long long v) {
#pragma unroll
    for (int off = 1; off <= 32; off <<= 1) {
        const int lo = (int)v, hi = (int)(v >> 32);
        const auto join = [](int h, int l) { return ((long long)h << 32) | (uint32_t)l; };
        if (off <= 8) {
            v += join(partner(hi, off), partner(lo, off));
        } else {
            int la, lb, ha, hb;
            pair_of(lo, off, la, lb);
            pair_of(hi, off, ha, hb);
            v = join(ha, la) + join(hb, lb);
        }
    }
    return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int off = 1; off <= 32; off <<= 1) {
        const long long bits = __double_as_longlong(v);
        const int lo = (int)bits, hi = (int)(bits >> 32);
        const auto join = [](int h, int l) { return __longlong_as_double(((long long)h << 32) | (uint32_t)l); };
        if (off <= 8) {
            v += join(partner(hi, off), partner(lo, off));
        } else {
            int la, lb, ha, hb;
            pair_of(lo, off, la, lb);
            pair_of(hi, off, ha, hb);
            v = join(ha, la) + join(hb, lb);
        }
    }
    return v;
}

template <bool kF16> __device__ __forceinline__ v4i nothing() {  // -infinity
    constexpr int kNone = kF16 ? (int)0xfc00fc00u : (int)0xff800000u;
    return v4i{kNone, kNone, kNone, kNone};
}
template <bool kF16> __device__ __forceinline__ float logit_of(const v4i& v, int j) {
    if constexpr (kF16) return h2f((uint16_t)((uint32_t)v[j >> 1] >> (16 * (j & 1))));
    else return __int_as_float(v[j]);
}

// The larger of each of two fp16 (the other one where one is a NaN), without the compiler's quieting of NaNs beforehand.
__device__ __forceinline__ int pk_max_f16(int a, int b) {
    int m;
    asm("v_pk_max_f16 %0, %1, %2" : "=v"(m) : "v"(a), "v"(b));
    return m;
}

template <bool kF16> __device__ __forceinline__ float largest_of(const v4i& v) {
    if constexpr (kF16) {
        const v2h m = __builtin_bit_cast(v2h, pk_max_f16(pk_max_f16(v[0], v[1]), pk_max_f16(v[2], v[3])));
        return __builtin_fmaxf((float)m[0], (float)m[1]);
    } else {
        return __builtin_fmaxf(__builtin_fmaxf(__int_as_float(v[0]), __int_as_float(v[1])), __builtin_fmaxf(__int_as_float(v[2]), __int_as_float(v[3])));
    }
}
template <int kLoads> __device__ __forceinline__ v4i pick(const v4i (&raw)[kLoads], int l) {  // raw[l] without an indexed register
    v4i v = raw[0];
#pragma unroll
    for (int i = 1; i < kLoads; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = l == i ? raw[i][j] : v[j];
    return v;
}
__device__ __forceinline__ unsigned long long key_of(float v, int i) { return ((unsigned long long)ordered(v) << 32) | (uint32_t)~(uint32_t)i; }

// What the kGroup threads that take a part share.
template <int kGroup> struct PartShared {
    static constexpr int kListed = 4 * kGroup, kRanked = kGroup > 128 ? kGroup : 128;  // candidates that are listed, and ranked as they are
    unsigned long long list[kListed];
    long long sum[kGroup / 64];
    float most[kGroup / 64];
    uint32_t bound[kGroup / 64];
    static constexpr int kTops = kGroup == 64 ? 2 : 1;  // more values than the most choices
    uint32_t top[kTops * kGroup];  // the threads' largest logits, ordered; 0: none
    int listed;
};

// The count-th largest of `size` different keys in LDS, or one below it that no more of them reach, by bisection of
// the bits in which they differ; each wave finds it by itself.  More than `count` keys: not all reach it.
template <int kMost> __device__ __forceinline__ unsigned long long bound_of_keys(const unsigned long long* list, int size, int count, int lane) {
    constexpr int kKeys = kMost / 64;
    const unsigned long long one = list[0];
    unsigned long long key[kKeys], differ = 0;
#pragma unroll
    for (int n = 0; n < kKeys; ++n) {
        key[n] = n * 64 + lane < size ? list[n * 64 + lane] : 0;
        differ |= n * 64 + lane < size ? key[n] ^ one : 0;
    }
#pragma unroll
    for (int off = 1; off <= 32; off <<= 1) differ |= (unsigned long long)__shfl_xor((long long)differ, off, 64);
    const int highest = 63 - __clzll((long long)differ);
    unsigned long long bound = one >> highest >> 1 << highest << 1;
    for (int bit = highest; bit >= 0; --bit) {
        const unsigned long long tried = bound | (1ull << bit);
        int reach = 0;
#pragma unroll
        for (int n = 0; n < kKeys; ++n) reach += __popcll(__builtin_amdgcn_ballot_w64(key[n] >= tried));
        if (reach >= count) bound = tried;
        if (reach == count) break;
    }
    return bound;
}

// The listed candidates in order, by counting those before each.
template <int kGroup>
__device__ __forceinline__ void rank_listed(const PartShared<kGroup>& shared, int count, int choices, int tid, unsigned long long* to) {
    if (tid >= count && tid < choices) to[tid] = 0;
    for (int i = tid; i < count; i += kGroup) {
        const unsigned long long key = shared.list[i];
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += shared.list[j] > key;
        if (rank < choices) to[rank] = key;
    }
}

// Part `part` of a row, by kGroup threads of a workgroup all of whose threads are here: its sum, and
// `choices` keys, best first, 0 where there are none (`to` null: neither is wanted).  `real` says, behind
// the loads, whether the row's logits are candidates.
//
// Logits are read 16 bytes at once at multiples of 16 (512 rows of 131071 fp16 logits: 29.4 us, 4.5
// TB/s; 33.4 with loads that straddle lines); those before the first and behind the last go to single threads.
// So a logit's thread depends on where its row lies, and the sum must not depend on the threads:
// equal rows have equal sums, and their candidates are ties.  It is therefore exact: a lane adds its
// terms (at most 1 each, 65 of them) to 384 in fp64, where a step is 2^-44 from 256 to 512, so that
// each term is rounded alike wherever it is added, and whole steps are added from there.  A term
// times 1 + 2^-52 is never half way between two steps, whose rounding would go by the sum before it:
// its lowest bit is 2^-52 of an fp32 term's, and half a step such a term's only from 128 on.
template <bool kF16, int kLoads, int kGroup, int kFew, typename Real>
__device__ __forceinline__ void best_of_part(const char* x, Real real, int vocab, int part, int choices, int tid, PartShared<kGroup>& shared,
                                             int& over, PartSum* sum_out, unsigned long long* to) {
    constexpr int kVec = kF16 ? 8 : 4, kWaves = kGroup / 64, kListed = PartShared<kGroup>::kListed, kRanked = PartShared<kGroup>::kRanked;
    constexpr int kTops = PartShared<kGroup>::kTops;
    constexpr bool kShort = kGroup == 64;  // rows are short, and loads without logits worth a branch
    constexpr int kPart = kGroup * kLoads * kVec, kBytes = kF16 ? 2 : 4;
    const int wave = tid >> 6, first = part * kPart, count_here = vocab - first < kPart ? vocab - first : kPart;
    const char* const here_x = x + (size_t)first * kBytes;
    const int gap = (int)(-(uintptr_t)here_x & 15) / kBytes, lead = gap < count_here ? gap : count_here;
    const int vectors = (count_here - lead) / kVec, tail = count_here - lead - vectors * kVec;
    v4i raw[kLoads];
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
        const int i = l * kGroup + tid;
        raw[l] = i < vectors ? *(const v4i*)(here_x + lead * kBytes + (size_t)i * 16) : nothing<kF16>();
    }
    const int extra_at = tid < lead ? first + tid : (tid >= 8 && tid < 8 + tail ? first + count_here - tail + tid - 8 : -1);
    float extra = -__builtin_inff();
    if (extra_at >= 0) extra = kF16 ? h2f(((const uint16_t*)x)[extra_at]) : ((const float*)x)[extra_at];
    const int filled = __builtin_amdgcn_readfirstlane(vectors);  // (of a wave: all its lanes are at one row)
    const bool candidates = real();
    const auto place = [&](int l, int j) { return first + lead + (l * kGroup + tid) * kVec + j; };
    float top[kLoads], mine = extra;  // of 16 bytes, of all
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
        top[l] = largest_of<kF16>(raw[l]);
        mine = __builtin_fmaxf(mine, top[l]);
    }
    const float wave_most = wave_max(mine);
    // (seven bits of the mantissa tell enough logits apart); 0: fewer than `choices` have a candidate
    const auto rated = [&](float v) { return candidates && v > -__builtin_inff() ? ordered(v) : 0; };
    const bool few = choices <= kFew;
    const uint32_t here = few ? wave_bound(rated(mine), choices, 16) : 0;
    if (!few) {
        float half[kTops];  // of every second 16 bytes, or of all
#pragma unroll
        for (int i = 0; i < kTops; ++i) half[i] = i ? -__builtin_inff() : extra;
#pragma unroll
        for (int l = 0; l < kLoads; ++l) half[l % kTops] = __builtin_fmaxf(half[l % kTops], top[l]);
#pragma unroll
        for (int i = 0; i < kTops; ++i) shared.top[i * kGroup + tid] = rated(half[i]);
    }
    if ((tid & 63) == 0) {
        shared.most[wave] = wave_most;
        shared.bound[wave] = here;
    }
    if (tid == 0) {
        shared.listed = 0;
        over = 0;  // (of all that are here)
    }
    __syncthreads();
    uint32_t found = shared.bound[0];
    float most = shared.most[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
        found = shared.bound[w] > found ? shared.bound[w] : found;
        most = __builtin_fmaxf(most, shared.most[w]);
    }
    if (!few) found = bound_of<kWaves * kTops>(shared.top, kWaves * kTops, tid & 63, choices, 16);
    const float bound = !candidates ? __builtin_nanf("") : (found ? unordered(found) : -3.402823466e38f);
    const float base = most > -__builtin_inff() ? most : 0.0f, c = base * kLog2e;
    const auto term = [&](float v) { return __builtin_amdgcn_exp2f(kF16 ? __builtin_fmaf(v, kLog2e, -c) : (v - base) * kLog2e); };
    const auto note = [&](float v, int i) {
        if (v >= bound) {
            const int k = atomicAdd(&shared.listed, 1);
            if (k < kListed) shared.list[k] = key_of(v, i);
            if (k >= kRanked) over = 1;
        }
    };
    constexpr double kNudge = 1.0 + 0x1p-52;
    static_assert(kLoads * kVec + 1 < 128);  // terms: the sum stays below 512
    double total = __builtin_fma((double)term(extra), kNudge, 384.0);
    uint32_t hits = 0;
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
        if (kShort && l * kGroup >= filled) break;
#pragma unroll
        for (int j = 0; j < kVec; ++j) total = __builtin_fma((double)term(logit_of<kF16>(raw[l], j)), kNudge, total);
        hits |= top[l] >= bound ? 1u << l : 0u;
    }
    note(extra, extra_at);
    while (hits) {  // most often one logit of a lane
        const int l = __ffs(hits) - 1;
        hits &= hits - 1;
        const v4i v = pick<kLoads>(raw, l);
        uint32_t which = 0;
#pragma unroll
        for (int j = 0; j < kVec; ++j) which |= logit_of<kF16>(v, j) >= bound ? 1u << j : 0u;
        int k = atomicAdd(&shared.listed, __popc(which));
        for (; which; which &= which - 1, ++k) {
            const int j = __ffs(which) - 1, w = kF16 ? j >> 1 : j;
            const int word = w & 2 ? (w & 1 ? v[3] : v[2]) : (w & 1 ? v[1] : v[0]);
            const float one = kF16 ? h2f((uint16_t)((uint32_t)word >> (16 * (j & 1)))) : __int_as_float(word);
            if (k < kListed) shared.list[k] = key_of(one, place(l, j));
            if (k >= kRanked) over = 1;
        }
    }
    const bool odd = __builtin_amdgcn_ballot_w64(total != total) != 0;
    const long long steps = wave_sum(__double_as_longlong(total) - __double_as_longlong(384.0));
    if ((tid & 63) == 0) shared.sum[wave] = odd ? -1 : steps;  // a NaN among the logits
    __syncthreads();
    if (tid == 0 && to) {
        long long sum = 0;
        bool some = false;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            some = some || shared.sum[w] < 0;
            sum += shared.sum[w];
        }
        *sum_out = PartSum{some ? __builtin_nan("") : (double)sum * 0x1p-44, most, 0};
    }
    if (!over) {
        if (to) rank_listed(shared, shared.listed, choices, tid, to);
        return;
    }
    // More than the list holds, often equal logits: 256 of those listed give a new bound, by value and index, and the
    // list is made again, until all fit: a few passes, each of which leaves about choices / 256 of those that are
    // equal (all logits of 64 sequences of 8 beams equal, 8 choices: 1025 of them 14 us, 131071 fp16 182).
    while (true) {
        const bool wide = shared.listed > kListed;
        __syncthreads();
        if (tid == 0) over = 0;
        __syncthreads();
        if (wide) over = 1;
        __syncthreads();
        if (!over) break;
        const unsigned long long at_least = wide ? bound_of_keys<256>(shared.list, 256, choices, tid & 63) : 0;
        __syncthreads();
        if (tid == 0 && wide) shared.listed = 0;
        __syncthreads();
        if (wide) {
            const auto reach = [&](float v, int i) {
                const unsigned long long key = key_of(v, i);
                if (v > -__builtin_inff() && key >= at_least) {
                    const int k = atomicAdd(&shared.listed, 1);
                    if (k < kListed) shared.list[k] = key;
                }
            };
#pragma unroll 1
            for (int l = 0; l * kGroup + tid < vectors; ++l) {  // (read again: little code that calls without it carry)
                const v4i v = *(const v4i*)(here_x + lead * kBytes + (size_t)(l * kGroup + tid) * 16);
#pragma unroll
                for (int j = 0; j < kVec; ++j) reach(logit_of<kF16>(v, j), place(l, j));
            }
            if (extra_at >= 0) reach(extra, extra_at);
        }
        __syncthreads();
    }
    // Still more than are ranked soon: the choices best of them alone.
    const int count = shared.listed;
    const bool narrow = count > kRanked;
    const unsigned long long at_least = narrow ? bound_of_keys<kListed>(shared.list, count, choices, tid & 63) : 0;
    unsigned long long key[kListed / kGroup];
#pragma unroll
    for (int n = 0; n < kListed / kGroup; ++n) key[n] = n * kGroup + tid < count ? shared.list[n * kGroup + tid] : 0;
    __syncthreads();
    if (tid == 0 && narrow) shared.listed = 0;
    __syncthreads();
    if (narrow)
#pragma unroll
        for (int n = 0; n < kListed / kGroup; ++n)
            if (n * kGroup + tid < count && key[n] >= at_least) shared.list[atomicAdd(&shared.listed, 1)] = key[n];
    __syncthreads();
    if (to) rank_listed(shared, shared.listed, choices, tid, to);
}

// A beam's candidates: 0 none, 1 of its logits, 2 ended.
__device__ __forceinline__ int beam_state(float score, const uint8_t* ended, size_t row) {
    return !(__builtin_fabsf(score) < __builtin_inff()) ? 0 : (ended && ended[row] ? 2 : 1);
}

template <bool kF16, int kLoads>
__global__ __launch_bounds__(256) __attribute__((amdgpu_num_sgpr(kSgprs))) void beam_part_kernel(BeamArgs a, int parts, PartSum* __restrict__ sums,
                                                                                                unsigned long long* __restrict__ best) {
    __shared__ PartShared<256> shared;
    __shared__ int over;
    const int row = blockIdx.x / parts, part = blockIdx.x % parts;
    if (beam_state(a.scores[row], a.ended, row) != 1) return;
    const size_t out = (size_t)row * parts + part;
    constexpr int kFew = kLoads == 1 ? kFewWhole : kFewChoices;
    best_of_part<kF16, kLoads, 256, kFew>((const char*)a.logits + (size_t)row * a.stride * (kF16 ? 2 : 4), [] { return true; }, a.vocab, part, a.choices,
                                          threadIdx.x, shared, over, sums + out, best + out * a.choices);
}

struct Candidate {
    unsigned long long score;  // ordered; 0 (a NaN's): none
    uint32_t place;            // beam * vocab + token
    __device__ __forceinline__ bool before(const Candidate& o) const { return score > o.score || (score == o.score && place < o.place); }
};

constexpr int kMostBeams = 32;

template <int kThreads, int kJoinListed> struct JoinShared {
    unsigned long long list_score[kJoinListed];
    double most[kMostBeams], rest[kMostBeams], have[kMostBeams];  // a beam's largest logit, log sum exp(x - most), its score
    unsigned long long wave_score[kThreads / 64];
    uint32_t list_place[kJoinListed];
    uint32_t wave_place[kThreads / 64], wave_bound[kThreads / 64];
    uint32_t top[kThreads];  // upper bits of the threads' best scores
    int state[kMostBeams];
    int listed;
};

// A sequence's answer, by a workgroup: the logarithms of the beams' sums, a wave a beam, then the
// best of all parts' candidates by the same bound, over the upper bits of their scores.  sums and keys are
// the sequence's, and need not be set for beams without candidates.
template <int kThreads, bool kF16, bool kOnePart, int kJoinListed>
__device__ __forceinline__ void join_parts(const BeamArgs& a, int seq, int parts, const PartSum* sums, const unsigned long long* keys,
                                           JoinShared<kThreads, kJoinListed>& shared) {
    constexpr int kWaves = kThreads / 64, kKept = 2;  // candidates a thread keeps between its two looks at them
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const size_t row0 = (size_t)seq * a.beams;
    // the first `depth` of each part: all threads have some to set the bound by; behind them a part goes on while it reaches it
    const int lists = a.beams * parts, enough = (kThreads + lists - 1) / lists, depth = enough < a.choices ? enough : a.choices, front = lists * depth;
    unsigned long long raw[kKept];
#pragma unroll
    for (int n = 0; n < kKept; ++n) {
        const int i = tid + n * kThreads;
        raw[n] = i < front ? keys[(size_t)(i / depth) * a.choices + i % depth] : 0;
    }
    if (tid == 0) shared.listed = 0;
    for (int b = wave; b < a.beams; b += kWaves) {
        const PartSum none{0.0, -__builtin_inff(), 0};
        const PartSum* const own = sums + (size_t)b * parts;
        const PartSum mine_of = lane < parts ? own[lane] : none;
        const float score = a.scores[row0 + b];
        int s = beam_state(score, a.ended, row0 + b);
        double rest = 0.0;
        float most = 0.0f;
        if (s == 1) {
            most = mine_of.most;
            for (int p = lane + 64; p < parts; p += 64) most = __builtin_fmaxf(most, own[p].most);
            most = wave_max(most);
            double mine = 0.0;
            for (int p = lane; p < parts; p += 64) {
                const PartSum one = p == lane ? mine_of : own[p];
                const bool some = one.most > -__builtin_inff() && one.most < __builtin_inff();
                // what c lacks of m log2e, in powers of 2
                const double lost = kF16 && some ? (double)(one.most * kLog2e) - (double)one.most * (double)kLog2e : 0.0;
                const double z = lost * 0.69314718055994530942;  // at most 94504 2^-24 ln 2 = 4e-3 off 0
                const double factor = kOnePart ? 1.0 + z * (1.0 + z * (0.5 + z * (1.0 / 6))) : exp(((double)one.most - (double)most) + z);
                mine += some ? one.sum * factor : one.sum;
            }
            // (kept apart from the maximum: beside one of 2^53 and more, an fp32 mask's lowest value, nothing of it would be left)
            rest = log(wave_sum(mine));
            s = most > -__builtin_inff() && most < __builtin_inff() && rest == rest;  // a NaN or an infinity: no candidates
        }
        if (lane == 0) {
            shared.most[b] = (double)most;
            shared.rest[b] = rest;
            shared.have[b] = (double)score;
            shared.state[b] = s;
        }
    }
    __syncthreads();
    const auto candidate_of = [&](int list, int c, unsigned long long key) {
        const int b = list / parts, s = shared.state[b];
        if (s == 2) return list == b * parts && c == 0 ? Candidate{ordered(shared.have[b]), (uint32_t)b * a.vocab + a.end_token} : Candidate{0, 0};
        if (!s || !key) return Candidate{0, 0};
        const double x = (double)unordered((uint32_t)(key >> 32));
        return Candidate{ordered(((x - shared.most[b]) - shared.rest[b]) + shared.have[b]), (uint32_t)b * a.vocab + ~(uint32_t)key};
    };
    const auto candidate = [&](int list, int c) { return candidate_of(list, c, keys[(size_t)list * a.choices + c]); };
    Candidate kept[kKept];
    uint32_t mine = 0;
    const auto larger = [&](const Candidate& one) {
        const uint32_t top = (uint32_t)(one.score >> 32);
        mine = top > mine ? top : mine;
    };
#pragma unroll
    for (int n = 0; n < kKept; ++n) {
        const int i = tid + n * kThreads;
        kept[n] = i < front ? candidate_of(i / depth, i % depth, raw[n]) : Candidate{0, 0};
        larger(kept[n]);
    }
    for (int i = tid + kKept * kThreads; i < front; i += kThreads) larger(candidate(i / depth, i % depth));
    uint32_t bound = 0;
    // a few are all ranked (16 of them 7.6 us of a call of one launch, 8.0 with a bound; 32 8.3 and 7.9; 128 7.9 us
    // of the join, 5.0 with a bound)
    if (front > 16 || depth < a.choices) {
        const bool few = a.choices <= (kOnePart ? kFewWhole : kFewChoices);
        const uint32_t here = few ? wave_bound(mine, a.choices, 12) : 0;  // eight bits of the mantissa
        if (few && lane == 0) shared.wave_bound[wave] = here;
        if (!few) shared.top[tid] = mine;
        __syncthreads();
        if (few) {
#pragma unroll
            for (int w = 0; w < kWaves; ++w) bound = shared.wave_bound[w] > bound ? shared.wave_bound[w] : bound;
        } else {
            bound = bound_of<kWaves>(shared.top, (front + 63) / 64, lane, a.choices, 12);
        }
    }
    const auto reaches = [&](const Candidate& one) {
        if (!one.score || (uint32_t)(one.score >> 32) < bound) return false;
        const int k = atomicAdd(&shared.listed, 1);
        if (k < kJoinListed) {
            shared.list_score[k] = one.score;
            shared.list_place[k] = one.place;
        }
        return true;
    };
    const auto note = [&](int i, const Candidate& one) {
        if (reaches(one) && i % depth == depth - 1)
            for (int c = depth; c < a.choices && reaches(candidate(i / depth, c)); ++c) {}
    };
#pragma unroll
    for (int n = 0; n < kKept; ++n) note(tid + n * kThreads, kept[n]);
    for (int i = tid + kKept * kThreads; i < front; i += kThreads) note(i, candidate(i / depth, i % depth));
    __syncthreads();
    const auto answer = [&](int c, const Candidate& one) {
        const size_t to = (size_t)seq * a.choices + c;
        const int b = one.score ? (int)(one.place / (uint32_t)a.vocab) : 0, token = one.score ? (int)(one.place % (uint32_t)a.vocab) : -1;
        a.out_scores[to] = one.score ? (float)unordered(one.score) : -__builtin_inff();
        a.out_tokens[to] = token;
        a.out_parents[to] = one.score ? (int)(row0 + b) : -1;
        if (a.out_ended) a.out_ended[to] = one.score && (shared.state[b] == 2 || token == a.end_token);
    };
    const int count = shared.listed;
    if (count <= kJoinListed) {
        if (tid >= count && tid < a.choices) answer(tid, Candidate{0, 0});
        for (int i = tid; i < count; i += kThreads) {
            const Candidate one{shared.list_score[i], shared.list_place[i]};
            int rank = 0;
            for (int j = 0; j < count; ++j) rank += Candidate{shared.list_score[j], shared.list_place[j]}.before(one);
            if (rank < a.choices) answer(rank, one);
        }
        return;
    }
    // Many candidates within a bound's last bits: the best one behind the last, `choices` times.
    Candidate last{~0ull, 0};
    for (int c = 0; c < a.choices; ++c) {
        Candidate top{0, 0};
        for (int i = tid; i < lists * a.choices; i += kThreads) {
            const Candidate one = candidate(i / a.choices, i % a.choices);
            if (one.score && last.before(one) && (!top.score || one.before(top))) top = one;
        }
#pragma unroll
        for (int off = 1; off <= 32; off <<= 1) {
            const Candidate other{(unsigned long long)__shfl_xor((long long)top.score, off, 64), (uint32_t)__shfl_xor((int)top.place, off, 64)};
            if (other.score && (!top.score || other.before(top))) top = other;
        }
        if (lane == 0) {
            shared.wave_score[wave] = top.score;
            shared.wave_place[wave] = top.place;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const Candidate other{shared.wave_score[w], shared.wave_place[w]};
            if (other.score && (!top.score || other.before(top))) top = other;
        }
        if (tid == 0) answer(c, top);
        last = top.score ? top : Candidate{0, 0xffffffffu};
        __syncthreads();
    }
}

constexpr int kJoinThreads = 512;

template <bool kF16>
__global__ __launch_bounds__(kJoinThreads) void beam_join_kernel(BeamArgs a, int parts, const PartSum* __restrict__ sums,
                                                                 const unsigned long long* __restrict__ best) {
    __shared__ JoinShared<kJoinThreads, 1024> shared;
    const size_t first = (size_t)blockIdx.x * a.beams;
    join_parts<kJoinThreads, kF16, false>(a, blockIdx.x, parts, sums + first * parts, best + first * parts * a.choices, shared);
}

// Both in one launch where the rows are short and a sequence has few beams: a wave a beam (4 waves a beam: 8
// sequences of 4 of 1025 logits 7.9 us instead of 7.6, 2048 of them 34 instead of 17, as fewer fit a CU at once).
constexpr int kWholeBeams = 16, kWholeVectors = 512;  // 16-byte loads a row

// (of 16 waves two workgroups a CU: 4096 sequences of 16 of 600 fp16 logits, 8 choices, 105 us instead of 141)
template <bool kF16, int kThreads>
__global__ __launch_bounds__(kThreads, kThreads == 1024 ? 8 : 1) __attribute__((amdgpu_num_sgpr(kSgprs))) void beam_whole_kernel(BeamArgs a) {
    constexpr int kGroup = 64;
    constexpr int kGroups = kThreads / kGroup;
    __shared__ PartShared<kGroup> part[kGroups];
    __shared__ int over;
    __shared__ JoinShared<kThreads, kGroups * 64> shared;  // (has room for all choices of all beams)
    __shared__ PartSum sums[kGroups];
    __shared__ unsigned long long keys[kGroups * 64];
    const int seq = blockIdx.x, b = threadIdx.x / kGroup;
    const size_t row = (size_t)seq * a.beams + (b < a.beams ? b : 0);
    const float score = a.scores[row];
    const uint8_t done = a.ended ? a.ended[row] : 0;
    const auto real = [&] { return b < a.beams && !done && __builtin_fabsf(score) < __builtin_inff(); };
    best_of_part<kF16, kWholeVectors / kGroup, kGroup, kFewWhole>((const char*)a.logits + row * a.stride * (kF16 ? 2 : 4), real, a.vocab, 0, a.choices,
                                                                  threadIdx.x % kGroup, part[b], over, sums + b, b < a.beams ? keys + b * a.choices : nullptr);
    __syncthreads();
    join_parts<kThreads, kF16, true>(a, seq, 1, sums, keys, shared);
}

// Loads a thread, and with them the parts: many workgroups where rows are few or short, else many
// loads, which hide what a part begins and ends with (512 rows of 131072 fp16 logits 28.6 us with 8 loads,
// 32.9 with 4, 31 with 16; 32 rows of 131071 7.3 with 2 loads, 64 rows 7.9 with 8).
constexpr long long kManyVectors = 1 << 20;  // of 16 bytes, of a call

template <bool kF16> static int beam_loads(int rows, int vocab) {
    const long long vectors = (vocab + (kF16 ? 7 : 3)) / (kF16 ? 8 : 4);
    return vectors <= 256 ? 1 : (vectors <= 512 || rows * vectors < kManyVectors ? 2 : kMostLoads);
}
template <bool kF16> static int beam_parts(int loads, int vocab) {
    const int part = 256 * loads * (kF16 ? 8 : 4);
    return (vocab + part - 1) / part;
}

// Enough for both kinds, and for fewer of everything: parts of the most loads, and those of two in a small call.
size_t beam_workspace(int sequences, int beams, int vocab, int choices) {
    const long long rows = (long long)sequences * beams, vectors = (vocab + 3) / 4, all = rows * vectors;
    const long long small = (all < kManyVectors ? all : kManyVectors) / 512, large = rows * (vectors / (256 * kMostLoads));
    return (size_t)(2 * rows + (small > large ? small : large)) * (sizeof(PartSum) + 8 * (size_t)choices);
}

template <bool kF16> static void select(const BeamArgs& a, hipStream_t s) {
    const int rows = a.sequences * a.beams, loads = beam_loads<kF16>(rows, a.vocab), parts = beam_parts<kF16>(loads, a.vocab);
    if (parts == 1 && loads <= 2 && a.beams <= kWholeBeams) {
        const auto whole = [&](auto kernel, int threads) { kernel<<<(unsigned)a.sequences, threads, 0, s>>>(a); };
        if (a.beams <= 4) whole(beam_whole_kernel<kF16, 256>, 256);
        else if (a.beams <= 8) whole(beam_whole_kernel<kF16, 512>, 512);
        else whole(beam_whole_kernel<kF16, 1024>, 1024);
        return;
    }
    PartSum* sums = (PartSum*)a.workspace;
    unsigned long long* best = (unsigned long long*)(sums + (size_t)rows * parts);
    const unsigned grid = (unsigned)rows * parts;
    if (loads == 1) beam_part_kernel<kF16, 1><<<grid, 256, 0, s>>>(a, parts, sums, best);  // more beams than the one launch takes
    else if (loads == 2) beam_part_kernel<kF16, 2><<<grid, 256, 0, s>>>(a, parts, sums, best);
    else beam_part_kernel<kF16, kMostLoads><<<grid, 256, 0, s>>>(a, parts, sums, best);
    beam_join_kernel<kF16><<<(unsigned)a.sequences, kJoinThreads, 0, s>>>(a, parts, sums, best);
}

void launch_beam_select(bool fp16, const BeamArgs& a, hipStream_t s) {
    if (fp16) select<true>(a, s);
    else select<false>(a, s);
}

// Rows in their beams' new order.  They go in units of 16 bytes, and where addresses or the row's bytes are no
// multiples of 16 the units lie at any address, which costs no more than lines touched twice (4096 x 8 rows of
// 4099 bytes 36 us, in single bytes 343; of 20004 183 us, in words of 4 511).  The last unit of a row ends where the
// row ends, and writes some bytes a second time.
typedef int AnyAddress __attribute__((ext_vector_type(4), aligned(1)));
struct Wide {
    static constexpr int kBytes = 16;
    v4i v;
    __device__ __forceinline__ void load(const char* p) { v = *(const AnyAddress*)p; }
    __device__ __forceinline__ void store(char* p) const { *(AnyAddress*)p = v; }
    __device__ __forceinline__ void store_past(char* p) const { __builtin_nontemporal_store(v, (AnyAddress*)p); }
};
struct Byte {
    static constexpr int kBytes = 1;
    uint8_t v;
    __device__ __forceinline__ void load(const char* p) { v = *(const uint8_t*)p; }
    __device__ __forceinline__ void store(char* p) const { *(uint8_t*)p = v; }
};

template <typename Unit> __device__ __forceinline__ long long unit_at(long long unit, long long row_bytes) {
    const long long at = unit * Unit::kBytes, last = row_bytes - Unit::kBytes;
    return at < last ? at : last;
}

// Into another array: a workgroup copies a chunk of a row.  Chunks of the same columns lie on one
// XCD, whose L2 then reads a parent's once for all its children (16 x 8 rows of 2 MB: 74 us, 80
// without; a copy of all of them 99).  Stores past the caches where the state is larger than they
// are (74 us against 80).
constexpr int kRowLoads = 2;

template <bool kPast>
__global__ __launch_bounds__(256) void beam_rows_kernel(const char* __restrict__ in, const int* __restrict__ parents, char* __restrict__ out, int beams,
                                                        long long row_bytes, long long units, int chunks, int step) {
    const long long row0 = (long long)blockIdx.y * beams;
    const int t = step >= 8 ? blockIdx.x >> 3 : blockIdx.x, b = t % beams;  // XCDs take workgroups in turn
    const long long p = (long long)parents[row0 + b] - row0;
    if (p < 0 || p >= beams) return;
    const char* const from = in + (row0 + p) * row_bytes;
    char* const to = out + (row0 + b) * row_bytes;
    for (int chunk = step >= 8 ? t / beams * 8 + (blockIdx.x & 7) : t / beams; chunk < chunks; chunk += step) {
        const long long first = (long long)chunk * 256 * kRowLoads + threadIdx.x;
        Wide held[kRowLoads];
#pragma unroll
        for (int n = 0; n < kRowLoads; ++n)
            if (first + n * 256 < units) held[n].load(from + unit_at<Wide>(first + n * 256, row_bytes));
#pragma unroll
        for (int n = 0; n < kRowLoads; ++n)
            if (first + n * 256 < units) {
                char* const at = to + unit_at<Wide>(first + n * 256, row_bytes);
                if constexpr (kPast) held[n].store_past(at);
                else held[n].store(at);
            }
    }
}

// Short rows: a thread a unit of all rows, one behind the other.
template <typename Unit>
__global__ __launch_bounds__(256) void beam_units_kernel(const char* __restrict__ in, const int* __restrict__ parents, char* __restrict__ out, uint32_t beams,
                                                         uint32_t row_bytes, uint32_t units, uint32_t all) {
    const uint32_t at = blockIdx.x * 256 + threadIdx.x;
    if (at >= all) return;
    const uint32_t row = at / units, parent = (uint32_t)parents[row];
    const long long in_row = unit_at<Unit>(at - row * units, row_bytes);
    if (parent / beams != row / beams) return;
    Unit one;
    one.load(in + (size_t)parent * row_bytes + in_row);
    one.store(out + (size_t)row * row_bytes + in_row);
}
// Units a row (32768 rows of 80 units 12.4 us, 25.2 with a workgroup a row; 250 33.2 and 34.0; 400 65 and 51).
constexpr long long kShortUnits = 256;

// In place: a thread owns a column of a sequence's rows, a unit wide, reads what they will hold and writes those that
// change then (the rows above: 66 us, for fewer of them are written).  From 9 beams on the places of 32 are read, those
// behind the last beam as its first row's (64 sequences, rows of 64 KB: 8 beams 7.3 us, 9 20.4, 16 22.7, 32 34.2).
template <typename Unit, int kBeams>
__device__ __forceinline__ void turn_column(char* column, const int* __restrict__ parents, long long row0, int beams, long long row_bytes) {
    Unit held[kBeams];
#pragma unroll
    for (int b = 0; b < kBeams; ++b) {
        const int at = b < beams ? b : 0;
        const long long p = (long long)parents[row0 + at] - row0;
        held[b].load(column + (p >= 0 && p < beams ? p : at) * row_bytes);
    }
#pragma unroll
    for (int b = 0; b < kBeams; ++b) {
        const long long p = b < beams ? (long long)parents[row0 + b] - row0 : -1;
        if (p >= 0 && p < beams && p != b) held[b].store(column + b * row_bytes);
    }
}

// No unit of a column may reach into another's: the `rest` bytes behind the last unit are columns of their own, which the
// last workgroup has (16 x 8 rows of 1 MB + 1 30 us, all in single bytes 134; 2 beams of 100 bytes 3.1 us, 5.2 with a launch
// for them, 64 x 16 of 100 9.1 and 15.0).
template <int kBeams>
__global__ __launch_bounds__(256) void beam_columns_kernel(char* state, const int* __restrict__ parents, int beams, long long row_bytes, long long units,
                                                           int rest) {
    const long long row0 = (long long)blockIdx.y * beams;
    char* const rows = state + row0 * row_bytes;
    const long long blocks = (long long)gridDim.x - (rest != 0);
    if (blockIdx.x >= blocks) {
        if ((int)threadIdx.x < rest) turn_column<Byte, kBeams>(rows + units * Wide::kBytes + threadIdx.x, parents, row0, beams, row_bytes);
        return;
    }
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < units; i += blocks * 256)
        turn_column<Wide, kBeams>(rows + i * Wide::kBytes, parents, row0, beams, row_bytes);
}

constexpr int kMostChunks = 1 << 16;  // of a row, in a launch: its threads in a dimension stay far below 2^32

template <bool kPast>
static void reorder_rows(const char* in, const int* parents, char* out, int sequences, int beams, long long row_bytes, long long units, hipStream_t s) {
    const int chunks = (int)((units + 256 * kRowLoads - 1) / (256 * kRowLoads)), once = chunks < kMostChunks ? chunks : kMostChunks;
    const int step = once >= 8 ? (once + 7) / 8 * 8 : once;
    beam_rows_kernel<kPast><<<dim3((unsigned)(step * beams), (unsigned)sequences), 256, 0, s>>>(in, parents, out, beams, row_bytes, units, chunks, step);
}

template <typename Unit> static void reorder_units(const char* in, const int* parents, char* out, int sequences, int beams, int row_bytes, hipStream_t s) {
    const uint32_t units = (row_bytes + Unit::kBytes - 1) / Unit::kBytes, all = units * sequences * beams;  // at most 2^25
    beam_units_kernel<Unit><<<(all + 255) / 256, 256, 0, s>>>(in, parents, out, beams, row_bytes, units, all);
}

static void reorder_columns(char* state, const int* parents, int sequences, int beams, long long row_bytes, hipStream_t s) {
    const long long units = row_bytes / Wide::kBytes, blocks = (units + 255) / 256;
    const int rest = (int)(row_bytes % Wide::kBytes);
    const dim3 grid((unsigned)((blocks < kMostChunks ? blocks : kMostChunks) + (rest != 0)), (unsigned)sequences);
    if (beams <= 8) beam_columns_kernel<8><<<grid, 256, 0, s>>>(state, parents, beams, row_bytes, units, rest);
    else beam_columns_kernel<32><<<grid, 256, 0, s>>>(state, parents, beams, row_bytes, units, rest);
}

void launch_beam_reorder(const void* state, const int* parents, void* out, int sequences, int beams, long long row_bytes, hipStream_t s) {
    const char* in = (const char*)state;
    char* to = (char*)out;
    if (in != to) {
        const long long units = (row_bytes + Wide::kBytes - 1) / Wide::kBytes;
        if (row_bytes < Wide::kBytes) reorder_units<Byte>(in, parents, to, sequences, beams, (int)row_bytes, s);
        else if (units <= kShortUnits) reorder_units<Wide>(in, parents, to, sequences, beams, (int)row_bytes, s);
        else if (row_bytes * sequences * beams > kCached) reorder_rows<true>(in, parents, to, sequences, beams, row_bytes, units, s);
        else reorder_rows<false>(in, parents, to, sequences, beams, row_bytes, units, s);
        return;
    }
    reorder_columns(to, parents, sequences, beams, row_bytes, s);
}

}  // namespace pk
