// A step of beam search: the best candidates over the beams of a sequence and the
// vocabulary, and rows of states put in their beams' new order.
//
//   score(b, t) = scores[b] + (x[b, t] - log sum_t exp x[b, t])
//
// Two launches.  The first reads the logits once, in parts of a row that a workgroup
// holds in registers: the part's maximum, its sum of exponentials, and its best `choices`
// logits, in order.  The second puts a sequence's parts together.
//
// The best of a part: a bound is the choices-th largest of the lanes' maxima of any one
// wave (as many logits at least reach it), found by bisection over the bits of the value
// with one ballot a bit; the few logits that reach it are listed in LDS and ranked by
// counting.  Keys are unique (value, then index), so the order of the list does not matter.
//
// The sum's terms are fp32, their sum and the scores 64 bits: beams are compared by
// differences of sums, and a rounding of 2^-24 of a score of -30 would change places of
// candidates that 64 bits tell apart.
#include "pk_kernels.hpp"

namespace pk {

constexpr int kPartElements = 64;                 // a lane's
constexpr int kPart = 256 * kPartElements;        // a workgroup's
constexpr int kListed = 1024;                     // candidates that are ranked; more of them are taken out one by one

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
        if (__popcll(__ballot(v >= tried)) >= count) bound = tried;
    }
    return bound;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// Eight fp16 or four fp32 logits at the alignment of one.
struct __attribute__((packed, aligned(2))) Eight { uint32_t w[4]; };
struct __attribute__((packed, aligned(4))) Four { uint32_t w[4]; };

template <bool kF16>
__global__ __launch_bounds__(256) void beam_part_kernel(const void* __restrict__ logits, long long stride, const float* __restrict__ scores,
                                                        const uint8_t* __restrict__ ended, int vocab, int choices, int parts,
                                                        PartSum* __restrict__ sums, unsigned long long* __restrict__ best) {
    constexpr int kVec = kF16 ? 8 : 4, kLoads = kPartElements / kVec;
    __shared__ unsigned long long list[kListed];
    __shared__ float part_most[4];
    __shared__ double part_sum[4];
    __shared__ uint32_t part_bound[4];
    __shared__ unsigned long long part_key[4];
    __shared__ int listed;
    const int row = blockIdx.x / parts, part = blockIdx.x % parts, wave = threadIdx.x >> 6;
    if ((ended && ended[row]) || !(__builtin_fabsf(scores[row]) < __builtin_inff())) return;  // no candidates from its logits
    const char* const x = (const char*)logits + (size_t)row * stride * (kF16 ? 2 : 4);
    const int start = part * kPart;
    uint32_t raw[kLoads][4];
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
        const int i = start + (l * 256 + (int)threadIdx.x) * kVec;
        if (i + kVec <= vocab) {
            if constexpr (kF16) {
                const Eight e = *(const Eight*)(x + (size_t)i * 2);
#pragma unroll
                for (int j = 0; j < 4; ++j) raw[l][j] = e.w[j];
            } else {
                const Four e = *(const Four*)(x + (size_t)i * 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) raw[l][j] = e.w[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (kF16) {
                    const uint32_t a = i + 2 * j < vocab ? ((const uint16_t*)x)[i + 2 * j] : 0xfc00u;
                    const uint32_t b = i + 2 * j + 1 < vocab ? ((const uint16_t*)x)[i + 2 * j + 1] : 0xfc00u;
                    raw[l][j] = a | (b << 16);
                } else {
                    raw[l][j] = i + j < vocab ? ((const uint32_t*)x)[i + j] : 0xff800000u;
                }
            }
        }
    }
    const auto at = [&](int l, int j) {
        if constexpr (kF16) return h2f((uint16_t)(raw[l][j >> 1] >> (16 * (j & 1))));
        else return __uint_as_float(raw[l][j]);
    };
    float mine = -__builtin_inff();
#pragma unroll
    for (int l = 0; l < kLoads; ++l)
#pragma unroll
        for (int j = 0; j < kVec; ++j) mine = __builtin_fmaxf(mine, at(l, j));
    const float wave_most = wave_max(mine);
    const bool any = mine > -__builtin_inff();
    const uint32_t bound_here = wave_bound(any ? ordered(mine) : 0, choices, kF16 ? 13 : 0);  // fp16 values end 13 bits earlier
    if ((threadIdx.x & 63) == 0) {
        part_most[wave] = wave_most;
        part_bound[wave] = bound_here;
    }
    if (threadIdx.x == 0) listed = 0;
    __syncthreads();
    const float most = __builtin_fmaxf(__builtin_fmaxf(part_most[0], part_most[1]), __builtin_fmaxf(part_most[2], part_most[3]));
    uint32_t bound = part_bound[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) bound = part_bound[w] > bound ? part_bound[w] : bound;
    const float base = most > -__builtin_inff() ? most : 0.0f;
    double total = 0.0;
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < kVec; ++j) sum += __builtin_amdgcn_exp2f((at(l, j) - base) * 1.44269504088896341f);
        total += (double)sum;
    }
    if (any && ordered(mine) >= bound) {
#pragma unroll
        for (int l = 0; l < kLoads; ++l)
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                const float v = at(l, j);
                if (v > -__builtin_inff() && ordered(v) >= bound) {
                    const int k = atomicAdd(&listed, 1);
                    if (k < kListed)
                        list[k] = ((unsigned long long)ordered(v) << 32) | (uint32_t)~(uint32_t)(start + (l * 256 + (int)threadIdx.x) * kVec + j);
                }
            }
    }
    total = wave_sum(total);
    if ((threadIdx.x & 63) == 0) part_sum[wave] = total;
    __syncthreads();
    const size_t out = (size_t)row * parts + part;
    if (threadIdx.x == 0) sums[out] = PartSum{(part_sum[0] + part_sum[1]) + (part_sum[2] + part_sum[3]), most, 0};
    unsigned long long* to = best + out * choices;
    const int count = listed;
    if (count <= kListed) {
        for (int i = threadIdx.x; i < choices; i += 256)
            if (i >= count) to[i] = 0;
        for (int i = threadIdx.x; i < count; i += 256) {
            const unsigned long long key = list[i];
            int rank = 0;
            for (int j = 0; j < count; ++j) rank += list[j] > key;
            if (rank < choices) to[rank] = key;
        }
        return;
    }
    // Many equal logits: the largest key below the last one, `choices` times.
    unsigned long long last = ~0ull;
    for (int c = 0; c < choices; ++c) {
        unsigned long long key = 0;
#pragma unroll
        for (int l = 0; l < kLoads; ++l)
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                const float v = at(l, j);
                const unsigned long long k =
                    ((unsigned long long)ordered(v) << 32) | (uint32_t)~(uint32_t)(start + (l * 256 + (int)threadIdx.x) * kVec + j);
                if (v > -__builtin_inff() && k < last && k > key) key = k;
            }
#pragma unroll
        for (int off = 1; off <= 32; off <<= 1) key = max_level(key, off);
        if ((threadIdx.x & 63) == 0) part_key[wave] = key;
        __syncthreads();
        key = part_key[0];
#pragma unroll
        for (int w = 1; w < 4; ++w) key = part_key[w] > key ? part_key[w] : key;
        if (threadIdx.x == 0) to[c] = key;
        last = key;
        __syncthreads();
    }
}

struct Candidate {
    unsigned long long score;  // ordered
    uint32_t place;            // beam * vocab + token
    __device__ __forceinline__ bool before(const Candidate& o) const { return score > o.score || (score == o.score && place < o.place); }
};

// A workgroup a sequence.  A thread has the lists (beam, part) it, it + 256, ...; each is in
// order, so that a list's first candidate is its best.
constexpr int kMostBeams = 32;

__global__ __launch_bounds__(256) void beam_join_kernel(BeamArgs a, int parts, const PartSum* __restrict__ sums,
                                                        const unsigned long long* __restrict__ best) {
    __shared__ double whole[kMostBeams];  // log of a beam's sum
    __shared__ int state[kMostBeams];     // 0 no candidates, 1 its logits, 2 ended
    __shared__ unsigned long long list_score[kListed];
    __shared__ uint32_t list_place[kListed];
    __shared__ uint32_t wave_part[4];
    __shared__ unsigned long long wave_score[4];
    __shared__ uint32_t wave_place[4];
    __shared__ int listed;
    const int seq = blockIdx.x, wave = threadIdx.x >> 6, lists = a.beams * parts;
    const size_t row0 = (size_t)seq * a.beams;
    if (threadIdx.x == 0) listed = 0;
    if ((int)threadIdx.x < a.beams) {
        const size_t row = row0 + threadIdx.x;
        const float score = a.scores[row];
        int s = 0;
        double log_sum = 0.0;
        if (__builtin_fabsf(score) < __builtin_inff()) {
            if (a.ended && a.ended[row]) {
                s = 2;
            } else {
                float most = -__builtin_inff();
                for (int p = 0; p < parts; ++p) most = __builtin_fmaxf(most, sums[row * parts + p].most);
                if (most > -__builtin_inff() && most < __builtin_inff()) {
                    double sum = 0.0;
                    for (int p = 0; p < parts; ++p) {
                        const PartSum& one = sums[row * parts + p];
                        if (one.most > -__builtin_inff()) sum += one.sum * exp((double)one.most - (double)most);
                        else if (one.sum != one.sum) sum = one.sum;
                    }
                    log_sum = (double)most + log(sum);
                    s = log_sum == log_sum ? 1 : 0;  // a NaN among the logits: no candidates
                }
            }
        }
        whole[threadIdx.x] = log_sum;
        state[threadIdx.x] = s;
    }
    __syncthreads();
    // candidate c of list i; score 0 stands for none (that of a NaN's bits)
    const auto candidate = [&](int i, int c) {
        const int b = i / parts, s = state[b];
        if (s == 2) return i % parts == 0 && c == 0 ? Candidate{ordered((double)a.scores[row0 + b]), (uint32_t)b * a.vocab + a.end_token} : Candidate{0, 0};
        const unsigned long long key = s ? best[(row0 * parts + i) * a.choices + c] : 0;
        if (!key) return Candidate{0, 0};
        const double x = (double)unordered((uint32_t)(key >> 32));
        return Candidate{ordered((x - whole[b]) + (double)a.scores[row0 + b]), (uint32_t)b * a.vocab + ~(uint32_t)key};
    };
    uint32_t mine = 0;
    for (int i = threadIdx.x; i < lists; i += 256) {
        const uint32_t top = (uint32_t)(candidate(i, 0).score >> 32);
        mine = top > mine ? top : mine;
    }
    const uint32_t here = wave_bound(mine, a.choices, 0);
    if ((threadIdx.x & 63) == 0) wave_part[wave] = here;
    __syncthreads();
    uint32_t bound = wave_part[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) bound = wave_part[w] > bound ? wave_part[w] : bound;
    for (int i = threadIdx.x; i < lists; i += 256)
        for (int c = 0; c < a.choices; ++c) {
            const Candidate one = candidate(i, c);
            if (!one.score || (uint32_t)(one.score >> 32) < bound) break;
            const int k = atomicAdd(&listed, 1);
            if (k < kListed) {
                list_score[k] = one.score;
                list_place[k] = one.place;
            }
        }
    __syncthreads();
    const auto answer = [&](int c, const Candidate& one) {
        const size_t to = (size_t)seq * a.choices + c;
        const int b = one.score ? (int)(one.place / (uint32_t)a.vocab) : 0, token = one.score ? (int)(one.place % (uint32_t)a.vocab) : -1;
        a.out_scores[to] = one.score ? (float)unordered(one.score) : -__builtin_inff();
        a.out_tokens[to] = token;
        a.out_parents[to] = one.score ? (int)(row0 + b) : -1;
        if (a.out_ended) a.out_ended[to] = one.score && (state[b] == 2 || token == a.end_token);
    };
    const int count = listed;
    if (count <= kListed) {
        for (int c = threadIdx.x; c < a.choices; c += 256)
            if (c >= count) answer(c, Candidate{0, 0});
        for (int i = threadIdx.x; i < count; i += 256) {
            const Candidate one{list_score[i], list_place[i]};
            int rank = 0;
            for (int j = 0; j < count; ++j) rank += Candidate{list_score[j], list_place[j]}.before(one);
            if (rank < a.choices) answer(rank, one);
        }
        return;
    }
    // Many candidates within a bound's last bits: the best one behind the last, `choices` times.
    Candidate last{~0ull, 0};
    for (int c = 0; c < a.choices; ++c) {
        Candidate top{0, 0};
        for (int i = threadIdx.x; i < lists; i += 256)
            for (int k = 0; k < a.choices; ++k) {
                const Candidate one = candidate(i, k);
                if (!one.score) break;
                if (last.before(one)) {  // the list's first that is left
                    if (!top.score || one.before(top)) top = one;
                    break;
                }
            }
#pragma unroll
        for (int off = 1; off <= 32; off <<= 1) {
            const Candidate other{(unsigned long long)__shfl_xor((long long)top.score, off, 64), (uint32_t)__shfl_xor((int)top.place, off, 64)};
            if (other.score && (!top.score || other.before(top))) top = other;
        }
        if ((threadIdx.x & 63) == 0) {
            wave_score[wave] = top.score;
            wave_place[wave] = top.place;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const Candidate other{wave_score[w], wave_place[w]};
            if (other.score && (!top.score || other.before(top))) top = other;
        }
        if (threadIdx.x == 0) answer(c, top);
        last = top;
        __syncthreads();
        if (!top.score) last = Candidate{0, 0xffffffffu};
    }
}

static int beam_parts(int vocab) { return (vocab + kPart - 1) / kPart; }

size_t beam_workspace(int sequences, int beams, int vocab, int choices) {
    return (size_t)sequences * beams * beam_parts(vocab) * (sizeof(PartSum) + 8 * (size_t)choices);
}

void launch_beam_select(bool fp16, const BeamArgs& a, hipStream_t s) {
    const int parts = beam_parts(a.vocab), rows = a.sequences * a.beams;
    PartSum* sums = (PartSum*)a.workspace;
    unsigned long long* best = (unsigned long long*)(sums + (size_t)rows * parts);
    const unsigned grid = (unsigned)rows * parts;
    if (fp16) beam_part_kernel<true><<<grid, 256, 0, s>>>(a.logits, a.stride, a.scores, a.ended, a.vocab, a.choices, parts, sums, best);
    else beam_part_kernel<false><<<grid, 256, 0, s>>>(a.logits, a.stride, a.scores, a.ended, a.vocab, a.choices, parts, sums, best);
    beam_join_kernel<<<(unsigned)a.sequences, 256, 0, s>>>(a, parts, sums, best);
}

// Rows in their beams' new order.  A thread owns a column of a sequence's rows, reads what
// all of them will hold and writes it then, so that the output may be the state itself.
template <typename Unit, int kBeams>
__global__ __launch_bounds__(256) void beam_reorder_kernel(const Unit* in, const int* __restrict__ parents, Unit* out, int beams, long long units) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const int seq = blockIdx.y;
    if (i >= units) return;
    const long long row0 = (long long)seq * beams;
    Unit held[kBeams];
#pragma unroll
    for (int b = 0; b < kBeams; ++b) {
        const long long p = b < beams ? (long long)parents[row0 + b] - row0 : -1;
        if (p >= 0 && p < beams) held[b] = in[(row0 + p) * units + i];
    }
#pragma unroll
    for (int b = 0; b < kBeams; ++b) {
        const long long p = b < beams ? (long long)parents[row0 + b] - row0 : -1;
        if (p >= 0 && p < beams) out[(row0 + b) * units + i] = held[b];
    }
}

template <typename Unit>
static void reorder(const void* in, const int* parents, void* out, int sequences, int beams, long long units, hipStream_t s) {
    const dim3 grid((unsigned)((units + 255) / 256), (unsigned)sequences);
    const auto launch = [&](auto kernel) { kernel<<<grid, 256, 0, s>>>((const Unit*)in, parents, (Unit*)out, beams, units); };
    if (beams <= 4) launch(beam_reorder_kernel<Unit, 4>);
    else if (beams <= 8) launch(beam_reorder_kernel<Unit, 8>);
    else if (beams <= 16) launch(beam_reorder_kernel<Unit, 16>);
    else launch(beam_reorder_kernel<Unit, 32>);
}

void launch_beam_reorder(const void* state, const int* parents, void* out, int sequences, int beams, long long row_bytes, hipStream_t s) {
    const uintptr_t all = (uintptr_t)state | (uintptr_t)out | (uintptr_t)row_bytes;
    if (all % 16 == 0) reorder<uint4>(state, parents, out, sequences, beams, row_bytes / 16, s);
    else if (all % 4 == 0) reorder<uint32_t>(state, parents, out, sequences, beams, row_bytes / 4, s);
    else reorder<uint8_t>(state, parents, out, sequences, beams, row_bytes, s);
}

}  // namespace pk
