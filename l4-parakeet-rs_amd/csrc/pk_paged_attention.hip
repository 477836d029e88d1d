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
#include "pk_kernels.hpp"

namespace pk {

constexpr float kNegInf = -__builtin_inff();

// Eight cache values of an operand -> fp16 (e4m3 values are exact in fp16).
template <bool kF8> __device__ __forceinline__ v8h operand(const uint4& raw, int half) {
    if constexpr (kF8) {
        const uint32_t w[2] = {half ? raw.z : raw.x, half ? raw.w : raw.y};
        v8h r;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const v2h a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.0f, false);
            const v2h b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.0f, true);
            r[4 * i] = a[0];
            r[4 * i + 1] = a[1];
            r[4 * i + 2] = b[0];
            r[4 * i + 3] = b[1];
        }
        return r;
    } else {
        return __builtin_bit_cast(v8h, raw);
    }
}

// Whether any of eight fp16 values is an infinity or a NaN (exponent all ones: adding
// one there carries into the sign bit, and nowhere else).
__device__ __forceinline__ uint32_t not_finite(const v8h& v) {
    const uint4 w = __builtin_bit_cast(uint4, v);
    const uint32_t e = 0x7c007c00u, one = 0x04000400u;
    return (((w.x & e) + one) | ((w.y & e) + one) | ((w.z & e) + one) | ((w.w & e) + one)) & 0x80008000u;
}

// o += V P for an operand with infinities or NaN in it, where a product with the
// zero of a masked key would spoil rows that do not see that key: the finite values
// are multiplied, and each kind of the others counted over the keys a row sees.
__device__ __forceinline__ v4f add_not_finite(const v8h& v, const v8h& p, uint32_t seen, v4f o) {
    const _Float16 one = (_Float16)1.0f, zero = (_Float16)0.0f, inf = (_Float16)__builtin_inff();
    v8h fin, pos, neg, nan, vis;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const bool is_pos = v[j] == inf, is_neg = v[j] == -inf, is_nan = v[j] != v[j];
        fin[j] = is_pos || is_neg || is_nan ? zero : v[j];
        pos[j] = is_pos ? one : zero;
        neg[j] = is_neg ? one : zero;
        nan[j] = is_nan ? one : zero;
        vis[j] = (seen >> j) & 1u ? one : zero;
    }
    const v4f none{};
    o = __builtin_amdgcn_mfma_f32_16x16x32_f16(fin, p, o, 0, 0, 0);
    const v4f up = __builtin_amdgcn_mfma_f32_16x16x32_f16(pos, vis, none, 0, 0, 0);
    const v4f down = __builtin_amdgcn_mfma_f32_16x16x32_f16(neg, vis, none, 0, 0, 0);
    const v4f bad = __builtin_amdgcn_mfma_f32_16x16x32_f16(nan, vis, none, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (up[r] > 0.0f) o[r] += __builtin_inff();
        if (down[r] > 0.0f) o[r] -= __builtin_inff();
        if (bad[r] > 0.0f) o[r] = __builtin_nanf("");
    }
    return o;
}

// One sequence's view for a tile of 16 query rows.
struct RowTile {
    int start, rows, length, first_pos;  // first_pos: position of the sequence's first new token
};

__device__ __forceinline__ RowTile sequence_of(const PagedArgs& a, int seq) {
    int s = a.starts[seq], e = a.starts[seq + 1], len = a.lengths[seq];
    s = s < 0 ? 0 : (s > a.tokens ? a.tokens : s);
    e = e < s ? s : (e > a.tokens ? a.tokens : e);
    const int most = a.max_pages << a.shift;
    len = len < 0 ? 0 : (len > most ? most : len);
    return {s, (e - s) * a.group, len, len - (e - s)};
}

// Keys [lo, hi) that a query at `pos` sees.
__device__ __forceinline__ void window(const PagedArgs& a, int pos, int length, int& lo, int& hi) {
    lo = a.left < 0 || pos < a.left ? 0 : pos - a.left;
    hi = a.right < 0 || length - pos <= a.right ? length : pos + a.right + 1;
    if (hi < 0) hi = 0;
}

template <int kD, bool kF8>
__global__ __launch_bounds__(256) void paged_attention_kernel(PagedArgs a) {
    constexpr int kSteps = kD / 32, kBlocks = kD / 16;  // MFMA steps of S over features, feature blocks of O
    constexpr int kU = kF8 ? 2 : 1, kKeys = 32 * kU;    // 16 bytes of a value row hold 8 * kU keys; keys a wave tile
    constexpr int kBytes = kF8 ? 1 : 2;
    constexpr int kLoads = kSteps / kU;                 // 16-byte loads of a key row
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x, seq = blockIdx.z;
    const RowTile t = sequence_of(a, seq);
    const int row0 = blockIdx.y * 16;
    if (row0 >= t.rows) return;
    const int last = t.rows - row0 < 16 ? t.rows - row0 - 1 : 15;
    const int row = row0 + (l16 < last ? l16 : last);  // rows behind the last repeat it and are not stored
    const int tok = row / a.group, head = kvh * a.group + row % a.group;
    int lo, hi, tile_lo, tile_hi, full_lo, full_hi;
    window(a, t.first_pos + tok, t.length, lo, hi);
    window(a, t.first_pos + row0 / a.group, t.length, tile_lo, full_hi);       // first row: lowest bounds
    window(a, t.first_pos + (row0 + last) / a.group, t.length, full_lo, tile_hi);  // last row: highest

    v8h qf[kSteps];
    const uint16_t* qp = a.query + (size_t)(t.start + tok) * a.query_stride + (size_t)head * kD;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const int d = kF8 ? (s >> 1) * 64 + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
        qf[s] = *(const v8h*)(qp + d);
    }

    v4f acc[kBlocks];
#pragma unroll
    for (int c = 0; c < kBlocks; ++c) acc[c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    float top = kNegInf, total = 0.0f;
    const int* table = a.table + (size_t)seq * a.max_pages;
    const int last_page = t.length > 0 ? (t.length - 1) >> a.shift : 0;
    const int in_page = (1 << a.shift) - 1;
    const size_t page_bytes = (size_t)kD * kBytes << a.shift;

    for (int k0 = (tile_lo & ~(kKeys - 1)) + wave * kKeys; k0 < tile_hi; k0 += 4 * kKeys) {
        // this lane's 8 * kU keys (its values and scores) lie in one page
        const int mine = k0 + 8 * kU * g;
        int col = mine >> a.shift;
        if (col > last_page) col = last_page;
        int id = table[col];
        const bool ok = (unsigned)id < (unsigned)a.pages;
        if (!ok) id = 0;
        const int there = ok ? t.length - mine : 0;  // keys from `mine` on that exist
        uint4 kraw[kU][2][kLoads], vraw[kBlocks];
        const uint8_t* vp = a.value + ((size_t)id * a.kv_heads + kvh) * page_bytes + (((size_t)l16 << a.shift) + (mine & in_page)) * kBytes;
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int key = k0 + 8 * kU * (l16 >> 2) + 8 * u + 4 * b + (l16 & 3);
                int kcol = key >> a.shift;
                if (kcol > last_page) kcol = last_page;
                int kid = table[kcol];
                if ((unsigned)kid >= (unsigned)a.pages) kid = 0;
                const uint8_t* kp = a.key + ((size_t)kid * a.kv_heads + kvh) * page_bytes + (size_t)(key & in_page) * kD * kBytes + 16 * g;
#pragma unroll
                for (int s = 0; s < kLoads; ++s) kraw[u][b][s] = *(const uint4*)(kp + 64 * s);
            }
#pragma unroll
        for (int c = 0; c < kBlocks; ++c) vraw[c] = *(const uint4*)(vp + (((size_t)c * 16) << a.shift) * kBytes);

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
        const bool whole = k0 >= full_lo && k0 + kKeys <= full_hi && __all(ok);
        uint32_t seen = 0;  // bit j: this lane's row sees key mine + j
        if (!whole) {
#pragma unroll
            for (int j = 0; j < 8 * kU; ++j) {
                const bool see = mine + j >= lo && mine + j < hi && j < there;
                seen |= (uint32_t)see << j;
                if (!see) p[j] = kNegInf;
            }
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
        if (whole) {
#pragma unroll
            for (int c = 0; c < kBlocks; ++c)
#pragma unroll
                for (int u = 0; u < kU; ++u)
                    acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand<kF8>(vraw[c], u), pf[u], acc[c], 0, 0, 0);
        } else {
            // keys that do not exist hold anything: their values are taken as zero
            v8h vf[kBlocks][kU];
            uint32_t odd = 0;
#pragma unroll
            for (int c = 0; c < kBlocks; ++c)
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    vf[c][u] = operand<kF8>(vraw[c], u);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (8 * u + j >= there) vf[c][u][j] = (_Float16)0.0f;
                    odd |= not_finite(vf[c][u]);
                }
            if (__any(odd != 0)) {
#pragma unroll
                for (int c = 0; c < kBlocks; ++c)
#pragma unroll
                    for (int u = 0; u < kU; ++u) acc[c] = add_not_finite(vf[c][u], pf[u], seen >> (8 * u), acc[c]);
            } else {
#pragma unroll
                for (int c = 0; c < kBlocks; ++c)
#pragma unroll
                    for (int u = 0; u < kU; ++u) acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[c][u], pf[u], acc[c], 0, 0, 0);
            }
        }
    }

    // join the four waves' parts
    total = add_level(add_level(total, 16), 32);
    __shared__ float part[4][16][kD + 4];
    __shared__ float part_top[4][16], part_total[4][16];
#pragma unroll
    for (int c = 0; c < kBlocks; ++c) *(v4f*)&part[wave][l16][16 * c + 4 * g] = acc[c];
    if (g == 0) {
        part_top[wave][l16] = top;
        part_total[wave][l16] = total;
    }
    __syncthreads();
    const int r = threadIdx.x >> 4;
    if (r > last) return;
    float best = part_top[0][r];
#pragma unroll
    for (int w = 1; w < 4; ++w) best = __builtin_fmaxf(best, part_top[w][r]);
    if (best == kNegInf) best = 0.0f;
    float f[4], sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        f[w] = __builtin_amdgcn_exp2f(part_top[w][r] - best);
        sum += part_total[w][r] * f[w];
    }
    const float inv = sum == 0.0f ? 0.0f : a.value_scale / sum;
    const int orow = row0 + r;
    uint16_t* op = a.out + (size_t)(t.start + orow / a.group) * a.out_stride + (size_t)(kvh * a.group + orow % a.group) * kD;
    constexpr int kEach = kD / 16;
    const int d0 = (threadIdx.x & 15) * kEach;
#pragma unroll
    for (int j = 0; j < kEach; j += 2) {
        float v[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float x2 = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) x2 += part[w][r][d0 + j + e] * f[w];
            v[e] = x2 * inv;
        }
        *(uint32_t*)(op + d0 + j) = (uint32_t)f2h(v[0]) | ((uint32_t)f2h(v[1]) << 16);
    }
}

void launch_paged_attention(int kind, const PagedArgs& a, int head_dim, int max_queries, hipStream_t s) {
    const dim3 grid((unsigned)a.kv_heads, (unsigned)((max_queries * a.group + 15) / 16), (unsigned)a.sequences);
    if (head_dim == 128) {
        if (kind == 1) paged_attention_kernel<128, true><<<grid, 256, 0, s>>>(a);
        else paged_attention_kernel<128, false><<<grid, 256, 0, s>>>(a);
    } else {
        if (kind == 1) paged_attention_kernel<64, true><<<grid, 256, 0, s>>>(a);
        else paged_attention_kernel<64, false><<<grid, 256, 0, s>>>(a);
    }
}

}  // namespace pk
