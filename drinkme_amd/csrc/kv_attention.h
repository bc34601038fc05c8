// The attention over the 4-bit cache (include/dmx_kv.h), included by
// kv_kernels.hip.
//
// The mathematics. A workgroup takes the query rows of one sequence that share
// a cache head (new tokens x query heads of the group) in tiles of 16, and
// walks the cached tokens 32 at a time: S^T = K Q^T and O^T += V^T P^T on
// v_mfma_f32_16x16x32_bf16, with the running maximum and sum of the softmax.
// The transposed products keep a query row in one column of every result, so
// a lane (i = lane & 15, j = lane >> 4) owns row i throughout: of a 32-token
// block it gets the scores of tokens 8 j .. 8 j + 7, which is the operand
// layout the second product wants them in. No score leaves its lane.
//
// The operands are exact: a code times its power of two is a bf16 number
// (v_cvt_scalef32_pk_bf16_fp4, two values an instruction). What is rounded:
// P, to bf16, whose error averages out over the tokens (2^-8 of a weight at
// most; the row's sum adds the unrounded ones); fp32 queries and their P go as
// three bf16 pieces, 24 bits, and lose nothing.

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kAttnWaves = 4;

struct AttnArgs {
    Cache cache;
    Seqs seqs;
    const void* q;
    int64_t q_token, q_head;  // strides, elements
    uint32_t q_heads, group;
    float scale;  // of the scores, times log2(e)
    uint32_t causal, window, splits;
    void* out;
    float* lse;
    float* part_o;   // [splits][total * q_heads][dim]
    float2* part_ml; // [splits][total * q_heads]: maximum (log2 domain), sum
};

// One lane's share of a 32-token block, as loaded.
template <int W>
struct Block {
    uint32_t k[2][W];  // tokens 8 (i >> 2) + 4 s + (i & 3): words W j .. W j + W - 1
    uint32_t ks[2][2]; // the exponent bytes of the first and the last of those words
    uint32_t v[W / 4 + (W & 3 ? (W & 3) == 3 ? 2 : 1 : 0)][8];  // per segment: tokens 8 j .. 8 j + 7
    uint32_t vs[W / 4 + (W & 3 ? (W & 3) == 3 ? 2 : 1 : 0)][2];
};

__device__ __forceinline__ float scale_of(uint32_t e) { return __uint_as_float(e << 23); }

template <int B>
__device__ __forceinline__ uint32_t pair_of(uint32_t word, float scale) {
    const bf16x2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, B);
    return __builtin_bit_cast(uint32_t, r);
}

// The maximum over the four lanes that share i.
__device__ __forceinline__ float max_over_j(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float sum_over_j(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// x as P bf16 pieces whose sum it is (to 8 P bits).
template <int P>
__device__ __forceinline__ void pieces(const float (&x)[8], bf16x8 (&out)[P]) {
    float rest[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) rest[e] = x[e];
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            out[p][e] = (__bf16)rest[e];
            if (p + 1 < P) rest[e] -= (float)out[p][e];
        }
}

// Segments of V: 128 channels (lane i reads word i, 8 channels), then 64
// (word i / 2, 4 channels) and 32 (word i / 4, 2 channels) for the rest of W.
template <int W>
struct Segments {
    static constexpr int wide = W / 4, rest = W & 3;
    static constexpr int count = wide + (rest ? rest == 3 ? 2 : 1 : 0);
    static constexpr int size(int s) { return s < wide ? 8 : s == wide && rest >= 2 ? 4 : 2; }  // channels a lane
    static constexpr int word(int s) { return s <= wide ? 16 * s : 16 * wide + 8; }             // first word
    static constexpr int tile(int s) { return s <= wide ? 8 * s : 8 * wide + 4; }               // first result tile
};

// W: dim / 32. P: bf16 pieces of the queries and weights (1: bf16, 3: fp32).
// NR: tiles of 16 query rows a wave. ROWS: the workgroup's waves take rows of
// their own and every token; else they share the rows and deal the tokens.
template <int W, int P, int NR, bool ROWS>
__global__ __launch_bounds__(64 * kAttnWaves) void k_attend(const AttnArgs a) {
    using S = Segments<W>;
    constexpr int D = 32 * W, NT = D / 16;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, j = lane >> 4;
    const uint32_t h = blockIdx.x, b = blockIdx.z / a.splits, split = blockIdx.z % a.splits;

    const Seq q = seq_of(a.seqs, b);
    const int rows = q.count * (int)a.group;
    const int r0 = (ROWS ? (int)blockIdx.y * kAttnWaves + (int)wave : (int)blockIdx.y) * 16 * NR;
    if (r0 >= rows) return;

    // what the rows see: [lo, hi) of each, and over all of them
    const int cap = a.seqs.cols << a.cache.page_shift;
    const int m0 = r0 / (int)a.group, m1 = (min(r0 + 16 * NR, rows) - 1) / (int)a.group;
    const auto hi_of = [&](int m) { return a.causal ? q.first + m + 1 : q.length; };
    const auto lo_of = [&](int m) { return a.window ? max(0, q.first + m + 1 - (int)a.window) : 0; };
    const int hi_all = min(hi_of(m1), cap), lo_all = lo_of(m0);
    const int full_hi = hi_of(m0), full_lo = lo_of(m1);  // every row sees what lies in between
    const int blk_lo = lo_all >> 5, blk_hi = hi_all > lo_all ? (hi_all + 31) >> 5 : blk_lo;
    const int per = (blk_hi - blk_lo + (int)a.splits - 1) / (int)a.splits;
    const int blk_first = blk_lo + (int)split * per, blk_end = min(blk_first + per, blk_hi);

    // this lane's row of each tile
    int hi[NR], lo[NR];
    int64_t row_out[NR];  // (token, head) in the output, -1: no row
    bf16x8 qf[NR][P][W];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        const int r = r0 + 16 * t + i;
        const bool ok = r < rows;
        const int m = ok ? r / (int)a.group : 0, g = ok ? r - m * (int)a.group : 0;
        hi[t] = ok ? hi_of(m) : 0;
        lo[t] = lo_of(m);
        const int64_t token = q.token + m, head = (int64_t)h * a.group + g;
        row_out[t] = ok ? token * a.q_heads + head : -1;
        const int64_t at = token * a.q_token + head * a.q_head + 8 * W * j;
#pragma unroll
        for (int c = 0; c < W; ++c) {
            if constexpr (P == 1) {
                u32x4 x = {0, 0, 0, 0};
                if (ok) __builtin_memcpy(&x, static_cast<const uint16_t*>(a.q) + at + 8 * c, 16);
                qf[t][0][c] = __builtin_bit_cast(bf16x8, x);
            } else {
                float x[8];
                for (int e = 0; e < 8; ++e) x[e] = ok ? static_cast<const float*>(a.q)[at + 8 * c + e] : 0.f;
                bf16x8 f[P];
                pieces<P>(x, f);
#pragma unroll
                for (int p = 0; p < P; ++p) qf[t][p][c] = f[p];
            }
        }
    }

    float mx[NR], sum[NR];
    f32x4 o[NR][NT];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        mx[t] = -INFINITY;
        sum[t] = 0.f;
#pragma unroll
        for (int c = 0; c < NT; ++c) o[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    const int g0 = (W * j) >> 2, g1 = (W * j + W - 1) >> 2;  // the blocks of this lane's first and last word of K
    const int step = ROWS ? 1 : kAttnWaves;
    for (int blk = blk_first + (ROWS ? 0 : (int)wave); blk < blk_end; blk += step) {
        Block<W> x;
        bool bad;
        {
            const Slot ko = slot_of(a.cache, a.seqs, b, h, (uint32_t)blk * 32 + 8 * (i >> 2));
            const Slot vo = slot_of(a.cache, a.seqs, b, h, (uint32_t)blk * 32 + 8 * j);
            bad = !ko.ok;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const uint64_t token = ko.token + 4 * s + (i & 3);
                __builtin_memcpy(x.k[s], a.cache.k_codes + token * (D / 8) + W * j, 4 * W);
                x.ks[s][0] = a.cache.k_scales[token * W + g0];
                x.ks[s][1] = g1 != g0 ? a.cache.k_scales[token * W + g1] : x.ks[s][0];
            }
#pragma unroll
            for (int s = 0; s < S::count; ++s) {
                const int lanes = 16 * S::size(s) / 8;  // words of the segment
                const int w = S::word(s) + i * lanes / 16;
                __builtin_memcpy(x.v[s], a.cache.v_codes + vo.token * (D / 8) + 8 * w, 32);
                __builtin_memcpy(x.vs[s], a.cache.v_scales + vo.token * W + 8 * (w >> 2), 8);
            }
        }
        const int t0 = blk * 32 + 8 * j;  // this lane's scores are of tokens t0 .. t0 + 7
        const bool part = blk * 32 < full_lo || blk * 32 + 32 > full_hi;
        const bool any_bad = __any(bad);

        // ------------------------------------------------ scores: S^T = K Q^T
        f32x4 sc[NR][2];
#pragma unroll
        for (int t = 0; t < NR; ++t) sc[t][0] = sc[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            if (any_bad && bad) x.ks[s][0] = x.ks[s][1] = 255;
            const float e0 = scale_of(x.ks[s][0]), e1 = scale_of(x.ks[s][1]);
#pragma unroll
            for (int c = 0; c < W; ++c) {
                const float e = ((W * j + c) >> 2) == g0 ? e0 : e1;
                const u32x4 f = {pair_of<0>(x.k[s][c], e), pair_of<1>(x.k[s][c], e), pair_of<2>(x.k[s][c], e),
                                 pair_of<3>(x.k[s][c], e)};
                const bf16x8 kf = __builtin_bit_cast(bf16x8, f);
#pragma unroll
                for (int t = 0; t < NR; ++t)
#pragma unroll
                    for (int p = 0; p < P; ++p)
                        sc[t][s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[t][p][c], sc[t][s], 0, 0, 0);
            }
        }

        // ------------------------------------------------------------ softmax
        bf16x8 pf[NR][P];
#pragma unroll
        for (int t = 0; t < NR; ++t) {
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = sc[t][e >> 2][e & 3] * a.scale;
            if (part) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (t0 + e < lo[t] || t0 + e >= hi[t]) p[e] = -INFINITY;
            }
            float top = p[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) top = fmaxf(top, p[e]);
            top = fmaxf(mx[t], max_over_j(top));
            if (__any(top > mx[t])) {
                const float alpha = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx[t] - top);
                sum[t] *= alpha;
#pragma unroll
                for (int c = 0; c < NT; ++c) o[t][c] *= alpha;
                mx[t] = top;
            }
            const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = __builtin_amdgcn_exp2f(p[e] - base);
                sum[t] += p[e];
            }
            pieces<P>(p, pf[t]);
        }

        // A weight of 0 does not hide a NaN in the product. Where some row does
        // not see some token of the block, values of no sequence and NaN blocks
        // go as zeros, and the NaN blocks' channels become NaN in the rows that
        // see one (an indicator's product says which).
        if (part) {
            bool nan = false;
#pragma unroll
            for (int s = 0; s < S::count; ++s)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t byte = (x.vs[s][e >> 2] >> (8 * (e & 3))) & 255u;
                    const bool out = t0 + e >= hi_all;
                    nan |= !out && byte == 255u;
                    if (out || byte == 255u) x.v[s][e] = 0;
                    if (out) x.vs[s][e >> 2] &= ~(255u << (8 * (e & 3)));
                }
            if (__any(nan)) {
#pragma unroll
                for (int t = 0; t < NR; ++t) {
                    bf16x8 seen;
#pragma unroll
                    for (int e = 0; e < 8; ++e) seen[e] = t0 + e >= lo[t] && t0 + e < hi[t] ? (__bf16)1.f : (__bf16)0.f;
#pragma unroll
                    for (int s = 0; s < S::count; ++s) {
                        bf16x8 is;
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            is[e] = ((x.vs[s][e >> 2] >> (8 * (e & 3))) & 255u) == 255u ? (__bf16)1.f : (__bf16)0.f;
                        const f32x4 n = __builtin_amdgcn_mfma_f32_16x16x32_bf16(is, seen, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                        for (int c = 0; c < S::size(s); ++c)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (n[r] > 0.f) o[t][S::tile(s) + c][r] = NAN;
                    }
                }
#pragma unroll
                for (int s = 0; s < S::count; ++s)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (((x.vs[s][e >> 2] >> (8 * (e & 3))) & 255u) == 255u) x.vs[s][e >> 2] &= ~(255u << (8 * (e & 3)));
            }
        }

        // ------------------------------------------------------ O^T += V^T P^T
#pragma unroll
        for (int s = 0; s < S::count; ++s) {
            float e[8];
#pragma unroll
            for (int n = 0; n < 8; ++n) e[n] = scale_of((x.vs[s][n >> 2] >> (8 * (n & 3))) & 255u);
            uint32_t w[8];
#pragma unroll
            for (int n = 0; n < 8; ++n)
                w[n] = S::size(s) == 8 ? x.v[s][n] : S::size(s) == 4 ? x.v[s][n] >> (16 * (i & 1)) : x.v[s][n] >> (8 * (i & 3));
#pragma unroll
            for (int c = 0; c < S::size(s); c += 2) {
                u32x4 even, odd;
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    uint32_t u, v;
                    switch (c) {
                        case 0: u = pair_of<0>(w[2 * n], e[2 * n]), v = pair_of<0>(w[2 * n + 1], e[2 * n + 1]); break;
                        case 2: u = pair_of<1>(w[2 * n], e[2 * n]), v = pair_of<1>(w[2 * n + 1], e[2 * n + 1]); break;
                        case 4: u = pair_of<2>(w[2 * n], e[2 * n]), v = pair_of<2>(w[2 * n + 1], e[2 * n + 1]); break;
                        default: u = pair_of<3>(w[2 * n], e[2 * n]), v = pair_of<3>(w[2 * n + 1], e[2 * n + 1]); break;
                    }
                    even[n] = __builtin_amdgcn_perm(v, u, 0x05040100u);
                    odd[n] = __builtin_amdgcn_perm(v, u, 0x07060302u);
                }
                const bf16x8 ve = __builtin_bit_cast(bf16x8, even), vo = __builtin_bit_cast(bf16x8, odd);
                const int n = S::tile(s) + c;
#pragma unroll
                for (int t = 0; t < NR; ++t)
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        o[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ve, pf[t][p], o[t][n], 0, 0, 0);
                        o[t][n + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vo, pf[t][p], o[t][n + 1], 0, 0, 0);
                    }
            }
        }
    }

#pragma unroll
    for (int t = 0; t < NR; ++t) sum[t] = sum_over_j(sum[t]);

    // the waves' results into wave 0's: 3 to 1 and 2 to 0, then 1 to 0
    if constexpr (!ROWS) {
        __shared__ float stat[kAttnWaves][NR][16][2];
        __shared__ f32x4 buf[2][NT][64];
        if (j == 0) {
#pragma unroll
            for (int t = 0; t < NR; ++t) {
                stat[wave][t][i][0] = mx[t];
                stat[wave][t][i][1] = sum[t];
            }
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < NR; ++t) {
            float top = -INFINITY, total = 0.f;
#pragma unroll
            for (int w = 0; w < kAttnWaves; ++w) top = fmaxf(top, stat[w][t][i][0]);
            const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int w = 0; w < kAttnWaves; ++w)
                total += stat[w][t][i][1] * __builtin_amdgcn_exp2f(stat[w][t][i][0] - base);
            const float own = __builtin_amdgcn_exp2f(mx[t] - base);
#pragma unroll
            for (int c = 0; c < NT; ++c) o[t][c] *= own;
            mx[t] = top;
            sum[t] = total;
        }
#pragma unroll
        for (int t = 0; t < NR; ++t) {
            if (wave >= 2)
#pragma unroll
                for (int c = 0; c < NT; ++c) buf[wave - 2][c][lane] = o[t][c];
            __syncthreads();
            if (wave < 2)
#pragma unroll
                for (int c = 0; c < NT; ++c) o[t][c] += buf[wave][c][lane];
            if (wave == 1)
#pragma unroll
                for (int c = 0; c < NT; ++c) buf[1][c][lane] = o[t][c];
            __syncthreads();
            if (wave == 0)
#pragma unroll
                for (int c = 0; c < NT; ++c) o[t][c] += buf[1][c][lane];
            __syncthreads();
        }
        if (wave != 0) return;
    }

    const int64_t all = (int64_t)a.seqs.total * a.q_heads;
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        if (row_out[t] < 0) continue;
        if (hi[t] > cap) sum[t] = NAN;  // it sees positions that the table has no page for
        const bool done = a.splits == 1;
        const float inv = !done || sum[t] == 0.f ? 1.f : 1.f / sum[t];
        if (j == 0) {
            if (!done)
                a.part_ml[split * all + row_out[t]] = make_float2(mx[t], sum[t]);
            else if (a.lse)
                a.lse[row_out[t]] = sum[t] == 0.f ? -INFINITY : (mx[t] + __builtin_amdgcn_logf(sum[t])) * 0.693147180559945309f;
        }
#pragma unroll
        for (int s = 0; s < S::count; ++s) {
            constexpr int most = 8;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int size = S::size(s), at = 8 * S::word(s) + size * (4 * j + r);
                float y[most];
#pragma unroll
                for (int c = 0; c < size; ++c) y[c] = o[t][S::tile(s) + c][r] * inv;
                if (!done) {
                    float* to = a.part_o + (split * all + row_out[t]) * D + at;
#pragma unroll
                    for (int c = 0; c < size; ++c) to[c] = y[c];
                } else {
                    if (sum[t] != sum[t])
#pragma unroll
                        for (int c = 0; c < size; ++c) y[c] = NAN;
                    if constexpr (P == 1) {
                        uint16_t* to = static_cast<uint16_t*>(a.out) + row_out[t] * D + at;
#pragma unroll
                        for (int c = 0; c < size; ++c) to[c] = __builtin_bit_cast(uint16_t, (__bf16)y[c]);
                    } else {
                        float* to = static_cast<float*>(a.out) + row_out[t] * D + at;
#pragma unroll
                        for (int c = 0; c < size; ++c) to[c] = y[c];
                    }
                }
            }
        }
    }
}

// The splits' results joined: a wave a row, in the order of the splits.
template <bool F32>
__global__ __launch_bounds__(256) void k_attend_join(const AttnArgs a, uint32_t dim) {
    const int64_t all = (int64_t)a.seqs.total * a.q_heads;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t lane = threadIdx.x & 63u;
    if (row >= all) return;
    float top = -INFINITY;
    for (uint32_t s = 0; s < a.splits; ++s) top = fmaxf(top, a.part_ml[s * all + row].x);
    const float base = top == -INFINITY ? 0.f : top;
    float total = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t s = 0; s < a.splits; ++s) {
        const float2 ml = a.part_ml[s * all + row];
        if (ml.y == 0.f) continue;  // nothing seen there
        const float w = __builtin_amdgcn_exp2f(ml.x - base);
        total += ml.y * w;
        const float* from = a.part_o + (s * all + row) * dim;
#pragma unroll
        for (int n = 0; n < 4; ++n)
            if (lane + 64 * n < dim) y[n] += from[lane + 64 * n] * w;
    }
    const float inv = total == 0.f ? 1.f : 1.f / total;
#pragma unroll
    for (int n = 0; n < 4; ++n)
        if (lane + 64 * n < dim) {
            const float v = total != total ? NAN : y[n] * inv;
            if constexpr (F32)
                static_cast<float*>(a.out)[row * dim + lane + 64 * n] = v;
            else
                static_cast<uint16_t*>(a.out)[row * dim + lane + 64 * n] = __builtin_bit_cast(uint16_t, (__bf16)v);
        }
    if (a.lse && lane == 0)
        a.lse[row] = total == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * 0.693147180559945309f;
}
