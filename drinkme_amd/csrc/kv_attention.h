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
// P, to bf16, 2^-8 of a weight at most, whose error averages out over the tokens
// (a row is divided by the sum of its rounded weights, so that the error cancels
// where few weights make the result: 0.0022 of the norm against 64 bits where the
// unrounded sum gave 0.0025, 0.0016 of both the result's own rounding; the logarithm
// takes the unrounded sum). fp32 queries and their P go as three bf16 pieces, 24
// bits: 4e-7 against 64 bits.

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
    uint32_t row_blocks;  // for each sequence's first seqs.each new tokens
    void* out;
    float* lse;
    float* part_o;   // [splits][total * q_heads][dim]
    f32x4* part_stat;  // [splits][total * q_heads]: reference (log2 domain), sum, sum of the rounded weights
};

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

// One lane's share of a 32-token block, as loaded.
template <int W>
struct Block {
    uint32_t k[2][W];   // tokens 8 (i >> 2) + 4 s + (i & 3): words W j .. W j + W - 1
    uint32_t ks[2][2];  // the exponent bytes of the first and the last of those words
    uint32_t v[Segments<W>::count][8];   // per segment: tokens 8 j .. 8 j + 7
    uint32_t vs[Segments<W>::count][2];  // their exponent bytes
    bool ok;                             // false: no page for this lane's K tokens
};

// Where tokens lie. WIDE: a page holds whole 32-token blocks, so that a block's
// place is the wave's and a lane's part in it an offset that stays; else each
// lane looks up the page of its own octet of the block. (In pages of 64, a decode
// step of 32 sequences of up to 8192 tokens 62 us by octets and 57 by blocks, a prompt
// of 2048 tokens after 8192 332 and 319, before the later steps.)
template <bool WIDE>
__device__ __forceinline__ uint32_t page_of(const AttnArgs& a, uint32_t b, uint32_t block, int octet) {
    const uint32_t col = (block * 32 + (WIDE ? 0 : 8 * octet)) >> a.cache.page_shift;
    return col >= (uint32_t)a.seqs.cols ? ~0u : (uint32_t)a.seqs.table[(int64_t)b * a.seqs.cols + col];
}

struct Place {
    uint64_t base;  // index of (page, head, slot): a block's (WIDE), or an octet's
    uint32_t in;    // the lane's octet after it, tokens
    bool ok;        // false: no page there, and the place is in page 0
};

template <bool WIDE>
__device__ __forceinline__ Place place_of(const AttnArgs& a, uint32_t h, uint32_t page, uint32_t block, int octet) {
    if (WIDE) page = __builtin_amdgcn_readfirstlane(page);
    const uint32_t shift = a.cache.page_shift, mask = (1u << shift) - 1u;
    const bool ok = page < a.cache.pages;
    const uint64_t base = (((uint64_t)(ok ? page : 0u) * a.cache.heads + h) << shift) + ((block * 32 + (WIDE ? 0 : 8 * octet)) & mask);
    return {base, WIDE ? 8u * octet : 0u, ok};
}

// The page numbers of a lane's K and V tokens in a block.
struct Entry {
    uint32_t k, v;
};

// The scale operand of the conversions takes the exponent bits alone; sign and
// mantissa may hold anything (measured over all exponents and codes).
template <int N>
__device__ __forceinline__ float scale_of(uint32_t bytes) {  // of byte N
    return __uint_as_float(N == 3 ? bytes >> 1 : bytes << (23 - 8 * N));
}

template <int B>
__device__ __forceinline__ uint32_t pair_of(uint32_t word, float scale) {
    const bf16x2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, B);
    return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ uint32_t pair_at(int b, uint32_t word, float scale) {  // b: a constant once unrolled
    return b == 0 ? pair_of<0>(word, scale) : b == 1 ? pair_of<1>(word, scale) : b == 2 ? pair_of<2>(word, scale) : pair_of<3>(word, scale);
}

// The maximum and the sum over the four lanes that share i.
__device__ __forceinline__ float max_over_j(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_over_j(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// sum plus the eight numbers of x.
__device__ __forceinline__ float plus_all(const bf16x8& x, float sum) {
    const u32x4 w = __builtin_bit_cast(u32x4, x);
    const bf16x2 ones = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
    for (int n = 0; n < 4; ++n) sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, (uint32_t)w[n]), ones, sum, false);
    return sum;
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

// What a wave keeps of its query rows: 16 a tile, lane (i, j) of row i.
template <int W, int P, int NR>
struct State {
    static constexpr int NT = 2 * W;
    int hi[NR], lo[NR];  // the positions that the lane's row sees
    bf16x8 q[NR][P][W];
    float mx[NR], sum[NR];  // the weights' reference (log2 domain) and the lane's share of their sum
    float norm[NR];         // the same of the weights as rounded
    f32x4 o[NR][NT];        // channels 4 j + r of tile n, in Segments' order
};

template <bool WIDE>
__device__ __forceinline__ Entry entries(const AttnArgs& a, uint32_t b, int blk, int i, int j) {
    Entry e;
    e.k = page_of<WIDE>(a, b, blk, i >> 2);
    e.v = WIDE ? e.k : page_of<WIDE>(a, b, blk, j);
    return e;
}

template <bool WIDE, int W>
__device__ __forceinline__ void fetch(const AttnArgs& a, uint32_t h, int blk, Entry e, int i, int j, Block<W>& x) {
    using S = Segments<W>;
    const Place k = place_of<WIDE>(a, h, e.k, blk, i >> 2), v = place_of<WIDE>(a, h, e.v, blk, j);
    const int g0 = (W * j) >> 2, g1 = (W * j + W - 1) >> 2;
    const uint32_t in = k.in + (i & 3);
    const uint32_t* kc = a.cache.k_codes + k.base * (4 * W);
    const uint8_t* ks = a.cache.k_scales + k.base * W;
    x.ok = k.ok;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        __builtin_memcpy(x.k[s], kc + ((in + 4 * s) * (4 * W) + W * j), 4 * W);
        x.ks[s][0] = ks[(in + 4 * s) * W + g0];
        if (W != 2 && W != 4) x.ks[s][1] = ks[(in + 4 * s) * W + g1];
    }
    const uint32_t* vc = a.cache.v_codes + v.base * (4 * W);
    const uint8_t* vs = a.cache.v_scales + v.base * W;
#pragma unroll
    for (int s = 0; s < S::count; ++s) {
        const uint32_t w = S::word(s) + (i * 2 * S::size(s) >> 4);
        __builtin_memcpy(x.v[s], vc + (v.in * (4 * W) + 8 * w), 32);
        __builtin_memcpy(x.vs[s], __builtin_assume_aligned(vs + (v.in * W + 8 * (w >> 2)), 8), 8);
    }
}

// Where some row does not see some token of the block. A weight of 0 does not
// hide a NaN or an infinity in the product: values of no sequence and blocks that
// may hold one (bytes over 252, the largest written for finite values) go as zeros,
// and those blocks' channels become NaN in the rows that see one (an indicator's
// product says which).
template <int W, int P, int NR>
__device__ __forceinline__ void hide_values(State<W, P, NR>& st, Block<W>& x, int t0, int hi_all) {
    using S = Segments<W>;
    bool nan = false;
#pragma unroll
    for (int s = 0; s < S::count; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t byte = (x.vs[s][e >> 2] >> (8 * (e & 3))) & 255u;
            const bool out = t0 + e >= hi_all;
            nan |= !out && byte > 252u;
            if (out || byte > 252u) x.v[s][e] = 0;
            if (out) x.vs[s][e >> 2] &= ~(255u << (8 * (e & 3)));
        }
    if (!__any(nan)) return;
#pragma unroll
    for (int s = 0; s < S::count; ++s) {
        bf16x8 is;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool n = ((x.vs[s][e >> 2] >> (8 * (e & 3))) & 255u) > 252u;
            is[e] = n ? (__bf16)1.f : (__bf16)0.f;
            if (n) x.vs[s][e >> 2] &= ~(255u << (8 * (e & 3)));
        }
#pragma unroll
        for (int t = 0; t < NR; ++t) {
            bf16x8 seen;
#pragma unroll
            for (int e = 0; e < 8; ++e) seen[e] = t0 + e >= st.lo[t] && t0 + e < st.hi[t] ? (__bf16)1.f : (__bf16)0.f;
            const f32x4 n = __builtin_amdgcn_mfma_f32_16x16x32_bf16(is, seen, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
            for (int c = 0; c < S::size(s); ++c)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (n[r] > 0.f) st.o[t][S::tile(s) + c][r] = NAN;
        }
    }
}

// A block's part of the rows' results.
template <int W, int P, int NR>
__device__ __forceinline__ void attend_block(State<W, P, NR>& st, Block<W>& x, float scale, int blk, int i, int j, bool fresh,
                                             bool part, int hi_all) {
    using S = Segments<W>;
    const int t0 = blk * 32 + 8 * j;  // this lane's scores are of tokens t0 .. t0 + 7

    // scores: S^T = K Q^T
    f32x4 sc[NR][2];
#pragma unroll
    for (int t = 0; t < NR; ++t) sc[t][0] = sc[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const float e0 = scale_of<0>(x.ok ? x.ks[s][0] : 255u);
        const float e1 = W == 2 || W == 4 ? e0 : scale_of<0>(x.ok ? x.ks[s][1] : 255u);
#pragma unroll
        for (int c = 0; c < W; ++c) {
            const float e = W == 8 ? (c < 4 ? e0 : e1) : W == 2 || W == 4 ? e0 : ((W * j + c) >> 2) == ((W * j) >> 2) ? e0 : e1;
            const u32x4 f = {pair_of<0>(x.k[s][c], e), pair_of<1>(x.k[s][c], e), pair_of<2>(x.k[s][c], e),
                             pair_of<3>(x.k[s][c], e)};
            const bf16x8 kf = __builtin_bit_cast(bf16x8, f);
#pragma unroll
            for (int t = 0; t < NR; ++t)
#pragma unroll
                for (int p = 0; p < P; ++p)
                    sc[t][s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, st.q[t][p][c], sc[t][s], 0, 0, 0);
        }
    }

    // Softmax. A row's reference is the maximum of the first scores that it sees;
    // later scores are weighed by it as they come, without a look at their maximum
    // (weights above 1 cost no precision, only range: values of 2^107 / tokens and more
    // may overflow in the sum, as those of 2^128 / tokens would under weights up to 1),
    // until a lane's sum passes 2^20: then the block is weighed again by a higher one. fresh: a row may see its first scores
    // of the wave's here.
    bf16x8 pf[NR][P];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = sc[t][e >> 2][e & 3];
        if (part) {
            int at = t0;
            asm volatile("" : "+v"(at));  // (a branch: else the comparisons are made for every block)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (at + e < st.lo[t] || at + e >= st.hi[t]) p[e] = -INFINITY;
        }
        const auto top_of = [&] {
            const float top = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
            return max_over_j(top * scale);
        };
        const auto refer_to = [&](float to) {
            const float alpha = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(st.mx[t] - to);
            st.sum[t] *= alpha;
            st.norm[t] *= alpha;
#pragma unroll
            for (int c = 0; c < 2 * W; ++c) st.o[t][c] *= alpha;
            st.mx[t] = to;
        };
        if (fresh) refer_to(fmaxf(st.mx[t], top_of()));
        float w[8], before = st.sum[t];
        const auto weigh = [&] {
            const float base = st.mx[t] == -INFINITY ? 0.f : -st.mx[t];
            st.sum[t] = before;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                w[e] = __builtin_amdgcn_exp2f(fmaf(p[e], scale, base));
                st.sum[t] += w[e];
            }
        };
        weigh();
        if (__any(st.sum[t] > 0x1p20f)) {
            const float top = top_of();
            st.sum[t] = before;
            refer_to(max_over_j(before + w[0] + w[1] + w[2] + w[3] + w[4] + w[5] + w[6] + w[7]) > 0x1p20f ? fmaxf(st.mx[t] + 16.f, top) : st.mx[t]);
            before = st.sum[t];
            weigh();
        }
        pieces<P>(w, pf[t]);
        if constexpr (P == 1) st.norm[t] = plus_all(pf[t][0], st.norm[t]);
    }

    if (part) hide_values(st, x, t0, hi_all);

    // O^T += V^T P^T
#pragma unroll
    for (int s = 0; s < S::count; ++s) {
        const uint32_t a = x.vs[s][0], b = x.vs[s][1];
        const float e[8] = {scale_of<0>(a), scale_of<1>(a), scale_of<2>(a), scale_of<3>(a),
                            scale_of<0>(b), scale_of<1>(b), scale_of<2>(b), scale_of<3>(b)};
        uint32_t w[8];
#pragma unroll
        for (int n = 0; n < 8; ++n)
            w[n] = S::size(s) == 8 ? x.v[s][n] : S::size(s) == 4 ? x.v[s][n] >> (16 * (i & 1)) : x.v[s][n] >> (8 * (i & 3));
#pragma unroll
        for (int c = 0; c < S::size(s); c += 2) {
            u32x4 even, odd;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const uint32_t u = pair_at(c / 2, w[2 * n], e[2 * n]), v = pair_at(c / 2, w[2 * n + 1], e[2 * n + 1]);
                even[n] = __builtin_amdgcn_perm(v, u, 0x05040100u);
                odd[n] = __builtin_amdgcn_perm(v, u, 0x07060302u);
            }
            const bf16x8 ve = __builtin_bit_cast(bf16x8, even), vo = __builtin_bit_cast(bf16x8, odd);
            const int n = S::tile(s) + c;
#pragma unroll
            for (int t = 0; t < NR; ++t)
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    st.o[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ve, pf[t][p], st.o[t][n], 0, 0, 0);
                    st.o[t][n + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vo, pf[t][p], st.o[t][n + 1], 0, 0, 0);
                }
        }
    }
}

// New tokens that no workgroup takes: a sequence's past the bound on them, and those before
// the first offset or after the last, become NaN: the result, or the first split's sum,
// which makes the join do so. (Offsets that decrease miss none: on the way from token 0
// to the last one each is passed upwards, here or by a sequence.) One workgroup of each
// sequence and head does it.
template <bool F32, int D>
__device__ __forceinline__ void leave_rest(const AttnArgs& a, const Seq& q, uint32_t h, uint32_t b) {
    const int end = q.token + q.count;
    int t = b == 0 ? 0 : q.token;
    const int last = b + 1 == a.seqs.batch ? (int)a.seqs.total : end, taken = q.token + min(q.count, (int)a.seqs.each.value);
    if (__builtin_expect(t == q.token && taken == last, 1)) return;
#pragma unroll 1
    for (;; ++t) {
        if (t == q.token) t = taken;
        if (t >= last) break;
        const int64_t row = (int64_t)t * a.q_heads + (int64_t)h * a.group;
#pragma unroll 1
        for (uint32_t n = threadIdx.x; n < a.group * D; n += blockDim.x) {
            if (a.splits > 1) {
                if (n < a.group) a.part_stat[row + n] = f32x4{-INFINITY, NAN, NAN, 0.f};
                continue;
            }
            if (a.lse && n < a.group) a.lse[row + n] = NAN;
            if constexpr (F32)
                static_cast<float*>(a.out)[row * D + n] = NAN;
            else
                static_cast<uint16_t*>(a.out)[row * D + n] = 0x7fc0;
        }
    }
}

// W: dim / 32. P: bf16 pieces of the queries and weights (1: bf16, 3: fp32).
// NR: tiles of 16 query rows a wave. ROWS (fp32 prompts): the workgroup's waves
// take rows of their own and every token; else they share the rows and deal the
// tokens, so that few rows still fill a CU. Two waves a SIMD where 256 registers
// are enough, else one.
//
// What bounds it: reading the cache where that is long, 48 us for 32 uneven
// sequences of up to 8192 tokens, 8 cache heads of 128 and 4 queries each, and 32 us
// for one of 131072 and 8 queries: 4.5 TB/s, the vector units 45% busy decoding,
// the matrix cores 14%. Short contexts wait for the chain of lengths, page and codes:
// 5.2 us for 1021 tokens, 17 us for 8 of 4097 in pages of 16 with 5 rows (eight
// blocks a wave, one wave a SIMD). fp32 queries, 4 of 4097 and one head of 256: 9.9 us.
// Two tiles of heads of 256 take 22 registers (pages of 32 and more) or 42 in scratch.
template <int W, int P, int NR, bool ROWS, bool WIDE>
__global__ __launch_bounds__(64 * kAttnWaves, W * NR * (P + 1) <= 16 ? 2 : 1) void k_attend(const AttnArgs a) {
    using S = Segments<W>;
    constexpr int D = 32 * W, NT = D / 16;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, j = lane >> 4;
    const uint32_t h = blockIdx.x, b = blockIdx.z / a.splits, split = blockIdx.z % a.splits;

    const Seq q = seq_of(a.seqs, b);
    if (a.seqs.cu && split == 0 && blockIdx.y + 1 == a.row_blocks) leave_rest<P != 1, D>(a, q, h, b);
    const int rows = min(q.count, (int)a.seqs.each.value) * (int)a.group;
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
    constexpr int step = ROWS ? 1 : kAttnWaves;
    int blk = blk_first + (ROWS ? 0 : (int)wave);

    // Loads run ahead of their use: page numbers two blocks, a block's codes one.
    Block<W> x[2];
    Entry e[2] = {};
    if (blk < blk_end) {
        e[0] = entries<WIDE>(a, b, blk, i, j);
        e[1] = entries<WIDE>(a, b, blk + step, i, j);
    }

    State<W, P, NR> st;
    int64_t row_out[NR];  // (token, head) in the output, -1: no row
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        const int r = r0 + 16 * t + i;
        const bool ok = r < rows;
        const int m = ok ? r / (int)a.group : 0, g = ok ? r - m * (int)a.group : 0;
        st.hi[t] = ok ? hi_of(m) : 0;
        st.lo[t] = lo_of(m);
        const int64_t token = q.token + m, head = (int64_t)h * a.group + g;
        row_out[t] = ok ? token * a.q_heads + head : -1;  // (past the last row: the first one's queries, unused)
        const int64_t at = token * a.q_token + head * a.q_head + 8 * W * j;
#pragma unroll
        for (int c = 0; c < W; ++c) {
            if constexpr (P == 1) {
                u32x4 f;
                __builtin_memcpy(&f, static_cast<const uint16_t*>(a.q) + at + 8 * c, 16);
                st.q[t][0][c] = __builtin_bit_cast(bf16x8, f);
            } else {
                float f[8];
                __builtin_memcpy(f, static_cast<const float*>(a.q) + at + 8 * c, 32);
                bf16x8 split_f[P];
                pieces<P>(f, split_f);
#pragma unroll
                for (int p = 0; p < P; ++p) st.q[t][p][c] = split_f[p];
            }
        }
        st.mx[t] = -INFINITY;
        st.sum[t] = st.norm[t] = 0.f;
#pragma unroll
        for (int c = 0; c < NT; ++c) st.o[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    const auto work = [&](Block<W>& y) {
        const bool part = blk * 32 < full_lo || blk * 32 + 32 > full_hi;
        // (a row that sees nothing of the wave's block before this one sees it from full_lo at the latest)
        const bool fresh = blk < blk_first + step || (blk - step) * 32 < full_lo;
        attend_block(st, y, a.scale, blk, i, j, fresh, part, hi_all);
        blk += step;
    };
    if (blk < blk_end) {
        fetch<WIDE>(a, h, blk, e[0], i, j, x[0]);
        for (;;) {
            const bool more = blk + step < blk_end;
            if (more) {
                fetch<WIDE>(a, h, blk + step, e[1], i, j, x[1]);
                e[0] = entries<WIDE>(a, b, blk + 2 * step, i, j);
            }
            work(x[0]);
            if (!more) break;
            const bool again = blk + step < blk_end;
            if (again) {
                fetch<WIDE>(a, h, blk + step, e[0], i, j, x[0]);
                e[1] = entries<WIDE>(a, b, blk + 2 * step, i, j);
            }
            work(x[1]);
            if (!again) break;
        }
    }

#pragma unroll
    for (int t = 0; t < NR; ++t) {
        st.sum[t] = sum_over_j(st.sum[t]);
        st.norm[t] = P == 1 ? sum_over_j(st.norm[t]) : st.sum[t];
    }

    // the waves' results into wave 0's: 3 to 1 and 2 to 0, then 1 to 0
    if constexpr (!ROWS) {
        __shared__ float stat[kAttnWaves][NR][16][3];
        __shared__ f32x4 buf[2][NT][64];
        if (j == 0) {
#pragma unroll
            for (int t = 0; t < NR; ++t) {
                stat[wave][t][i][0] = st.mx[t];
                stat[wave][t][i][1] = st.sum[t];
                stat[wave][t][i][2] = st.norm[t];
            }
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < NR; ++t) {
            float top = -INFINITY, total = 0.f, norm = 0.f;
#pragma unroll
            for (int w = 0; w < kAttnWaves; ++w) top = fmaxf(top, stat[w][t][i][0]);
            const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int w = 0; w < kAttnWaves; ++w) {
                const float weight = __builtin_amdgcn_exp2f(stat[w][t][i][0] - base);
                total += stat[w][t][i][1] * weight;
                norm += stat[w][t][i][2] * weight;
            }
            const float own = __builtin_amdgcn_exp2f(st.mx[t] - base);
#pragma unroll
            for (int c = 0; c < NT; ++c) st.o[t][c] *= own;
            st.mx[t] = top;
            st.sum[t] = total;
            st.norm[t] = norm;
        }
#pragma unroll
        for (int t = 0; t < NR; ++t) {
            if (wave >= 2)
#pragma unroll
                for (int c = 0; c < NT; ++c) buf[wave - 2][c][lane] = st.o[t][c];
            __syncthreads();
            if (wave < 2)
#pragma unroll
                for (int c = 0; c < NT; ++c) st.o[t][c] += buf[wave][c][lane];
            if (wave == 1)
#pragma unroll
                for (int c = 0; c < NT; ++c) buf[1][c][lane] = st.o[t][c];
            __syncthreads();
            if (wave == 0)
#pragma unroll
                for (int c = 0; c < NT; ++c) st.o[t][c] += buf[1][c][lane];
            __syncthreads();
        }
        if (wave != 0) return;
    }

    const int64_t all = (int64_t)a.seqs.total * a.q_heads;
    const bool done = a.splits == 1;
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        if (row_out[t] < 0) continue;
        float sum = st.sum[t];
        if (st.hi[t] > cap) sum = NAN;  // it sees positions that the table has no page for
        const float inv = !done || st.norm[t] == 0.f ? 1.f : 1.f / st.norm[t];
        if (j == 0) {
            if (!done)
                a.part_stat[split * all + row_out[t]] = f32x4{st.mx[t], sum, st.norm[t], 0.f};
            else if (a.lse)
                a.lse[row_out[t]] = sum == 0.f ? -INFINITY : (st.mx[t] + __builtin_amdgcn_logf(sum)) * 0.693147180559945309f;
        }
#pragma unroll
        for (int s = 0; s < S::count; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int size = S::size(s), at = 8 * S::word(s) + size * (4 * j + r);
                float y[8];
#pragma unroll
                for (int c = 0; c < size; ++c) y[c] = done && sum != sum ? NAN : st.o[t][S::tile(s) + c][r] * inv;
                if (!done) {
                    float* to = a.part_o + (split * all + row_out[t]) * D + at;
#pragma unroll
                    for (int c = 0; c < size; ++c) to[c] = y[c];
                } else if constexpr (P == 1) {
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

// ------------------------------------------------------------------ prompts --
//
// Many rows to a cache head: a workgroup's waves, 32 rows each, decode every
// token once for all of them, a part each: codes to operands in LDS, 64 tokens
// a step. The products are v_mfma_f32_32x32x16_bf16's, transposed as above: lane
// (i, f), i = lane & 31, f = lane >> 5, owns row i and gets of a 32-token block
// the scores of tokens 16 m + 8 f .. + 7, m = 0, 1, which the second product
// wants there; operand row n of K is token
// 16 (n >> 4) + 8 (n >> 2 & 1) + 4 (n >> 3 & 1) + (n & 3).
//
// While a block's weights are taken (vector instructions) the next block's
// scores and the last one's products run on the matrix core, in one straight
// piece of code. So a step reads keys of blocks 2 s + 1 and 2 s + 2 and values of
// 2 s - 1 and 2 s: set s. Meanwhile set s + 1 is written, from codes loaded a
// step before.
//
// What bounds it: a prompt of 2048 tokens after 8192, 32 query and 8 cache heads of
// 128, takes 307 us, 1.01 PFLOP/s: the matrix cores are busy 47% and the vector
// units 45% of the time; a wave issues 38% of its life, waits 27% for a slot and
// 36% for LDS, loads and the barrier. Six prompts with a window of 512 and heads of 64,
// 41 us: nine steps of 1.3 us after a start of 6.

typedef float f32x16 __attribute__((ext_vector_type(16)));

// Waves of a workgroup: eight, two a SIMD, which share a decoded token among 256
// rows; four, one a SIMD with 512 registers a lane, for heads of 256. (Eight take 256
// registers, which heads of 192 exceed by 25 to 29, in scratch, and still gain.) TFLOP/s
// of a prompt of 1024 tokens in a context of 4096 with eight and with four: heads of 192
// 570 and 409, of 256 433 and 520; us of the prompt above, heads of 128: 305 and 350.
constexpr int prompt_waves(int W) { return W <= 6 ? 8 : 4; }

// Where leave_rest is done: by a block of rows more than there are, or, where its code costs
// the kernel's registers (heads of 96 and 192, 5% of a prompt), by a launch of its own.
constexpr bool rest_inside(int W) { return W != 3 && W != 6; }
template <int W>
__global__ __launch_bounds__(256) void k_attend_rest(const AttnArgs a) {
    leave_rest<false, 32 * W>(a, seq_of(a.seqs, blockIdx.y), blockIdx.x, blockIdx.y);
}

template <int W>
struct Set {
    static constexpr int frag = 1024;           // bytes of an operand: 16 a lane
    static constexpr int block = 2 * W * frag;  // of 32 tokens' keys (one per 16 channels) or values (one per 32 channels
                                                // and 16 tokens)
    static constexpr int bytes = 4 * block;     // two blocks of keys, two of values
    static constexpr int nan = 2 * bytes;       // two sets; then whether values of a set hold a NaN, by part
    static constexpr int lds = nan + 8 * (int)sizeof(int);
    static constexpr int raw = 10 * Segments<W>::count > W + 2 ? 10 * Segments<W>::count : W + 2;
};

// Part 0..7 of set s: 0..3 values, 4..7 keys; of the set's block part >> 1 & 1
// the half part & 1 of the channels (keys: of each lane's words).
__device__ __forceinline__ int part_block(int s, int part) { return 2 * s + (part >> 1 & 1) + (part < 4 ? -1 : 1); }

// The octet of its block that a lane's part concerns: its eight tokens' values or
// its token's key.
__device__ __forceinline__ int part_octet(int part, int lane) { return part < 4 ? lane >> 4 : 2 * (lane >> 4 & 1) + (lane >> 2 & 1); }

// (blocks before the first one count as that)
template <bool WIDE>
__device__ __forceinline__ uint32_t part_page(const AttnArgs& a, uint32_t b, int s, int part, int lane) {
    return page_of<WIDE>(a, b, max(part_block(s, part), 0), part_octet(part, lane));
}

template <bool WIDE, int W>
__device__ __forceinline__ void part_load(const AttnArgs& a, uint32_t h, int s, int part, int lane, uint32_t page,
                                          uint32_t (&raw)[Set<W>::raw]) {
    using S = Segments<W>;
    const Place p = place_of<WIDE>(a, h, page, max(part_block(s, part), 0), part_octet(part, lane));
    if (part < 4) {
        const int i = lane & 15;
        const uint32_t* codes = a.cache.v_codes + p.base * (4 * W);
        const uint8_t* scales = a.cache.v_scales + p.base * W;
#pragma unroll
        for (int n = 0; n < S::count; ++n) {
            const uint32_t w = S::word(n) + (i * 2 * S::size(n) >> 4);
            __builtin_memcpy(&raw[10 * n], codes + (p.in * (4 * W) + 8 * w), 32);
            __builtin_memcpy(&raw[10 * n + 8], __builtin_assume_aligned(scales + (p.in * W + 8 * (w >> 2)), 8), 8);
        }
    } else {
        const int j = 2 * (lane >> 5) + (part & 1);
        const uint32_t in = p.in + 4 * (lane >> 3 & 1) + (lane & 3);
        const int g0 = (W * j) >> 2, g1 = (W * j + W - 1) >> 2;
        const uint8_t* scales = a.cache.k_scales + p.base * W;
        __builtin_memcpy(&raw[0], a.cache.k_codes + p.base * (4 * W) + (in * (4 * W) + W * j), 4 * W);
        raw[W] = scales[in * W + g0];
        if (W != 2 && W != 4) raw[W + 1] = scales[in * W + g1];
        if (!p.ok) raw[W] = raw[W + 1] = 255;  // no page: NaN
    }
}

// Pairs [first, first + count) of a segment's values (even and odd channels) to
// their operands. Octet j = 2 m + f: lane slot 32 f of operand m; channels of
// both parities 16 lanes apart.
template <int W, int SEG, int FIRST, int COUNT>
__device__ __forceinline__ void write_values(char* to, int lane, const uint32_t (&raw)[Set<W>::raw]) {
    using S = Segments<W>;
    const int i = lane & 15, j = lane >> 4;
    const uint32_t a = raw[10 * SEG + 8], b = raw[10 * SEG + 9];
    const float e[8] = {scale_of<0>(a), scale_of<1>(a), scale_of<2>(a), scale_of<3>(a),
                        scale_of<0>(b), scale_of<1>(b), scale_of<2>(b), scale_of<3>(b)};
    to += (j >> 1) * Set<W>::frag + ((j & 1) * 32 + i) * 16;
    uint32_t w[8];
#pragma unroll
    for (int n = 0; n < 8; ++n)
        w[n] = S::size(SEG) == 8   ? raw[10 * SEG + n]
               : S::size(SEG) == 4 ? raw[10 * SEG + n] >> (16 * (i & 1))
                                   : raw[10 * SEG + n] >> (8 * (i & 3));
#pragma unroll
    for (int c = FIRST; c < FIRST + COUNT; ++c) {
        u32x4 even, odd;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const uint32_t u = pair_at(c, w[2 * n], e[2 * n]), v = pair_at(c, w[2 * n + 1], e[2 * n + 1]);
            even[n] = __builtin_amdgcn_perm(v, u, 0x05040100u);
            odd[n] = __builtin_amdgcn_perm(v, u, 0x07060302u);
        }
        char* tile = to + (S::tile(SEG) + 2 * c) * Set<W>::frag;
        *reinterpret_cast<u32x4*>(tile) = even;
        *reinterpret_cast<u32x4*>(tile + 256) = odd;
    }
}

template <int W, int HALF, int SEG = 0>
__device__ __forceinline__ void write_half(char* to, int lane, const uint32_t (&raw)[Set<W>::raw]) {
    if constexpr (SEG < Segments<W>::count) {
        constexpr int units = Segments<W>::size(SEG) / 2, some = units > 1 ? units / 2 : HALF;
        if constexpr (some > 0) write_values<W, SEG, (units > 1 ? HALF * some : 0), some>(to, lane, raw);
        write_half<W, HALF, SEG + 1>(to, lane, raw);
    }
}

// The loaded codes as operands in LDS. Values of no token (before the first or
// from `hi` on), and blocks that may hold a NaN or an infinity (hide_values), go as
// zeros; the set's flags say that there were some of the latter.
template <int W>
__device__ __forceinline__ void part_write(char* lds, int s, int part, int lane, int hi, uint32_t (&raw)[Set<W>::raw]) {
    using S = Segments<W>;
    using G = Set<W>;
    char* to = lds + (s & 1) * G::bytes + (part >> 1 & 1) * G::block;
    if (part >= 4) {
        const int j = 2 * (lane >> 5) + (part & 1);
        const float e0 = scale_of<0>(raw[W]), e1 = W == 2 || W == 4 ? e0 : scale_of<0>(raw[W + 1]);
        to += (part & 1) * W * G::frag + lane * 16;
#pragma unroll
        for (int c = 0; c < W; ++c) {
            const float e = W == 8 ? (c < 4 ? e0 : e1) : W == 2 || W == 4 ? e0 : ((W * j + c) >> 2) == ((W * j) >> 2) ? e0 : e1;
            const uint32_t w = raw[c];
            *reinterpret_cast<u32x4*>(to + c * G::frag) = u32x4{pair_of<0>(w, e), pair_of<1>(w, e), pair_of<2>(w, e), pair_of<3>(w, e)};
        }
        return;
    }
    const int block = part_block(s, part);
    const int t0 = block * 32 + 8 * (lane >> 4);
    if (block < 0 || block * 32 + 32 > hi) {
#pragma unroll
        for (int x = 0; x < S::count; ++x)
#pragma unroll
            for (int n = 0; n < 8; ++n)
                if (block < 0 || t0 + n >= hi) {
                    raw[10 * x + n] = 0;
                    raw[10 * x + 8 + (n >> 2)] &= ~(255u << (8 * (n & 3)));
                }
    }
    uint32_t all = 0;  // the top bit of each byte over 252
#pragma unroll
    for (int x = 0; x < S::count; ++x)
#pragma unroll
        for (int n = 8; n < 10; ++n) {
            const uint32_t y = raw[10 * x + n];
            all |= y & ((y & 0x7f7f7f7fu) + 0x03030303u) & 0x80808080u;
        }
    const bool any = __any(all != 0);
    if (any) {
#pragma unroll
        for (int x = 0; x < S::count; ++x)
#pragma unroll
            for (int n = 0; n < 8; ++n)
                if ((raw[10 * x + 8 + (n >> 2)] >> (8 * (n & 3)) & 255u) > 252u) {
                    raw[10 * x + n] = 0;
                    raw[10 * x + 8 + (n >> 2)] &= ~(255u << (8 * (n & 3)));
                }
    }
    if (lane == 0) reinterpret_cast<int*>(lds + G::nan)[4 * (s & 1) + part] = any;
    to += 2 * G::block;
    if (part & 1)
        write_half<W, 1>(to, lane, raw);
    else
        write_half<W, 0>(to, lane, raw);
}

// LSE: the unrounded weights are summed, too (without it their sum is not needed).
template <int W, bool WIDE, bool LSE>
__global__ __launch_bounds__(64 * prompt_waves(W), prompt_waves(W) / 4) void k_attend_prompt(const AttnArgs a) {
    using S = Segments<W>;
    using G = Set<W>;
    constexpr int D = 32 * W, waves = prompt_waves(W), parts = 8 / waves, half = waves / 2;
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 31, f = lane >> 5;
    const uint32_t h = blockIdx.x, b = blockIdx.z / a.splits, split = blockIdx.z % a.splits;

    const Seq q = seq_of(a.seqs, b);
    constexpr int unit = 32 * half;  // the rows of half of the waves
    const int rows = min(q.count, (int)a.seqs.each.value) * (int)a.group, units = (rows + unit - 1) / unit, y = blockIdx.y;
    if (2 * y >= units) {
        if constexpr (rest_inside(W))
            if (y == (int)a.row_blocks && split == 0) leave_rest<false, D>(a, q, h, b);
        return;
    }
    // Half of the waves take a unit of rows, half another: of a causal prompt the
    // one as far from its end as the first is from its start, so that workgroups
    // get alike, else the neighbour.
    const bool far = a.causal && !a.window;
    const int low = far ? y : 2 * y, high = far ? units - 1 - y : 2 * y + 1;
    const int first = (wave < half ? high : low) * unit + 32 * (wave % half);
    const int cap = a.seqs.cols << a.cache.page_shift;
    const auto hi_of = [&](int m) { return a.causal ? q.first + m + 1 : q.length; };
    const auto lo_of = [&](int m) { return a.window ? max(0, q.first + m + 1 - (int)a.window) : 0; };
    const auto new_of = [&](int r) { return r / (int)a.group; };
    // the steps of the workgroup, and what this wave's rows see of their tokens
    const int hi_all = min(hi_of(new_of(min(high * unit + unit, rows) - 1)), cap), lo_all = lo_of(new_of(low * unit));
    const int s_lo = lo_all >> 6, s_hi = hi_all > lo_all ? (hi_all + 63) >> 6 : s_lo;
    const int per = (s_hi - s_lo + (int)a.splits - 1) / (int)a.splits;
    const int s_first = s_lo + (int)split * per, s_end = min(s_first + per, s_hi);
    const bool some = first < rows && (wave < half || low != high);  // (an odd unit in the middle is the first waves')
    const int m0 = some ? new_of(first) : 0, m1 = some ? new_of(min(first + 32, rows) - 1) : 0;
    const int full_hi = some ? hi_of(m0) : 0, full_lo = lo_of(m1);  // every row sees what lies in between,
    const int see_hi = some ? min(hi_of(m1), cap) : 0, see_lo = lo_of(m0);  // and none what lies outside of these

    // Parts of the work on a set: values by four waves, keys by the other four (or
    // by the same). Values are written when a step begins and keys in its middle,
    // so that of a SIMD's two waves one has products to run meanwhile.
    const int vpart = wave & 3, kpart = 4 + (wave & 3);
    const bool does_v = wave < 4, does_k = waves == 4 || wave >= 4;
    uint32_t page[2], raw[parts][G::raw];
    uint32_t(&vraw)[G::raw] = raw[0];
    uint32_t(&kraw)[G::raw] = raw[parts - 1];
    const auto next_v = [&](int s) {  // loads set s, then the page numbers of the next
        part_load<WIDE, W>(a, h, s, vpart, lane, page[0], vraw);
        page[0] = part_page<WIDE>(a, b, s + 1, vpart, lane);
    };
    const auto next_k = [&](int s) {
        part_load<WIDE, W>(a, h, s, kpart, lane, page[1], kraw);
        page[1] = part_page<WIDE>(a, b, s + 1, kpart, lane);
    };
    const auto write_v = [&](int s) { part_write<W>(lds, s, vpart, lane, hi_all, vraw); };
    const auto write_k = [&](int s) { part_write<W>(lds, s, kpart, lane, hi_all, kraw); };
    uint32_t early[G::raw];  // keys of the set before the first: of its second block are the first scores
    if (s_first < s_end) {
        if (does_k) {
            const uint32_t p = part_page<WIDE>(a, b, s_first - 1, kpart, lane);
            page[1] = part_page<WIDE>(a, b, s_first, kpart, lane);
            part_load<WIDE, W>(a, h, s_first - 1, kpart, lane, p, early);
            next_k(s_first);
        }
        if (does_v) {
            page[0] = part_page<WIDE>(a, b, s_first, vpart, lane);
            next_v(s_first);
        }
    }

    const int r = first + i;
    const bool mine = some && r < rows;
    const int m = mine ? new_of(r) : 0, g = mine ? r - m * (int)a.group : 0;
    const int hi = mine ? hi_of(m) : 0, lo = lo_of(m);
    // (past the last row: the first one's queries, unused)
    const int64_t token = q.token + m, head = (int64_t)h * a.group + g, row_out = token * a.q_heads + head;
    bf16x8 qf[2 * W];
    {
        const uint16_t* at = static_cast<const uint16_t*>(a.q) + token * a.q_token + head * a.q_head + 16 * W * f;
#pragma unroll
        for (int c = 0; c < 2 * W; ++c) {
            u32x4 x;
            __builtin_memcpy(&x, at + 8 * c, 16);
            qf[c] = __builtin_bit_cast(bf16x8, x);
        }
    }
    float mx = -INFINITY, sum = 0.f, norm = 0.f;  // (the reference; the lane's share of the sums)
    f32x16 o[W], sc[2];
    bf16x8 pf[2];  // the last block's weights
#pragma unroll
    for (int c = 0; c < W; ++c) o[c] = f32x16{};
    pf[0] = pf[1] = __builtin_bit_cast(bf16x8, u32x4{0, 0, 0, 0});

    // a block's scores (keys k of a set), and the last block's products (values v)
    const auto score = [&](const char* from, f32x16& to) {
        to = f32x16{};
#pragma unroll
        for (int c = 0; c < 2 * W; ++c)
            to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(from + c * G::frag), qf[c], to, 0, 0, 0);
    };
    const auto add_up = [&](const char* from) {
        norm = plus_all(pf[1], plus_all(pf[0], norm));
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int c = 0; c < W; ++c)
                o[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(from + (2 * c + z) * G::frag), pf[z],
                                                               o[c], 0, 0, 0);
    };
    const auto keys = [&](int s, int n) { return lds + (s & 1) * G::bytes + n * G::block + lane * 16; };
    const auto values = [&](int s, int n) { return lds + (s & 1) * G::bytes + (2 + n) * G::block + lane * 16; };
    const auto top_of = [&](const f32x16& x) {
        float top = x[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, x[e]);
        top *= a.scale;
        const auto swap = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
        return fmaxf(__uint_as_float(swap[0]), __uint_as_float(swap[1]));
    };
    const auto refer_to = [&](float to) {
        const float alpha = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx - to);
        sum *= alpha;
        norm *= alpha;
#pragma unroll
        for (int c = 0; c < W; ++c) o[c] *= alpha;
        mx = to;
    };
    // Of block n's scores what a row does not see, and where rows may see their
    // first ones (in the first block, and up to the one after the last that begins
    // before full_lo) their references. Weights taken before (of the block whose
    // values are at `from`) go into the products first.
    const auto turn_to = [&](int n, f32x16& x, const char* from, bool start) {
        const bool part = n * 32 < full_lo || n * 32 + 32 > full_hi;
        if (part) {
            int t = n * 32 + 8 * f;
            asm volatile("" : "+v"(t));  // (a branch: else the comparisons are made for every block)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int at = t + 16 * (e >> 3) + (e & 7);
                if (at < lo || at >= hi) x[e] = -INFINITY;
            }
        }
        if (!start && (n - 1) * 32 >= full_lo) return;
        const float top = top_of(x);
        if (!__any(top > mx + 8.f)) return;
        asm volatile("" : "+v"(from));  // (else the operands are read ahead of the branch, for both sides)
        add_up(from);
        pf[0] = pf[1] = __builtin_bit_cast(bf16x8, u32x4{0, 0, 0, 0});
        refer_to(fmaxf(mx, top));
    };
    const auto weigh = [&](const f32x16& x) {  // -> the lane's largest weight
        const float base = mx == -INFINITY ? 0.f : -mx;
        float most = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float p = __builtin_amdgcn_exp2f(fmaf(x[e], a.scale, base));
            if constexpr (LSE) sum += p;
            most = fmaxf(most, p);
            pf[e >> 3][e & 7] = (__bf16)p;
        }
        asm volatile("" : "+v"(pf[0]), "+v"(pf[1]), "+v"(sum), "+v"(most));  // (here, beside the products, not where they are used)
        return most;
    };
    // block x's weights; the scores of the block after it, and the products of the one before
    // (later scores are weighed by a row's reference as they come, until a weight
    // passes 2^20: k_attend)
    const auto block = [&](f32x16& x, f32x16& next, const char* k, const char* v) {
        const float before = sum;
        norm = plus_all(pf[1], plus_all(pf[0], norm));
        next = f32x16{};
#pragma unroll
        for (int n = 0; n < 2 * W; ++n) {
            next = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(k + n * G::frag), qf[n], next, 0, 0, 0);
            const int c = n % W, z = n / W;
            o[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(v + (2 * c + z) * G::frag), pf[z], o[c], 0, 0, 0);
        }
        const float most = weigh(x);
        if (__any(most > 0x1p20f)) {
            const auto swap = __builtin_amdgcn_permlane32_swap(__float_as_uint(most), __float_as_uint(most), false, false);
            const bool over = fmaxf(__uint_as_float(swap[0]), __uint_as_float(swap[1])) > 0x1p20f;
            sum = before;
            refer_to(over ? fmaxf(mx, top_of(x)) : mx);
            weigh(x);
        }
    };
    // NaN blocks among a set's values: NaN in the rows that see one
    const auto mark_nan = [&](int s) {
        const int* nan = reinterpret_cast<const int*>(lds + G::nan) + 4 * (s & 1);
        if (!__builtin_amdgcn_readfirstlane(nan[0] | nan[1] | nan[2] | nan[3])) return;
#pragma unroll 1
        for (int n = 0; n < 4; ++n) {
            const int t = (2 * s - 1) * 32 + 16 * n + 8 * f;
            const Slot slot = slot_of(a.cache, a.seqs, b, h, (uint32_t)max(t, 0));
            bf16x8 seen;
#pragma unroll
            for (int x = 0; x < 8; ++x) seen[x] = t + x >= lo && t + x < hi ? (__bf16)1.f : (__bf16)0.f;
#pragma unroll
            for (int x = 0; x < S::count; ++x) {
                const int w = S::word(x) + ((i & 15) * 2 * S::size(x) >> 4);
                const uint8_t* e = a.cache.v_scales + slot.token * W + 8 * (w >> 2);
                bf16x8 is;
#pragma unroll
                for (int z = 0; z < 8; ++z) is[z] = e[z] > 252 && t + z < hi_all ? (__bf16)1.f : (__bf16)0.f;
                const f32x16 hit = __builtin_amdgcn_mfma_f32_32x32x16_bf16(is, seen, f32x16{}, 0, 0, 0);
#pragma unroll
                for (int c = 0; c < S::size(x) / 2; ++c)
#pragma unroll
                    for (int z = 0; z < 16; ++z)
                        if (hit[z] > 0.f) o[S::tile(x) / 2 + c][z] = NAN;
            }
        }
    };

    if (s_first < s_end) {
        if (does_k) {
            part_write<W>(lds, s_first - 1, kpart, lane, hi_all, early);
            write_k(s_first);
            next_k(s_first + 1);
        }
        if (does_v) {
            write_v(s_first);
            next_v(s_first + 1);
        }
        __syncthreads();
        score(keys(s_first - 1, 1), sc[0]);
        for (int s = s_first; s < s_end; ++s) {
            __syncthreads();  // (set s is written, and set s - 1 read)
            if (does_v) {
                write_v(s + 1);
                next_v(s + 2);
            }
            // (blocks 2 s - 1 .. 2 s + 2)
            const bool seen = 64 * s - 32 < see_hi && 64 * s + 96 > see_lo;
            if (seen) {
                mark_nan(s);
                turn_to(2 * s, sc[0], values(s, 0), s == s_first);
                block(sc[0], sc[1], keys(s, 0), values(s, 0));
            }
            if (does_k) {
                write_k(s + 1);
                next_k(s + 2);
            }
            if (seen) {
                turn_to(2 * s + 1, sc[1], values(s, 1), false);
                block(sc[1], sc[0], keys(s, 1), values(s, 1));
            }
        }
        __syncthreads();
        mark_nan(s_end);
        add_up(values(s_end, 0));
    }
    {
        const auto both = [](float x) {
            const auto swap = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
            return __uint_as_float(swap[0]) + __uint_as_float(swap[1]);
        };
        norm = both(norm);
        sum = LSE ? both(sum) : norm;
    }
    if (!mine) return;
    if (hi > cap) sum = NAN;  // it sees positions that the table has no page for
    const bool done = a.splits == 1;
    const int64_t at = done ? row_out : (int64_t)split * a.seqs.total * a.q_heads + row_out;
    const float inv = !done || norm == 0.f ? 1.f : 1.f / norm;
    if (f == 0) {
        if (!done)
            a.part_stat[at] = f32x4{mx, sum, norm, 0.f};
        else if (LSE)
            a.lse[at] = sum == 0.f ? -INFINITY : (mx + __builtin_amdgcn_logf(sum)) * 0.693147180559945309f;
    }
#pragma unroll
    for (int s = 0; s < S::count; ++s)
#pragma unroll
        for (int x = 0; x < 8; ++x) {  // operand row 8 (x >> 2) + 4 f + (x & 3), and 16 more for odd channels
            const int size = S::size(s), ch = 8 * S::word(s) + size * (8 * (x >> 2) + 4 * f + (x & 3));
            float v[8];
#pragma unroll
            for (int c = 0; c < size; ++c) {
                v[c] = o[S::tile(s) / 2 + c / 2][8 * (c & 1) + x] * inv;
                if (done && sum != sum) v[c] = NAN;
            }
            if (!done) {
#pragma unroll
                for (int c = 0; c < size; ++c) a.part_o[at * D + ch + c] = v[c];
            } else {
                uint16_t* to = static_cast<uint16_t*>(a.out) + at * D + ch;
#pragma unroll
                for (int c = 0; c < size; ++c) to[c] = __builtin_bit_cast(uint16_t, (__bf16)v[c]);
            }
        }
}

// The splits' results joined, in the order of the splits. A row is a wave's, or
// with `ways` 4 a workgroup's: lane n of a wave weighs split n (64 at most),
// then dim / 4 lanes add a split's row, 16 bytes a lane, as many splits at a
// time as lanes allow, and the partial sums meet at the end. Bound by its start
// and two dependent loads: 2.7 us for 32 rows of 8 splits, 4.8 for 1024 of 2, 5.4
// for 64 of 64 (heads of 128). The last workgroup's joining instead would need
// counters kept between calls.
template <bool F32>
__global__ __launch_bounds__(256) void k_attend_join(const AttnArgs a, int dim, int ways) {
    __shared__ f32x4 part[3][64];
    const int64_t all = (int64_t)a.seqs.total * a.q_heads;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = ways == 4 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
    if (row >= all) return;
    const int splits = (int)a.splits, per = dim / 4, groups = 64 / per;
    f32x4 stat = {-INFINITY, 0.f, 0.f, 0.f};
    if (lane < splits) stat = a.part_stat[lane * all + row];
    float top = stat[0];
#pragma unroll
    for (int n = 32; n; n >>= 1) top = fmaxf(top, __shfl_xor(top, n));
    const float weight = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(stat[0] - top);
    float total = stat[1] != stat[1] ? NAN : stat[1] * weight, norm = stat[2] * weight;
#pragma unroll
    for (int n = 32; n; n >>= 1) {
        total += __shfl_xor(total, n);
        norm += __shfl_xor(norm, n);
    }

    const int group = lane / per, col = lane - group * per;
    const int stride = groups * (ways == 4 ? 4 : 1);
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
    const f32x4* from = reinterpret_cast<const f32x4*>(a.part_o + row * dim) + (group < groups ? col : 0);
    // (no branch, so that loads go ahead of the weights: past the last split, and in
    // lanes past the last group, a row is read again with weight 0)
#pragma unroll 4
    for (int s0 = ways == 4 ? wave * groups : 0; s0 < splits; s0 += stride) {
        const int s = s0 + group;
        const bool in = group < groups && s < splits;
        const float w = __shfl(weight, s & 63);
        y += from[min(s, splits - 1) * (all * per)] * (in ? w : 0.f);
    }
    f32x4 sum = y;
    for (int g = 1; g < groups; ++g)
#pragma unroll
        for (int n = 0; n < 4; ++n) sum[n] += __shfl(y[n], (lane + g * per) & 63);
    if (ways == 4) {
        if (wave) part[wave - 1][lane] = sum;
        __syncthreads();
        if (wave) return;
        sum += part[0][lane] + part[1][lane] + part[2][lane];
    }
    const float inv = norm == 0.f ? 1.f : 1.f / norm;
    if (lane < per) {
        f32x4 v = sum * inv;
        if (total != total) v = f32x4{NAN, NAN, NAN, NAN};
        if constexpr (F32) {
            reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + row * dim)[lane] = v;
        } else {
            typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
            const bf16x4 r = __builtin_convertvector(v, bf16x4);
            reinterpret_cast<bf16x4*>(static_cast<uint16_t*>(a.out) + row * dim)[lane] = r;
        }
    }
    if (a.lse && lane == 0)
        a.lse[row] = total == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * 0.693147180559945309f;
}
