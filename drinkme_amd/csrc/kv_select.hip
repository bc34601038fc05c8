// Summaries of the 4-bit cache's pages, and the pages that a cheap score selects
// for each query (include/dmx_kv.h).
//
//   k_summarize          the bounds of the keys in a page
//   k_select, k_choose   scores of a token's pages, and the best of them
//   k_select_tokens      the same for a prompt's tokens together
#include "kv_common.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// --------------------------------------------------------------- summaries --
//
// Every channel's largest and smallest key of a page bound its product with any
// query there. They are exact (a code times its power of two is an fp32 number,
// and neither depends on an order), and rounded outwards to 8 bits.
//
// Waits bound it: lengths, page number, the look for a shared page, codes, then three barriers: 4.75 us for the last
// pages of 32 sequences (8 heads of 128, 64 tokens a page), 9.3 for the 16 of a chunk of 1024 tokens, 107 for the
// 8192 pages of 16 of a prompt, from a graph.

struct Summarize {
    Cache cache;
    Seqs seqs;
    int8_t* bounds;
    uint8_t* scales;
    uint32_t run;  // new tokens a workgroup looks at, 64 at most
    uint32_t team;  // 2^team lanes look through a sequence's columns (fuller_elsewhere)
};

// A page that several of the sequences have, or one has twice, is written by who holds most tokens there: those
// bounds hold for the others', too, and equal numbers write equal bytes; of different ones the bytes could mix.
// Looking for them takes 0.4 us of a step, 4 to 8 of 4 to 64 prompts' (their last workgroups'), 1 of 1024 sequences',
// 15 of 4096's.
// -> The bits of `partial` (lanes whose page, number `number`, holds less than it may: `tokens`) that a lane
// finds to hold more somewhere else.
__device__ __forceinline__ uint64_t fuller_elsewhere(const Summarize& a, uint64_t partial, int tokens, int number) {
    const int shift = a.cache.page_shift;
    uint64_t out = 0;
    for (uint32_t b0 = 0; b0 < a.seqs.batch; b0 += 256u >> a.team) {  // (loops of whole waves: readlane reads every lane)
        const uint32_t b = b0 + (threadIdx.x >> a.team);
        const Seq q = seq_of(a.seqs, min(b, a.seqs.batch - 1));
        const int end = b < a.seqs.batch && q.count && q.length ? min(((q.length - 1) >> shift) + 1, a.seqs.cols) : 0;
        int col = (max(q.first, 0) >> shift) + (int)(threadIdx.x & ((1u << a.team) - 1));
        for (; __any(col < end); col += 1 << a.team) {
            const int page = col < end ? a.seqs.table[(int64_t)b * a.seqs.cols + col] : -1;
            for (uint64_t m = partial; m; m &= m - 1) {
                const int l = __builtin_ctzll(m), count = __builtin_amdgcn_readlane(tokens, l);
                // (where offsets decrease, the token that would find the column may be another sequence's)
                if (page == __builtin_amdgcn_readlane(number, l) && min(1 << shift, q.length - (col << shift)) > count &&
                    seq_at(a.seqs, q.token + max((col << shift) - q.first, 0)) == b)
                    out |= 1ull << l;
            }
        }
    }
    return out;
}

// A workgroup takes a head of the pages that begin among its new tokens (or in
// which their sequence's first one lies), one after the other: a lane finds a token's, then a thread
// takes a word of eight channels, of every 256 / words-th token, then a channel.
// (eight workgroups a CU: a prompt of 8192 pages takes 114 us with the seven that more registers leave)
template <int D>
__global__ __launch_bounds__(256, 8) void k_summarize(const Summarize a) {
    constexpr int words = D / 8, groups = 256 / words;
    __shared__ float part[groups][2][D];
    __shared__ float tops[4];
    __shared__ uint64_t fuller[4];
    const int x = threadIdx.x, w = x % words, g = x / words;
    const uint32_t h = blockIdx.y, heads = a.cache.heads, shift = a.cache.page_shift;
    const uint32_t t = blockIdx.x * a.run + (x & 63);
    int start = -1, tokens = 0, number = 0;  // a page's first position, how many tokens it holds, which it is
    if ((uint32_t)(x & 63) < a.run && t < a.seqs.total) {
        int p;
        const Slot at = slot_of_new(a.cache, a.seqs, t, p);
        const uint32_t b = seq_at(a.seqs, t);
        const Seq q = seq_of(a.seqs, b);
        const int in = p & ((1 << shift) - 1);
        if (at.ok && (!in || (int)t == q.token)) {  // (the first of its page, or of its sequence's new ones)
            start = p - in;
            tokens = min(1 << shift, q.length - start);
            number = a.seqs.table[(int64_t)b * a.seqs.cols + (p >> shift)];
        }
    }
    const uint64_t partial = __ballot(start >= 0 && tokens < 1 << shift);
    if (partial) {
        uint64_t elsewhere = fuller_elsewhere(a, partial, tokens, number);
        if (__any(elsewhere != 0)) {  // (rare: the lanes' bits together)
#pragma unroll
            for (int n = 32; n; n >>= 1) elsewhere |= __shfl_xor(elsewhere, n);
        }
        if ((x & 63) == 0) fuller[x >> 6] = elsewhere;  // (read behind the first page's barrier)
    }
    for (uint64_t found = __ballot(start >= 0); found; found &= found - 1) {
        const int l = __builtin_ctzll(found), count = __builtin_amdgcn_readlane(tokens, l);
        const uint64_t page = (uint32_t)__builtin_amdgcn_readlane(number, l);
        const uint64_t first = (page * heads + h) << shift;
        float hi[8], lo[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) hi[n] = -INFINITY, lo[n] = INFINITY;
        if (g < groups) {
#pragma unroll 4
            for (int m = g; m < count; m += groups) {
                const uint32_t e = a.cache.k_scales[(first + m) * (D / 32) + w / 4];
                const uint32_t word = a.cache.k_codes[(first + m) * words + w];
                const float once = e > 252 ? NAN : 1.f;  // (which a maximum passes over; no branch, so that loads go ahead)
                const float unit = __uint_as_float(e << 23);
                const f32x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, unit, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, unit, 1),
                                    __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, unit, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, unit, 3)};
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    hi[n] = fmaxf(hi[n], v[n / 2][n & 1] * once);
                    lo[n] = fminf(lo[n], v[n / 2][n & 1] * once);
                }
            }
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                part[g][0][8 * w + n] = hi[n];
                part[g][1][8 * w + n] = lo[n];
            }
        }
        __syncthreads();
        if (partial >> l & 1 && (fuller[0] | fuller[1] | fuller[2] | fuller[3]) >> l & 1) continue;
        float most = -INFINITY, least = INFINITY;
        if (x < D) {
#pragma unroll
            for (int n = 0; n < groups; ++n) {
                most = fmaxf(most, part[n][0][x]);
                least = fminf(least, part[n][1][x]);
            }
        }
        if (most == -INFINITY) most = least = 0.f;  // no number there
        float top = fmaxf(fabsf(most), fabsf(least));
#pragma unroll
        for (int n = 32; n; n >>= 1) top = fmaxf(top, __shfl_xor(top, n));
        if ((x & 63) == 0) tops[x >> 6] = top;
        __syncthreads();
        top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        // 127 / 64 and less of a power of two: 127 of its 64th; above, of its 32nd
        const int e = max((int)((__float_as_uint(top) + 0x1ffffu) >> 23) - 133, -126);
        const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
        if (x < D) {
            int8_t* to = a.bounds + (page * heads + h) * (2 * D) + x;
            // (a quotient may vanish: what is above 0 rounds up to 1 all the same)
            to[0] = (int8_t)(most > 0.f ? fmaxf(ceilf(most * inv), 1.f) : ceilf(most * inv));
            to[D] = (int8_t)(least < 0.f ? fminf(floorf(least * inv), -1.f) : floorf(least * inv));
        }
        if (x == 0) a.scales[page * heads + h] = (uint8_t)(e + 127);
        __syncthreads();
    }
}

// --------------------------------------------------------------- selection --
//
// The score of a page is a product of two vectors of 2 D whole numbers of 8
// bits: the query's positive and negative parts against the page's largest and
// smallest keys. On v_mfma_i32_16x16x64_i8 16 pages meet 16 query rows, in
// whole numbers, which no order of summation changes: ties are ties, and go
// to the lower column whatever computes them.
//
// The best `count` keys (a score's bits, ordered as numbers) are those from a
// threshold on, the largest that `count` keys reach: found from the bits that all share
// downwards, by counting, one bit at a time in a wave's registers or eight in a
// workgroup's histogram.

struct Select {
    Cache cache;  // (page numbers and sizes alone)
    Seqs seqs;
    const int8_t* bounds;
    const uint8_t* scales;
    const void* q;
    int64_t q_token, q_head;  // strides, elements
    uint32_t group, count, first, last, causal;
    int32_t* blocks;
    uint32_t tokens, slots, stride;  // k_select_tokens: tokens a workgroup, rows a token, keys a token
    uint32_t* keys;  // k_select's SPLIT: [heads, total, columns]
    uint32_t tiles;  // of a workgroup there
};

constexpr uint32_t kForced = 0xffffffffu, kLost = 1;  // keys above and below every score's; 0: no column

__device__ __forceinline__ uint32_t key_of(int score, int scale) {
    const uint32_t bits = __float_as_uint(__builtin_ldexpf((float)score, scale - 127));
    return bits ^ (bits >> 31 ? 0xffffffffu : 0x80000000u);
}

// Sixteen adjacent channels as fp32, 0 for what is no number.
template <bool F32>
__device__ __forceinline__ void load16(const void* base, int64_t at, float (&x)[16]) {
    if constexpr (F32) {
        __builtin_memcpy(x, static_cast<const float*>(base) + at, 64);
    } else {
        uint32_t w[8];
        __builtin_memcpy(w, static_cast<const uint16_t*>(base) + at, 32);
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            x[2 * n] = __uint_as_float(w[n] << 16);
            x[2 * n + 1] = __uint_as_float(w[n] & 0xffff0000u);
        }
    }
#pragma unroll
    for (int n = 0; n < 16; ++n) x[n] = (__float_as_uint(x[n]) & 0x7fffffffu) >= 0x7f800000u ? 0.f : x[n];
}

// Piece c of lane (i, j)'s share of a row: 16 channels, of the positive side's D / 16
// pieces and then of the negative one's.
template <int D>
struct Piece {
    bool negative;
    int channel;
    __device__ __forceinline__ Piece(int c, int j) : negative(4 * c + j >= D / 16), channel(16 * (4 * c + j - (negative ? D / 16 : 0))) {}
};

__device__ __forceinline__ uint32_t largest(const float (&x)[16], uint32_t top) {
#pragma unroll
    for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
    return top;
}

// The factor of whole numbers: 255 / 128 of a power of two and above round to 128 of
// its 64th, and take its 32nd.
__device__ __forceinline__ float factor_of(uint32_t top) {
    return __uint_as_float((uint32_t)(127 - max((int)((top + 0x10000u) >> 23) - 133, -126)) << 23);
}

__device__ __forceinline__ i32x4 whole(const float (&x)[16], float factor, bool negative) {
    i32x4 out;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        uint32_t word = 0;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const int v = (int)rintf(x[4 * w + y] * factor);
            word |= (uint32_t)((negative ? min(v, 0) : max(v, 0)) & 255) << (8 * y);
        }
        out[w] = (int)word;
    }
    return out;
}

// What a lane reads of a tile of 16 pages: page i's pieces, and its scale.
template <int D>
struct PageTile {
    i32x4 bounds[D / 32];
    int scale;
    bool ok;
};
template <int D>
__device__ __forceinline__ void load_tile(const Select& a, uint32_t h, uint32_t page, int j, PageTile<D>& x) {
    x.ok = page < a.cache.pages;
    const uint64_t at = (uint64_t)(x.ok ? page : 0u) * a.cache.heads + h;
    const i32x4* from = reinterpret_cast<const i32x4*>(a.bounds + at * (2 * D) + 16 * j);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) x.bounds[c] = from[4 * c];
    x.scale = a.scales[at];
}

// The largest (MAX) or smallest over a wave, in every lane of it.
template <bool MAX>
__device__ __forceinline__ uint32_t over_lanes(uint32_t x) {
    const auto of = [](uint32_t a, uint32_t b) { return MAX ? max(a, b) : min(a, b); };
    x = of(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xF, 0xF, true));
    x = of(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xF, 0xF, true));
    x = of(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xF, 0xF, true));
    x = of(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x140, 0xF, 0xF, true));
    auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = of(r[0], r[1]);
    r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return __builtin_amdgcn_readfirstlane(of(r[0], r[1]));
}

// A wave's choice: the count largest of keys [0, n) in LDS (more than count of them, 64 R
// at most), ties to the first, their indexes to `out` in ascending order.
template <int R>
__device__ __forceinline__ void choose(const uint32_t* keys, int n, int count, int lane, int32_t* out) {
    uint32_t key[R];
#pragma unroll
    for (int x = 0; x < R; ++x) key[x] = 64 * x + lane < n ? keys[64 * x + lane] : 0;
    // What all scores begin with, the threshold does: of 18 rounds or so that leaves ten.
    uint32_t most = 0, least = ~0u;
#pragma unroll
    for (int x = 0; x < R; ++x) {
        most = max(most, key[x] == kForced ? 0 : key[x]);
        least = min(least, key[x] ? key[x] : ~0u);
    }
    most = over_lanes<true>(most);
    least = over_lanes<false>(least);
    const uint32_t differ = most ^ min(least, most);
    uint32_t bit = differ ? 1u << (31 - __clz(differ)) : 0, at_least = bit ? most & ~(2 * bit - 1) : most;
    for (; bit; bit >>= 1) {
        const uint32_t to = at_least | bit;
        int have = 0;
#pragma unroll
        for (int x = 0; x < R; ++x) have += __popcll(__ballot(key[x] >= to));
        if (have >= count) at_least = to;
        if (have == count) break;
    }
    int above = 0;
#pragma unroll
    for (int x = 0; x < R; ++x) above += __popcll(__ballot(key[x] > at_least));
    const int fill = count - above;  // (of those at the threshold)
    int over = 0, level = 0;
#pragma unroll
    for (int x = 0; x < R; ++x) {
        const bool up = key[x] > at_least, even = key[x] == at_least;
        const uint64_t u = __ballot(up), v = __ballot(even);
        const int o = over + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(u >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)u, 0));
        const int l = level + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(v >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)v, 0));
        if (up || (even && l < fill)) out[o + min(l, fill)] = 64 * x + lane;
        over += __popcll(u);
        level += __popcll(v);
    }
}

// As choose, by a workgroup of WAVES waves, a run of keys each: eight bits of the threshold at a
// time, by a histogram of the keys that share the bits above.
template <int WAVES>
__device__ __forceinline__ void choose_together(const uint32_t* keys, int n, int count, int32_t* out) {
    __shared__ int bins[256], before[2][WAVES], found[2];
    __shared__ uint32_t ends[2][WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rows = (n + 64 * WAVES - 1) / (64 * WAVES), c0 = wave * rows * 64 + lane;
    const auto key_at = [&](int x) { return c0 + 64 * x < n ? keys[c0 + 64 * x] : 0u; };
    uint32_t most = 0, least = ~0u;
    int forced = 0;
    for (int x = 0; x < rows; ++x) {
        const uint32_t key = key_at(x);
        most = max(most, key == kForced ? 0 : key);
        least = min(least, key ? key : ~0u);
        forced += __popcll(__ballot(key == kForced));
    }
    most = over_lanes<true>(most);
    least = over_lanes<false>(least);
    if (lane == 0) ends[0][wave] = most, ends[1][wave] = least, before[0][wave] = forced;
    __syncthreads();
    int need = count;  // of the keys that share the threshold's bits so far
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        most = max(most, ends[0][w]);
        least = min(least, ends[1][w]);
        need -= before[0][w];
    }
    const uint32_t differ = most ^ min(least, most);
    int top = differ ? 31 - __clz(differ) : -1;  // the highest bit not yet known
    uint32_t at_least = top < 0 ? most : top == 31 ? 0 : most & ~((2u << top) - 1);
    while (top >= 0 && need > 0) {
        const int low = max(top - 7, 0);
        for (int c = threadIdx.x; c < 256; c += 64 * WAVES) bins[c] = 0;
        __syncthreads();
        for (int x = 0; x < rows; ++x) {
            const uint32_t key = key_at(x), apart = key ^ at_least;
            if (key && key != kForced && (top == 31 || apart >> (top + 1) == 0)) atomicAdd(&bins[(key >> low) & 255 & ((2u << (top - low)) - 1)], 1);
        }
        __syncthreads();
        if (wave == 0) {  // lane l: bins 4 l .. 4 l + 3; those above them, from the highest down
            int mine[4], sum = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += mine[e] = bins[4 * lane + e];
            int upto = sum;  // with the lanes above
#pragma unroll
            for (int m = 1; m < 64; m *= 2) {
                const int y = __shfl_down(upto, m);
                if (lane + m < 64) upto += y;
            }
            int over = upto - sum;
#pragma unroll
            for (int e = 3; e >= 0; --e) {
                if (over < need && over + mine[e] >= need) found[0] = 4 * lane + e, found[1] = over;
                over += mine[e];
            }
        }
        __syncthreads();
        const int bin = found[0];
        need -= found[1];
        at_least |= (uint32_t)bin << low;
        if (bins[bin] == need) break;  // (all of them)
        top = low - 1;
        __syncthreads();
    }
    if (need <= 0) at_least = kForced;  // (forced ones alone)
    int above = 0, equal = 0;
    for (int x = 0; x < rows; ++x) {
        const uint32_t key = key_at(x);
        above += __popcll(__ballot(key > at_least));
        equal += __popcll(__ballot(key == at_least));
    }
    __syncthreads();
    if (lane == 0) before[0][wave] = above, before[1][wave] = equal;
    __syncthreads();
    int fill = count, over = 0, level = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        fill -= before[0][w];
        over += w < wave ? before[0][w] : 0;
        level += w < wave ? before[1][w] : 0;
    }
    for (int x = 0; x < rows; ++x) {
        const uint32_t key = key_at(x);
        const bool up = key > at_least, even = key == at_least;
        const uint64_t u = __ballot(up), v = __ballot(even);
        const int o = over + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(u >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)u, 0));
        const int l = level + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(v >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)v, 0));
        if (up || (even && l < fill)) out[o + min(l, fill)] = c0 + 64 * x;
        over += __popcll(u);
        level += __popcll(v);
    }
}

// The same for as few keys as a wave takes, by the workgroup's first.
template <int WAVES>
__device__ __forceinline__ void choose_any(const uint32_t* keys, int n, int count, int32_t* out) {
    const int lane = threadIdx.x & 63;
    if (n > 1024) {
        choose_together<WAVES>(keys, n, count, out);
    } else if (threadIdx.x < 64) {
        n <= 128   ? choose<2>(keys, n, count, lane, out)
        : n <= 256 ? choose<4>(keys, n, count, lane, out)
        : n <= 512 ? choose<8>(keys, n, count, lane, out)
                   : choose<16>(keys, n, count, lane, out);
    }
}

// The largest of each of x over `slots` neighbouring lanes, a power of two up to 16: in every one of them.
template <int DPP, int N>
__device__ __forceinline__ void max_with(int (&x)[N]) {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = max(x[e], __builtin_amdgcn_mov_dpp(x[e], DPP, 0xF, 0xF, true));
}
template <int N>
__device__ __forceinline__ void max_over_slots(int (&x)[N], uint32_t slots) {
    if (slots > 1) max_with<0xB1>(x);   // lane ^ 1
    if (slots > 2) max_with<0x4E>(x);   // lane ^ 2
    if (slots > 4) max_with<0x141>(x);  // the other four of eight
    if (slots > 8) max_with<0x140>(x);  // the other eight
}

// The columns that token t sees, and its sequence.
__device__ __forceinline__ int columns_seen(const Select& a, uint32_t t, uint32_t& b) {
    b = seq_at(a.seqs, t);
    const Seq q = seq_of(a.seqs, b);
    const int m = (int)t - q.token, p = a.causal ? q.first + m : q.length - 1;
    const bool inside = (uint32_t)m < (uint32_t)q.count && q.first + m >= 0;
    return inside ? min((p >> a.cache.page_shift) + 1, a.seqs.cols) : 0;
}

// Fewer columns than are asked for: all of them.
__device__ __forceinline__ void list_all(int32_t* out, int n, int count) {
    for (int c = threadIdx.x; c < count; c += blockDim.x) out[c] = c < n ? c : -1;
}

// Single tokens: a workgroup to a token and head. A wave takes tiles of 16 pages, the next
// one's loads ahead of this one's product. SPLIT: a run of tiles to a workgroup, the keys go to
// the workspace, and k_choose chooses.
//
// Waits bound it: lengths, page numbers, summaries in turn, then the choice. One token over 128 pages 6.6
// us, 32 uneven sequences of up to 256 pages 8.3 (12.5 MB, 2.6 us at a copy's rate), eight heads of 128 each, in a
// graph; 7.2 and 10 as launches alone.
template <bool F32, int D, int WAVES, bool SPLIT>
__global__ __launch_bounds__(64 * WAVES) void k_select(const Select a) {
    constexpr int chunks = D / 32;
    extern __shared__ __align__(16) uint32_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, j = lane >> 4;
    // (neighbours, which different XCDs run, are tokens: a head's summaries alone would meet in two of an L2's 16 channels)
    const uint32_t heads = a.cache.heads, h = blockIdx.y, t = blockIdx.x;
    int32_t* out = a.blocks + ((int64_t)t * heads + h) * a.count;
    uint32_t* const keys = SPLIT ? a.keys + ((int64_t)h * a.seqs.total + t) * a.seqs.cols : lds;

    uint32_t b;
    const int n = columns_seen(a, t, b), count = a.count;
    if (n <= count) {
        if (!SPLIT) list_all(out, n, count);
        return;
    }
    const int first = SPLIT ? blockIdx.z * a.tiles : 0, tiles = SPLIT ? min(first + (int)a.tiles, (n + 15) / 16) : (n + 15) / 16;
    if (SPLIT && first >= tiles) return;
    const auto page_at = [&](int tile) { return (uint32_t)a.seqs.table[(int64_t)b * a.seqs.cols + min(16 * tile + i, n - 1)]; };
    const auto load = [&](int r, int c, float (&x)[16]) {  // of query head r of the group
        load16<F32>(a.q, t * a.q_token + ((int64_t)h * a.group + r) * a.q_head + Piece<D>(c, j).channel, x);
    };
    for (uint32_t r0 = 0; r0 < a.group; r0 += 16) {
        PageTile<D> x[2];
        uint32_t page = page_at(min(first + wave, tiles - 1));
        uint32_t top = 0;
        for (uint32_t r = i; r < a.group; r += 16)
#pragma unroll
            for (int c = 0; c < chunks; ++c) {
                float y[16];
                load(r, c, y);
                top = largest(y, top);
            }
        load_tile(a, h, page, j, x[0]);
        page = page_at(min(first + wave + WAVES, tiles - 1));
#pragma unroll
        for (int s = 32; s; s >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, s));
        const float factor = factor_of(top);
        const uint32_t r = r0 + i;
        i32x4 qf[chunks];
#pragma unroll
        for (int c = 0; c < chunks; ++c) {
            float y[16] = {};
            if (r < a.group) load(r, c, y);
            qf[c] = whole(y, factor, Piece<D>(c, j).negative);
        }
        const auto work = [&](int tile, const PageTile<D>& y) {
            i32x4 s = {0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < chunks; ++c) s = __builtin_amdgcn_mfma_i32_16x16x64_i8(y.bounds[c], qf[c], s, 0, 0, 0);
            int v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = r < a.group ? s[e] : -(1 << 30);
            max_over_slots(v, 16);
            const int best = i & 2 ? (i & 1 ? v[3] : v[2]) : (i & 1 ? v[1] : v[0]);  // of page 4 j + (i & 3)
            const int c = 16 * tile + i;
            if (i >> 2 == j && c < n) {
                uint32_t key = y.ok ? key_of(best, y.scale) : kLost;
                if (c < (int)a.first || c >= n - (int)a.last) key = kForced;
                keys[c] = r0 ? max(keys[c], key) : key;
            }
        };
        for (int tile = first + wave; tile < tiles; tile += 2 * WAVES) {
            load_tile(a, h, page, j, x[1]);  // (past the last tile: the last page again)
            page = page_at(min(tile + 2 * WAVES, tiles - 1));
            work(tile, x[0]);
            if (tile + WAVES >= tiles) break;
            load_tile(a, h, page, j, x[0]);
            page = page_at(min(tile + 3 * WAVES, tiles - 1));
            work(tile + WAVES, x[1]);
        }
    }
    if constexpr (!SPLIT) {
        __syncthreads();
        choose_any<WAVES>(keys, n, count, out);
    }
}

__global__ __launch_bounds__(1024) void k_choose(const Select a) {
    extern __shared__ __align__(16) uint32_t lds[];
    const uint32_t h = blockIdx.y, t = blockIdx.x;
    int32_t* out = a.blocks + ((int64_t)t * a.cache.heads + h) * a.count;
    uint32_t b;
    const int n = columns_seen(a, t, b), count = a.count;
    if (n <= count) {
        list_all(out, n, count);
        return;
    }
    const uint32_t* from = a.keys + ((int64_t)h * a.seqs.total + t) * a.seqs.cols;
    for (int c = threadIdx.x; c < n; c += 1024) lds[c] = from[c];
    __syncthreads();
    choose_any<16>(lds, n, count, out);
}

// Prompts: a workgroup to a head and up to 16 tokens in a row, which share the reading of
// their sequence's summaries: 64 query rows (`slots` to a token, a power of two), four tiles that a wave
// each made whole numbers of, meet a tile of pages. Then the waves choose for the tokens in turn.
//
// 1024 tokens of 32 query and 8 cache heads of 128 over 512 pages: 33 us in a graph, 36 as a launch alone, of which the
// products and their keys take 6, the choices 14, queries and starts the rest; a workgroup to each token 158, eight waves
// in 128 registers, some of them in scratch, 44, two tiles of rows 42. 141 to 151 scalar registers live in
// vector registers' lanes (the choices of five sizes are all in here), and with heads of 256 ten vector registers in 44
// bytes of scratch. A table of 2048 columns takes 43 us and one of 4096 61 for the same pages: fewer tokens' keys fit.
constexpr int kSelectWaves = 4;
template <bool F32, int D>
__global__ __launch_bounds__(64 * kSelectWaves, 2) void k_select_tokens(const Select a) {
    constexpr int chunks = D / 32, WAVES = kSelectWaves;
    extern __shared__ __align__(16) uint32_t keys[];  // [tokens][stride]; before them, there, the queries: [4][chunks][64]
    i32x4* const rows = reinterpret_cast<i32x4*>(keys);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, j = lane >> 4;
    const uint32_t heads = a.cache.heads, h = blockIdx.y, slot = i & (a.slots - 1), per = 16 / a.slots;  // tokens a tile of rows
    const int shift = a.cache.page_shift, count = a.count, row_tiles = (int)((a.tokens * a.slots + 15) / 16);
    const int t_end = (int)min(blockIdx.x * a.tokens + a.tokens, a.seqs.total);
    int t0 = (int)(blockIdx.x * a.tokens);
    while (t0 < t_end) {  // (a turn for each sequence)
        const uint32_t b = seq_at(a.seqs, t0);
        const Seq q = seq_of(a.seqs, b);
        const bool inside = (uint32_t)(t0 - q.token) < (uint32_t)q.count;
        const int t1 = inside ? min(t_end, q.token + q.count) : t0 + 1, first = t0;
        t0 = t1;
        const auto columns_of = [&](int t) {  // that token t sees
            const int at = q.first + (t - q.token), p = a.causal ? at : q.length - 1;
            return inside && at >= 0 ? min((p >> shift) + 1, a.seqs.cols) : 0;
        };
        const int most = columns_of(t1 - 1);
        if (most > count) {
            const int tiles = (most + 15) / 16;
            const auto page_at = [&](int tile) { return (uint32_t)a.seqs.table[(int64_t)b * a.seqs.cols + min(16 * tile + i, most - 1)]; };
            uint32_t page = page_at(min(wave, tiles - 1));
            if (wave < row_tiles) {
                const uint32_t token = first + wave * per + i / a.slots;
                const bool mine = (int)token < t1 && slot < a.group;
                float y[chunks][16] = {};
                uint32_t top = 0;
                if (mine)
#pragma unroll
                    for (int c = 0; c < chunks; ++c) {
                        load16<F32>(a.q, token * a.q_token + ((int64_t)h * a.group + slot) * a.q_head + Piece<D>(c, j).channel, y[c]);
                        top = largest(y[c], top);
                    }
                int of[1] = {(int)top};
                max_over_slots(of, a.slots);
                top = max((uint32_t)of[0], (uint32_t)__shfl_xor(of[0], 16));
                top = max(top, (uint32_t)__shfl_xor((int)top, 32));
                const float factor = factor_of(top);
#pragma unroll
                for (int c = 0; c < chunks; ++c) rows[(wave * chunks + c) * 64 + lane] = whole(y[c], factor, Piece<D>(c, j).negative);
            }
            __syncthreads();
            i32x4 qf[4][chunks];
#pragma unroll
            for (int y = 0; y < 4; ++y)
#pragma unroll
                for (int c = 0; c < chunks; ++c) qf[y][c] = y < row_tiles ? rows[(y * chunks + c) * 64 + lane] : i32x4{0, 0, 0, 0};
            __syncthreads();
            int seen[4];  // columns of the lane's token in each tile of rows, -1: no token
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int token = first + y * per + i / a.slots;
                seen[y] = token < t1 ? columns_of(token) : -1;
            }
            uint32_t* const mine = keys + i / a.slots * a.stride;
            const auto key = [&](int score, int scale, int c, int n) {
                return c < (int)a.first || c >= n - (int)a.last ? kForced : scale < 0 ? kLost : key_of(score, scale);
            };
            const auto work = [&](int tile, const PageTile<D>& y) {
                const int scale = y.ok ? y.scale : -1, c = 16 * tile + 4 * j;
                const int own = 4 * j + (i & 3);  // (a lane's page of the four whose results it holds)
                int of[4];
                if (a.slots >= 4)
                    of[0] = __shfl(scale, own);
                else
#pragma unroll
                    for (int e = 0; e < 4; ++e) of[e] = __shfl(scale, 4 * j + e);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    if (x >= row_tiles) break;
                    i32x4 s = {0, 0, 0, 0};
#pragma unroll
                    for (int c = 0; c < chunks; ++c) s = __builtin_amdgcn_mfma_i32_16x16x64_i8(y.bounds[c], qf[x][c], s, 0, 0, 0);
                    int v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = slot < a.group ? s[e] : -(1 << 30);
                    max_over_slots(v, a.slots);
                    if (seen[x] < 0) continue;
                    uint32_t* const to = mine + x * per * a.stride;  // (what goes past `seen` is not read)
                    if (a.slots >= 4) {  // a page a lane
                        if (slot < 4) to[16 * tile + own] = key(i & 2 ? (i & 1 ? v[3] : v[2]) : (i & 1 ? v[1] : v[0]), of[0], 16 * tile + own, seen[x]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (slot == 0) to[c + e] = key(v[e], of[e], c + e, seen[x]);
                    }
                }
            };
            for (int tile = wave; tile < tiles; tile += WAVES) {
                PageTile<D> y;
                load_tile(a, h, page, j, y);
                page = page_at(min(tile + WAVES, tiles - 1));
                work(tile, y);
            }
            __syncthreads();
        }
        for (int t = first + wave; t < t1; t += WAVES) {
            const int n = columns_of(t);
            int32_t* out = a.blocks + ((int64_t)t * heads + h) * count;
            const uint32_t* mine = keys + (t - first) * a.stride;
            if (n <= count) {
                for (int c = lane; c < count; c += 64) out[c] = c < n ? c : -1;
            } else {
                n <= 128    ? choose<2>(mine, n, count, lane, out)
                : n <= 256  ? choose<4>(mine, n, count, lane, out)
                : n <= 512  ? choose<8>(mine, n, count, lane, out)
                : n <= 1024 ? choose<16>(mine, n, count, lane, out)
                            : choose<64>(mine, n, count, lane, out);
            }
        }
        if (most > count) __syncthreads();
    }
}

// -------------------------------------------------------------- host side --

int check_summaries(const dmx_kv_summaries* s, char* err, size_t errn) {
    if (!s || !s->bounds || !s->scales) return fail(err, errn, "null summaries");
    if (!aligned(s->bounds, 16)) return fail(err, errn, "summaries not 16-byte aligned");
    return 0;
}

constexpr uint32_t kTokenColumns = 4096;  // of k_select_tokens, at most: 64 keys a lane

// How a call is laid out: prompts' tokens together (tokens > 0), a workgroup to a
// token and head, or several (tiles > 0).
struct Plan {
    uint32_t tokens, slots, tiles;
};

Plan plan_of(const dmx_kv_cache* c, const dmx_kv_seqs* s, uint32_t q_heads) {
    Plan p = {0, 1, 0};
    while (p.slots < q_heads / c->heads) p.slots *= 2;
    // Tokens of a prompt share their sequence's summaries where there are eight or more to a sequence on the mean (the
    // host knows no more of them), and keys and rows fit. Where one call mixes them, some go the wrong way: 31 single
    // tokens and 512 of a prompt take 161 us in one call (a workgroup's 16 tokens of as many sequences come one after the
    // other), 9 and 21 in two; 200 and 512, below eight, 47. Past 4096 columns of the table 1024 tokens over 512 pages
    // take 210 us, whatever of the table is in use.
    if (s->total / s->batch >= 8 && s->table_cols <= kTokenColumns && p.slots <= 16) {
        p.tokens = std::min(16u, 64 / p.slots);
        return p;
    }
    // Few tokens over many columns: workgroups of four waves, a tile of 16 columns a wave or more, to
    // fill the CUs, and a second launch that chooses. us with one workgroup to a token and head, and so:
    // 1 token over 2048 columns 32 and 12, over 8192 87 and 17, 8 over 1024 19.5 and 16, 4 over 512 11.9
    // and 10.7, 1 over 313 9.0 and 9.4; 160 rows over 513 11.6 and 15. (Of the table's width, too: 8 sequences of ten
    // columns 6.0 in a table of 384 and 8.3 in a wider one.)
    const uint64_t rows = (uint64_t)s->total * c->heads, tiles = (s->table_cols + 15) / 16;
    if (rows <= 128 && s->table_cols > 384) p.tiles = (uint32_t)std::max<uint64_t>(4, (tiles * rows + 255) / 256);
    return p;
}

uint64_t workspace_of(const Plan& p, const dmx_kv_cache* c, const dmx_kv_seqs* s) {
    return p.tiles ? 4ull * c->heads * s->total * s->table_cols : 0;
}

template <bool F32, int D>
int launch_select(Select& a, hipStream_t stream, char* err, size_t errn) {
    static std::atomic<uint64_t> allowed[4] = {};
    const uint32_t cols = a.seqs.cols, total = a.seqs.total, heads = a.cache.heads;
    if (a.tokens) {
        // (64 KB of keys: two workgroups a CU; a tile's last columns and a shift of the banks between tokens)
        a.stride = (cols + 15) / 16 * 16 + 4;
        while (a.tokens > 1 && a.tokens * a.stride * 4 > 66000) a.tokens /= 2;
        const auto kern = k_select_tokens<F32, D>;
        const uint32_t groups = (total + a.tokens - 1) / a.tokens;
        if (check_lanes(groups, 64 * kSelectWaves, err, errn)) return 1;
        const uint32_t rows = 4 * (D / 32) * 64 * sizeof(i32x4), bytes = std::max(rows, 4 * a.tokens * a.stride);
        if (allow_lds(reinterpret_cast<const void*>(kern), 66000, allowed[2], err, errn)) return 1;
        hipLaunchKernelGGL(kern, dim3(groups, heads), dim3(64 * kSelectWaves), bytes, stream, a);
    } else if (a.tiles) {
        hipLaunchKernelGGL((k_select<F32, D, 4, true>), dim3(total, heads, ((cols + 15) / 16 + a.tiles - 1) / a.tiles), dim3(256), 0, stream, a);
        if (launch_check(err, errn, "kv score launch")) return 1;
        if (allow_lds(reinterpret_cast<const void*>(k_choose), 4 * DMX_KV_MAX_COLUMNS, allowed[3], err, errn)) return 1;
        hipLaunchKernelGGL(k_choose, dim3(total, heads), dim3(1024), 4 * cols, stream, a);
    } else {
        // (every wave makes the queries whole numbers for itself: eight waves gain from 1025 columns on, 32
        // sequences of up to 256 columns take 8.5 us with four and 9.2 with eight)
        const bool many = cols > 1024;
        const auto kern = many ? k_select<F32, D, 8, false> : k_select<F32, D, 4, false>;
        if (allow_lds(reinterpret_cast<const void*>(kern), 4 * DMX_KV_MAX_COLUMNS, allowed[many], err, errn)) return 1;
        if (check_lanes(total, many ? 512 : 256, err, errn)) return 1;
        hipLaunchKernelGGL(kern, dim3(total, heads), dim3(many ? 512 : 256), 4 * cols, stream, a);
    }
    return launch_check(err, errn, "kv select launch");
}

}  // namespace

extern "C" int dmx_kv_summarize(const dmx_kv_cache* cache, const dmx_kv_summaries* summaries, const dmx_kv_seqs* seqs,
                                void* stream, char* err, size_t errn) {
    if (check_cache(cache, err, errn) || check_seqs(cache, seqs, err, errn) || check_summaries(summaries, err, errn)) return 1;
    if (seqs->total == 0) return 0;
    Summarize a = {cache_of(cache), seqs_of(seqs), summaries->bounds, summaries->scales, 1, 0};
    while (a.team < 8 && ((uint64_t)cache->page * seqs->batch << a.team) < seqs->total) ++a.team;
    // (tokens that begin no page cost a workgroup's start: a few thousand workgroups look at several tokens each)
    a.run = (uint32_t)std::min<uint64_t>({64, cache->page, std::max<uint64_t>(1, (uint64_t)seqs->total * cache->heads / 2048)});
    const dim3 grid((seqs->total + a.run - 1) / a.run, cache->heads);
    if (check_lanes(grid.x, 256, err, errn)) return 1;
    const auto launch = [&](auto d) {
        hipLaunchKernelGGL(k_summarize<decltype(d)::value>, grid, dim3(256), 0, static_cast<hipStream_t>(stream), a);
    };
    cache->dim == 64    ? launch(std::integral_constant<int, 64>{})
    : cache->dim == 96  ? launch(std::integral_constant<int, 96>{})
    : cache->dim == 128 ? launch(std::integral_constant<int, 128>{})
    : cache->dim == 192 ? launch(std::integral_constant<int, 192>{})
                        : launch(std::integral_constant<int, 256>{});
    return launch_check(err, errn, "kv summarize launch");
}

extern "C" uint64_t dmx_kv_select_workspace(const dmx_kv_cache* cache, const dmx_kv_seqs* seqs, uint32_t q_heads) {
    if (check_cache(cache, nullptr, 0) || check_seqs(cache, seqs, nullptr, 0) || seqs->table_cols > DMX_KV_MAX_COLUMNS || q_heads == 0 ||
        q_heads % cache->heads || q_heads > 65535)
        return 0;
    return workspace_of(plan_of(cache, seqs, q_heads), cache, seqs);
}

extern "C" int dmx_kv_select(const dmx_kv_cache* cache, const dmx_kv_summaries* summaries, const dmx_kv_seqs* seqs,
                             const dmx_rows* q, int dtype, uint32_t count, uint32_t first, uint32_t last, int causal,
                             int32_t* blocks, void* workspace, uint64_t workspace_bytes, void* stream, char* err, size_t errn) {
    if (check_cache(cache, err, errn) || check_seqs(cache, seqs, err, errn) || check_dtype(dtype, err, errn) ||
        check_summaries(summaries, err, errn))
        return 1;
    if (!q) return fail(err, errn, "null queries");
    if (q->heads == 0 || q->heads % cache->heads || q->heads > 65535)
        return fail(err, errn, "query heads not a multiple of the cache's, or too many");
    if (seqs->table_cols > DMX_KV_MAX_COLUMNS) return fail(err, errn, "a block table of more columns than can be listed (16384)");
    if (count == 0 || count > DMX_KV_MAX_COLUMNS) return fail(err, errn, "lists of no columns, or more than 16384");
    if (first > count || last > count || first + last > count) return fail(err, errn, "first and last are more than count");
    if (seqs->total == 0) return 0;
    if (!q->at || !blocks) return fail(err, errn, "null queries or lists");
    Select a = {};
    a.cache = cache_of(cache);
    a.seqs = seqs_of(seqs);
    a.bounds = summaries->bounds, a.scales = summaries->scales;
    a.q = q->at, a.q_token = q->token_stride, a.q_head = q->head_stride;
    a.group = q->heads / cache->heads;
    a.count = count, a.first = first, a.last = last, a.causal = causal != 0;
    a.blocks = blocks;
    const Plan p = plan_of(cache, seqs, q->heads);
    if (workspace_bytes < workspace_of(p, cache, seqs) || (p.tiles && (!workspace || !aligned(workspace, 16))))
        return fail(err, errn, "workspace missing, short or not 16-byte aligned");
    a.tokens = p.tokens, a.slots = p.slots, a.tiles = p.tiles;
    a.keys = static_cast<uint32_t*>(workspace);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const auto by_type = [&](auto d) {
        constexpr int D = decltype(d)::value;
        return dtype == DMX_F32 ? launch_select<true, D>(a, st, err, errn) : launch_select<false, D>(a, st, err, errn);
    };
    return cache->dim == 64    ? by_type(std::integral_constant<int, 64>{})
           : cache->dim == 96  ? by_type(std::integral_constant<int, 96>{})
           : cache->dim == 128 ? by_type(std::integral_constant<int, 128>{})
           : cache->dim == 192 ? by_type(std::integral_constant<int, 192>{})
                               : by_type(std::integral_constant<int, 256>{});
}
