// Summaries of the 4-bit cache's pages, and the pages that a cheap score selects
// for each query (include/dmx_kv.h).
//
//   k_summarize   the bounds of the keys in a page
//   k_select      scores of a token's pages, and the best of them
#include "kv_common.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// --------------------------------------------------------------- summaries --
//
// Every channel's largest and smallest key of a page bound its product with any
// query there. They are exact (a code times its power of two is an fp32 number,
// and neither depends on an order), and rounded outwards to 8 bits.

struct Summarize {
    Cache cache;
    Seqs seqs;
    int8_t* bounds;
    uint8_t* scales;
    uint32_t run;  // new tokens a workgroup looks at
};

// A workgroup takes a head of the pages that begin among its new tokens (or in
// which their sequence's first one lies): a thread a word of eight channels, of
// every 256 / words-th token, then a channel.
template <int D>
__global__ __launch_bounds__(256) void k_summarize(const Summarize a) {
    constexpr int words = D / 8, groups = 256 / words;
    __shared__ float part[groups][2][D];
    __shared__ float tops[4];
    const int x = threadIdx.x, w = x % words, g = x / words;
    const uint32_t h = blockIdx.y, heads = a.cache.heads, shift = a.cache.page_shift;
    for (uint32_t t = blockIdx.x * a.run; t < min((blockIdx.x + 1) * a.run, a.seqs.total); ++t) {
        int p;
        const Slot at = slot_of_new(a.cache, a.seqs, t, p);
        if (!at.ok) continue;
        const uint32_t b = seq_at(a.seqs, t);
        const Seq q = seq_of(a.seqs, b);
        const int in = p & ((1 << shift) - 1);
        if (in && (int)t != q.token) continue;  // (not the first of its page, nor of its sequence's new ones)
        const uint64_t page = a.seqs.table[(int64_t)b * a.seqs.cols + (p >> shift)];
        const int count = min(1 << shift, q.length - (p - in));
        const uint64_t first = (page * heads + h) << shift;
        float hi[8], lo[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) hi[n] = -INFINITY, lo[n] = INFINITY;
        if (g < groups) {
#pragma unroll 4
            for (int m = g; m < count; m += groups) {
                const uint32_t e = a.cache.k_scales[(first + m) * (D / 32) + w / 4];
                const uint32_t word = a.cache.k_codes[(first + m) * words + w];
                if (e > 252) continue;  // NaN
                const float unit = __uint_as_float(e << 23);
                const f32x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, unit, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, unit, 1),
                                    __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, unit, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, unit, 3)};
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    hi[n] = fmaxf(hi[n], v[n / 2][n & 1]);
                    lo[n] = fminf(lo[n], v[n / 2][n & 1]);
                }
            }
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                part[g][0][8 * w + n] = hi[n];
                part[g][1][8 * w + n] = lo[n];
            }
        }
        __syncthreads();
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
// smallest keys. On v_mfma_i32_16x16x64_i8 16 pages meet up to 16 query heads, in
// whole numbers, which no order of summation changes: ties are ties, and go
// to the lower column whatever computes them.
//
// The best `count` keys (a score's bits, ordered as numbers) are those from a
// threshold on, found three of its bits at a time by counting: the largest one that
// `count` keys reach.

struct Select {
    Cache cache;  // (page numbers and sizes alone)
    Seqs seqs;
    const int8_t* bounds;
    const uint8_t* scales;
    const void* q;
    int64_t q_token, q_head;  // strides, elements
    uint32_t group, count, first, last, causal;
    int32_t* blocks;
};

__device__ __forceinline__ int max_over_16(int x) {
    x = max(x, __builtin_amdgcn_mov_dpp(x, 0x128, 0xF, 0xF, true));  // a row of 16 lanes, turned by 8, 4, 2, 1
    x = max(x, __builtin_amdgcn_mov_dpp(x, 0x124, 0xF, 0xF, true));
    x = max(x, __builtin_amdgcn_mov_dpp(x, 0x122, 0xF, 0xF, true));
    return max(x, __builtin_amdgcn_mov_dpp(x, 0x121, 0xF, 0xF, true));
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

// WAVES: of a token and head. One: four of them to a workgroup, 512 columns at most.
template <bool F32, int D, int WAVES>
__global__ __launch_bounds__(64 * (WAVES == 1 ? 4 : WAVES)) void k_select(const Select a) {
    constexpr int chunks = D / 32, R = WAVES == 1 ? 8 : 16, kRounds = 11;
    extern __shared__ __align__(16) uint32_t lds[];
    __shared__ int counts[kRounds][8];
    __shared__ int before[2][WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, j = lane >> 4;
    const int team = WAVES == 1 ? wave : 0, member = WAVES == 1 ? 0 : wave;
    const uint32_t heads = a.cache.heads, row = blockIdx.x * (WAVES == 1 ? 4 : 1) + team;
    if (row >= a.seqs.total * heads) return;
    const uint32_t t = row / heads, h = row - t * heads;
    uint32_t* keys = lds + team * a.seqs.cols;
    int32_t* out = a.blocks + (int64_t)row * a.count;

    const uint32_t b = seq_at(a.seqs, t);
    const Seq q = seq_of(a.seqs, b);
    const int m = (int)t - q.token, p = a.causal ? q.first + m : q.length - 1;
    const bool inside = (uint32_t)m < (uint32_t)q.count && q.first + m >= 0;
    const int n = inside ? min((p >> a.cache.page_shift) + 1, a.seqs.cols) : 0, count = a.count;
    if (n <= count) {
        for (int c = threadIdx.x - 64 * team; c < count; c += 64 * WAVES) out[c] = c < n ? c : -1;
        return;
    }
    if constexpr (WAVES > 1)
        for (int c = threadIdx.x; c < kRounds * 8; c += 64 * WAVES) (&counts[0][0])[c] = 0;

    // piece c of a lane: 16 channels, of the positive side's D / 16 pieces and then of the negative one's
    const auto side_of = [&](int c) { return 4 * c + j >= D / 16; };
    const auto channel = [&](int c) { return 16 * (4 * c + j - (side_of(c) ? D / 16 : 0)); };
    const auto load = [&](int r, int c, float (&x)[16]) {  // of query head r of the group
        load16<F32>(a.q, t * a.q_token + ((int64_t)h * a.group + r) * a.q_head + channel(c), x);
    };
    uint32_t top = 0;
    for (uint32_t r = i; r < a.group; r += 16)
#pragma unroll
        for (int c = 0; c < chunks; ++c) {
            float x[16];
            load(r, c, x);
#pragma unroll
            for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
        }
#pragma unroll
    for (int s = 32; s; s >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, s));
    // 255 / 128 of a power of two and above round to 128 of its 64th: of its 32nd
    const int e = max((int)((top + 0x10000u) >> 23) - 133, -126);
    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);

    for (uint32_t r0 = 0; r0 < a.group; r0 += 16) {
        const uint32_t r = r0 + i;
        i32x4 qf[chunks];
#pragma unroll
        for (int c = 0; c < chunks; ++c) {
            float x[16] = {};
            if (r < a.group) load(r, c, x);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t word = 0;
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const int v = (int)rintf(x[4 * w + y] * inv);
                    word |= (uint32_t)((side_of(c) ? min(v, 0) : max(v, 0)) & 255) << (8 * y);
                }
                qf[c][w] = (int)word;
            }
        }
        const auto page_at = [&](int tile) { return (uint32_t)a.seqs.table[(int64_t)b * a.seqs.cols + min(16 * tile + i, n - 1)]; };
        const int tiles = (n + 15) / 16;
        uint32_t next = member < tiles ? page_at(member) : 0;
        for (int tile = member; tile < tiles; tile += WAVES) {
            const uint32_t page = next;
            if (tile + WAVES < tiles) next = page_at(tile + WAVES);
            const bool ok = page < a.cache.pages;
            const uint64_t at = (uint64_t)(ok ? page : 0u) * heads + h;
            const i32x4* from = reinterpret_cast<const i32x4*>(a.bounds + at * (2 * D) + 16 * j);
            const int scale = a.scales[at];
            i32x4 s = {0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < chunks; ++c) s = __builtin_amdgcn_mfma_i32_16x16x64_i8(from[4 * c], qf[c], s, 0, 0, 0);
            int best = 0;  // of page i, in the lanes of its row of results
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int v = max_over_16(r < a.group ? s[y] : -(1 << 30));
                if ((i & 3) == y) best = v;
            }
            const int c = 16 * tile + i;
            if (i >> 2 == j && c < n) {
                const uint32_t bits = __float_as_uint(__builtin_ldexpf((float)best, scale - 127));
                uint32_t key = bits ^ (bits >> 31 ? 0xffffffffu : 0x80000000u);
                if (!ok) key = 1;  // below every number
                if (c < (int)a.first || c >= n - (int)a.last) key = 0xffffffffu;
                keys[c] = r0 ? max(keys[c], key) : key;
            }
        }
    }
    if constexpr (WAVES > 1)
        __syncthreads();
    else
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");

    // a wave's keys: `rows` times 64 columns in a row
    const int rows = (n + 64 * WAVES - 1) / (64 * WAVES), c0 = member * rows * 64 + lane;
    uint32_t key[R];
#pragma unroll
    for (int x = 0; x < R; ++x) key[x] = x < rows && c0 + 64 * x < n ? keys[c0 + 64 * x] : 0;
    uint32_t at_least = 0;
    if constexpr (WAVES == 1) {
        for (uint32_t bit = 1u << 31; bit; bit >>= 1) {
            const uint32_t to = at_least | bit;
            int have = 0;
#pragma unroll
            for (int x = 0; x < R; ++x)
                if (x < rows) have += __popcll(__ballot(key[x] >= to));
            if (have >= count) at_least = to;
            if (have == count) break;
        }
    } else {
        for (int round = 0; round < kRounds; ++round) {
            const int shift = 30 - 3 * round;
            int mine = 0;  // lane k: how many reach at_least + k << shift
#pragma unroll
            for (int k = 1; k < 8; ++k) {
                if (round == 0 && k > 3) break;
                const uint32_t to = at_least + ((uint32_t)k << shift);
                int have = 0;
#pragma unroll
                for (int x = 0; x < R; ++x)
                    if (x < rows) have += __popcll(__ballot(key[x] >= to));
                if (lane == k) mine = have;
            }
            if (mine) atomicAdd(&counts[round][lane], mine);
            __syncthreads();
            int k = 0, reach = 0;
#pragma unroll
            for (int y = 1; y < 8; ++y) {
                const int have = counts[round][y];
                if (have >= count) k = y, reach = have;
            }
            at_least += (uint32_t)k << shift;
            if (reach == count) break;
        }
    }

    // those above the threshold, and of those at it the first ones
    int above = 0, equal = 0;
#pragma unroll
    for (int x = 0; x < R; ++x)
        if (x < rows) {
            above += __popcll(__ballot(key[x] > at_least));
            equal += __popcll(__ballot(key[x] == at_least && key[x]));
        }
    int all_above = above, over = 0, level = 0;
    if constexpr (WAVES > 1) {
        if (lane == 0) before[0][wave] = above, before[1][wave] = equal;
        __syncthreads();
        all_above = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            all_above += before[0][w];
            over += w < wave ? before[0][w] : 0;
            level += w < wave ? before[1][w] : 0;
        }
    }
    const int fill = count - all_above;
#pragma unroll
    for (int x = 0; x < R; ++x) {
        const bool up = key[x] > at_least, even = key[x] == at_least && key[x];
        const uint64_t u = __ballot(up), v = __ballot(even);
        const int o = over + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(u >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)u, 0));
        const int l = level + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(v >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)v, 0));
        if (up || (even && l < fill)) out[o + min(l, fill)] = c0 + 64 * x;
        over += __popcll(u);
        level += __popcll(v);
    }
}

// -------------------------------------------------------------- host side --

int check_summaries(const dmx_kv_summaries* s, char* err, size_t errn) {
    if (!s || !s->bounds || !s->scales) return fail(err, errn, "null summaries");
    if (!aligned(s->bounds, 16)) return fail(err, errn, "summaries not 16-byte aligned");
    return 0;
}

template <bool F32, int D, int WAVES>
int launch_select(const Select& a, uint32_t rows, hipStream_t stream, char* err, size_t errn) {
    constexpr int teams = WAVES == 1 ? 4 : 1;
    static std::atomic<uint64_t> allowed = {};
    const auto kern = k_select<F32, D, WAVES>;
    if (allow_lds(reinterpret_cast<const void*>(kern), 4 * DMX_KV_MAX_COLUMNS, allowed, err, errn)) return 1;
    hipLaunchKernelGGL(kern, dim3((rows + teams - 1) / teams), dim3(64 * teams * WAVES), 4 * teams * a.seqs.cols, stream, a);
    return launch_check(err, errn, "kv select launch");
}

}  // namespace

extern "C" int dmx_kv_summarize(const dmx_kv_cache* cache, const dmx_kv_summaries* summaries, const dmx_kv_seqs* seqs,
                                void* stream, char* err, size_t errn) {
    if (check_cache(cache, err, errn) || check_seqs(cache, seqs, err, errn) || check_summaries(summaries, err, errn)) return 1;
    if (seqs->total == 0) return 0;
    Summarize a = {cache_of(cache), seqs_of(seqs), summaries->bounds, summaries->scales, 1};
    // (tokens that begin no page cost a workgroup's start: a few thousand workgroups look at several tokens each)
    a.run = (uint32_t)std::min<uint64_t>({64, cache->page, std::max<uint64_t>(1, (uint64_t)seqs->total * cache->heads / 2048)});
    const dim3 grid((seqs->total + a.run - 1) / a.run, cache->heads);
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

extern "C" int dmx_kv_select(const dmx_kv_cache* cache, const dmx_kv_summaries* summaries, const dmx_kv_seqs* seqs,
                             const dmx_rows* q, int dtype, uint32_t count, uint32_t first, uint32_t last, int causal,
                             int32_t* blocks, void* stream, char* err, size_t errn) {
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
    const uint64_t rows = (uint64_t)seqs->total * cache->heads;
    if (rows >= 1ull << 31) return fail(err, errn, "too many tokens and heads");
    Select a = {};
    a.cache = cache_of(cache);
    a.seqs = seqs_of(seqs);
    a.bounds = summaries->bounds, a.scales = summaries->scales;
    a.q = q->at, a.q_token = q->token_stride, a.q_head = q->head_stride;
    a.group = q->heads / cache->heads;
    a.count = count, a.first = first, a.last = last, a.causal = causal != 0;
    a.blocks = blocks;
    const uint32_t cols = seqs->table_cols;
    const int waves = cols <= 512 && rows >= 2048 ? 1 : cols <= 512 || (cols <= 4096 && rows >= 512) ? 4 : 16;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const auto by_waves = [&](auto f32, auto d) {
        constexpr bool F32 = decltype(f32)::value;
        constexpr int D = decltype(d)::value;
        return waves == 1   ? launch_select<F32, D, 1>(a, (uint32_t)rows, st, err, errn)
               : waves == 4 ? launch_select<F32, D, 4>(a, (uint32_t)rows, st, err, errn)
                            : launch_select<F32, D, 16>(a, (uint32_t)rows, st, err, errn);
    };
    const auto by_type = [&](auto d) { return dtype == DMX_F32 ? by_waves(std::true_type{}, d) : by_waves(std::false_type{}, d); };
    return cache->dim == 64    ? by_type(std::integral_constant<int, 64>{})
           : cache->dim == 96  ? by_type(std::integral_constant<int, 96>{})
           : cache->dim == 128 ? by_type(std::integral_constant<int, 128>{})
           : cache->dim == 192 ? by_type(std::integral_constant<int, 192>{})
                               : by_type(std::integral_constant<int, 256>{});
}
