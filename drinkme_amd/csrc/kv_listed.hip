// The attention over listed pages of the 4-bit cache (include/dmx_kv.h):
// kv_attention.h's k_attend, whose tiles walk the pages that any of their tokens
// lists, and its join.
//
// A tile is 16 rows: with four query heads to a cache head, four tokens, whose lists
// of 32 pages of 512 join to 65 where neighbours look for the same things (a chunk of 1024 tokens: 156 us in a
// graph over one set of inputs, 176 as a launch alone over three, the vector units 74% busy, decoding first; 32 rows, whose eight
// tokens' lists join to 97, take 217 beside 177 at the time). Decoding each block once for 64 rows, in LDS, took 345: too few
// waves to wait with. fp32 queries (three times the products): 512 tokens after 15 872, four heads of 128, 77 us in a
// graph. A step of 32 sequences, 32 of up to 256 pages each, takes 19 us in a graph and 20.6 alone, 3.7 TB/s of the
// listed pages' codes.
//
// A row's weights go to the matrix cores in as many bf16 pieces as its queries have (one of bf16; three, 24 bits,
// of fp32), as in the attention over everything: bf16 results are off by 2.1e-3 to 2.3e-3 of their norm, where the
// rounding of the results alone makes 1.7e-3.
#include "kv_common.h"

namespace {

#include "kv_attention.h"

// Waves of a workgroup: eight for a call of few tiles of rows to a sequence and head, where
// two fit a SIMD (256 registers a lane); else four.
constexpr int few_waves(int W, int P) { return W * (P + 1) <= 16 ? 8 : 4; }

// How a call is laid out: splits of each tile's pages.
struct Plan {
    int waves;
    uint32_t tokens, row_blocks, splits;  // tokens: of a sequence, at most
    uint32_t listed;                      // columns that a tile may list, at most
};

Plan plan_of(const dmx_kv_cache* c, const dmx_kv_seqs* s, uint32_t q_heads, int dtype, uint32_t count, uint32_t max_length) {
    Plan p;
    const uint32_t group = q_heads / c->heads;
    p.tokens = s->cu ? std::min(s->max_tokens, s->total) : s->total / s->batch;
    const uint64_t rows = (uint64_t)p.tokens * group;
    const uint32_t tile_tokens = std::min(p.tokens, 1 + (16 + group - 2) / group);
    p.row_blocks = (uint32_t)((rows + 15) / 16);
    p.listed = (uint32_t)std::min<uint64_t>(s->table_cols, (uint64_t)tile_tokens * count);
    uint64_t length = (uint64_t)p.listed * c->page;
    if (max_length) length = std::min<uint64_t>(length, max_length);
    // Splits to fill the CUs once, each of a block of 32 tokens a wave at least. Eight waves where
    // half of the CUs have a workgroup without splits (us a step of 32 sequences, 32 pages of 64 each: 36,
    // and 41 with four; 8 of 5 tokens 26 and 33; one sequence of 16 pages, split in 8: 21, in 4 of eight
    // waves 22), and not for prompts (a chunk of 1024 tokens 235, and 177 with four).
    const uint64_t groups = (uint64_t)c->heads * s->batch * std::max(1u, p.row_blocks);
    p.waves = p.row_blocks <= 4 && groups >= 128 ? few_waves(c->dim / 32, dtype == DMX_F32 ? 3 : 1) : 4;
    const uint64_t wanted = std::max<uint64_t>(1, 256 / groups), possible = std::max<uint64_t>(1, length / (32 * p.waves));
    p.splits = (uint32_t)std::min<uint64_t>({wanted, possible, 64, 65535 / s->batch});
    return p;
}

uint64_t workspace_of(const Plan& p, const dmx_kv_cache* c, const dmx_kv_seqs* s, uint32_t q_heads) {
    return p.splits == 1 ? 0 : (uint64_t)p.splits * s->total * q_heads * (c->dim + 4) * 4;
}

int check_listed(const dmx_kv_cache* c, const dmx_kv_seqs* s, uint32_t count, char* err, size_t errn) {
    if (s->table_cols > DMX_KV_MAX_COLUMNS) return fail(err, errn, "a block table of more columns than can be listed (16384)");
    if (count == 0 || count > DMX_KV_MAX_COLUMNS) return fail(err, errn, "lists of no columns, or more than 16384");
    return 0;
}

template <int W, int P, bool WIDE, int WAVES>
int launch(dim3 grid, int lds, hipStream_t stream, ListedArgs a, char* err, size_t errn) {
    // (the most that any call takes: 16384 columns' bits, and as many 16-bit entries; in their
    // place half of the waves' results at the end)
    static std::atomic<uint64_t> allowed = {};
    constexpr uint32_t most = 65535;  // workgroups along a grid's second axis
    constexpr int results = WAVES / 2 * 2 * W * 64 * (int)sizeof(f32x4);
    static_assert(results <= 6 * DMX_KV_MAX_COLUMNS);
    const auto kern = k_attend<W, P, 1, false, WIDE, true, WAVES>;
    if (allow_lds(reinterpret_cast<const void*>(kern), 6 * DMX_KV_MAX_COLUMNS, allowed, err, errn)) return 1;
    for (; a.first_block < a.row_blocks; a.first_block += most) {  // (65535 tiles are 262 140 tokens of four rows)
        grid.y = std::min(most, a.row_blocks - a.first_block);
        hipLaunchKernelGGL(kern, grid, dim3(64 * WAVES), std::max(lds, results), stream, a);
    }
    return launch_check(err, errn, "kv attention launch");
}

}  // namespace

extern "C" uint64_t dmx_kv_attention_blocks_workspace(const dmx_kv_cache* cache, const dmx_kv_seqs* seqs, uint32_t q_heads,
                                                      int dtype, uint32_t count, uint32_t max_length) {
    if (check_cache(cache, nullptr, 0) || check_seqs(cache, seqs, nullptr, 0) || check_listed(cache, seqs, count, nullptr, 0) ||
        q_heads == 0 || q_heads % cache->heads)
        return 0;
    return workspace_of(plan_of(cache, seqs, q_heads, dtype, count, max_length), cache, seqs, q_heads);
}

extern "C" int dmx_kv_attention_blocks(const dmx_kv_cache* cache, const dmx_kv_seqs* seqs, const dmx_rows* q, int dtype,
                                       float scale, int causal, const int32_t* blocks, uint32_t count, uint32_t max_length,
                                       void* out, float* lse, void* workspace, uint64_t workspace_bytes, void* stream,
                                       char* err, size_t errn) {
    if (check_cache(cache, err, errn) || check_seqs(cache, seqs, err, errn) || check_dtype(dtype, err, errn) ||
        check_listed(cache, seqs, count, err, errn))
        return 1;
    if (!q) return fail(err, errn, "null queries");
    if (q->heads == 0 || q->heads % cache->heads || q->heads > 65535)
        return fail(err, errn, "query heads not a multiple of the cache's, or too many");
    const float scale2 = scale * 1.44269504088896341f;  // (the kernels' exponentials are of 2)
    if (!(scale > 0) || !std::isfinite(scale2)) return fail(err, errn, "scale not a positive number, or too large");
    if (seqs->total == 0) return 0;
    if (!q->at || !out || !blocks) return fail(err, errn, "null queries, lists or output");
    if ((uint64_t)seqs->total * cache->heads * count >= 1ull << 62) return fail(err, errn, "too many lists");
    const Plan p = plan_of(cache, seqs, q->heads, dtype, count, max_length);
    if (p.tokens == 0) return fail(err, errn, "max_tokens is 0");
    // (the kernel numbers a sequence's rows in 31 bits; so many have 256 GiB of results at least)
    if ((uint64_t)p.tokens * (q->heads / cache->heads) >= 1ull << 31) return fail(err, errn, "too many query rows of one sequence");
    if (workspace_bytes < workspace_of(p, cache, seqs, q->heads) || (p.splits > 1 && (!workspace || !aligned(workspace, 16))))
        return fail(err, errn, "workspace missing, short or not 16-byte aligned");
    ListedArgs a = {};
    a.cache = cache_of(cache);
    a.seqs = seqs_of(seqs);
    a.q = q->at, a.q_token = q->token_stride, a.q_head = q->head_stride;
    a.q_heads = q->heads, a.group = q->heads / cache->heads;
    a.scale = scale2;
    a.causal = causal != 0, a.splits = p.splits;
    a.seqs.each = divisor_of(p.tokens);
    a.row_blocks = p.row_blocks;
    a.out = out, a.lse = lse;
    a.blocks = blocks, a.count = divisor_of(count);
    const uint64_t all = (uint64_t)seqs->total * q->heads;
    a.part_o = static_cast<float*>(workspace);
    a.part_stat = reinterpret_cast<f32x4*>(a.part_o + (p.splits > 1 ? p.splits * all * cache->dim : 0));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid(cache->heads, p.row_blocks, seqs->batch * p.splits);
    const int lds = 4 * (int)seqs->table_cols + 2 * (int)p.listed;
    const auto by_type = [&](auto w, auto wide) {
        constexpr int W = decltype(w)::value;
        constexpr bool WIDE = decltype(wide)::value;
        const auto by_waves = [&](auto pieces) {
            constexpr int P = decltype(pieces)::value;
            return p.waves == 4 ? launch<W, P, WIDE, 4>(grid, lds, st, a, err, errn) : launch<W, P, WIDE, few_waves(W, P)>(grid, lds, st, a, err, errn);
        };
        return dtype == DMX_F32 ? by_waves(std::integral_constant<int, 3>{}) : by_waves(std::integral_constant<int, 1>{});
    };
    const auto by_page = [&](auto w) { return cache->page >= 32 ? by_type(w, std::true_type{}) : by_type(w, std::false_type{}); };
    const int rc = cache->dim == 64    ? by_page(std::integral_constant<int, 2>{})
                   : cache->dim == 96  ? by_page(std::integral_constant<int, 3>{})
                   : cache->dim == 128 ? by_page(std::integral_constant<int, 4>{})
                   : cache->dim == 192 ? by_page(std::integral_constant<int, 6>{})
                                       : by_page(std::integral_constant<int, 8>{});
    if (rc) return 1;
    if (p.splits == 1) return 0;
    const int ways = p.splits > 8 ? 4 : 1;
    hipLaunchKernelGGL((dtype == DMX_F32 ? k_attend_join<true> : k_attend_join<false>),
                       dim3((uint32_t)(ways == 4 ? all : (all + 3) / 4)), dim3(256), 0, st,
                       static_cast<const AttnArgs&>(a), (int)cache->dim, ways);
    return launch_check(err, errn, "kv attention join launch");
}
