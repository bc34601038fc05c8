// The operators between a decoder's q/k/v and o projections (include/dmx_kv.h):
// gfx950 kernels and the C-ABI entry points that launch them.
//
//   k_rotary, k_rotary_any   rotary positions, of one axis or several
//   k_append                 keys (rotated) and values into the 4-bit cache
//   k_read                   cached tokens back to bf16
//   k_attend, k_attend_join  the attention over the cache (kv_attention.h)
#include "kv_common.h"

namespace {

// ----------------------------------------------------------------- rotary --

// (a, b) turned: each product and the sum rounded on its own, so that a result
// does not depend on which operations a compiler joins.
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
#pragma clang fp contract(off)
    const float x = a * c - b * s, y = b * c + a * s;
    a = x;
    b = y;
}

// N (cos, sin) pairs from angle `first` of a position's row; NaN outside the table.
template <int N>
__device__ __forceinline__ void angles(const Table& t, int64_t position, uint32_t first, float (&c)[8], float (&s)[8]) {
    const bool ok = position >= 0 && position < (int64_t)t.positions;
    const float4* p = reinterpret_cast<const float4*>(t.at + 2 * ((ok ? position : 0) * t.half + first));
#pragma unroll
    for (int n = 0; n < N / 2; ++n) {
        const float4 v = p[n];
        c[2 * n] = ok ? v.x : NAN, s[2 * n] = ok ? v.y : NAN;
        c[2 * n + 1] = ok ? v.z : NAN, s[2 * n + 1] = ok ? v.w : NAN;
    }
}

// Items of a rotation: (token, run of heads, c). A lane keeps its token's
// position and angles for a run of heads.
struct Rotation {
    Rows in[2], out[2];
    uint32_t n, tokens, dim;
    const void* positions;  // null: the tokens' places in seqs
    int wide;
    Table table;
    Seqs seqs;
    Divisor per, runs;  // items of a head, runs of a token
    uint32_t run;       // heads of a run
};

__device__ __forceinline__ int64_t position_of(const Rotation& r, uint32_t t) {
    if (r.positions)
        return r.wide ? static_cast<const int64_t*>(r.positions)[t] : static_cast<const int32_t*>(r.positions)[t];
    const Seq q = seq_of(r.seqs, seq_at(r.seqs, t));
    return (int64_t)q.first + ((int)t - q.token);
}

// Positions of several axes, [axes, tokens]: angle i follows axis of[i / 16] >> 2 (i % 16) & 3.
struct AxesRotation : Rotation {
    uint32_t axes;
    uint32_t of[16];
};

// Eight angles' cos and sin from angle 8 c of token t, and the one of angle c.
__device__ __forceinline__ void angles_of(const Rotation& r, uint32_t t, uint32_t c, float (&cs)[8], float (&sn)[8]) {
    angles<8>(r.table, position_of(r, t), 8 * c, cs, sn);
}
__device__ __forceinline__ void angle_of(const Rotation& r, uint32_t t, uint32_t c, float& cs, float& sn) {
    const int64_t p = position_of(r, t);
    const bool ok = p >= 0 && p < (int64_t)r.table.positions;
    const float* at = r.table.at + 2 * ((ok ? p : 0) * r.table.half + c);
    cs = ok ? at[0] : NAN, sn = ok ? at[1] : NAN;
}

__device__ __forceinline__ int64_t position_of(const AxesRotation& r, uint32_t t, uint32_t axis) {
    const int64_t at = (int64_t)axis * r.tokens + t;
    return r.wide ? static_cast<const int64_t*>(r.positions)[at] : static_cast<const int32_t*>(r.positions)[at];
}
// (eight angles of one axis are one piece of a row of the table; of several, each its own)
__device__ __forceinline__ void angles_of(const AxesRotation& r, uint32_t t, uint32_t c, float (&cs)[8], float (&sn)[8]) {
    const uint32_t of = r.of[c >> 1] >> (16 * (c & 1)) & 0xffffu;
    if (of == (of & 3) * 0x5555u) {
        angles<8>(r.table, position_of(r, t, of & 3), 8 * c, cs, sn);
        return;
    }
    int64_t p[4];
#pragma unroll
    for (uint32_t x = 0; x < 4; ++x) p[x] = x < r.axes ? position_of(r, t, x) : 0;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
        const uint32_t x = of >> (2 * n) & 3;
        const int64_t at = x == 0 ? p[0] : x == 1 ? p[1] : x == 2 ? p[2] : p[3];
        const bool ok = at >= 0 && at < (int64_t)r.table.positions;
        const float2 v = *reinterpret_cast<const float2*>(r.table.at + 2 * ((ok ? at : 0) * r.table.half + 8 * c + n));
        cs[n] = ok ? v.x : NAN, sn[n] = ok ? v.y : NAN;
    }
}
__device__ __forceinline__ void angle_of(const AxesRotation& r, uint32_t t, uint32_t c, float& cs, float& sn) {
    const int64_t p = position_of(r, t, r.of[c >> 4] >> (2 * (c & 15)) & 3);
    const bool ok = p >= 0 && p < (int64_t)r.table.positions;
    const float* at = r.table.at + 2 * ((ok ? p : 0) * r.table.half + c);
    cs = ok ? at[0] : NAN, sn = ok ? at[1] : NAN;
}

struct RotaryItem {
    uint32_t c, t, first, end;  // heads of both tensors, in's first
};
__device__ __forceinline__ RotaryItem rotary_item_of(const Rotation& r, uint32_t n) {
    const uint32_t c = take(n, r.per), k = take(n, r.runs), all = r.in[0].heads + (r.n > 1 ? r.in[1].heads : 0);
    return {c, n, k * r.run, min(k * r.run + r.run, all)};
}

struct RowAt {
    void *in, *out;
    int64_t from, to;
};
__device__ __forceinline__ RowAt row_at(const Rotation& r, uint32_t t, uint32_t h) {
    const bool other = h >= r.in[0].heads;
    const int64_t k = other ? h - r.in[0].heads : h;
    return {other ? r.in[1].at : r.in[0].at, other ? r.out[1].at : r.out[0].at,
            t * (other ? r.in[1].token : r.in[0].token) + k * (other ? r.in[1].head : r.in[0].head),
            t * (other ? r.out[1].token : r.out[0].token) + k * (other ? r.out[1].head : r.out[0].head)};
}

// c: 16 channels, two runs of 8. In the turned part the eight pairs of angles
// 8 c .. 8 c + 7, else 16 channels to copy. Takes 16-byte aligned rows, dim and
// the turned channels multiples of 16.
template <bool F32, typename R>
__device__ __forceinline__ void rotate(const R& r, uint32_t item) {
    const auto [c, t, first, end] = rotary_item_of(r, item);
    if (t >= r.tokens) return;
    const bool turned = 8 * c < r.table.half, split = turned && r.table.layout == DMX_ROTARY_HALF;
    const uint32_t x = split ? 8 * c : 16 * c, y = split ? 8 * c + r.table.half : 16 * c + 8;
    float cs[8], sn[8];
    if (turned) angles_of(r, t, c, cs, sn);
    for (uint32_t h = first; h < end; ++h) {
        const RowAt row = row_at(r, t, h);
        float a[8], b[8];
        load8<F32>(row.in, row.from + x, a);
        load8<F32>(row.in, row.from + y, b);
        if (split) {
#pragma unroll
            for (int e = 0; e < 8; ++e) turn(a[e], b[e], cs[e], sn[e]);
        } else if (turned) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                turn(a[2 * e], a[2 * e + 1], cs[e], sn[e]);
                turn(b[2 * e], b[2 * e + 1], cs[4 + e], sn[4 + e]);
            }
        }
        store8<F32>(row.out, row.to + x, a);
        store8<F32>(row.out, row.to + y, b);
    }
}

// Any sizes, strides and alignment. c: a pair of channels.
template <bool F32, typename R>
__device__ __forceinline__ void rotate_any(const R& r, uint32_t item) {
    const auto [c, t, first, end] = rotary_item_of(r, item);
    if (t >= r.tokens) return;
    const bool turned = c < r.table.half, split = turned && r.table.layout == DMX_ROTARY_HALF;
    const uint32_t x = split ? c : 2 * c, y = split ? c + r.table.half : 2 * c + 1;
    float cs = 0.f, sn = 0.f;
    if (turned) angle_of(r, t, c, cs, sn);
    for (uint32_t h = first; h < end; ++h) {
        const RowAt row = row_at(r, t, h);
        float a = load1<F32>(row.in, row.from + x), b = load1<F32>(row.in, row.from + y);
        if (turned) turn(a, b, cs, sn);
        store1<F32>(row.out, row.to + x, a);
        store1<F32>(row.out, row.to + y, b);
    }
}

// Memory bounds it: 8192 tokens of 40 heads of 128 out of a fused product, 172 MB
// read and written, take 30.5 us (5.6 TB/s, part of the reads cached). A lane takes
// two runs of 8 channels of a pair, 16 bytes each way, and its angles serve a run of
// heads; one token takes 2.6 us, its launch. Of several axes: 8064 tokens 28.9 us in blocks, 30.1 with the
// axes dealt in turn, whose angles come one by one; 1147 tokens of 32 heads of 96 in fp32 10. Turned parts of no whole
// 16 channels go a pair of values at a time, two bytes a load: 4096 tokens of 40 heads of 72 25, 16.5 of heads of 80.
template <bool F32, typename R>
__global__ __launch_bounds__(256) void k_rotary(const R r) {
    rotate<F32>(r, blockIdx.x * 256 + threadIdx.x);
}
// (what k_rotary does not take, a value at a time)
template <bool F32, typename R>
__global__ __launch_bounds__(256) void k_rotary_any(const R r) {
    rotate_any<F32>(r, blockIdx.x * 256 + threadIdx.x);
}

// ----------------------------------------------------------------- append --

// Items of a call's keys: (token, run of heads, word), words fastest, which lie
// side by side in the cache and in the activations; of its values: (eight tokens,
// run of heads, word, token), as the cache has them. A lane keeps its token's
// place for a run of heads.
struct Items {
    Divisor words, runs;
    uint32_t run;
};

struct Append {
    Cache cache;
    Seqs seqs;
    Rows k, v;
    Items items;
    Table table;  // at null: keys as they are
    Rotation q;   // the queries' (n 0: none)
    uint32_t key_blocks, cached_blocks;  // blocks of keys; of keys and values
};

// The maximum over the four lanes of a block of 32: adjacent (STRIDE 1), or
// eight lanes apart.
template <int STRIDE>
__device__ __forceinline__ uint32_t max_of_block(uint32_t x) {
    if constexpr (STRIDE == 1) {
        x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xF, 0xF, true));  // lane ^ 1
        return max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xF, 0xF, true));  // lane ^ 2
    } else {
        x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x128, 0xF, 0xF, true));  // lane ^ 8
        const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);            // lane ^ 16
        return max(r[0], r[1]);
    }
}

// The codes of a lane's eight channels, and the exponent byte of the block that
// it holds with three more lanes.
template <int STRIDE>
__device__ __forceinline__ uint32_t coded(const float (&x)[8], uint32_t& e) {
    uint32_t top = 0;  // as integers, NaN above infinity above every number
#pragma unroll
    for (int n = 0; n < 8; ++n) top = max(top, __float_as_uint(x[n]) & 0x7fffffffu);
    top = max_of_block<STRIDE>(top);
    const int exponent = (int)((top + 0x200000u) >> 23) - 2;  // 1.75 and above: the next power's
    const uint32_t unit = (uint32_t)min(max(exponent, 2), 252);
    e = top >= 0x7f800000u ? 255u : unit;
    const float scale = __uint_as_float(unit << 23);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
}

struct Item {
    uint32_t w, t, first;
};
__device__ __forceinline__ Item key_item(const Items& d, uint32_t n) {
    const uint32_t w = take(n, d.words), k = take(n, d.runs);
    return {w, n, k * d.run};
}
__device__ __forceinline__ Item value_item(const Items& d, uint32_t n) {
    const uint32_t t = n & 7;
    n >>= 3;
    const uint32_t w = take(n, d.words), k = take(n, d.runs);
    return {w, n * 8 + t, k * d.run};
}

// Words of the keys. VEC: 16-byte aligned rows, and the turned channels a
// multiple of 16.
template <bool F32, bool VEC>
__device__ __forceinline__ void append_keys(const Append& a, uint32_t item) {
    const auto [w, t, first] = key_item(a.items, item);
    if (t >= a.seqs.total) return;
    int p;
    const Slot at = slot_of_new(a.cache, a.seqs, t, p);
    const uint32_t words = a.items.words.value, half = a.table.at ? a.table.half : 0;
    const bool inter = a.table.layout != DMX_ROTARY_HALF, turned = VEC && 4 * w < half, second = !inter && 8 * w >= half;
    const uint32_t other = second ? 8 * w - half : 8 * w + half;  // (half layout: the word's partner)
    float c[8], s[8];
    if (turned && inter)
        angles<4>(a.table, p, 4 * w, c, s);
    else if (turned)
        angles<8>(a.table, p, second ? other : 8 * w, c, s);
    for (uint32_t h = first; h < min(first + a.items.run, a.cache.heads); ++h) {
        const int64_t row = t * a.k.token + h * a.k.head;
        float k[8];
        if constexpr (VEC) {
            load8<F32>(a.k.at, row + 8 * w, k);
            if (turned && !inter) {
                float y[8];
                load8<F32>(a.k.at, row + other, y);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float lo = second ? y[e] : k[e], hi = second ? k[e] : y[e];
                    turn(lo, hi, c[e], s[e]);
                    k[e] = second ? hi : lo;
                }
            } else if (turned) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    turn(k[2 * e], k[2 * e + 1], c[e], s[e]);
            }
        } else {
            const bool in = p >= 0 && p < (int)a.table.positions;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t ch = 8 * w + e;
                k[e] = load1<F32>(a.k.at, row + ch);
                if (ch < 2 * half) {
                    const bool high = inter ? ch & 1 : ch >= half;
                    const uint32_t partner = inter ? ch ^ 1 : high ? ch - half : ch + half;
                    const uint32_t angle = inter ? ch / 2 : high ? partner : ch;
                    const float* cs = a.table.at + 2 * ((int64_t)(in ? p : 0) * half + angle);
                    const float y = load1<F32>(a.k.at, row + partner);
                    float lo = high ? y : k[e], hi = high ? k[e] : y;
                    turn(lo, hi, in ? cs[0] : NAN, in ? cs[1] : NAN);
                    k[e] = high ? hi : lo;
                }
            }
        }
        uint32_t e;
        const uint32_t word = coded<1>(k, e);
        if (!at.ok) continue;
        const uint64_t token = at.token + ((uint64_t)h << a.cache.page_shift);
        a.cache.k_codes[token * words + w] = word;
        if ((w & 3) == 0) a.cache.k_scales[token * (words / 4) + w / 4] = (uint8_t)e;
    }
}

template <bool F32, bool VEC>
__device__ __forceinline__ void append_values(const Append& a, uint32_t item) {
    const auto [w, t, first] = value_item(a.items, item);
    if (t >= a.seqs.total) return;
    int p;
    const Slot at = slot_of_new(a.cache, a.seqs, t, p);
    const uint32_t words = a.items.words.value;
    for (uint32_t h = first; h < min(first + a.items.run, a.cache.heads); ++h) {
        const int64_t from = t * a.v.token + h * a.v.head + 8 * w;
        float v[8];
        if constexpr (VEC)
            load8<F32>(a.v.at, from, v);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = load1<F32>(a.v.at, from + e);
        uint32_t e;
        const uint32_t word = coded<8>(v, e);
        if (!at.ok) continue;
        const uint64_t token = at.token + ((uint64_t)h << a.cache.page_shift), octet = token >> 3, in = token & 7;
        a.cache.v_codes[(octet * words + w) * 8 + in] = word;
        if ((w & 3) == 0) a.cache.v_scales[(octet * (words / 4) + w / 4) * 8 + in] = (uint8_t)e;
    }
}

// Keys, values and queries are separate blocks of one launch. Loads bound it: 6743
// tokens of 32 query and 8 + 8 cache heads of 128 take 34 us, 75% of a wave's life
// waiting on them, the vector units 55% busy (rotation, codes and indexes); 32
// tokens 3.2 us. A block of 32 channels is four lanes of a wave, whose maximum needs no
// LDS, and each lane writes a word of its own.
template <bool F32, bool VEC>
__global__ __launch_bounds__(256) void k_append(const Append a) {
    const uint32_t x = threadIdx.x;
    if (blockIdx.x < a.key_blocks) return append_keys<F32, VEC>(a, blockIdx.x * 256 + x);
    if (blockIdx.x < a.cached_blocks) return append_values<F32, VEC>(a, (blockIdx.x - a.key_blocks) * 256 + x);
    const uint32_t item = (blockIdx.x - a.cached_blocks) * 256 + x;
    if constexpr (VEC)
        rotate<F32>(a.q, item);
    else
        rotate_any<F32>(a.q, item);
}

// ------------------------------------------------------------------- read --

__device__ __forceinline__ uint4 decoded(uint32_t word, uint32_t e) {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    const float scale = __uint_as_float(e << 23);
    const pair a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 0);
    const pair b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 1);
    const pair c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 2);
    const pair d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 3);
    return make_uint4(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, c),
                      __builtin_bit_cast(uint32_t, d));
}

// Blocks of keys, then (from the key_blocks-th) of values. 6743 tokens of 8 + 8
// heads of 128 take 11 us, 28 MB written: short for the chain of sequence, page and
// codes that each lane waits for; 32 tokens 2.5 us.
__global__ __launch_bounds__(256) void k_read(const Cache c, const Seqs s, const Items items, uint32_t key_blocks, uint16_t* k,
                                              uint16_t* v) {
    const uint32_t words = items.words.value;
    const bool keys = blockIdx.x < key_blocks;
    const uint32_t n = (keys ? blockIdx.x : blockIdx.x - key_blocks) * 256 + threadIdx.x;
    const auto [w, t, first] = keys ? key_item(items, n) : value_item(items, n);
    if (t >= s.total) return;
    int p;
    const Slot at = slot_of_new(c, s, t, p);
    for (uint32_t h = first; h < min(first + items.run, c.heads); ++h) {
        const uint64_t token = at.token + ((uint64_t)h << c.page_shift), octet = token >> 3, in = token & 7;
        const uint32_t e = keys ? c.k_scales[token * (words / 4) + w / 4] : c.v_scales[(octet * (words / 4) + w / 4) * 8 + in];
        const uint32_t word = keys ? c.k_codes[token * words + w] : c.v_codes[(octet * words + w) * 8 + in];
        reinterpret_cast<uint4*>(keys ? k : v)[((uint64_t)t * c.heads + h) * words + w] = decoded(word, at.ok ? e : 255u);
    }
}

// -------------------------------------------------------------- attention --

#include "kv_attention.h"

// Heads that a lane takes one after the other, so that its token's place and angles
// serve them all: more than one where there are lanes enough to fill the device
// without (256 CUs of 2048, half of them). us of 6743 tokens appended and read, and
// of 8192 rotated, with items >> 17, 18, 19: 51.8 45.8 52.4, and 33.8 30.9 30.7.
uint32_t run_of(uint64_t items, uint32_t heads) { return (uint32_t)std::min<uint64_t>({heads, 8, std::max<uint64_t>(1, items >> 18)}); }

// Completes a rotation; its items.
uint64_t rotary_items(Rotation& r, bool wide) {
    const uint32_t heads = r.in[0].heads + (r.n > 1 ? r.in[1].heads : 0), per = wide ? r.dim / 16 : r.dim / 2;
    r.run = run_of((uint64_t)r.tokens * heads * per, heads);
    const uint32_t runs = (heads + r.run - 1) / r.run;
    r.per = divisor_of(per);
    r.runs = divisor_of(runs);
    return (uint64_t)r.tokens * runs * per;
}

// The items of a call's keys and values, and their blocks.
int cached_items(const dmx_kv_cache* c, uint32_t total, Items& d, uint32_t& keys, uint32_t& values, char* err, size_t errn) {
    const uint32_t words = c->dim / 8;
    d.run = run_of((uint64_t)total * c->heads * words, c->heads);
    const uint32_t runs = (c->heads + d.run - 1) / d.run;
    d.words = divisor_of(words);
    d.runs = divisor_of(runs);
    const uint64_t each = (uint64_t)runs * words;
    return launch_blocks(total * each, keys, err, errn) || launch_blocks((total + 7ull) / 8 * 8 * each, values, err, errn);
}

}  // namespace

namespace {

// (before a call of no tokens returns)
int check_rotation(const dmx_rows* in, const dmx_rows* out, uint32_t n, uint32_t tokens, uint32_t dim, int dtype,
                   const dmx_rotary_table* table, char* err, size_t errn) {
    if (!in || !out || !table) return fail(err, errn, "null rows or table");
    if (n < 1 || n > 2) return fail(err, errn, "one or two tensors");
    if (dim == 0 || dim % 2 || dim > 65536) return fail(err, errn, "head dim odd, zero or over 65536");
    return check_dtype(dtype, err, errn) || check_table(table, dim, err, errn);
}

template <typename R>
int launch_rotation(R& r, const dmx_rows* in, const dmx_rows* out, uint32_t n, uint32_t tokens, uint32_t dim, int dtype,
                    const void* positions, int wide, const dmx_rotary_table* table, void* stream, char* err, size_t errn) {
    if (tokens >= (1u << 30)) return fail(err, errn, "too many tokens");
    if (!positions) return fail(err, errn, "null positions");
    bool vec = dim % 16 == 0 && table->dim % 16 == 0;
    for (uint32_t i = 0; i < n; ++i) {
        if (!in[i].at || !out[i].at) return fail(err, errn, "null rows");
        if (in[i].heads == 0 || in[i].heads > 65535 || in[i].heads != out[i].heads)
            return fail(err, errn, "no heads, too many, or not as many out as in");
        r.in[i] = rows_of(in + i);
        r.out[i] = rows_of(out + i);
        vec = vec && wide_rows(in + i, dtype) && wide_rows(out + i, dtype);
    }
    r.n = n, r.tokens = tokens, r.dim = dim;
    r.positions = positions, r.wide = wide;
    r.table = table_of(table);
    uint32_t blocks;
    if (launch_blocks(rotary_items(r, vec), blocks, err, errn)) return 1;
    const auto kern = vec ? (dtype == DMX_F32 ? k_rotary<true, R> : k_rotary<false, R>)
                          : (dtype == DMX_F32 ? k_rotary_any<true, R> : k_rotary_any<false, R>);
    hipLaunchKernelGGL(kern, dim3(blocks), dim3(256), 0, static_cast<hipStream_t>(stream), r);
    return launch_check(err, errn, "rotary launch");
}

}  // namespace

extern "C" int dmx_rotary(const dmx_rows* in, const dmx_rows* out, uint32_t n, uint32_t tokens, uint32_t dim, int dtype,
                          const void* positions, int wide, const dmx_rotary_table* table, void* stream, char* err,
                          size_t errn) {
    if (check_rotation(in, out, n, tokens, dim, dtype, table, err, errn)) return 1;
    if (tokens == 0) return 0;
    Rotation r = {};
    return launch_rotation(r, in, out, n, tokens, dim, dtype, positions, wide, table, stream, err, errn);
}

extern "C" int dmx_rotary_by_axes(const dmx_rows* in, const dmx_rows* out, uint32_t n, uint32_t tokens, uint32_t dim, int dtype,
                                  const void* positions, int wide, const dmx_rotary_axes* axes, const dmx_rotary_table* table,
                                  void* stream, char* err, size_t errn) {
    if (check_rotation(in, out, n, tokens, dim, dtype, table, err, errn)) return 1;
    if (!axes) return fail(err, errn, "null axes");
    if (axes->count < 1 || axes->count > 4) return fail(err, errn, "no axes, or more than 4");
    if (table->dim > 512) return fail(err, errn, "more than 256 angles");
    AxesRotation r = {};
    r.axes = axes->count;
    for (uint32_t i = 0; i < table->dim / 2; ++i) {
        const uint32_t axis = axes->of[i / 16] >> (2 * (i % 16)) & 3;
        if (axis >= axes->count) return fail(err, errn, "an angle of an axis that there is not");
        r.of[i / 16] |= axis << (2 * (i % 16));
    }
    if (tokens == 0) return 0;
    return launch_rotation(r, in, out, n, tokens, dim, dtype, positions, wide, table, stream, err, errn);
}

extern "C" int dmx_kv_append(const dmx_kv_cache* cache, const dmx_kv_seqs* seqs, const dmx_rows* k, const dmx_rows* v,
                             const dmx_rows* q, const dmx_rows* q_out, int dtype, const dmx_rotary_table* table,
                             void* stream, char* err, size_t errn) {
    if (check_cache(cache, err, errn) || check_seqs(cache, seqs, err, errn) || check_dtype(dtype, err, errn)) return 1;
    if (!k || !v || !q != !q_out) return fail(err, errn, "null keys or values, or queries without their output");
    if (q && !table) return fail(err, errn, "queries without a rotary table");
    if (table && check_table(table, cache->dim, err, errn)) return 1;
    if (k->heads != cache->heads || v->heads != cache->heads) return fail(err, errn, "keys or values of other heads than the cache's");
    if (q && (q->heads == 0 || q->heads > 65535 || q->heads != q_out->heads))
        return fail(err, errn, "no query heads, too many, or not as many out as in");
    if (seqs->total == 0) return 0;
    if (!k->at || !v->at || (q && (!q->at || !q_out->at))) return fail(err, errn, "null rows");
    Append a = {};
    a.cache = cache_of(cache);
    a.seqs = seqs_of(seqs);
    a.k = rows_of(k), a.v = rows_of(v);
    bool vec = wide_rows(k, dtype) && wide_rows(v, dtype);
    if (table) {
        a.table = table_of(table);
        vec = vec && table->dim % 16 == 0;
    }
    if (q) {
        vec = vec && wide_rows(q, dtype) && wide_rows(q_out, dtype);
        a.q.in[0] = rows_of(q), a.q.out[0] = rows_of(q_out);
        a.q.n = 1, a.q.tokens = seqs->total, a.q.dim = cache->dim;
        a.q.table = a.table;
        a.q.seqs = a.seqs;
    }
    uint32_t values, more = 0;
    if (cached_items(cache, seqs->total, a.items, a.key_blocks, values, err, errn) ||
        (q && launch_blocks(rotary_items(a.q, vec), more, err, errn)))
        return 1;
    a.cached_blocks = a.key_blocks + values;
    const auto kern = vec ? (dtype == DMX_F32 ? k_append<true, true> : k_append<false, true>)
                          : (dtype == DMX_F32 ? k_append<true, false> : k_append<false, false>);
    hipLaunchKernelGGL(kern, dim3(a.cached_blocks + more), dim3(256), 0, static_cast<hipStream_t>(stream), a);
    return launch_check(err, errn, "kv append launch");
}

extern "C" int dmx_kv_read(const dmx_kv_cache* cache, const dmx_kv_seqs* seqs, uint16_t* k, uint16_t* v, void* stream,
                           char* err, size_t errn) {
    if (check_cache(cache, err, errn) || check_seqs(cache, seqs, err, errn)) return 1;
    if (seqs->total == 0) return 0;
    if (!k || !v) return fail(err, errn, "null output");
    if (!aligned(k, 16) || !aligned(v, 16)) return fail(err, errn, "outputs not 16-byte aligned");
    Items items;
    uint32_t keys, values;
    if (cached_items(cache, seqs->total, items, keys, values, err, errn)) return 1;
    hipLaunchKernelGGL(k_read, dim3(keys + values), dim3(256), 0, static_cast<hipStream_t>(stream), cache_of(cache),
                       seqs_of(seqs), items, keys, k, v);
    return launch_check(err, errn, "kv read launch");
}

namespace {

// How a call of the attention is laid out: tiles of rows a wave, whether the
// waves take rows or tokens (over 64 rows to a cache head), and the splits of each
// sequence. fp32 takes one tile, of three pieces.
struct Plan {
    int tiles;
    bool rows;
    uint32_t tokens, row_blocks, splits;  // tokens: of a sequence, at most
};

Plan plan_of(const dmx_kv_cache* c, const dmx_kv_seqs* s, uint32_t q_heads, int dtype, uint32_t max_length,
             uint32_t window) {
    Plan p;
    const uint32_t tokens = p.tokens = s->cu ? std::min(s->max_tokens, s->total) : s->total / s->batch;
    const uint64_t rows = (uint64_t)tokens * (q_heads / c->heads);
    p.rows = rows > 64;
    p.tiles = rows <= 16 || dtype == DMX_F32 ? 1 : 2;
    const uint32_t a_block = !p.rows ? 16u * p.tiles : dtype == DMX_F32 ? 16u * kAttnWaves : 32u * prompt_waves(c->dim / 32);
    p.row_blocks = (uint32_t)((rows + a_block - 1) / a_block);
    uint64_t length = (uint64_t)s->table_cols * c->page;
    if (max_length) length = std::min<uint64_t>(length, max_length);
    if (window) length = std::min<uint64_t>(length, (uint64_t)window + tokens + 31);
    // Splits: a workgroup a CU, two where a split is still longer than 2048
    // tokens (an even deal of uneven sequences, and more loads in flight), each of
    // 128 tokens at least; contexts up to 512 tokens go unsplit, without the join.
    // Measured, 32 query and 8 key heads of 128, us by splits: 1021 tokens 10.3 (1)
    // 9.0 (8); 16384 90 (1) 14.9 (16) 13.1 (32) 15.0 (64); 32 sequences of 1024
    // 12.3 (1) 17.0 (4), of 8192 64.7 (1) 53.4 (2) 56.1 (4); 8 of 4096 27.4 (1)
    // 15.7 (4) 20.5 (32). Prompts are split only where they fill half of the CUs.
    const uint64_t groups = (uint64_t)c->heads * s->batch * std::max(1u, p.row_blocks);
    uint64_t wanted = std::max<uint64_t>(1, 256 / groups);
    if (!p.rows && length / wanted > 2048) wanted = std::max<uint64_t>(1, 512 / groups);
    const uint64_t possible = length <= 512 ? 1 : length / 128;
    p.splits = (uint32_t)std::min<uint64_t>({wanted, possible, 64, 65535 / s->batch});
    return p;
}

uint64_t workspace_of(const Plan& p, const dmx_kv_cache* c, const dmx_kv_seqs* s, uint32_t q_heads) {
    return p.splits == 1 ? 0 : (uint64_t)p.splits * s->total * q_heads * (c->dim + 4) * 4;
}

template <int W, bool WIDE>
int launch_attend(const Plan& p, int dtype, dim3 grid, hipStream_t stream, const AttnArgs& a, char* err, size_t errn) {
    const dim3 block(64 * kAttnWaves);
    if (dtype == DMX_F32) {
        if (p.rows)
            hipLaunchKernelGGL((k_attend<W, 3, 1, true, WIDE>), grid, block, 0, stream, a);
        else
            hipLaunchKernelGGL((k_attend<W, 3, 1, false, WIDE>), grid, block, 0, stream, a);
    } else if (p.rows) {
        static std::atomic<uint64_t> allowed[2] = {};
        const auto kern = a.lse ? k_attend_prompt<W, WIDE, true> : k_attend_prompt<W, WIDE, false>;
        if (allow_lds(reinterpret_cast<const void*>(kern), Set<W>::lds, allowed[a.lse != nullptr], err, errn)) return 1;
        const dim3 more(grid.x, grid.y + (rest_inside(W) && a.seqs.cu), grid.z);
        hipLaunchKernelGGL(kern, more, dim3(64 * prompt_waves(W)), Set<W>::lds, stream, a);
        if constexpr (!rest_inside(W))
            if (a.seqs.cu) hipLaunchKernelGGL(k_attend_rest<W>, dim3(grid.x, a.seqs.batch), block, 0, stream, a);
    } else if (p.tiles == 1) {
        hipLaunchKernelGGL((k_attend<W, 1, 1, false, WIDE>), grid, block, 0, stream, a);
    } else {
        hipLaunchKernelGGL((k_attend<W, 1, 2, false, WIDE>), grid, block, 0, stream, a);
    }
    return launch_check(err, errn, "kv attention launch");
}

}  // namespace

extern "C" uint64_t dmx_kv_attention_workspace(const dmx_kv_cache* cache, const dmx_kv_seqs* seqs, uint32_t q_heads,
                                               int dtype, uint32_t max_length, uint32_t window) {
    if (check_cache(cache, nullptr, 0) || check_seqs(cache, seqs, nullptr, 0) || q_heads == 0 || q_heads % cache->heads)
        return 0;
    return workspace_of(plan_of(cache, seqs, q_heads, dtype, max_length, window), cache, seqs, q_heads);
}

extern "C" int dmx_kv_attention(const dmx_kv_cache* cache, const dmx_kv_seqs* seqs, const dmx_rows* q, int dtype,
                                float scale, int causal, uint32_t window, uint32_t max_length, void* out, float* lse,
                                void* workspace, uint64_t workspace_bytes, void* stream, char* err, size_t errn) {
    if (check_cache(cache, err, errn) || check_seqs(cache, seqs, err, errn) || check_dtype(dtype, err, errn)) return 1;
    if (!q) return fail(err, errn, "null queries");
    if (q->heads == 0 || q->heads % cache->heads || q->heads > 65535)
        return fail(err, errn, "query heads not a multiple of the cache's, or too many");
    const float scale2 = scale * 1.44269504088896341f;  // (the kernels' exponentials are of 2)
    if (!(scale > 0) || !std::isfinite(scale2)) return fail(err, errn, "scale not a positive number, or too large");
    if (window >= (1u << 30)) return fail(err, errn, "window of 2^30 or more");
    if (seqs->total == 0) return 0;
    if (!q->at || !out) return fail(err, errn, "null queries or output");
    const Plan p = plan_of(cache, seqs, q->heads, dtype, max_length, window);
    if (p.row_blocks == 0) return fail(err, errn, "max_tokens is 0");
    if (p.row_blocks > 65534) return fail(err, errn, "too many query rows of one sequence");
    if (workspace_bytes < workspace_of(p, cache, seqs, q->heads) || (p.splits > 1 && !aligned(workspace, 16)) ||
        (p.splits > 1 && !workspace))
        return fail(err, errn, "workspace missing, short or not 16-byte aligned");
    AttnArgs a = {};
    a.cache = cache_of(cache);
    a.seqs = seqs_of(seqs);
    a.q = q->at, a.q_token = q->token_stride, a.q_head = q->head_stride;
    a.q_heads = q->heads, a.group = q->heads / cache->heads;
    a.scale = scale2;
    a.causal = causal != 0, a.window = window, a.splits = p.splits;
    a.seqs.each = divisor_of(p.tokens);
    a.row_blocks = p.row_blocks;
    a.out = out, a.lse = lse;
    const uint64_t all = (uint64_t)seqs->total * q->heads;
    a.part_o = static_cast<float*>(workspace);
    a.part_stat = reinterpret_cast<f32x4*>(a.part_o + (p.splits > 1 ? p.splits * all * cache->dim : 0));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid(cache->heads, p.row_blocks, seqs->batch * p.splits);
    const bool wide = cache->page >= 32;
    const auto launch = [&](auto w) {
        constexpr int W = decltype(w)::value;
        return wide ? launch_attend<W, true>(p, dtype, grid, st, a, err, errn) : launch_attend<W, false>(p, dtype, grid, st, a, err, errn);
    };
    const int rc = cache->dim == 64    ? launch(std::integral_constant<int, 2>{})
                   : cache->dim == 96  ? launch(std::integral_constant<int, 3>{})
                   : cache->dim == 128 ? launch(std::integral_constant<int, 4>{})
                   : cache->dim == 192 ? launch(std::integral_constant<int, 6>{})
                                       : launch(std::integral_constant<int, 8>{});
    if (rc) return 1;
    if (p.splits == 1) return 0;
    const int ways = p.splits > 8 ? 4 : 1;
    hipLaunchKernelGGL((dtype == DMX_F32 ? k_attend_join<true> : k_attend_join<false>),
                       dim3((uint32_t)(ways == 4 ? all : (all + 3) / 4)), dim3(256), 0, st, a, (int)cache->dim, ways);
    return launch_check(err, errn, "kv attention join launch");
}
