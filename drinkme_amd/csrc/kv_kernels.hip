// The operators between a decoder's q/k/v and o projections (include/dmx_kv.h):
// gfx950 kernels and the C-ABI entry points that launch them.
//
//   k_rotary, k_rotary_any   rotary positions
//   k_append                 keys (rotated) and values into the 4-bit cache
//   k_read                   cached tokens back to bf16
//   k_attend, k_attend_join  the attention over the cache (kv_attention.h)
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "dmx_kv.h"
#include "dmx_radix.h"

namespace {

struct Cache {
    uint32_t* k_codes;
    uint32_t* v_codes;
    uint8_t* k_scales;
    uint8_t* v_scales;
    uint32_t pages, heads, page_shift;
};

struct Seqs {
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* cu;
    uint32_t batch, total;
    int cols;
};

struct Rows {
    void* at;
    int64_t token, head;  // strides, elements
    uint32_t heads;
};

struct Table {
    const float* at;
    uint32_t positions, half;  // half: angles
    int layout;
};

// ------------------------------------------------------------- sequences --

struct Seq {
    int token, count;   // its new tokens in [total]: the first one, how many
    int first, length;  // position of the first one; tokens in all
};

// Sequence b of a call. cu is clamped to [0, total], so that no token index
// leaves the call's tensors whatever it holds.
__device__ __forceinline__ Seq seq_of(const Seqs& s, uint32_t b) {
    Seq q;
    if (s.cu) {
        q.token = min(max(s.cu[b], 0), (int)s.total);
        q.count = min(max(s.cu[b + 1], q.token), (int)s.total) - q.token;
    } else {
        q.count = s.total / s.batch;
        q.token = b * q.count;
    }
    q.length = max(s.lengths[b], 0);
    q.first = q.length - q.count;
    return q;
}

// The sequence of new token t: the last one that begins at or before it.
__device__ __forceinline__ uint32_t seq_at(const Seqs& s, uint32_t t) {
    if (!s.cu) return t / (s.total / s.batch);
    uint32_t lo = 0, hi = s.batch - 1;
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) >> 1;
        if (s.cu[mid] <= (int)t)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

struct Slot {
    uint64_t token;  // (page, head, slot) as one index
    bool ok;         // false: no page there, and the index is page 0's
};

// Where position p of sequence b and a cache head lies.
__device__ __forceinline__ Slot slot_of(const Cache& c, const Seqs& s, uint32_t b, uint32_t head, uint32_t p) {
    const uint32_t col = p >> c.page_shift;
    uint32_t page = ~0u;
    if (col < (uint32_t)s.cols) page = (uint32_t)s.table[(int64_t)b * s.cols + col];
    const bool ok = page < c.pages;
    const uint32_t slot = p & ((1u << c.page_shift) - 1u);
    return {(((uint64_t)(ok ? page : 0u) * c.heads + head) << c.page_shift) + slot, ok};
}

// ------------------------------------------------------------ activations --

// Eight adjacent channels as fp32.
template <bool F32>
__device__ __forceinline__ void load8(const void* base, int64_t at, float (&x)[8]) {
    if constexpr (F32) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
        const float4 a = p[0], b = p[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            x[2 * n] = __uint_as_float(w[n] << 16);
            x[2 * n + 1] = __uint_as_float(w[n] & 0xffff0000u);
        }
    }
}

template <bool F32>
__device__ __forceinline__ void store8(void* base, int64_t at, const float (&x)[8]) {
    if constexpr (F32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + at);
        p[0] = make_float4(x[0], x[1], x[2], x[3]);
        p[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            typedef __bf16 pair __attribute__((ext_vector_type(2)));
            const pair b = {(__bf16)x[2 * n], (__bf16)x[2 * n + 1]};
            w[n] = __builtin_bit_cast(uint32_t, b);
        }
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + at) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <bool F32>
__device__ __forceinline__ float load1(const void* base, int64_t at) {
    if constexpr (F32) return static_cast<const float*>(base)[at];
    return __uint_as_float((uint32_t) static_cast<const uint16_t*>(base)[at] << 16);
}

template <bool F32>
__device__ __forceinline__ void store1(void* base, int64_t at, float x) {
    if constexpr (F32)
        static_cast<float*>(base)[at] = x;
    else
        static_cast<uint16_t*>(base)[at] = __builtin_bit_cast(uint16_t, (__bf16)x);
}

// ----------------------------------------------------------------- rotary --

// (a, b) turned: each product and the sum rounded on its own, so that a result
// does not depend on which operations a compiler joins.
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
#pragma clang fp contract(off)
    const float x = a * c - b * s, y = b * c + a * s;
    a = x;
    b = y;
}

// Eight (cos, sin) pairs from angle `first` of a position's row; NaN outside the table.
__device__ __forceinline__ void angles(const Table& t, int64_t position, uint32_t first, float (&c)[8], float (&s)[8]) {
    const bool ok = position >= 0 && position < (int64_t)t.positions;
    const float4* p = reinterpret_cast<const float4*>(t.at + 2 * ((ok ? position : 0) * t.half + first));
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const float4 v = p[n];
        c[2 * n] = ok ? v.x : NAN, s[2 * n] = ok ? v.y : NAN;
        c[2 * n + 1] = ok ? v.z : NAN, s[2 * n + 1] = ok ? v.w : NAN;
    }
}

struct Rotation {
    Rows in[2], out[2];
    uint32_t n, tokens, dim;
    const void* positions;  // null: the tokens' places in seqs
    int wide;
    Table table;
    Seqs seqs;
};

__device__ __forceinline__ int64_t position_of(const Rotation& r, uint32_t t) {
    if (r.positions)
        return r.wide ? static_cast<const int64_t*>(r.positions)[t] : static_cast<const int32_t*>(r.positions)[t];
    const Seq q = seq_of(r.seqs, seq_at(r.seqs, t));
    return (int64_t)q.first + ((int)t - q.token);
}

// Item (token, head, c) of 16 channels: two runs of 8. In the turned part the
// eight pairs of angles 8 c .. 8 c + 7, else 16 channels to copy. Takes 16-byte
// aligned rows, dim and the turned channels multiples of 16.
template <bool F32>
__device__ __forceinline__ void rotary_item(const Rotation& r, uint64_t item) {
    const uint32_t per = r.dim / 16, heads = r.in[0].heads + (r.n > 1 ? r.in[1].heads : 0);
    const uint32_t c = item % per;
    const uint64_t th = item / per;
    uint32_t h = th % heads;
    const uint32_t t = th / heads;
    if (t >= r.tokens) return;
    const int which = h >= r.in[0].heads;
    if (which) h -= r.in[0].heads;
    const Rows &in = r.in[which], &out = r.out[which];
    const int64_t from = t * in.token + h * in.head, to = t * out.token + h * out.head;
    const bool turned = 8 * c < r.table.half, split = turned && r.table.layout == DMX_ROTARY_HALF;
    const uint32_t x = split ? 8 * c : 16 * c, y = split ? 8 * c + r.table.half : 16 * c + 8;
    float a[8], b[8];
    load8<F32>(in.at, from + x, a);
    load8<F32>(in.at, from + y, b);
    if (turned) {
        float cs[8], sn[8];
        angles(r.table, position_of(r, t), 8 * c, cs, sn);
        if (split) {
#pragma unroll
            for (int e = 0; e < 8; ++e) turn(a[e], b[e], cs[e], sn[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                turn(a[2 * e], a[2 * e + 1], cs[e], sn[e]);
                turn(b[2 * e], b[2 * e + 1], cs[4 + e], sn[4 + e]);
            }
        }
    }
    store8<F32>(out.at, to + x, a);
    store8<F32>(out.at, to + y, b);
}

template <bool F32>
__global__ __launch_bounds__(256) void k_rotary(const Rotation r) {
    rotary_item<F32>(r, (uint64_t)blockIdx.x * 256 + threadIdx.x);
}

// Any sizes, strides and alignment: item (token, head, pair), a pair of
// channels an item.
template <bool F32>
__device__ __forceinline__ void rotary_item_any(const Rotation& r, uint64_t item) {
    const uint32_t per = r.dim / 2, heads = r.in[0].heads + (r.n > 1 ? r.in[1].heads : 0);
    const uint32_t c = item % per;
    const uint64_t th = item / per;
    uint32_t h = th % heads;
    const uint32_t t = th / heads;
    if (t >= r.tokens) return;
    const int which = h >= r.in[0].heads;
    if (which) h -= r.in[0].heads;
    const Rows &in = r.in[which], &out = r.out[which];
    const int64_t from = t * in.token + h * in.head, to = t * out.token + h * out.head;
    const bool turned = c < r.table.half, split = turned && r.table.layout == DMX_ROTARY_HALF;
    const uint32_t x = split ? c : 2 * c, y = split ? c + r.table.half : 2 * c + 1;
    float a = load1<F32>(in.at, from + x), b = load1<F32>(in.at, from + y);
    if (turned) {
        const int64_t p = position_of(r, t);
        const bool ok = p >= 0 && p < (int64_t)r.table.positions;
        const float* cs = r.table.at + 2 * ((ok ? p : 0) * r.table.half + c);
        turn(a, b, ok ? cs[0] : NAN, ok ? cs[1] : NAN);
    }
    store1<F32>(out.at, to + x, a);
    store1<F32>(out.at, to + y, b);
}

template <bool F32>
__global__ __launch_bounds__(256) void k_rotary_any(const Rotation r) {
    rotary_item_any<F32>(r, (uint64_t)blockIdx.x * 256 + threadIdx.x);
}

// ----------------------------------------------------------------- append --

struct Append {
    Cache cache;
    Seqs seqs;
    Rows k, v;
    uint32_t dim;
    Table table;  // at null: keys as they are
    Rotation q;   // the queries' (n 0: none)
    uint64_t cached;  // words of keys (and as many of values) that the first blocks code
    uint32_t cached_blocks;
};

// The codes of a lane's eight channels; four adjacent lanes hold a block of 32,
// whose exponent byte each of them returns.
__device__ __forceinline__ uint32_t coded(const float (&x)[8], uint32_t& e) {
    uint32_t top = 0;  // as integers, NaN above infinity above every number
#pragma unroll
    for (int n = 0; n < 8; ++n) top = max(top, __float_as_uint(x[n]) & 0x7fffffffu);
    top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xB1, 0xF, 0xF, true));  // lane ^ 1
    top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4E, 0xF, 0xF, true));  // lane ^ 2
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

// Word (token, head, w) of the keys and of the values. VEC: 16-byte aligned
// rows, and the turned channels a multiple of 16.
template <bool F32, bool VEC>
__device__ __forceinline__ void append_word(const Append& a, uint64_t item) {
    if (item >= a.cached) return;
    const uint32_t words = a.dim / 8, w = item % words;
    const uint64_t th = item / words;
    const uint32_t h = th % a.cache.heads, t = th / a.cache.heads;
    const uint32_t b = seq_at(a.seqs, t);
    const Seq q = seq_of(a.seqs, b);
    const int p = q.first + ((int)t - q.token);
    const Slot at = slot_of(a.cache, a.seqs, b, h, (uint32_t)max(p, 0));
    const bool ok = at.ok && p >= 0;
    const int64_t kat = t * a.k.token + h * a.k.head, vat = t * a.v.token + h * a.v.head;
    float k[8], v[8];
    if constexpr (VEC) {
        load8<F32>(a.k.at, kat + 8 * w, k);
        load8<F32>(a.v.at, vat + 8 * w, v);
        if (a.table.at && 4 * w < a.table.half) {
            const uint32_t half = a.table.half;
            float c[8], s[8];
            if (a.table.layout == DMX_ROTARY_HALF) {
                const bool second = 8 * w >= half;
                const uint32_t other = second ? 8 * w - half : 8 * w + half;
                float y[8];
                load8<F32>(a.k.at, kat + other, y);
                angles(a.table, p, second ? other : 8 * w, c, s);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float lo = second ? y[e] : k[e], hi = second ? k[e] : y[e];
                    turn(lo, hi, c[e], s[e]);
                    k[e] = second ? hi : lo;
                }
            } else {
                angles(a.table, p, (4 * w) & ~7u, c, s);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    turn(k[2 * e], k[2 * e + 1], (w & 1) ? c[4 + e] : c[e], (w & 1) ? s[4 + e] : s[e]);
            }
        }
    } else {
        const bool in = a.table.at && p >= 0 && p < (int)a.table.positions;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t ch = 8 * w + e, half = a.table.half;
            k[e] = load1<F32>(a.k.at, kat + ch);
            v[e] = load1<F32>(a.v.at, vat + ch);
            if (a.table.at && ch < 2 * half) {
                const bool inter = a.table.layout != DMX_ROTARY_HALF, second = inter ? ch & 1 : ch >= half;
                const uint32_t other = inter ? ch ^ 1 : second ? ch - half : ch + half;
                const uint32_t angle = inter ? ch / 2 : second ? other : ch;
                const float* cs = a.table.at + 2 * ((int64_t)(in ? p : 0) * half + angle);
                const float y = load1<F32>(a.k.at, kat + other);
                float lo = second ? y : k[e], hi = second ? k[e] : y;
                turn(lo, hi, in ? cs[0] : NAN, in ? cs[1] : NAN);
                k[e] = second ? hi : lo;
            }
        }
    }
    uint32_t ke, ve;
    const uint32_t kw = coded(k, ke), vw = coded(v, ve);
    if (!ok) return;
    a.cache.k_codes[at.token * words + w] = kw;
    const uint64_t octet = at.token >> 3, in_octet = at.token & 7;
    a.cache.v_codes[(octet * words + w) * 8 + in_octet] = vw;
    if ((w & 3) == 0) {
        a.cache.k_scales[at.token * (words / 4) + w / 4] = (uint8_t)ke;
        a.cache.v_scales[(octet * (words / 4) + w / 4) * 8 + in_octet] = (uint8_t)ve;
    }
}

template <bool F32, bool VEC>
__global__ __launch_bounds__(256) void k_append(const Append a) {
    if (blockIdx.x < a.cached_blocks) {
        append_word<F32, VEC>(a, (uint64_t)blockIdx.x * 256 + threadIdx.x);
        return;
    }
    const uint64_t item = (uint64_t)(blockIdx.x - a.cached_blocks) * 256 + threadIdx.x;
    if constexpr (VEC)
        rotary_item<F32>(a.q, item);
    else
        rotary_item_any<F32>(a.q, item);
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

__global__ __launch_bounds__(256) void k_read(const Cache c, const Seqs s, uint32_t dim, uint16_t* k, uint16_t* v) {
    const uint64_t item = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    const uint32_t words = dim / 8, w = item % words;
    const uint64_t th = item / words;
    const uint32_t h = th % c.heads;
    if (th / c.heads >= s.total) return;
    const uint32_t t = th / c.heads, b = seq_at(s, t);
    const Seq q = seq_of(s, b);
    const int p = q.first + ((int)t - q.token);
    const Slot at = slot_of(c, s, b, h, (uint32_t)max(p, 0));
    const bool ok = at.ok && p >= 0;
    const uint64_t octet = at.token >> 3, in_octet = at.token & 7;
    const uint32_t ke = c.k_scales[at.token * (words / 4) + w / 4];
    const uint32_t ve = c.v_scales[(octet * (words / 4) + w / 4) * 8 + in_octet];
    reinterpret_cast<uint4*>(k)[item] = decoded(c.k_codes[at.token * words + w], ok ? ke : 255u);
    reinterpret_cast<uint4*>(v)[item] = decoded(c.v_codes[(octet * words + w) * 8 + in_octet], ok ? ve : 255u);
}

// -------------------------------------------------------------- attention --

#include "kv_attention.h"

// -------------------------------------------------------------- host side --

int fail(char* err, size_t n, const char* msg) {
    if (err && n) {
        strncpy(err, msg, n - 1);
        err[n - 1] = 0;
    }
    return 1;
}

int launch_check(char* err, size_t errn, const char* what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    char msg[256];
    snprintf(msg, sizeof msg, "%s: %s", what, hipGetErrorString(e));
    return fail(err, errn, msg);
}

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int check_cache(const dmx_kv_cache* c, char* err, size_t errn) {
    if (!c) return fail(err, errn, "null cache");
    if (!c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales) return fail(err, errn, "null cache buffer");
    if (!aligned(c->k_codes, 16) || !aligned(c->v_codes, 16) || !aligned(c->k_scales, 8) || !aligned(c->v_scales, 8))
        return fail(err, errn, "cache buffers not aligned (codes 16 bytes, scales 8)");
    if (c->pages == 0 || c->heads == 0) return fail(err, errn, "empty cache");
    if (c->pages >= (1u << 31) || c->heads > 65535) return fail(err, errn, "cache of too many pages or heads");
    if (c->page < 8 || c->page > 1024 || (c->page & (c->page - 1))) return fail(err, errn, "page not a power of two, 8..1024");
    if (c->dim != 64 && c->dim != 96 && c->dim != 128 && c->dim != 192 && c->dim != 256)
        return fail(err, errn, "head dim not 64, 96, 128, 192 or 256");
    return 0;
}

int check_seqs(const dmx_kv_cache* c, const dmx_kv_seqs* s, char* err, size_t errn) {
    if (!s) return fail(err, errn, "null sequences");
    if (!s->table || !s->lengths) return fail(err, errn, "null block table or lengths");
    if (s->batch == 0 || s->table_cols == 0) return fail(err, errn, "no sequences, or a block table without columns");
    if (s->batch > 65535 || s->total >= (1u << 30)) return fail(err, errn, "too many sequences or tokens");
    if ((uint64_t)s->table_cols * c->page >= (1ull << 30)) return fail(err, errn, "a block table of 2^30 positions or more");
    if (!s->cu && s->total % s->batch) return fail(err, errn, "tokens not a multiple of the sequences, and no cu");
    return 0;
}

int check_dtype(int dtype, char* err, size_t errn) {
    return dtype == DMX_BF16 || dtype == DMX_F32 ? 0 : fail(err, errn, "dtype must be DMX_BF16 or DMX_F32");
}

int check_table(const dmx_rotary_table* t, uint32_t dim, char* err, size_t errn) {
    if (!t->at) return fail(err, errn, "null rotary table");
    if (!aligned(t->at, 16)) return fail(err, errn, "rotary table not 16-byte aligned");
    if (t->positions == 0 || t->positions >= (1u << 31)) return fail(err, errn, "rotary table without positions, or too many");
    if (t->dim == 0 || t->dim % 2 || t->dim > dim) return fail(err, errn, "rotary dim odd, zero or over the head's");
    if (t->layout != DMX_ROTARY_HALF && t->layout != DMX_ROTARY_INTERLEAVED) return fail(err, errn, "unknown rotary layout");
    return 0;
}

Cache cache_of(const dmx_kv_cache* c) {
    return {c->k_codes, c->v_codes, c->k_scales, c->v_scales, c->pages, c->heads, (uint32_t)__builtin_ctz(c->page)};
}
Seqs seqs_of(const dmx_kv_seqs* s) { return {s->table, s->lengths, s->cu, s->batch, s->total, (int)s->table_cols}; }
Rows rows_of(const dmx_rows* r) { return {r->at, r->token_stride, r->head_stride, r->heads}; }
Table table_of(const dmx_rotary_table* t) { return {t->at, t->positions, t->dim / 2, t->layout}; }

// Whether rows can be read and written 16 bytes at a time.
bool wide_rows(const dmx_rows* r, int dtype) {
    const int64_t n = dtype == DMX_F32 ? 4 : 8;
    return aligned(r->at, 16) && r->token_stride % n == 0 && r->head_stride % n == 0;
}

int launch_blocks(uint64_t items, uint32_t& blocks, char* err, size_t errn) {
    const uint64_t n = (items + 255) / 256;
    if (n >= (1ull << 31)) return fail(err, errn, "too many values for one launch");
    blocks = (uint32_t)n;
    return 0;
}

uint64_t rotary_items(const Rotation& r, bool wide) {
    const uint64_t heads = r.in[0].heads + (r.n > 1 ? r.in[1].heads : 0);
    return (uint64_t)r.tokens * heads * (wide ? r.dim / 16 : r.dim / 2);
}

}  // namespace

extern "C" int dmx_rotary(const dmx_rows* in, const dmx_rows* out, uint32_t n, uint32_t tokens, uint32_t dim, int dtype,
                          const void* positions, int wide, const dmx_rotary_table* table, void* stream, char* err,
                          size_t errn) {
    if (!in || !out || !table) return fail(err, errn, "null rows or table");
    if (n < 1 || n > 2) return fail(err, errn, "one or two tensors");
    if (dim == 0 || dim % 2 || dim > 65536) return fail(err, errn, "head dim odd, zero or over 65536");
    if (check_dtype(dtype, err, errn) || check_table(table, dim, err, errn)) return 1;
    if (tokens == 0) return 0;
    if (tokens >= (1u << 30)) return fail(err, errn, "too many tokens");
    if (!positions) return fail(err, errn, "null positions");
    Rotation r = {};
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
    const auto kern = vec ? (dtype == DMX_F32 ? k_rotary<true> : k_rotary<false>)
                          : (dtype == DMX_F32 ? k_rotary_any<true> : k_rotary_any<false>);
    hipLaunchKernelGGL(kern, dim3(blocks), dim3(256), 0, static_cast<hipStream_t>(stream), r);
    return launch_check(err, errn, "rotary launch");
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
    a.dim = cache->dim;
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
    a.cached = (uint64_t)seqs->total * cache->heads * (cache->dim / 8);
    uint32_t more = 0;
    if (launch_blocks(a.cached, a.cached_blocks, err, errn) || (q && launch_blocks(rotary_items(a.q, vec), more, err, errn)))
        return 1;
    if ((uint64_t)a.cached_blocks + more >= (1ull << 31)) return fail(err, errn, "too many values for one launch");
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
    uint32_t blocks;
    if (launch_blocks((uint64_t)seqs->total * cache->heads * (cache->dim / 8), blocks, err, errn)) return 1;
    hipLaunchKernelGGL(k_read, dim3(blocks), dim3(256), 0, static_cast<hipStream_t>(stream), cache_of(cache),
                       seqs_of(seqs), cache->dim, k, v);
    return launch_check(err, errn, "kv read launch");
}

namespace {

// How a call of the attention is laid out: tiles of rows a wave, whether the
// waves take rows or tokens, and the splits of each sequence.
struct Plan {
    int tiles;
    bool rows;
    uint32_t row_blocks, splits;
};

Plan plan_of(const dmx_kv_cache* c, const dmx_kv_seqs* s, uint32_t q_heads, int dtype, uint32_t max_length,
             uint32_t window) {
    Plan p;
    const uint32_t tokens = s->cu ? s->max_tokens : s->total / s->batch;
    const uint64_t rows = (uint64_t)tokens * (q_heads / c->heads);
    const int most = dtype == DMX_F32 ? 1 : 2;
    p.rows = rows > 64;
    p.tiles = p.rows ? most : (int)std::min<uint64_t>(most, rows <= 16 ? 1 : rows <= 32 ? 2 : 4);
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
    return p.splits == 1 ? 0 : (uint64_t)p.splits * s->total * q_heads * (c->dim + 2) * 4;
}

// Lets a kernel have `bytes` of dynamic LDS on the current device (over 64 KB
// takes an opt-in), once for each device.
int allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>& devices, char* err, size_t errn) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev > 63) return fail(err, errn, "no current device");
    if (devices.load() >> dev & 1) return 0;
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return fail(err, errn, "kv attention LDS opt-in refused");
    devices.fetch_or(1ull << dev);
    return 0;
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
        static std::atomic<uint64_t> allowed{0};
        if (allow_lds(reinterpret_cast<const void*>(k_attend_prompt<W, WIDE>), Set<W>::lds, allowed, err, errn)) return 1;
        hipLaunchKernelGGL((k_attend_prompt<W, WIDE>), grid, dim3(64 * prompt_waves(W)), Set<W>::lds, stream, a);
    } else if (p.tiles == 1) {
        hipLaunchKernelGGL((k_attend<W, 1, 1, false, WIDE>), grid, block, 0, stream, a);
    } else if (p.tiles == 2) {
        hipLaunchKernelGGL((k_attend<W, 1, 2, false, WIDE>), grid, block, 0, stream, a);
    } else if constexpr (W <= 4) {
        hipLaunchKernelGGL((k_attend<W, 1, 4, false, WIDE>), grid, block, 0, stream, a);
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
    if (!(scale > 0) || !std::isfinite(scale)) return fail(err, errn, "scale not a positive number");
    if (window >= (1u << 30)) return fail(err, errn, "window of 2^30 or more");
    if (seqs->total == 0) return 0;
    if (!q->at || !out) return fail(err, errn, "null queries or output");
    const Plan p = plan_of(cache, seqs, q->heads, dtype, max_length, window);
    if (p.row_blocks == 0) return fail(err, errn, "max_tokens is 0");
    if (p.row_blocks > 65535) return fail(err, errn, "too many query rows of one sequence");
    if (workspace_bytes < workspace_of(p, cache, seqs, q->heads) || (p.splits > 1 && !aligned(workspace, 16)) ||
        (p.splits > 1 && !workspace))
        return fail(err, errn, "workspace missing, short or not 16-byte aligned");
    AttnArgs a = {};
    a.cache = cache_of(cache);
    a.seqs = seqs_of(seqs);
    a.q = q->at, a.q_token = q->token_stride, a.q_head = q->head_stride;
    a.q_heads = q->heads, a.group = q->heads / cache->heads;
    a.scale = scale * 1.44269504088896341f;
    a.causal = causal != 0, a.window = window, a.splits = p.splits;
    a.out = out, a.lse = lse;
    const uint64_t all = (uint64_t)seqs->total * q->heads;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + (p.splits > 1 ? p.splits * all * cache->dim : 0));
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
