// What the kernels between a decoder's projections share: how sequences, cache
// and activations are seen on the device, and the checks on the host. Included by
// each of their sources.
#pragma once
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

// A divisor known to the host: n / d, n < 2^31, by a multiplication. With s the
// least for which 2^s >= d, 2^(32 + s) / d lies between 2^32 and 2^33; mul is
// its excess over 2^32, rounded up, and the error stays below 1 / d.
struct Divisor {
    uint32_t mul, shift, value;
};
__device__ __forceinline__ uint32_t operator/(uint32_t n, const Divisor& d) { return (__umulhi(n, d.mul) + n) >> d.shift; }

// n = a * d + b: a into n, b returned.
__device__ __forceinline__ uint32_t take(uint32_t& n, const Divisor& d) {
    const uint32_t a = n / d, b = n - a * d.value;
    n = a;
    return b;
}

struct Seqs {
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* cu;
    uint32_t batch, total;
    int cols;
    Divisor each;  // new tokens of each sequence (attention with cu: at most)
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
        q.count = s.each.value;
        q.token = b * q.count;
    }
    q.length = max(s.lengths[b], 0);
    q.first = q.length - q.count;
    return q;
}

// The sequence of new token t: the last one that begins at or before it.
__device__ __forceinline__ uint32_t seq_at(const Seqs& s, uint32_t t) {
    if (!s.cu) return t / s.each;
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

// The place of new token t in head 0, and its position; a further head is a
// page's tokens on. A token of no sequence (before the first offset, after the
// last, or where offsets decrease) has none.
__device__ __forceinline__ Slot slot_of_new(const Cache& c, const Seqs& s, uint32_t t, int& p) {
    const uint32_t b = seq_at(s, t);
    const Seq q = seq_of(s, b);
    p = q.first + ((int)t - q.token);
    Slot at = slot_of(c, s, b, 0, (uint32_t)max(p, 0));
    at.ok = at.ok && p >= 0 && (!s.cu || (uint32_t)((int)t - q.token) < (uint32_t)q.count);
    return at;
}

// -------------------------------------------------------------- host side --

inline int fail(char* err, size_t n, const char* msg) {
    if (err && n) {
        strncpy(err, msg, n - 1);
        err[n - 1] = 0;
    }
    return 1;
}

inline int launch_check(char* err, size_t errn, const char* what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    char msg[256];
    snprintf(msg, sizeof msg, "%s: %s", what, hipGetErrorString(e));
    return fail(err, errn, msg);
}

inline bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

inline int check_cache(const dmx_kv_cache* c, char* err, size_t errn) {
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

inline int check_seqs(const dmx_kv_cache* c, const dmx_kv_seqs* s, char* err, size_t errn) {
    if (!s) return fail(err, errn, "null sequences");
    if (!s->table || !s->lengths) return fail(err, errn, "null block table or lengths");
    if (s->batch == 0 || s->table_cols == 0) return fail(err, errn, "no sequences, or a block table without columns");
    if (s->batch > 65535 || s->total >= (1u << 30)) return fail(err, errn, "too many sequences or tokens");
    if ((uint64_t)s->table_cols * c->page >= (1ull << 30)) return fail(err, errn, "a block table of 2^30 positions or more");
    if (!s->cu && s->total % s->batch) return fail(err, errn, "tokens not a multiple of the sequences, and no cu");
    return 0;
}

inline int check_dtype(int dtype, char* err, size_t errn) {
    return dtype == DMX_BF16 || dtype == DMX_F32 ? 0 : fail(err, errn, "dtype must be DMX_BF16 or DMX_F32");
}

inline int check_table(const dmx_rotary_table* t, uint32_t dim, char* err, size_t errn) {
    if (!t->at) return fail(err, errn, "null rotary table");
    if (!aligned(t->at, 16)) return fail(err, errn, "rotary table not 16-byte aligned");
    if (t->positions == 0 || t->positions >= (1u << 31)) return fail(err, errn, "rotary table without positions, or too many");
    if (t->dim == 0 || t->dim % 2 || t->dim > dim) return fail(err, errn, "rotary dim odd, zero or over the head's");
    if (t->layout != DMX_ROTARY_HALF && t->layout != DMX_ROTARY_INTERLEAVED) return fail(err, errn, "unknown rotary layout");
    return 0;
}

inline Cache cache_of(const dmx_kv_cache* c) {
    return {c->k_codes, c->v_codes, c->k_scales, c->v_scales, c->pages, c->heads, (uint32_t)__builtin_ctz(c->page)};
}
inline Divisor divisor_of(uint32_t d) {
    uint32_t shift = 0;
    while ((1ull << shift) < d) ++shift;
    return {(uint32_t)((((1ull << shift) - d) << 32) / d + 1), shift, d};
}
inline Seqs seqs_of(const dmx_kv_seqs* s) {
    return {s->table, s->lengths, s->cu, s->batch, s->total, (int)s->table_cols, divisor_of(s->cu ? 1 : std::max(1u, s->total / s->batch))};
}
inline Rows rows_of(const dmx_rows* r) { return {r->at, r->token_stride, r->head_stride, r->heads}; }
inline Table table_of(const dmx_rotary_table* t) { return {t->at, t->positions, t->dim / 2, t->layout}; }

// Whether rows can be read and written 16 bytes at a time.
inline bool wide_rows(const dmx_rows* r, int dtype) {
    const int64_t n = dtype == DMX_F32 ? 4 : 8;
    return aligned(r->at, 16) && r->token_stride % n == 0 && r->head_stride % n == 0;
}

// Blocks of 256 for `items`, whose numbers the kernels hold in 31 bits.
inline int launch_blocks(uint64_t items, uint32_t& blocks, char* err, size_t errn) {
    if (items >= (1ull << 31) - 256) return fail(err, errn, "too many values for one launch");
    blocks = (uint32_t)((items + 255) / 256);
    return 0;
}

// A launch has fewer than 2^32 lanes along an axis.
inline int check_lanes(uint64_t groups, uint32_t threads, char* err, size_t errn) {
    return groups * threads < 1ull << 32 ? 0 : fail(err, errn, "too many tokens for one launch");
}

// Lets a kernel have `bytes` of dynamic LDS on the current device (over 64 KB
// takes an opt-in), once for each device.
inline int allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>& devices, char* err, size_t errn) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev > 63) return fail(err, errn, "no current device");
    if (devices.load() >> dev & 1) return 0;
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return fail(err, errn, "kv attention LDS opt-in refused");
    devices.fetch_or(1ull << dev);
    return 0;
}

}  // namespace
