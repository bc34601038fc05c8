// The norms around a decoder's blocks (include/dmx_norm.h).
//
// A row stays in the registers of its lanes (16, a wave, or a workgroup, 8 N
// channels a lane) from its read to its result, through as many sums over the row as
// its form takes: one read of each input, one write of each output. Memory bounds it:
// 8192 rows of 4096, norms before and after, fp32 residual, 403 MB in 79 us (5.1 TB/s, part of the reads
// cached); 4084 of 1536 with layer norm, gate, scale and shift 50 MB in 12.6; the heads of 8192 x 40 x 128
// 168 MB in 26. fp32 rows: 8192 of 4096, both norms, 537 MB in 103, the heads of 8192 x 40 x 128 336 MB in 60.
// Rows of no whole eights go a value at a time, lanes side by side: fp32 ones of 4095 111, a wave's 256 bytes a load; bf16 ones,
// 128 bytes a load and eight times the loads, 82 us for 8192 of 4095 with one norm and a bf16 residual, 42 for
// 4096 (142 with a lane's eight values side by side). One row takes 3.5 us, its launch.
#include "dmx_norm.h"

#include "kv_common.h"

namespace {

struct Vectors {
    const void* at;
    int f32;
    int by;        // row of them: 0 the only one, 1 the row divided by `per`, 2 its sequence's
    Divisor per;
};

struct Norm {
    Rows x;           // dmx_norm: rows (token, head); dmx_block_norm: the block's output
    Divisor heads;
    const void* residual;
    int64_t residual_stride;
    void *residual_out, *out;
    uint32_t rows, dim;
    uint32_t first;  // row of a launch
    int layer;
    float eps, offset, factor, inv_dim;
    Vectors weight, bias, post, gate, scale, shift;
    const int32_t* cu;
    uint32_t batch;
};

// The sum over a row's LANES lanes. `part` is one of the caller's, used once.
template <int LANES>
__device__ __forceinline__ float sum_of_row(float x, float* part) {
#pragma unroll
    for (int n = (LANES < 64 ? LANES : 64) / 2; n; n >>= 1) x += __shfl_xor(x, n);
    if constexpr (LANES > 64) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
        __syncthreads();
        x = 0.f;
#pragma unroll
        for (int w = 0; w < LANES / 64; ++w) x += part[w];
    }
    return x;
}

// load8 and store8 at any address: the machine takes 16 bytes wherever they begin, so that a
// view's rows go the way of dense ones, and sum in their order.
template <bool F32>
__device__ __forceinline__ void load8_anywhere(const void* base, int64_t at, float (&x)[8]) {
    if constexpr (F32) {
        __builtin_memcpy(x, static_cast<const float*>(base) + at, 32);
    } else {
        uint32_t w[4];
        __builtin_memcpy(w, static_cast<const uint16_t*>(base) + at, 16);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            x[2 * n] = __uint_as_float(w[n] << 16);
            x[2 * n + 1] = __uint_as_float(w[n] & 0xffff0000u);
        }
    }
}
template <bool F32>
__device__ __forceinline__ void store8_anywhere(void* base, int64_t at, const float (&x)[8]) {
    if constexpr (F32) {
        __builtin_memcpy(static_cast<float*>(base) + at, x, 32);
    } else {
        typedef __bf16 eight __attribute__((ext_vector_type(8)));
        const eight y = {(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3], (__bf16)x[4], (__bf16)x[5], (__bf16)x[6], (__bf16)x[7]};
        __builtin_memcpy(static_cast<uint16_t*>(base) + at, &y, 16);
    }
}

// Eight channels of a row of vectors, adjacent ones from `at` (STEP 1: whole rows of eight, 16 bytes
// a load), or STEP apart, so that lanes side by side read and write side by side; past `dim` 0.
template <uint32_t STEP>
__device__ __forceinline__ void vector8(const Vectors& v, int64_t row, uint32_t at, uint32_t dim, float (&x)[8]) {
    const int64_t from = row * dim + at;
    if constexpr (STEP == 1) {
        if (v.f32)
            load8_anywhere<true>(v.at, from, x);
        else
            load8_anywhere<false>(v.at, from, x);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = at + e * STEP >= dim ? 0.f : v.f32 ? load1<true>(v.at, from + e * STEP) : load1<false>(v.at, from + e * STEP);
    }
}

template <bool F32, uint32_t STEP>
__device__ __forceinline__ void row8(const void* base, int64_t row, uint32_t at, uint32_t dim, float (&x)[8]) {
    if constexpr (STEP == 1) {
        load8_anywhere<F32>(base, row + at, x);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = at + e * STEP >= dim ? 0.f : load1<F32>(base, row + at + e * STEP);
    }
}

template <bool F32, uint32_t STEP>
__device__ __forceinline__ void put8(void* base, int64_t row, uint32_t at, uint32_t dim, const float (&x)[8]) {
    if constexpr (STEP == 1) {
        store8_anywhere<F32>(base, row + at, x);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (at + e * STEP < dim) store1<F32>(base, row + at + e * STEP, x[e]);
    }
}

__device__ __forceinline__ int64_t row_of(const Norm& a, const Vectors& v, uint32_t row) {
    if (v.by == 0) return 0;
    if (v.by == 1) return row / v.per;
    uint32_t lo = 0, hi = a.batch - 1;  // the last sequence that begins at or before it
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) >> 1;
        if (a.cu[mid] <= (int)row)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

// BLOCK: dmx_block_norm, else dmx_norm. F32X, F32R: fp32 rows, fp32 residual.
template <bool BLOCK, bool F32X, bool F32R, bool VEC, int LANES, int N>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void k_norm(const Norm a) {
    __shared__ float part[4][LANES > 64 ? LANES / 64 : 1];
    const uint32_t lane = threadIdx.x % LANES;
    const uint32_t row = a.first + (LANES < 256 ? blockIdx.x * (256 / LANES) + threadIdx.x / LANES : blockIdx.x);
    if (row >= a.rows) return;
    constexpr uint32_t STEP = VEC ? 1 : LANES;
    const auto channel = [&](int n) { return 8 * n * LANES + (VEC ? 8 : 1) * lane; };

    float v[N][8], r[N][8];
    uint32_t head = row;
    int64_t from;
    if constexpr (BLOCK) {
        from = row * a.x.token;
    } else {
        const uint32_t h = take(head, a.heads);
        from = head * a.x.token + h * a.x.head;
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const uint32_t c = channel(n);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[n][e] = r[n][e] = 0.f;
        if (c >= a.dim) continue;
        row8<F32X, STEP>(a.x.at, from, c, a.dim, v[n]);
        if constexpr (BLOCK) row8<F32R, STEP>(a.residual, row * a.residual_stride, c, a.dim, r[n]);
    }

    // x less its mean (layer norm), and the factor that gives it a norm of 1
    const auto standard = [&](float (&x)[N][8], float* first, float* second) {
        if (a.layer) {
            float sum = 0.f;
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int e = 0; e < 8; ++e) sum += x[n][e];
            const float mean = sum_of_row<LANES>(sum, first) * a.inv_dim;
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int e = 0; e < 8; ++e) x[n][e] = channel(n) + e * STEP < a.dim ? x[n][e] - mean : 0.f;
        }
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(x[n][e], x[n][e], sum);
        return 1.f / sqrtf(sum_of_row<LANES>(sum, second) * a.inv_dim + a.eps);
    };

    if constexpr (BLOCK) {
        if (a.post.at) {
            const float inv = standard(v, part[0], part[1]);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                if (channel(n) >= a.dim) continue;
                float w[8];
                vector8<STEP>(a.post, 0, channel(n), a.dim, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[n][e] *= inv * (w[e] + a.offset);
            }
        }
        const int64_t gate = a.gate.at ? row_of(a, a.gate, row) : 0;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if (channel(n) >= a.dim) continue;
            if (a.gate.at) {
                float g[8];
                vector8<STEP>(a.gate, gate, channel(n), a.dim, g);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[n][e] *= g[e];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) r[n][e] = fmaf(a.factor, v[n][e], r[n][e]);
            put8<F32R, STEP>(a.residual_out, (int64_t)row * a.dim, channel(n), a.dim, r[n]);
        }
    }
    float(&x)[N][8] = BLOCK ? r : v;
    const float inv = standard(x, part[2], part[3]);
    const int64_t scale = BLOCK && a.scale.at ? row_of(a, a.scale, row) : 0;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const uint32_t c = channel(n);
        if (c >= a.dim) continue;
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[n][e] *= inv;
        if (a.weight.at) {
            vector8<STEP>(a.weight, 0, c, a.dim, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[n][e] *= w[e] + a.offset;
        }
        if (a.bias.at) {
            vector8<STEP>(a.bias, 0, c, a.dim, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[n][e] += w[e];
        }
        if (BLOCK && a.scale.at) {
            float s[8];
            vector8<STEP>(a.scale, scale, c, a.dim, s);
            vector8<STEP>(a.shift, scale, c, a.dim, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[n][e] = fmaf(x[n][e], 1.f + s[e], w[e]);
        }
        put8<F32X, STEP>(a.out, (int64_t)row * a.dim, c, a.dim, x[n]);
    }
}

// -------------------------------------------------------------- host side --

int vectors_of(const dmx_vectors& v, const char* what, uint32_t rows, const dmx_norm_form* f, Vectors& to, char* err, size_t errn) {
    to = {};
    if (!v.at) return 0;
    char msg[128];
    if (v.dtype != DMX_BF16 && v.dtype != DMX_F32) {
        snprintf(msg, sizeof msg, "%s: dtype must be DMX_BF16 or DMX_F32", what);
        return fail(err, errn, msg);
    }
    to.at = v.at, to.f32 = v.dtype == DMX_F32;
    if (v.rows == 1) return 0;
    if (f->cu && v.rows == f->batch) {
        to.by = 2;
        return 0;
    }
    if (v.rows == 0 || rows % v.rows) {
        snprintf(msg, sizeof msg, "%s: %u rows for a call of %u", what, v.rows, rows);
        return fail(err, errn, msg);
    }
    to.by = 1, to.per = divisor_of(std::max(1u, rows / v.rows));  // (a call of no rows divides by none)
    return 0;
}

int form_of(const dmx_norm_form* f, bool block, uint32_t rows, uint32_t dim, Norm& a, char* err, size_t errn) {
    if (!f) return fail(err, errn, "null form");
    if (f->kind != DMX_NORM_RMS && f->kind != DMX_NORM_LAYER) return fail(err, errn, "unknown kind of norm");
    if (!(f->eps >= 0) || !std::isfinite(f->eps)) return fail(err, errn, "eps not a number of 0 or more");
    if (!std::isfinite(f->offset) || (block && !std::isfinite(f->factor))) return fail(err, errn, "offset or factor not finite");
    if (dim == 0 || dim > DMX_NORM_MAX_DIM) return fail(err, errn, "rows of no channels, or more than 32768");
    if (rows >= (1u << 31)) return fail(err, errn, "too many rows");
    for (const dmx_vectors* v : {&f->weight, &f->bias, &f->post})
        if (v->at && v->rows != 1) return fail(err, errn, "weight, bias and post have one row");
    if (block && !f->scale.at != !f->shift.at) return fail(err, errn, "a scale without a shift, or a shift without a scale");
    if (block && f->scale.at && f->scale.rows != f->shift.rows) return fail(err, errn, "scale and shift of different rows");
    if (block && f->cu && f->batch == 0) return fail(err, errn, "offsets of no sequences");
    if (vectors_of(f->weight, "weight", rows, f, a.weight, err, errn) || vectors_of(f->bias, "bias", rows, f, a.bias, err, errn)) return 1;
    if (block && (vectors_of(f->post, "post", rows, f, a.post, err, errn) || vectors_of(f->gate, "gate", rows, f, a.gate, err, errn) ||
                  vectors_of(f->scale, "scale", rows, f, a.scale, err, errn) || vectors_of(f->shift, "shift", rows, f, a.shift, err, errn)))
        return 1;
    a.rows = rows, a.dim = dim;
    a.layer = f->kind == DMX_NORM_LAYER;
    a.eps = f->eps, a.offset = f->offset, a.factor = f->factor;
    a.inv_dim = 1.f / (float)dim;
    a.cu = f->cu, a.batch = f->batch;
    return 0;
}

template <bool BLOCK, bool F32X, bool F32R, bool VEC>
int launch(Norm a, hipStream_t stream, char* err, size_t errn) {
    const auto go = [&](auto lanes, auto runs) {
        constexpr int LANES = decltype(lanes)::value, N = decltype(runs)::value, threads = LANES < 256 ? 256 : LANES;
        constexpr uint32_t each = threads / LANES, most = 0xffffffffu / threads;  // workgroups of a launch
        for (uint64_t first = 0; first < a.rows; first += (uint64_t)most * each) {
            a.first = (uint32_t)first;
            const uint32_t groups = (a.rows - a.first + each - 1) / each;
            hipLaunchKernelGGL((k_norm<BLOCK, F32X, F32R, VEC, LANES, N>), dim3(std::min(groups, most)), dim3(threads), 0, stream, a);
        }
    };
    using std::integral_constant;
    const integral_constant<int, 1> one;
    const integral_constant<int, 2> two;
    const integral_constant<int, 4> four;
    if (a.dim <= 128) go(integral_constant<int, 16>{}, one);
    else if (a.dim <= 512) go(integral_constant<int, 64>{}, one);
    else if (a.dim <= 1024) go(integral_constant<int, 64>{}, two);
    else if (a.dim <= 2048) go(integral_constant<int, 256>{}, one);
    else if (a.dim <= 4096) go(integral_constant<int, 256>{}, two);
    else if (a.dim <= 8192) go(integral_constant<int, 1024>{}, one);
    else if (a.dim <= 16384) go(integral_constant<int, 1024>{}, two);
    else go(integral_constant<int, 1024>{}, four);
    return launch_check(err, errn, "norm launch");
}

template <bool BLOCK, bool F32X, bool F32R>
int launch(const Norm& a, hipStream_t stream, char* err, size_t errn) {
    return a.dim % 8 == 0 ? launch<BLOCK, F32X, F32R, true>(a, stream, err, errn) : launch<BLOCK, F32X, F32R, false>(a, stream, err, errn);
}

}  // namespace

extern "C" int dmx_norm(const dmx_rows* x, void* out, uint32_t tokens, uint32_t dim, int dtype, const dmx_norm_form* form,
                        void* stream, char* err, size_t errn) {
    if (check_dtype(dtype, err, errn)) return 1;
    if (!x) return fail(err, errn, "null rows");
    if (x->heads == 0 || (uint64_t)tokens * x->heads >= (1ull << 31)) return fail(err, errn, "no heads, or too many rows");
    Norm a = {};
    if (form_of(form, false, tokens * x->heads, dim, a, err, errn)) return 1;
    if (tokens == 0) return 0;
    if (!x->at || !out) return fail(err, errn, "null rows");
    a.x = rows_of(x);
    a.heads = divisor_of(x->heads);
    a.out = out;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return dtype == DMX_F32 ? launch<false, true, true>(a, st, err, errn) : launch<false, false, false>(a, st, err, errn);
}

extern "C" int dmx_block_norm(const void* y, int64_t y_stride, const void* residual, int64_t residual_stride, void* residual_out,
                              void* out, uint32_t rows, uint32_t dim, int dtype, int residual_dtype, const dmx_norm_form* form,
                              void* stream, char* err, size_t errn) {
    if (check_dtype(dtype, err, errn) || check_dtype(residual_dtype, err, errn)) return 1;
    if (dtype == DMX_F32 && residual_dtype != DMX_F32) return fail(err, errn, "a bf16 residual beside fp32 rows");
    Norm a = {};
    if (form_of(form, true, rows, dim, a, err, errn)) return 1;
    if (rows == 0) return 0;
    if (!y || !residual || !residual_out || !out) return fail(err, errn, "null rows");
    a.x = {const_cast<void*>(y), y_stride, 0, 1};
    a.residual = residual, a.residual_stride = residual_stride, a.residual_out = residual_out, a.out = out;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return dtype == DMX_F32            ? launch<true, true, true>(a, st, err, errn)
           : residual_dtype == DMX_F32 ? launch<true, false, true>(a, st, err, errn)
                                       : launch<true, false, false>(a, st, err, errn);
}
