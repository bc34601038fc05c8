// The pages of the 4-bit cache handed out and taken back on the device
// (include/dmx_kv.h).
//
//   k_reserve, k_slots   pages, offsets, positions and slots of a step's new tokens
//   k_trim               sequences cut back, their pages to the pool
//
// Running sums over the sequences order everything, so one workgroup makes them;
// what it does for each page and token is spread over its 1024 lanes, which find
// their sequence in the sums by bisection. Its start and dependent loads bound it: 32 sequences of 5 tokens
// 4.2 us and 3.6 to trim them; 64 prompts of 58 000 tokens in pages of 16 5.7, 3.6 for the slots, 7.0.
#include "kv_common.h"

namespace {

constexpr int kLanes = 1024, kWaves = kLanes / 64;
constexpr int kCap = (1 << 30) - 1;  // sums of pages stop here, which no pool reaches, and lengths

struct Pages {
    int32_t* free;
    int32_t* count;
    int32_t* lacking;
    int pages;
    int32_t* table;
    int32_t* lengths;
    const int32_t* given;  // new tokens (k_reserve, null: `each` of them), tokens kept (k_trim)
    int each, batch, cols, shift, total;
    int32_t* cu;
    int32_t* positions;
    int64_t* slots;
};

// x plus those of the lanes before it, over the workgroup, at most `cap` (x in 0 .. cap,
// below 2^30). `part` is the caller's; its next use lies a barrier away.
__device__ __forceinline__ int running_sum(int x, int cap, int (&part)[kWaves]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int n = 1; n < 64; n *= 2) {
        const int y = __shfl_up(x, n);
        if (lane >= n) x = min(x + y, cap);
    }
    if (lane == 63) part[wave] = x;
    __syncthreads();
    int y = lane < wave && lane < kWaves ? part[lane] : 0;  // (a lane each: up to 15 waves before this one)
#pragma unroll
    for (int n = kWaves / 2; n; n >>= 1) y = min(y + __shfl_xor(y, n), cap);
    return min(x + __shfl(y, 0), cap);
}

// The first of sums [0, n) that is over x (there is one).
__device__ __forceinline__ int first_over(const int* sums, int n, int x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] > x)
            hi = mid;
        else
            lo = mid + 1;
    }
    return lo;
}

// Where new token t of a sequence of `length` tokens before `first` lies.
__device__ __forceinline__ void place(const Pages& a, int t, int b, int first, int length) {
    const int p = length + (t - first), col = p >> a.shift;
    int page = -1;
    if (col < a.cols) page = a.table[(int64_t)b * a.cols + col];
    a.positions[t] = p;
    a.slots[t] = page >= 0 && page < a.pages ? ((int64_t)page << a.shift) + (p & ((1 << a.shift) - 1)) : -1;
}

// TOKENS: this launch places the tokens, too; else k_slots does.
template <bool TOKENS>
__global__ __launch_bounds__(kLanes) void k_reserve(const Pages a) {
    __shared__ int part[2][kWaves], tokens[kLanes], pages[kLanes], held[kLanes];
    const int x = threadIdx.x, round = (1 << a.shift) - 1;
    const int have = min(max(*a.count, 0), a.pages);
    int token = 0, page = 0;  // of the sequences before this turn's
    if (x == 0) a.cu[0] = 0;
    for (int b0 = 0; b0 < a.batch; b0 += kLanes) {
        const int b = b0 + x, n = min(kLanes, a.batch - b0);
        int length = 0, count = 0;
        if (b < a.batch) {
            length = min(max(a.lengths[b], 0), kCap);
            count = min(a.given ? max(a.given[b], 0) : a.each, a.total);
        }
        const int end = min(token + running_sum(count, a.total, part[0]), a.total);
        tokens[x] = end;
        held[x] = length;
        __syncthreads();
        const int first = x ? tokens[x - 1] : token;
        count = end - first;
        const int from = (length + round) >> a.shift, need = max(min((int)((uint32_t)(length + count + round) >> a.shift), a.cols) - from, 0);
        pages[x] = running_sum(need, kCap, part[1]);
        if (b < a.batch) {
            a.cu[b + 1] = end;
            a.lengths[b] = length + count;
        }
        __syncthreads();
        const int wanted = pages[n - 1];
        for (int k = x; k < wanted; k += kLanes) {
            const int s = first_over(pages, n, k), before = s ? pages[s - 1] : 0;
            const int at = have - 1 - min(page + k, kCap);
            a.table[(int64_t)(b0 + s) * a.cols + ((held[s] + round) >> a.shift) + (k - before)] = at >= 0 ? a.free[at] : -1;
        }
        const int last = tokens[n - 1];
        if constexpr (TOKENS) {
            __syncthreads();
            for (int t = token + x; t < last; t += kLanes) {
                const int s = first_over(tokens, n, t);
                place(a, t, b0 + s, s ? tokens[s - 1] : token, held[s]);
            }
        }
        token = last;
        page = min(page + wanted, kCap);
        __syncthreads();
    }
    if constexpr (TOKENS)
        for (int t = token + x; t < a.total; t += kLanes) {
            a.positions[t] = -1;
            a.slots[t] = -1;
        }
    if (x == 0) {
        *a.count = max(have - page, 0);
        *a.lacking = max(page - have, 0);
    }
}

__global__ __launch_bounds__(256) void k_slots(const Pages a) {
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= a.total) return;
    if (t >= a.cu[a.batch]) {
        a.positions[t] = -1;
        a.slots[t] = -1;
        return;
    }
    const int b = first_over(a.cu + 1, a.batch, t), first = a.cu[b];
    place(a, t, b, first, a.lengths[b] - (a.cu[b + 1] - first));
}

// From the last sequence's last column backwards, so that the stack's top is
// the first sequence's first.
__global__ __launch_bounds__(kLanes) void k_trim(const Pages a) {
    __shared__ int part[kWaves], columns[kLanes], first[kLanes], found[2][kWaves];
    const int x = threadIdx.x, lane = x & 63, wave = x >> 6, round = (1 << a.shift) - 1;
    int have = min(max(*a.count, 0), a.pages), turn = 0;
    for (int b0 = 0; b0 < a.batch; b0 += kLanes) {
        // (lane x: sequence b, the last one first)
        const int b = a.batch - 1 - b0 - x, n = min(kLanes, a.batch - b0);
        int gone = 0, from = 0;
        if (b >= 0) {
            const int length = min(max(a.lengths[b], 0), kCap), keep = min(max(a.given[b], 0), length);
            from = min((keep + round) >> a.shift, a.cols);
            gone = min((length + round) >> a.shift, a.cols) - from;
            a.lengths[b] = keep;
        }
        columns[x] = running_sum(gone, kCap, part);
        first[x] = from;
        __syncthreads();
        const int all = columns[n - 1];
        for (int k0 = 0; k0 < all; k0 += kLanes, turn ^= 1) {
            const int k = k0 + x;
            int page = -1;
            if (k < all) {
                const int s = first_over(columns, n, k), before = s ? columns[s - 1] : 0;
                int32_t* at = a.table + (int64_t)(a.batch - 1 - b0 - s) * a.cols + first[s] + (columns[s] - before - 1 - (k - before));
                page = *at;
                *at = -1;
            }
            const bool back = page >= 0 && page < a.pages;
            const uint64_t m = __ballot(back);
            if (lane == 0) found[turn][wave] = __popcll(m);
            __syncthreads();
            int at = have, here = 0;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                at += w < wave ? found[turn][w] : 0;
                here += found[turn][w];
            }
            at += (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
            if (back && at < a.pages) a.free[at] = page;
            have = min(have + here, a.pages);
        }
        __syncthreads();
    }
    if (x == 0) *a.count = have;
}

// -------------------------------------------------------------- host side --

int check_pages(const dmx_kv_pool* pool, const int32_t* table, const int32_t* lengths, uint32_t batch, uint32_t table_cols,
                uint32_t page, char* err, size_t errn) {
    if (!pool || !pool->free || !pool->count || !pool->lacking) return fail(err, errn, "null pool");
    if (pool->pages == 0 || pool->pages >= (1u << 30)) return fail(err, errn, "pool of no pages, or too many");
    if (!table || !lengths) return fail(err, errn, "null block table or lengths");
    if (batch == 0 || table_cols == 0) return fail(err, errn, "no sequences, or a block table without columns");
    if (batch > 65535) return fail(err, errn, "too many sequences");
    if (page < 8 || page > 1024 || (page & (page - 1))) return fail(err, errn, "page not a power of two, 8..1024");
    if ((uint64_t)table_cols * page >= (1ull << 30)) return fail(err, errn, "a block table of 2^30 positions or more");
    return 0;
}

Pages pages_of(const dmx_kv_pool* pool, int32_t* table, int32_t* lengths, const int32_t* given, uint32_t batch,
               uint32_t table_cols, uint32_t page) {
    Pages a = {};
    a.free = pool->free, a.count = pool->count, a.lacking = pool->lacking, a.pages = (int)pool->pages;
    a.table = table, a.lengths = lengths, a.given = given;
    a.batch = (int)batch, a.cols = (int)table_cols, a.shift = __builtin_ctz(page);
    return a;
}

}  // namespace

extern "C" int dmx_kv_reserve(const dmx_kv_pool* pool, int32_t* table, int32_t* lengths, const int32_t* added, uint32_t batch,
                              uint32_t table_cols, uint32_t page, uint32_t total, int32_t* cu, int32_t* positions,
                              int64_t* slots, void* stream, char* err, size_t errn) {
    if (check_pages(pool, table, lengths, batch, table_cols, page, err, errn)) return 1;
    if (total >= (1u << 30)) return fail(err, errn, "too many tokens");
    if (!added && total % batch) return fail(err, errn, "tokens not a multiple of the sequences, and no numbers of them");
    if (!cu || (total && (!positions || !slots))) return fail(err, errn, "null offsets, positions or slots");
    Pages a = pages_of(pool, table, lengths, added, batch, table_cols, page);
    a.total = (int)total, a.each = (int)(total / batch);
    a.cu = cu, a.positions = positions, a.slots = slots;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool one = total <= 4096;  // (four tokens a lane; a second launch takes 2 us at least)
    hipLaunchKernelGGL((one ? k_reserve<true> : k_reserve<false>), dim3(1), dim3(kLanes), 0, st, a);
    if (launch_check(err, errn, "kv reserve launch")) return 1;
    if (one) return 0;
    hipLaunchKernelGGL(k_slots, dim3((total + 255) / 256), dim3(256), 0, st, a);
    return launch_check(err, errn, "kv slots launch");
}

extern "C" int dmx_kv_trim(const dmx_kv_pool* pool, int32_t* table, int32_t* lengths, const int32_t* keep, uint32_t batch,
                           uint32_t table_cols, uint32_t page, void* stream, char* err, size_t errn) {
    if (check_pages(pool, table, lengths, batch, table_cols, page, err, errn)) return 1;
    if (!keep) return fail(err, errn, "null numbers of tokens to keep");
    const Pages a = pages_of(pool, table, lengths, keep, batch, table_cols, page);
    hipLaunchKernelGGL(k_trim, dim3(1), dim3(kLanes), 0, static_cast<hipStream_t>(stream), a);
    return launch_check(err, errn, "kv trim launch");
}
