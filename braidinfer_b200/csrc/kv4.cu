// A cache held in 4 bits (kv4.cuh has the format): the tables of a step, the write of new keys and values, their reading
// back, and the plain attention that the tensor-core kernel (attn_kv4.cu) is checked against.
#include "kv4.cuh"
#include <cuda_fp16.h>
#include <type_traits>

// ------------------------------------------------------------------ tables of a step
// From the lengths of n requests (q_len new tokens behind kv_before cached ones) and their pages, packed one request after
// another (request i has ceil((kv_before + q_len) / 64) of them, -1 where a block was given back):
//   q_start[i]       sum of q_len before i
//   page_table[i, c] the request's pages, -1 beyond
//   positions[r], token_seq[r], place[r] = page * 64 + position % 64 of every row (0, -1, -1 for rows past the requests')
// Every CTA adds the lengths up itself (n of them, in shared memory) and then fills its share of the tables, so that one launch does.
struct TablesArgs {
    const int* q_len;
    const int* kv_before;
    const int* pages;
    int* page_table;
    int* place;
    int* positions;              // these three may be null
    int* token_seq;
    int* q_start;
    int n, n_pages_listed, rows, cols, num_pages;
    int* error_flag;
};

#define TABLES_THREADS 256
#define TABLES_PER_THREAD 4
#define TABLES_MAX_REQUESTS 12288

__global__ void __launch_bounds__(TABLES_THREADS)
step_tables_kernel(TablesArgs a) {
    pdl_trigger();
    pdl_wait();
    extern __shared__ int tab_smem[];
    int* q0 = tab_smem;                                       // [n + 1] rows before request i
    int* b0 = q0 + a.n + 1;                                   // [n + 1] pages before request i
    __shared__ long long part[2][TABLES_THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    bool bad = false;
    const int per = (a.n + TABLES_THREADS - 1) / TABLES_THREADS;
    const int lo = min(a.n, tid * per), hi = min(a.n, lo + per);
    auto lengths = [&](int i, long long& q, long long& b) {
        q = a.q_len[i];
        long long before = a.kv_before[i];
        if (q < 0 || before < 0) { bad = true; q = max(q, 0LL); before = max(before, 0LL); }
        b = (q + before + BRAID_PAGE_SIZE - 1) / BRAID_PAGE_SIZE;
        if (b > a.cols) { bad = true; }
    };
    long long sq = 0, sb = 0;
    for (int i = lo; i < hi; ++i) {
        long long q, b;
        lengths(i, q, b);
        sq += q;
        sb += b;
    }
    long long iq = sq, ib = sb;                               // inclusive sums over the warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long uq = __shfl_up_sync(0xffffffffu, iq, o), ub = __shfl_up_sync(0xffffffffu, ib, o);
        if (lane >= o) { iq += uq; ib += ub; }
    }
    if (lane == 31) { part[0][warp] = iq; part[1][warp] = ib; }
    __syncthreads();
    long long tq = iq - sq, tb = ib - sb;                     // exclusive
    for (int w = 0; w < warp; ++w) { tq += part[0][w]; tb += part[1][w]; }
    for (int i = lo; i < hi; ++i) {
        long long q, b;
        lengths(i, q, b);
        q0[i] = (int)min(tq, (long long)a.rows);              // what does not fit is cut off, and flagged
        b0[i] = (int)min(tb, (long long)a.n_pages_listed);
        if (a.q_start && blockIdx.x == 0) a.q_start[i] = q0[i];
        tq += q;
        tb += b;
        if (tq > a.rows || tb > a.n_pages_listed) bad = true;
        if (i == a.n - 1) { q0[a.n] = (int)min(tq, (long long)a.rows); b0[a.n] = (int)min(tb, (long long)a.n_pages_listed); }
    }
    if (a.n == 0 && tid == 0) q0[0] = b0[0] = 0;              // no request: all rows are padding
    if (bad) atomicExch(a.error_flag, 1);
    __syncthreads();
    auto page_of = [&](int i, long long c) {
        if (c >= b0[i + 1] - b0[i]) return -1;
        const int p = a.pages[b0[i] + c];
        if (p < -1 || p >= a.num_pages) { atomicExch(a.error_flag, 1); return -1; }
        return p;
    };
    const long long items = (long long)a.rows + (long long)a.n * a.cols;
    const long long base = (long long)blockIdx.x * (TABLES_THREADS * TABLES_PER_THREAD) + tid;
#pragma unroll
    for (int k = 0; k < TABLES_PER_THREAD; ++k) {
        const long long it = base + k * TABLES_THREADS;
        if (it >= items) break;
        if (it < a.rows) {
            const int r = (int)it;
            int pos = 0, seq = -1, place = -1;
            if (r < q0[a.n]) {
                int x = 0, y = a.n;                           // the last request whose first row is not after r
                while (y - x > 1) {
                    const int m = (x + y) >> 1;
                    if (q0[m] <= r) x = m; else y = m;
                }
                seq = x;
                const long long at = (long long)max(a.kv_before[x], 0) + (r - q0[x]);
                pos = (int)at;
                const int page = page_of(x, at / BRAID_PAGE_SIZE);
                if (page >= 0) place = page * BRAID_PAGE_SIZE + (int)(at % BRAID_PAGE_SIZE);
                else atomicExch(a.error_flag, 1);             // a new token needs its page
            }
            a.place[r] = place;
            if (a.positions) a.positions[r] = pos;
            if (a.token_seq) a.token_seq[r] = seq;
        } else {
            const long long cell = it - a.rows;
            const int i = (int)(cell / a.cols), c = (int)(cell - (long long)i * a.cols);
            a.page_table[cell] = page_of(i, c);
        }
    }
}

// The entry points take their arguments as one structure that the caller fills in (csrc/api.py has the layouts): a call with one pointer
// costs the host a fraction of one with twenty arguments.
extern "C" int braid_step_tables(const TablesArgs* args, void* stream) {
    const TablesArgs& a = *args;
    if (a.n < 0 || a.rows < 0 || a.cols < 0 || a.n_pages_listed < 0) BRAID_REFUSE("step_tables: negative sizes");
    if (a.n > TABLES_MAX_REQUESTS) BRAID_REFUSE("step_tables: %d requests exceed %d", a.n, TABLES_MAX_REQUESTS);
    if ((long long)a.num_pages * BRAID_PAGE_SIZE > 0x7fffffffLL) BRAID_REFUSE("step_tables: places in %d pages pass 32 bits", a.num_pages);
    const long long items = (long long)a.rows + (long long)a.n * a.cols;
    if (items == 0 && a.n == 0) return BRAID_OK;
    // (requests without rows and columns still have their first rows written and their lengths looked at)
    const long long ctas = items == 0 ? 1 : (items + TABLES_THREADS * TABLES_PER_THREAD - 1) / (TABLES_THREADS * TABLES_PER_THREAD);
    if (ctas > 0x7fffffffLL) BRAID_REFUSE("step_tables: the tables exceed the grid limit");
    const size_t smem = 2 * ((size_t)a.n + 1) * sizeof(int);
    cudaError_t e = cudaSuccess;
    if (smem > 40 * 1024) e = cudaFuncSetAttribute(step_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(2 * (TABLES_MAX_REQUESTS + 1) * sizeof(int)));
    if (e != cudaSuccess) { braid_set_error("step_tables: cannot reserve shared memory: %s", cudaGetErrorString(e)); return (int)e; }
    braid_launch(step_tables_kernel, dim3((unsigned)ctas), dim3(TABLES_THREADS), smem, (cudaStream_t)stream, a);
    BRAID_LAUNCH_CHECK();
}

// ------------------------------------------------------------------ write
// Two lanes a group: lane h takes its numbers 16 h .. 16 h + 15, which are two words of key codes, or four 16-bit words of value
// codes.  `place` < 0: a row of padding, nothing is written.  Places must differ from one another.
//
// A code is the quotient (x - lo) / step rounded to the nearest whole number, ties to even.  The quotient is taken as a product with 1 / step,
// which may miss a number next to a tie, and then put right by the remainder x - lo - code step: that is exact (the code has
// 4 bits, the step 8, and the remainder is at most about step), so ties are ties.  Instructions bound it, some 15 a number.  (5,845 rows of 8
// heads of 128, keys and values, bfloat16: 23 us with 8 numbers a thread and tests of each for NaN, 15 us so; what is read and
// written takes 5 us.)
struct StoreArgs {
    const void* k;
    const void* v;
    const int* place;
    uint8_t* cache;
    int* error_flag;
    long long k_stride, v_stride;
    int rows, nkh, hd, num_pages, dtype;
};

template <typename T, bool WIDE>
__device__ __forceinline__ void load8(const T* p, float* x) {
    if constexpr (WIDE) {
        constexpr int VW = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 8; i += VW) load_run<T, VW>(p + i, x + i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(p[i]);
    }
}

__device__ __forceinline__ float min_nan(float a, float b) { float y; asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b)); return y; }
__device__ __forceinline__ float max_nan(float a, float b) { float y; asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b)); return y; }

// A row takes 2 nkh hd / 16 threads: a CTA holds several rows, or a row passes through it 256 threads at a time.
template <typename T, int W, bool WIDE>
__global__ void __launch_bounds__(256)
kv4_store_kernel(const StoreArgs a, int row_threads, int rows_cta) {
    pdl_trigger();
    pdl_wait();
    constexpr int hd = 32 * W, per = 2 * W;                   // lanes a (row, plane, kv head)
    const int nkh = a.nkh;
    const int r_cta = rows_cta > 1 ? threadIdx.x / row_threads : 0;
    const long long row = (long long)blockIdx.x * rows_cta + r_cta;
    const bool here = row < a.rows && r_cta < rows_cta;
    const int at = here ? a.place[row] : -1;
    for (int it0 = rows_cta > 1 ? threadIdx.x - r_cta * row_threads : threadIdx.x, turn = 0; turn < row_threads; it0 += 256, turn += rows_cta > 1 ? row_threads : 256) {
        const bool live = here && it0 < row_threads;
        const int it = live ? it0 : 0;
        const int ph = it / per, c16 = it - ph * per;         // numbers 16 c16 .. 16 c16 + 15
        const bool value = ph >= nkh;
        const int kvh = value ? ph - nkh : ph, w = c16 >> 1, h = c16 & 1;
        float x[16];
        if (live) {                                           // (asked for beside the row's place, not after it)
            const T* src = (value ? (const T*)a.v + row * a.v_stride : (const T*)a.k + row * a.k_stride) + (long long)kvh * hd + 16 * c16;
            load8<T, WIDE>(src, x);
            load8<T, WIDE>(src + 8, x + 8);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = 0.f;
        }
        if (sizeof(T) == 4)
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = __bfloat162float(__float2bfloat16_rn(x[i]));
        float lo = x[0], hi = x[0];                           // NaN if one is
#pragma unroll
        for (int i = 1; i < 16; ++i) { lo = min_nan(lo, x[i]); hi = max_nan(hi, x[i]); }
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, 1));                 // rows and heads take whole pairs of lanes
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, 1));
        if (!live || at < 0) continue;
        const int page = at / BRAID_PAGE_SIZE, off = at % BRAID_PAGE_SIZE, t = off % KV4_REC;
        if (page >= a.num_pages) {
            if (it == 0) atomicExch(a.error_flag, 1);
            continue;
        }
        const float span = hi - lo;
        const bool bad = !(span <= 3.4028234663852886e38f);
        const __nv_bfloat16 nan = __ushort_as_bfloat16(0x7fff);
        const __nv_bfloat16 step16 = bad ? nan : __float2bfloat16_rn(span / 15.f);
        const float step = __bfloat162float(step16);
        // codes in the lowest bits of 1.5 2^23 + code
        uint32_t code[16];
        constexpr float base = 12582912.f;
        if (step >= 1e-36f) {
            const float inv = 1.f / step;
            const uint32_t half = __float_as_uint(0.5f * step);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float d = x[i] - lo;
                float u = fmaf(d, inv, base);
                const float rem = fmaf(base - u, step, d);    // d - code step
                // too far off, or a tie and an odd code: the next one (half a step less one unit is the bound for odd codes)
                const float limit = __uint_as_float(half - (__float_as_uint(u) & 1u));
                u += fabsf(rem) > limit ? copysignf(1.f, rem) : 0.f;
                code[i] = __float_as_uint(fminf(u, base + 15.f));
            }
        } else {                                              // no range (or NaN): code 0; or one that 1 / step would leave float32's with
#pragma unroll
            for (int i = 0; i < 16; ++i) code[i] = __float_as_uint(base) + (step > 0.f ? (uint32_t)fminf(fmaxf(rintf((x[i] - lo) / step), 0.f), 15.f) : 0u);
        }
        uint8_t* rec = a.cache + ((long long)page * nkh + kvh) * kv4_page_bytes(hd) + (off / KV4_REC) * kv4_record_bytes(hd);
        // sums of codes at their places, with what they have too much taken off at the end
        constexpr uint32_t C = 0x4b400000u;
        if (!value) {
            uint32_t* words = reinterpret_cast<uint32_t*>(rec + t * (hd / 2)) + w;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                uint32_t word = 0;
#pragma unroll
                for (int n = 0; n < 4; ++n) word += (code[8 * g + 2 * n] - C) * (1u << (4 * n)) + (code[8 * g + 2 * n + 1] - C) * (1u << (16 + 4 * n));
                words[(2 * h + g) * W] = word;
            }
        } else {
            uint16_t* codes = reinterpret_cast<uint16_t*>(rec + kv4_value_codes(hd) + t * (hd / 2)) + w;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                uint32_t word = 0;
#pragma unroll
                for (int n = 0; n < 4; ++n) word += (code[4 * g + n] - C) * (1u << (4 * n));
                codes[(4 * h + g) * W] = (uint16_t)word;
            }
        }
        if (h == 0)
            reinterpret_cast<uint32_t*>(rec + (value ? kv4_value_groups(hd) : kv4_key_groups(hd)))[t * W + w] =
                (uint32_t)__bfloat16_as_ushort(step16) | ((uint32_t)__bfloat16_as_ushort(bad ? nan : __float2bfloat16_rn(lo)) << 16);
    }
}

static int kv4_check(const char* what, int nkh, int hd, const void* cache) {
    if (nkh <= 0) BRAID_REFUSE("%s: %d kv heads", what, nkh);
    if (hd <= 0 || hd % KV4_GROUP || hd > 256) BRAID_REFUSE("%s: heads of %d numbers; groups of %d up to 256 are taken", what, hd, KV4_GROUP);
    if ((uintptr_t)cache & 15) BRAID_REFUSE("%s: the cache must start on 16 bytes", what);
    return BRAID_OK;
}

template <typename T, bool WIDE>
static int launch_store(const StoreArgs& a, cudaStream_t s) {
    const long long threads = (long long)2 * a.nkh * (a.hd / 16);
    if (threads > 0x3fffffffLL) BRAID_REFUSE("kv4_store: %d kv heads exceed the kernel's limit", a.nkh);
    const int rows_cta = threads <= 128 ? (int)(256 / threads) : 1;
    const int ctas = (a.rows + rows_cta - 1) / rows_cta;
    void (*const kernels[8])(const StoreArgs, int, int) = {kv4_store_kernel<T, 1, WIDE>, kv4_store_kernel<T, 2, WIDE>, kv4_store_kernel<T, 3, WIDE>,
                                                           kv4_store_kernel<T, 4, WIDE>, kv4_store_kernel<T, 5, WIDE>, kv4_store_kernel<T, 6, WIDE>,
                                                           kv4_store_kernel<T, 7, WIDE>, kv4_store_kernel<T, 8, WIDE>};
    braid_launch(kernels[a.hd / KV4_GROUP - 1], dim3(ctas), dim3(256), 0, s, a, (int)threads, rows_cta);
    BRAID_LAUNCH_CHECK();
}

extern "C" int braid_kv4_store(const StoreArgs* a, void* stream) {
    if (a->rows <= 0) return BRAID_OK;
    if (int rc = kv4_check("kv4_store", a->nkh, a->hd, a->cache)) return rc;
    const int size = a->dtype == BRAID_F32 ? 4 : 2;
    const bool wide = !(((uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)(a->k_stride * size) | (uintptr_t)(a->v_stride * size)) & 15);
    cudaStream_t s = (cudaStream_t)stream;
    if (a->dtype == BRAID_F32) return wide ? launch_store<float, true>(*a, s) : launch_store<float, false>(*a, s);
    if (a->dtype == BRAID_BF16) return wide ? launch_store<__nv_bfloat16, true>(*a, s) : launch_store<__nv_bfloat16, false>(*a, s);
    BRAID_REFUSE("kv4_store: unknown dtype code %d", a->dtype);
}

// ------------------------------------------------------------------ reading back
// The pages of a step's sequences as values, into pages [page][2][kv head][64][hd]: what a sequence's queries see (from its window's first
// position, and its kept first ones, up to its new tokens); other places of those pages come out zero.  The
// pages are numbered as the cache's, or (out_cols > 0) block c of sequence i is page i * out_cols + c.  A page belongs to one sequence.
//
// A CTA takes one page of one kv head, four lanes a token: lane j reads the W neighbouring words that hold its numbers 32 w + 8 j .. + 7
// (of a value: the two 16-bit words a group that do), so that codes and groups come in one wide load each and the values leave 16
// bytes at a time.  Bytes bound it: the values that it writes are 3.2 times (bfloat16) the codes that it reads.
struct ExpandArgs {
    const uint8_t* cache;
    void* out;
    const int* page_table;
    const int* q_len;
    const int* kv_before;
    int* error_flag;
    int* repair;                 // given: groups of values that are NaN come out zero, and repair[0] and [1 + seq0 + sequence] become 1
    int* out_table;              // (out_cols > 0) [n_seqs, out_cols]: the numbers of the pages, for whoever reads them
    int* scales;                 // given: float16 numbers, rows of 64, 128 or 256, scaled a page and kv head: [pages, nkh, 2] exponents + KV4_EXPONENT of keys, values (0: all zero)
    int* top;                    // (scales) [n_seqs, nkh] from sequence seq0 on: the largest of a sequence's values' exponents; zeros before
    int n_seqs, nkh, hd, cols, num_pages, window, keep_first, out_cols, seq0, dtype;
    int q_from;                  // only the pages of sequences that bring at least so many tokens
};

template <int N>
__device__ __forceinline__ void load_words(const void* p, uint32_t* x) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) *reinterpret_cast<uint4*>(x + i) = reinterpret_cast<const uint4*>(p)[i / 4];
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) *reinterpret_cast<uint2*>(x + i) = reinterpret_cast<const uint2*>(p)[i / 2];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = reinterpret_cast<const uint32_t*>(p)[i];
    }
}

// lowest + step * code of codes n (first) and 4 + n (second) of a word, n 0 .. 3
template <typename T>
struct Kv4Pairs;
template <>
struct Kv4Pairs<__nv_bfloat16> {
    using Pair = uint32_t;
    // one multiply-add of the pair in bfloat16: the code and 128 + code are exact, the sum is rounded once
    static __device__ __forceinline__ void make(uint32_t word, uint32_t group, uint32_t* y, float) {
        const uint32_t s2 = __byte_perm(group, group, 0x1010), l2 = __byte_perm(group, group, 0x3232);
        const __nv_bfloat162 base(__float2bfloat16(128.f), __float2bfloat16(128.f));
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const uint32_t c = ((word >> (4 * n)) & 0x000f000fu) | 0x43004300u;
            const __nv_bfloat162 v = __hfma2(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&c), base), *reinterpret_cast<const __nv_bfloat162*>(&s2),
                                             *reinterpret_cast<const __nv_bfloat162*>(&l2));
            y[n] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
    static __device__ __forceinline__ uint32_t lows(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
    static __device__ __forceinline__ uint32_t highs(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }
};
template <>
struct Kv4Pairs<__half> {
    using Pair = uint32_t;
    // the same in float16, step and lowest value times a power of two: they keep their 8 bits but for what is below 2^-24
    static __device__ __forceinline__ void make(uint32_t word, uint32_t group, uint32_t* y, float factor) {
        const __half2 s2 = __float2half2_rn(kv4_step(group) * factor), l2 = __float2half2_rn(kv4_lowest(group) * factor);
        const __half2 base = __float2half2_rn(1024.f);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const uint32_t c = ((word >> (4 * n)) & 0x000f000fu) | 0x64006400u;
            const __half2 v = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&c), base), s2, l2);
            y[n] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
    static __device__ __forceinline__ uint32_t lows(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
    static __device__ __forceinline__ uint32_t highs(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }
};
template <>
struct Kv4Pairs<float> {
    using Pair = float2;
    static __device__ __forceinline__ void make(uint32_t word, uint32_t group, float2* y, float) {
        const float step = kv4_step(group), low = kv4_lowest(group);
#pragma unroll
        for (int n = 0; n < 4; ++n) {                          // a code under the lowest bits of 2^23 is 2^23 + code
            const float a = __uint_as_float(((word >> (4 * n)) & 15u) | 0x4b000000u) - 8388608.f;
            const float b = __uint_as_float(((word >> (16 + 4 * n)) & 15u) | 0x4b000000u) - 8388608.f;
            y[n] = make_float2(fmaf(step, a, low), fmaf(step, b, low));
        }
    }
    static __device__ __forceinline__ float2 lows(float2 a, float2 b) { return make_float2(a.x, b.x); }
    static __device__ __forceinline__ float2 highs(float2 a, float2 b) { return make_float2(a.y, b.y); }
};

template <typename T, int W>
__global__ void __launch_bounds__(256)
kv4_expand_kernel(const ExpandArgs a) {
    pdl_trigger();
    pdl_wait();
    constexpr int HD = 32 * W;
    using P = typename Kv4Pairs<T>::Pair;
    const int kvh = blockIdx.y, seq = blockIdx.z;
    const int before = a.kv_before[seq], end = before + a.q_len[seq];
    if (a.out_table && kvh == 0)
        for (int c = blockIdx.x + gridDim.x * threadIdx.x; c < a.out_cols; c += gridDim.x * blockDim.x)
            a.out_table[(size_t)seq * a.out_cols + c] = seq * a.out_cols + c;
    if (end - before < a.q_from) return;
    // a table that ends before the sequence (whoever reads pages of the other numbering looks after that itself)
    if (a.out_cols <= 0 && blockIdx.x == 0 && kvh == 0 && threadIdx.x == 0 && end > (long long)a.cols * BRAID_PAGE_SIZE) atomicExch(a.error_flag, 1);
    constexpr bool SCALED = sizeof(T) == 2 && !std::is_same<T, __nv_bfloat16>::value;
    constexpr int OUT = !SCALED ? HD : HD <= 64 ? 64 : HD <= 128 ? 128 : 256;       // numbers of a row that is written, zeros behind the head's
    __shared__ float3 sizes[2][8];
    int turn = 0;
    const int lo = a.window > 0 ? max(0, before - a.window + 1) : 0, cols = a.out_cols > 0 ? min(a.cols, a.out_cols) : a.cols;
    for (int c = blockIdx.x; c < cols; c += gridDim.x) {
        const int key0 = c * BRAID_PAGE_SIZE;
        if (key0 >= end) return;
        if (key0 + BRAID_PAGE_SIZE <= lo && key0 >= a.keep_first) continue;
        const int page = a.page_table[(size_t)seq * a.cols + c];
        if (page < 0 || page >= a.num_pages) {
            if (threadIdx.x == 0) atomicExch(a.error_flag, 1);
            continue;
        }
        const size_t out_page = a.out_cols > 0 ? (size_t)seq * a.out_cols + c : (size_t)page;
        const int t = threadIdx.x >> 2, j = threadIdx.x & 3, tr = t % KV4_REC;
        const uint8_t* rec = a.cache + ((size_t)page * a.nkh + kvh) * kv4_page_bytes(HD) + (t / KV4_REC) * kv4_record_bytes(HD);
        const bool in = key0 + t < end && (key0 + t >= lo || key0 + t < a.keep_first);
        T* dst = (T*)a.out + ((out_page * 2 * a.nkh + kvh) * BRAID_PAGE_SIZE + t) * OUT + 8 * j;
        const size_t plane = (size_t)a.nkh * BRAID_PAGE_SIZE * OUT;
        uint32_t kc[W], kg[W], vc[W], vg[W];
        load_words<W>(rec + tr * (HD / 2) + 4 * W * j, kc);
        load_words<W>(rec + kv4_key_groups(HD) + 4 * W * tr, kg);
        load_words<W>(rec + kv4_value_codes(HD) + tr * (HD / 2) + 4 * W * j, vc);
        load_words<W>(rec + kv4_value_groups(HD) + 4 * W * tr, vg);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if (!in) kc[w] = kg[w] = vg[w] = 0u;                   // a group of step 0 and lowest value 0
            if (a.repair && ((vg[w] & 0x7f80u) == 0x7f80u || (vg[w] & 0x7f800000u) == 0x7f800000u)) {
                vg[w] = 0u;
                a.repair[1 + a.seq0 + seq] = 1;
                a.repair[0] = 1;
            }
        }
        float kf = 1.f, vf = 1.f;
        if constexpr (SCALED) {
            // the page's largest key and value become numbers of 2^14 .. 2^15
            float k = 0.f, v = 0.f, least = INFINITY;              // (least: of a group's largest value)
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float a0 = fmaxf(fabsf(kv4_lowest(kg[w])), fabsf(fmaf(15.f, kv4_step(kg[w]), kv4_lowest(kg[w]))));
                const float a1 = fmaxf(fabsf(kv4_lowest(vg[w])), fabsf(fmaf(15.f, kv4_step(vg[w]), kv4_lowest(vg[w]))));
                if (a0 < INFINITY) k = fmaxf(k, a0);
                v = fmaxf(v, a1);
                if (a1 > 0.f) least = fminf(least, a1);
            }
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                k = fmaxf(k, __shfl_xor_sync(0xffffffffu, k, o));
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
                least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
            }
            if ((threadIdx.x & 31) == 0) sizes[turn][threadIdx.x >> 5] = make_float3(k, v, least);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float3 x = sizes[turn][i];
                k = fmaxf(k, x.x); v = fmaxf(v, x.y); least = fminf(least, x.z);
            }
            turn ^= 1;
            const int ke = max(kv4_exponent(k) - 14, -112), ve = max(kv4_exponent(v) - 14, -112);
            if (k > 0.f) kf = kv4_pow2(-ke);
            if (v > 0.f) vf = kv4_pow2(-ve);
            if (threadIdx.x == 0) {
                *reinterpret_cast<int2*>(a.scales + (out_page * a.nkh + kvh) * 2) =
                    make_int2(k > 0.f ? ke + KV4_EXPONENT : 0, v > 0.f ? ve + KV4_EXPONENT : 0);
                if (v > 0.f) atomicMax(&a.top[(size_t)(a.seq0 + seq) * a.nkh + kvh], ve + KV4_EXPONENT);
                // a group whose largest value is 2^26 times smaller than the page's would lose bits
                if (least * 67108864.f < v || !(v < INFINITY)) {
                    a.repair[1 + a.seq0 + seq] = 1;
                    a.repair[0] = 1;
                }
            }
        }
#pragma unroll
        for (int w = 0; w < W; ++w) {
            // the 16 bits of group w in the lane's first and second half of value words
            const int h0 = w, h1 = W + w;
            const uint32_t v0 = (vc[h0 / 2] >> (16 * (h0 & 1))) & 0xffffu, v1 = (vc[h1 / 2] >> (16 * (h1 & 1))) & 0xffffu;
            const uint32_t both = in ? v0 | (v1 << 16) : 0u;
            __align__(16) P y[4];
            P z[4];
            Kv4Pairs<T>::make(kc[w], kg[w], y, kf);                  // pairs of neighbours, in order
            *reinterpret_cast<uint4*>(dst + 32 * w) = *reinterpret_cast<const uint4*>(y);
            if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(dst + 32 * w + 4) = *reinterpret_cast<const uint4*>(y + 2);
            Kv4Pairs<T>::make(both, vg[w], z, vf);                   // numbers n and 4 + n
            y[0] = Kv4Pairs<T>::lows(z[0], z[1]);
            y[1] = Kv4Pairs<T>::lows(z[2], z[3]);
            y[2] = Kv4Pairs<T>::highs(z[0], z[1]);
            y[3] = Kv4Pairs<T>::highs(z[2], z[3]);
            *reinterpret_cast<uint4*>(dst + plane + 32 * w) = *reinterpret_cast<const uint4*>(y);
            if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(dst + plane + 32 * w + 4) = *reinterpret_cast<const uint4*>(y + 2);
        }
#pragma unroll
        for (int w = W; w < OUT / 32; ++w)
            *reinterpret_cast<uint4*>(dst + 32 * w) = *reinterpret_cast<uint4*>(dst + plane + 32 * w) = make_uint4(0u, 0u, 0u, 0u);
    }
}

template <typename T>
static int launch_expand(const ExpandArgs& a, cudaStream_t s) {
    const int cols = a.out_cols > 0 ? min(a.cols, a.out_cols) : a.cols;
    // A CTA a page; where most sequences may be passed over, some pages a CTA.  (512 tokens beside 63 single ones behind 8,000, attention as a
    // whole: 285 us with a CTA a page, 225 with 4,096 CTAs; 512 behind 16,000 beside 15 behind 2,000: 210, 186.)
    const int x = a.q_from > 1 ? min(cols, max(1, 4096 / (a.nkh * a.n_seqs))) : cols;
    const dim3 grid(x, a.nkh, a.n_seqs);
    void (*const kernels[8])(const ExpandArgs) = {kv4_expand_kernel<T, 1>, kv4_expand_kernel<T, 2>, kv4_expand_kernel<T, 3>, kv4_expand_kernel<T, 4>,
                                                  kv4_expand_kernel<T, 5>, kv4_expand_kernel<T, 6>, kv4_expand_kernel<T, 7>, kv4_expand_kernel<T, 8>};
    braid_launch(kernels[a.hd / KV4_GROUP - 1], grid, dim3(256), 0, s, a);
    BRAID_LAUNCH_CHECK();
}

extern "C" int braid_kv4_expand(const ExpandArgs* args, void* stream) {
    ExpandArgs a = *args;
    if (a.n_seqs <= 0 || a.cols <= 0) return BRAID_OK;
    if (int rc = kv4_check("kv4_expand", a.nkh, a.hd, a.cache)) return rc;
    if ((uintptr_t)a.out & 15) BRAID_REFUSE("kv4_expand: the pages must start on 16 bytes");
    if (a.nkh > 65535 || a.n_seqs > 65535) BRAID_REFUSE("kv4_expand: the step exceeds the grid limits (%d kv heads, %d sequences)", a.nkh, a.n_seqs);
    if (a.window <= 0) a.window = a.keep_first = 0;
    if (a.scales) {
        if (!a.repair || !a.top || a.out_cols <= 0) BRAID_REFUSE("kv4_expand: scaled pages want pages of their own, the largest exponents and the flags");
        return launch_expand<__half>(a, (cudaStream_t)stream);
    }
    if (a.dtype == BRAID_F32) return launch_expand<float>(a, (cudaStream_t)stream);
    if (a.dtype == BRAID_BF16) return launch_expand<__nv_bfloat16>(a, (cudaStream_t)stream);
    BRAID_REFUSE("kv4_expand: unknown dtype code %d", a.dtype);
}

// ------------------------------------------------------------------ plain attention
// One warp per (row, query head), 32 keys at a time: a lane a key for the scores, a lane a number of the head for the values.  All
// arithmetic float32.  Options as in attn_simple.cu.  Rows of padding (token_seq < 0) are left as they were.
// With `repair` ([0]: whether to work at all, [1 + i]: whether for sequence i) it goes over the result of a product that multiplies masked
// values by 0 (the attention of ordinary pages): a NaN among them would make all of it NaN, so they were taken out, and the rows of
// those sequences are computed here.
struct Kv4SimpleArgs {
    const void* q;
    void* out;
    const uint8_t* cache;
    const int* page_table;
    const int* token_seq;
    const int* q_start;
    const int* kv_before;
    long long q_stride, out_stride;
    int rows, nqh, nkh, hd, cols, num_pages, window, keep_first;
    float scale;
    int has_sink;
    float sink, out_scale;
    const float* head_sinks;
    const void* head_gate;
    long long gate_stride;
    const float* head_scale;
    const float* bias_slope;
    const float* bias_rate;
    float softcap;
    int dtype;
    int* error_flag;
    const int* repair;
};

template <typename T>
__device__ void attn_kv4_item(const Kv4SimpleArgs& a, long long item, float* qs, int lane) {
    const int row = (int)(item / a.nqh), head = (int)(item - (long long)row * a.nqh);
    const int seq = a.token_seq[row];
    if (seq < 0 || (a.repair && !a.repair[1 + seq])) return;
    const int hd = a.hd, W = hd / KV4_GROUP, kvh = head / (a.nqh / a.nkh);
    __syncwarp();
    const T* q = (const T*)a.q + (size_t)row * a.q_stride + (size_t)head * hd;
    for (int d = lane; d < hd; d += 32) qs[d] = to_f32(q[d]);
    __syncwarp();
    const int pos = a.kv_before[seq] + (row - a.q_start[seq]);
    const float scale = a.head_scale ? a.scale * a.head_scale[head] : a.scale;
    const float r1 = a.bias_slope ? a.bias_slope[head] : 0.f, r2 = a.bias_slope ? a.bias_rate[head] : 0.f;
    const int lo = (a.window > 0 && pos - a.window + 1 > 0) ? pos - a.window + 1 : 0;
    const int kept = min(a.keep_first, lo);
    const int* table = a.page_table + (size_t)seq * a.cols;
    float m = -INFINITY, l = 0.f, acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    for (int part = kept > 0 ? 0 : 1; part < 2; ++part) {
        const int end = part ? pos + 1 : kept;
        for (int j0 = part ? lo : 0; j0 < end; j0 += 32) {
            const int key = j0 + lane;
            float s = -INFINITY;
            const uint8_t* rec = nullptr;
            if (key < end) {
                const int block = key / BRAID_PAGE_SIZE, off = key % BRAID_PAGE_SIZE;
                int page = block < a.cols ? table[block] : -1;
                if (page < 0 || page >= a.num_pages) { atomicExch(a.error_flag, 1); page = 0; }
                rec = a.cache + ((size_t)page * a.nkh + kvh) * kv4_page_bytes(hd) + (off / KV4_REC) * kv4_record_bytes(hd);
                const int tr = off % KV4_REC;
                float dot = 0.f;
                for (int w = 0; w < W; ++w) {
                    const uint32_t group = reinterpret_cast<const uint32_t*>(rec + kv4_key_groups(hd))[tr * W + w];
                    const float step = kv4_step(group), low = kv4_lowest(group);
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t word = reinterpret_cast<const uint32_t*>(rec + tr * (hd / 2))[j * W + w];
#pragma unroll
                        for (int n = 0; n < 8; ++n)
                            dot = fmaf(qs[32 * w + 8 * j + n], fmaf(step, (float)((word >> (16 * (n & 1) + 4 * (n >> 1))) & 15u), low), dot);
                    }
                }
                s = dot * scale;
                if (a.softcap > 0.f) s = a.softcap * tanhf(s / a.softcap);
                if (a.bias_slope) s -= r1 * log1pf(r2 * (float)(pos - key));
            }
            const float m_new = fmaxf(m, warp_max(s));
            const float ref = m_new == -INFINITY ? 0.f : m_new;
            const float corr = m == -INFINITY ? 0.f : expf(m - m_new);
            const float p = key < end ? expf(s - ref) : 0.f;
            l = l * corr + warp_sum(p);
            m = m_new;
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] *= corr;
            for (int k = 0; k < min(32, end - j0); ++k) {
                const float pk = __shfl_sync(0xffffffffu, p, k);
                const uint8_t* rk = (const uint8_t*)__shfl_sync(0xffffffffu, (unsigned long long)rec, k);
                const int tr = (j0 + k) % KV4_REC;
                const uint32_t* groups = reinterpret_cast<const uint32_t*>(rk + kv4_value_groups(hd)) + tr * W;
                const uint16_t* codes = reinterpret_cast<const uint16_t*>(rk + kv4_value_codes(hd) + tr * (hd / 2)) + (lane >> 2) * W;
#pragma unroll
                for (int w = 0; w < 8; ++w)
                    if (w < W) acc[w] = fmaf(pk, fmaf(kv4_step(groups[w]), (float)((codes[w] >> (4 * (lane & 3))) & 15), kv4_lowest(groups[w])), acc[w]);
            }
        }
    }
    if (a.has_sink) {
        const float sk = a.head_sinks ? a.head_sinks[head] : a.sink;
        const float m_new = fmaxf(m, sk), corr = m == -INFINITY ? 0.f : expf(m - m_new);
        l = l * corr + expf(sk - m_new);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] *= corr;
    }
    float inv = a.out_scale / l;
    if (a.head_gate) inv *= 1.f / (1.f + expf(-to_f32(((const T*)a.head_gate)[(size_t)row * a.gate_stride + head])));
    T* o = (T*)a.out + (size_t)row * a.out_stride + (size_t)head * hd;
#pragma unroll
    for (int w = 0; w < 8; ++w)
        if (w < W) o[32 * w + lane] = from_f32<T>(acc[w] * inv);
}

template <typename T>
__global__ void __launch_bounds__(128)
attn_kv4_simple_kernel(const Kv4SimpleArgs a) {
    pdl_trigger();
    pdl_wait();
    __shared__ float qs_all[4][256];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (a.repair && a.repair[0] == 0) return;
    for (long long item = (long long)blockIdx.x * 4 + warp; item < (long long)a.rows * a.nqh; item += (long long)gridDim.x * 4)
        attn_kv4_item<T>(a, item, qs_all[warp], lane);
}

// `args`: a Kv4SimpleArgs, filled in by the caller (csrc/api.py has its layout).
extern "C" int braid_attn_kv4_simple(const Kv4SimpleArgs* args, void* stream) {
    Kv4SimpleArgs a = *args;
    if (a.rows <= 0) return BRAID_OK;
    if (int rc = kv4_check("attn_kv4", a.nkh, a.hd, a.cache)) return rc;
    if (a.nqh <= 0 || a.nqh % a.nkh) BRAID_REFUSE("attn_kv4: %d query heads do not divide into %d kv heads", a.nqh, a.nkh);
    if (a.num_pages <= 0 || a.cols <= 0) BRAID_REFUSE("attn_kv4: the cache has no pages (pages=%d, table columns=%d)", a.num_pages, a.cols);
    long long ctas = ((long long)a.rows * a.nqh + 3) / 4;
    if (a.repair) ctas = min(ctas, 148LL);                    // one an SM: they hardly ever have anything to do
    if (ctas > 0x7fffffffLL) BRAID_REFUSE("attn_kv4: the rows exceed the grid limit");
    if (a.window <= 0) a.window = a.keep_first = 0;
    if (a.head_sinks) a.has_sink = 1;
    if (a.dtype == BRAID_F32) braid_launch(attn_kv4_simple_kernel<float>, dim3((unsigned)ctas), dim3(128), 0, (cudaStream_t)stream, a);
    else if (a.dtype == BRAID_BF16) braid_launch(attn_kv4_simple_kernel<__nv_bfloat16>, dim3((unsigned)ctas), dim3(128), 0, (cudaStream_t)stream, a);
    else BRAID_REFUSE("attn_kv4: unknown dtype code %d", a.dtype);
    BRAID_LAUNCH_CHECK();
}

// Bytes of the argument structures: tables, write, reading back, plain attention.
extern "C" int braid_kv4_args_bytes(int which) {
    return which == 0 ? (int)sizeof(TablesArgs) : which == 1 ? (int)sizeof(StoreArgs) : which == 2 ? (int)sizeof(ExpandArgs) : (int)sizeof(Kv4SimpleArgs);
}
