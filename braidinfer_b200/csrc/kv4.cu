// A cache held in 4 bits (kv4.cuh has the format): the tables of a step, the write of new keys and values, their reading
// back, and the plain attention that the tensor-core kernel (attn_kv4.cu) is checked against.
#include "kv4.cuh"

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

extern "C" int braid_step_tables(const int* q_len, const int* kv_before, const int* pages, int* page_table, int* place, int* positions,
                                 int* token_seq, int* q_start, int n, int n_pages_listed, int rows, int cols, int num_pages,
                                 int* error_flag, void* stream) {
    if (n < 0 || rows < 0 || cols < 0 || n_pages_listed < 0) BRAID_REFUSE("step_tables: negative sizes");
    if (n > TABLES_MAX_REQUESTS) BRAID_REFUSE("step_tables: %d requests exceed %d", n, TABLES_MAX_REQUESTS);
    if ((long long)num_pages * BRAID_PAGE_SIZE > 0x7fffffffLL) BRAID_REFUSE("step_tables: places in %d pages pass 32 bits", num_pages);
    const long long items = (long long)rows + (long long)n * cols;
    if (items == 0) return BRAID_OK;
    const long long ctas = (items + TABLES_THREADS * TABLES_PER_THREAD - 1) / (TABLES_THREADS * TABLES_PER_THREAD);
    if (ctas > 0x7fffffffLL) BRAID_REFUSE("step_tables: the tables exceed the grid limit");
    const size_t smem = 2 * ((size_t)n + 1) * sizeof(int);
    cudaError_t e = cudaSuccess;
    if (smem > 40 * 1024) e = cudaFuncSetAttribute(step_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(2 * (TABLES_MAX_REQUESTS + 1) * sizeof(int)));
    if (e != cudaSuccess) { braid_set_error("step_tables: cannot reserve shared memory: %s", cudaGetErrorString(e)); return (int)e; }
    TablesArgs a{q_len, kv_before, pages, page_table, place, positions, token_seq, q_start, n, n_pages_listed, rows, cols, num_pages, error_flag};
    braid_launch(step_tables_kernel, dim3((unsigned)ctas), dim3(TABLES_THREADS), smem, (cudaStream_t)stream, a);
    BRAID_LAUNCH_CHECK();
}

// ------------------------------------------------------------------ write
// Four lanes a group: lane j takes its numbers 8 j .. 8 j + 7, which are one word of key codes, or two 16-bit words of value
// codes.  `place` < 0: a row of padding, nothing is written.  Places must differ from one another.
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

template <typename T, bool WIDE>
__global__ void __launch_bounds__(256)
kv4_store_kernel(const T* __restrict__ k, long long k_stride, const T* __restrict__ v, long long v_stride, const int* __restrict__ place,
                 uint8_t* __restrict__ cache, int rows, int nkh, int hd, long long places, int* error_flag) {
    pdl_trigger();
    pdl_wait();
    const int per = hd / 8, W = hd / KV4_GROUP;               // lanes a (row, plane, kv head)
    const long long it = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long heads = it / per;
    const int c8 = (int)(it - heads * per);                   // numbers 8 c8 .. 8 c8 + 7
    const long long row = heads / (2 * nkh);
    const int ph = (int)(heads - row * (2 * nkh));
    const bool value = ph >= nkh;
    const int kvh = value ? ph - nkh : ph;
    const int w = c8 >> 2, j = c8 & 3;
    long long at = -1;
    if (row < rows) {
        at = place[row];
        if (at >= places) { if (c8 == 0) atomicExch(error_flag, 1); at = -1; }
    }
    float x[8];
    bool bad = false;
    float lo = INFINITY, hi = -INFINITY;
    if (at >= 0) {
        load8<T, WIDE>((value ? v + row * v_stride : k + row * k_stride) + (long long)kvh * hd + 8 * c8, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = __bfloat162float(__float2bfloat16_rn(x[i]));
            bad |= x[i] != x[i];
            lo = fminf(lo, x[i]);
            hi = fmaxf(hi, x[i]);
        }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {                         // per is a multiple of 4: the four lanes are of one warp and one group
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        bad |= __shfl_xor_sync(0xffffffffu, (int)bad, o) != 0;
    }
    if (at < 0) return;
    const float span = hi - lo;
    bad |= !(span <= 3.4028234663852886e38f);
    const __nv_bfloat16 nan = __ushort_as_bfloat16(0x7fff);
    const __nv_bfloat16 step16 = bad ? nan : __float2bfloat16_rn(span / 15.f);
    const float step = __bfloat162float(step16);
    uint32_t code[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)                               // the quotient is rounded as IEEE has it: ties are ties in every form
        code[i] = step > 0.f ? (uint32_t)fminf(fmaxf(rintf((x[i] - lo) / step), 0.f), 15.f) : 0u;
    const uint32_t group = (uint32_t)__bfloat16_as_ushort(step16) | ((uint32_t)__bfloat16_as_ushort(bad ? nan : __float2bfloat16_rn(lo)) << 16);
    const long long page = at / BRAID_PAGE_SIZE;
    const int off = (int)(at - page * BRAID_PAGE_SIZE), t = off % KV4_REC;
    uint8_t* rec = cache + (page * nkh + kvh) * kv4_page_bytes(hd) + (off / KV4_REC) * kv4_record_bytes(hd);
    if (!value) {
        uint32_t word = 0;
#pragma unroll
        for (int n = 0; n < 4; ++n) word |= (code[2 * n] << (4 * n)) | (code[2 * n + 1] << (16 + 4 * n));
        reinterpret_cast<uint32_t*>(rec + t * (hd / 2))[j * W + w] = word;
    } else {
        uint16_t* codes = reinterpret_cast<uint16_t*>(rec + kv4_value_codes(hd) + t * (hd / 2));
#pragma unroll
        for (int h = 0; h < 2; ++h)
            codes[(2 * j + h) * W + w] = (uint16_t)(code[4 * h] | (code[4 * h + 1] << 4) | (code[4 * h + 2] << 8) | (code[4 * h + 3] << 12));
    }
    if (j == 0) reinterpret_cast<uint32_t*>(rec + (value ? kv4_value_groups(hd) : kv4_key_groups(hd)))[t * W + w] = group;
}

template <typename T>
static int launch_store(const void* k, long long ks, const void* v, long long vs, const int* place, void* cache, int rows, int nkh, int hd,
                        long long places, int* flag, cudaStream_t s) {
    const long long items = (long long)rows * 2 * nkh * (hd / 8), ctas = (items + 255) / 256;
    if (ctas > 0x7fffffffLL) BRAID_REFUSE("kv4_store: the rows exceed the grid limit");
    const bool wide = !(((uintptr_t)k | (uintptr_t)v | (uintptr_t)(ks * sizeof(T)) | (uintptr_t)(vs * sizeof(T))) & 15);
    braid_launch(wide ? kv4_store_kernel<T, true> : kv4_store_kernel<T, false>, dim3((unsigned)ctas), dim3(256), 0, s, (const T*)k, ks, (const T*)v, vs,
                 place, (uint8_t*)cache, rows, nkh, hd, places, flag);
    BRAID_LAUNCH_CHECK();
}

static int kv4_check(const char* what, int nkh, int hd, const void* cache) {
    if (nkh <= 0) BRAID_REFUSE("%s: %d kv heads", what, nkh);
    if (hd <= 0 || hd % KV4_GROUP || hd > 256) BRAID_REFUSE("%s: heads of %d numbers; groups of %d up to 256 are taken", what, hd, KV4_GROUP);
    if ((uintptr_t)cache & 15) BRAID_REFUSE("%s: the cache must start on 16 bytes", what);
    return BRAID_OK;
}

extern "C" int braid_kv4_store(const void* k, long long k_stride, const void* v, long long v_stride, int dtype, const int* place, void* cache,
                               int rows, int nkh, int hd, int num_pages, int* error_flag, void* stream) {
    if (rows <= 0) return BRAID_OK;
    if (int rc = kv4_check("kv4_store", nkh, hd, cache)) return rc;
    const long long places = (long long)num_pages * BRAID_PAGE_SIZE;
    if (dtype == BRAID_F32) return launch_store<float>(k, k_stride, v, v_stride, place, cache, rows, nkh, hd, places, error_flag, (cudaStream_t)stream);
    if (dtype == BRAID_BF16) return launch_store<__nv_bfloat16>(k, k_stride, v, v_stride, place, cache, rows, nkh, hd, places, error_flag, (cudaStream_t)stream);
    BRAID_REFUSE("kv4_store: unknown dtype code %d", dtype);
}

// ------------------------------------------------------------------ reading back
// The pages of a step's sequences as values, into pages [page][2][kv head][64][hd]: what a sequence's queries see (from its window's first
// position, and its kept first ones, up to its new tokens); other places of those pages come out zero.  The
// pages are numbered as the cache's, or (out_cols > 0) block c of sequence i is page i * out_cols + c.  A CTA takes one page of one kv
// head.  A page belongs to one sequence.
struct ExpandArgs {
    const uint8_t* cache;
    void* out;
    const int* page_table;
    const int* q_len;
    const int* kv_before;
    int nkh, hd, cols, num_pages, window, keep_first, out_cols;
    int* error_flag;
    int* repair;                 // given: groups of values that are NaN come out zero, and repair[0] and [2 + seq0 + sequence] become 1
    int seq0;
};

template <typename T>
__global__ void __launch_bounds__(256)
kv4_expand_kernel(ExpandArgs a) {
    pdl_trigger();
    pdl_wait();
    const int c = blockIdx.x, kvh = blockIdx.y, seq = blockIdx.z;
    const int before = a.kv_before[seq], end = before + a.q_len[seq];
    const int key0 = c * BRAID_PAGE_SIZE;
    if (key0 >= end) return;
    const int lo = a.window > 0 ? max(0, before - a.window + 1) : 0;
    if (key0 + BRAID_PAGE_SIZE <= lo && key0 >= a.keep_first) return;
    const int page = a.page_table[(size_t)seq * a.cols + c];
    if (page < 0 || page >= a.num_pages) {
        if (threadIdx.x == 0) atomicExch(a.error_flag, 1);
        return;
    }
    const size_t out_page = a.out_cols > 0 ? (size_t)seq * a.out_cols + c : (size_t)page;
    const int hd = a.hd, W = hd / KV4_GROUP, per = hd / 8;
    const uint8_t* src = a.cache + ((size_t)page * a.nkh + kvh) * kv4_page_bytes(hd);
    const int n_here = min(BRAID_PAGE_SIZE, end - key0);
    for (int it = threadIdx.x; it < 2 * BRAID_PAGE_SIZE * per; it += 256) {
        const int c8 = it % per, tp = it / per, t = tp % BRAID_PAGE_SIZE, value = tp / BRAID_PAGE_SIZE;
        const int w = c8 >> 2, j = c8 & 3;
        float x[8];
        if (t < n_here && (key0 + t >= lo || key0 + t < a.keep_first)) {
            const uint8_t* rec = src + (t / KV4_REC) * kv4_record_bytes(hd);
            const int tr = t % KV4_REC;
            const uint32_t group = reinterpret_cast<const uint32_t*>(rec + (value ? kv4_value_groups(hd) : kv4_key_groups(hd)))[tr * W + w];
            float step = kv4_step(group), low = kv4_lowest(group);
            if (value && a.repair && !(fabsf(step) + fabsf(low) < INFINITY)) {
                step = low = 0.f;
                a.repair[2 + a.seq0 + seq] = 1;
                a.repair[0] = 1;
            }
            if (!value) {
                const uint32_t word = reinterpret_cast<const uint32_t*>(rec + tr * (hd / 2))[j * W + w];
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    x[2 * n] = fmaf(step, (float)((word >> (4 * n)) & 15u), low);
                    x[2 * n + 1] = fmaf(step, (float)((word >> (16 + 4 * n)) & 15u), low);
                }
            } else {
                const uint16_t* codes = reinterpret_cast<const uint16_t*>(rec + kv4_value_codes(hd) + tr * (hd / 2));
                const uint32_t word = codes[2 * j * W + w] | ((uint32_t)codes[(2 * j + 1) * W + w] << 16);
#pragma unroll
                for (int n = 0; n < 8; ++n) x[n] = fmaf(step, (float)((word >> (4 * n)) & 15u), low);
            }
        } else {
#pragma unroll
            for (int n = 0; n < 8; ++n) x[n] = 0.f;
        }
        T* dst = (T*)a.out + (((out_page * 2 + value) * a.nkh + kvh) * BRAID_PAGE_SIZE + t) * hd + 8 * c8;
        constexpr int VW = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 8; i += VW) store_run<T, VW>(dst + i, x + i);
    }
}

extern "C" int braid_kv4_expand(const void* cache, void* out, int dtype, const int* page_table, const int* q_len, const int* kv_before,
                                int n_seqs, int cols, int nkh, int hd, int num_pages, int window, int keep_first, int out_cols, int* repair,
                                int seq0, int* error_flag, void* stream) {
    if (n_seqs <= 0 || cols <= 0) return BRAID_OK;
    if (int rc = kv4_check("kv4_expand", nkh, hd, cache)) return rc;
    if ((uintptr_t)out & 15) BRAID_REFUSE("kv4_expand: the pages must start on 16 bytes");
    if (nkh > 65535 || n_seqs > 65535) BRAID_REFUSE("kv4_expand: the step exceeds the grid limits (%d kv heads, %d sequences)", nkh, n_seqs);
    ExpandArgs a{(const uint8_t*)cache, out, page_table, q_len, kv_before, nkh, hd, cols, num_pages, window, window > 0 ? keep_first : 0, out_cols, error_flag, repair, seq0};
    const dim3 grid(out_cols > 0 ? min(cols, out_cols) : cols, nkh, n_seqs);
    if (dtype == BRAID_F32) braid_launch(kv4_expand_kernel<float>, grid, dim3(256), 0, (cudaStream_t)stream, a);
    else if (dtype == BRAID_BF16) braid_launch(kv4_expand_kernel<__nv_bfloat16>, grid, dim3(256), 0, (cudaStream_t)stream, a);
    else BRAID_REFUSE("kv4_expand: unknown dtype code %d", dtype);
    BRAID_LAUNCH_CHECK();
}

// ------------------------------------------------------------------ plain attention
// One warp per (row, query head), 32 keys at a time: a lane a key for the scores, a lane a number of the head for the values.  All
// arithmetic float32.  Options as in attn_simple.cu.  Rows of padding (token_seq < 0) are left as they were.
// With `repair` ([0]: whether to work at all, [1]: CTAs that are done, [2 + i]: whether for sequence i; all 0 before) it goes over the
// result of a product that multiplies masked values by 0 (the attention of ordinary pages): a NaN among them would make all of it NaN, so
// they were taken out, and the rows of those sequences are computed here.  The last CTA to end leaves all numbers 0 again.
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
    int* error_flag;
    int* repair;
    int n_seqs;
};

template <typename T>
__device__ void attn_kv4_item(const Kv4SimpleArgs& a, long long item, float* qs, int lane) {
    const int row = (int)(item / a.nqh), head = (int)(item - (long long)row * a.nqh);
    const int seq = a.token_seq[row];
    if (seq < 0 || (a.repair && !a.repair[2 + seq])) return;
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
    if (a.repair && *(volatile int*)a.repair == 0) return;
    for (long long item = (long long)blockIdx.x * 4 + warp; item < (long long)a.rows * a.nqh; item += (long long)gridDim.x * 4)
        attn_kv4_item<T>(a, item, qs_all[warp], lane);
    if (a.repair) {
        __syncthreads();
        if (threadIdx.x == 0 && atomicAdd(a.repair + 1, 1) == (int)gridDim.x - 1) {      // every CTA has looked at the flag
            for (int i = 0; i < a.n_seqs + 2; ++i) a.repair[i] = 0;
        }
    }
}

extern "C" int braid_attn_kv4_simple(const void* q, long long q_stride, void* out, long long out_stride, int dtype, const void* cache,
                                     const int* page_table, const int* token_seq, const int* q_start, const int* kv_before, int rows, int nqh,
                                     int nkh, int hd, int cols, int num_pages, int window, int keep_first, float scale, int has_sink, float sink,
                                     float out_scale, const float* head_sinks, const void* head_gate, long long gate_stride, const float* head_scale,
                                     const float* bias_slope, const float* bias_rate, float softcap, int* repair, int n_seqs, int* error_flag, void* stream) {
    if (rows <= 0) return BRAID_OK;
    if (int rc = kv4_check("attn_kv4", nkh, hd, cache)) return rc;
    if (nqh <= 0 || nqh % nkh) BRAID_REFUSE("attn_kv4: %d query heads do not divide into %d kv heads", nqh, nkh);
    if (num_pages <= 0 || cols <= 0) BRAID_REFUSE("attn_kv4: the cache has no pages (pages=%d, table columns=%d)", num_pages, cols);
    long long ctas = ((long long)rows * nqh + 3) / 4;
    if (repair) ctas = min(ctas, 148LL);                      // one an SM: they hardly ever have anything to do
    if (ctas > 0x7fffffffLL) BRAID_REFUSE("attn_kv4: the rows exceed the grid limit");
    Kv4SimpleArgs a{q, out, (const uint8_t*)cache, page_table, token_seq, q_start, kv_before, q_stride, out_stride, rows, nqh, nkh, hd, cols, num_pages,
                    window, window > 0 ? keep_first : 0, scale, has_sink || head_sinks, sink, out_scale, head_sinks, head_gate, gate_stride, head_scale,
                    bias_slope, bias_rate, softcap, error_flag, repair, n_seqs};
    if (dtype == BRAID_F32) braid_launch(attn_kv4_simple_kernel<float>, dim3((unsigned)ctas), dim3(128), 0, (cudaStream_t)stream, a);
    else if (dtype == BRAID_BF16) braid_launch(attn_kv4_simple_kernel<__nv_bfloat16>, dim3((unsigned)ctas), dim3(128), 0, (cudaStream_t)stream, a);
    else BRAID_REFUSE("attn_kv4: unknown dtype code %d", dtype);
    BRAID_LAUNCH_CHECK();
}
