// Attention over a cache held in 4 bits (kv4.cuh), compiled for one head size: -DBRAID_HD=<32, 64, ... 256>.
//
// softmax over the visible keys of scale * q . k_j, with k_j = lowest + step * code a group of 32 numbers, so that
//   q . k_j = sum over groups g of  step_jg (q_g . code_jg) + lowest_jg sum(q_g)
//   out     = sum over keys of  (p_j step_jg) code_jg + sum over keys of p_j lowest_jg                         (for the numbers of group g)
//           = sum over keys of  (p_j step_jg) (code_jg - 8) + sum over keys of p_j (lowest_jg + 8 step_jg)
// Each sum of the first form is some 2 standard deviations of the values, and the result what is left of them; those of the second are about as
// small as the result.  bfloat16 runs take the first, whose codes cost less, with p step in float16 (FAST below; in bfloat16 it made errors
// of 0.0046 of the result behind 128k tokens).  Float32 runs take the second (the first: 7e-6 behind 3k tokens), and so does a warp of a
// bfloat16 run whose values float16 does not hold.
// The codes themselves are the tensor cores' operand (mma.sync m16n8k16, float32 sums): a mask makes two of them a pair of 16-bit
// numbers, exact, straight from the bytes as they are stored (`codes`).  So neither keys nor values are ever rounded, and what scales
// them is applied to a group's sums (keys) or to the probabilities (values).  Keys and value columns are the 16 rows of a product and the
// queries its 8 columns (query heads of one kv head, of up to 8 tokens), so that few queries waste little.
//
// What bounds it: reading the cache, 1.25 head-size bytes a token and kv head, at about two instructions a code of which the masks and
// shifts are half (64 requests of 8,000 in bfloat16: 135 us, 3.9 TB/s).  Every warp walks units of 32 or 64 tokens of its own through a ring of its own in shared memory, filled by one bulk copy a unit
// (the units are contiguous), so that warps never wait for one another before the end, where a CTA's warps merge their maxima, sums
// and results.  A context is sliced over CTAs where few would work on it: a few slices are a cluster, whose CTAs read one another's
// results and end together; those of more are merged by a second kernel.
// The running maximum of a column is raised only when a unit's scores exceed it by more than 4 (in powers of two): a vote instead
// of a reduction over the warp; sums are taken against the same maximum, so nothing is lost.
//
// float32 runs (PARTS 3): queries and scaled probabilities are three bfloat16 numbers each, whose products with the codes are exact, so
// that the result has float32's precision.
#include "kv4.cuh"
#include "tcgen05.cuh"
#include "softcap.cuh"
#include <cuda_fp16.h>
#include <type_traits>

#ifndef BRAID_HD
#error "compile with -DBRAID_HD=<head_dim>"
#endif
static_assert(BRAID_HD % 32 == 0 && BRAID_HD >= 32 && BRAID_HD <= 256, "head_dim must be a multiple of 32 in [32, 256]");

struct Kv4Args {
    const void* q;
    void* out;
    float* partial;              // n_splits > 1: [rows * nqh][n_splits][HD] results, then [rows * nqh][n_splits][2] maxima and sums
    const uint8_t* cache;
    const int* page_table;
    const int* q_start;
    const int* q_len;
    const int* kv_before;
    const int* token_seq;
    const float* head_sinks;
    const void* head_gate;
    const float* head_scale;
    const float* bias_slope;
    const float* bias_rate;
    int* error_flag;
    long long q_stride, out_stride, gate_stride;
    int rows, n_seqs, max_q_len, nqh, nkh, cols, num_pages, window, keep_first, n_splits, has_sink, settled;
    float scale, sink, out_scale, softcap;
    int f32;                     // float32 rows
    int cluster;                 // the slices are CTAs of a cluster, which merges them
    int q_from, q_to;            // (0: no bound) only sequences that bring at least, at most so many tokens
    int partial_rows;            // rows of `partial`: `rows`, or with q_to n_seqs * q_to (sequence, token)
};

#define LOG2E 1.4426950408889634f
#define KV4_RAISE 4.f

// What a merged row is multiplied by: 1 / its sum, the sink's share in it, and the head's gate.
template <typename T>
__device__ __forceinline__ float kv4_finish(const Kv4Args& a, float M, float L, int row, int head, const T*) {
    float f = 1.f;
    if (a.has_sink) {                                          // one more score, with no value
        const float sk = (a.head_sinks ? a.head_sinks[head] : a.sink) * LOG2E, mn = fmaxf(M, sk);
        f = exp2f(M - mn);
        L = L * f + exp2f(sk - mn);
    }
    float inv = f * a.out_scale / L;
    if (a.head_gate) inv *= 1.f / (1.f + expf(-to_f32(((const T*)a.head_gate)[(size_t)row * a.gate_stride + head])));
    return inv;
}

// The row whose slices are row `prow` of `partial`, or -1: none.
__device__ __forceinline__ int kv4_merged_row(const Kv4Args& a, int prow) {
    if (a.q_to > 0) {
        const int seq = prow / a.q_to, t = prow - seq * a.q_to, n = a.q_len[seq];
        return n <= a.q_to && t < n ? a.q_start[seq] + t : -1;
    }
    const int seq = a.token_seq[prow];
    return seq < 0 || (a.q_from > 0 && a.q_len[seq] < a.q_from) ? -1 : prow;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_zero(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
// Codes n and 4 + n of a word as a pair of 16-bit numbers.  FAST: the code's bits are left where they are and read as a number below
// the normal ones (or just at their start): the lowest 8 bits of bfloat16 count in steps of 2^-133, the lowest 11 of float16 in
// steps of 2^-24, so the pair is the codes times that, or 16 times that for odd n, in one instruction (and a shift for two of four).
// The products' other operand is scaled up by a power of two instead, and the results are scaled back.  (With 128 added to the code, the usual
// way, a code took 1.75 instructions and the 128 had to be taken off again: 64 requests of 8k 167 us instead of 140.)  Otherwise: the
// codes less 8, as they are, in bfloat16.
#define KV4_UNIT 133
#define KV4_NO_STEP 101                                       // step_exp of a group whose first unit has no range
template <bool FAST, int N> __device__ __forceinline__ uint32_t codes(uint32_t x) {
    if constexpr (FAST) {
        return (N & 2 ? x >> 8 : x) & (N & 1 ? 0x00f000f0u : 0x000f000fu);
    } else {
        const uint32_t y = ((x >> (4 * N)) & 0x000f000fu) | 0x43004300u;
        const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&y), __nv_bfloat162(__float2bfloat16(136.f), __float2bfloat16(136.f)));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((min(max(e, -126), 127) + 127) << 23); }
__device__ __forceinline__ int exponent(float x) { return (int)((__float_as_uint(x) >> 23) & 255u) - 127; }
// x * 2^e for any e
__device__ __forceinline__ float scaled(float x, int e) { const int h = e / 2; return x * pow2(h) * pow2(e - h); }
// The CTAs of a cluster: all have come here, and see what the others wrote before.
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// Shared memory at the address `at` of CTA `rank` of the cluster (`cluster` false: of this CTA).
__device__ __forceinline__ float2 ld_cluster2(uint32_t at, int rank, int cluster) {
    float2 v;
    if (cluster) {
        uint32_t p;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(p) : "r"(at), "r"(rank));
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(p) : "memory");
    } else {
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
    }
    return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t at, int rank, int cluster) {
    float4 v;
    if (cluster) {
        uint32_t p;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(p) : "r"(at), "r"(rank));
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(p) : "memory");
    } else {
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    }
    return v;
}
__device__ __forceinline__ float exp2_ftz(float x) {        // to 2 units of the last place; 0 below 2^-126
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// N neighbouring 32-bit words of shared memory, in the widest loads that their count allows
template <int N>
__device__ __forceinline__ void lds_words(const void* p, uint32_t* x) {
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
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// a bfloat16 pair from two float32 numbers, and what the rounding leaves
__device__ __forceinline__ uint32_t split_pair(float& a, float& b) {
    const uint32_t w = pack2(a, b);
    a -= __uint_as_float(w << 16);
    b -= __uint_as_float(w & 0xffff0000u);
    return w;
}

// The parity of a stage's last use, of `uses` that went through the stages in turn.
__host__ __device__ constexpr uint32_t kv4_last_parity(int uses, int stage, int stages) { return (uint32_t)((uses - 1 - stage) / stages) & 1u; }

template <int PARTS, int NW, int SR, int ST>
struct Kv4Cfg {
    static constexpr int HD = BRAID_HD, W = HD / 32;
    static constexpr int US = 16 * SR;                       // tokens a unit
    static constexpr int SB = SR * kv4_record_bytes(HD);     // bytes a unit
    static constexpr int BM = 8;                             // columns a CTA
    static constexpr int RING = NW * ST * SB;
    static constexpr int MERGE = NW * BM * (HD + 4) * 4;
    static constexpr int SMEM = RING > MERGE ? RING : MERGE;
    static_assert(BRAID_PAGE_SIZE % US == 0, "a unit must not straddle a page");
};

template <int PARTS, int NW, int SR, int ST>
__global__ void __launch_bounds__(NW * 32, SR == 4 ? 2 : 1)
attn_kv4_kernel(const Kv4Args a) {
    using C = Kv4Cfg<PARTS, NW, SR, ST>;
    using T = typename std::conditional<PARTS == 3, float, __nv_bfloat16>::type;
    constexpr int HD = C::HD, W = C::W;
    pdl_trigger();
    // a caller that has made the tables, or this step's older keys, with kernels of this library right before does not say `settled`
    if (!a.settled) pdl_wait();
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint64_t full[NW][ST];
    __shared__ int abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int r = lane >> 2, j = lane & 3;
    const int g = a.nqh / a.nkh;
    const int hpc = min(g, C::BM), tpc = C::BM / hpc, hchunks = (g + hpc - 1) / hpc;
    const int seq = blockIdx.y;
    const int heads = a.nkh * hchunks, part = blockIdx.x / heads, hx = blockIdx.x - part * heads;
    const int kvh = hx / hchunks, hchunk = hx - kvh * hchunks;
    // late tokens, which see the most, first (and more than 65,535 tiles in parts along x)
    const int unit = (int)(gridDim.x / heads - part) * (int)gridDim.z - 1 - (int)blockIdx.z;
    const int tile = unit / a.n_splits, split = unit - tile * a.n_splits;
    const int q_len = a.q_len[seq], tok0 = tile * tpc;
    if (tok0 >= q_len || (a.q_to > 0 && q_len > a.q_to)) {
        pdl_wait();                                            // all CTAs may leave here, and a grid ends after what is ahead of it (common.cuh)
        return;
    }
    const int q_start = a.q_start[seq], kv_before = a.kv_before[seq];
    const int n_tok = min(tpc, q_len - tok0);
    const int head0 = kvh * g + hchunk * hpc, n_heads = min(hpc, g - hchunk * hpc);
    const int pos_min = kv_before + tok0, pos_max = pos_min + n_tok - 1;
    const int k_lo = (a.window > 0 && pos_min - a.window + 1 > 0) ? pos_min - a.window + 1 : 0;
    const int t_win = k_lo / C::US;                            // the units walked: kept first ones that the window has left, then the window's
    const int n_first = min((a.keep_first + C::US - 1) / C::US, t_win);
    int i_lo = 0, i_hi = n_first + pos_max / C::US + 1 - t_win;
    if (a.n_splits > 1) {
        const int per = (i_hi + a.n_splits - 1) / a.n_splits;
        i_lo = min(i_hi, split * per);
        i_hi = min(i_hi, i_lo + per);
    }
    const int n_mine = max(0, (i_hi - i_lo - warp + NW - 1) / NW);
    auto tile_of = [&](int k) { const int i = i_lo + warp + k * NW; return i < n_first ? i : t_win + (i - n_first); };

    uint8_t* ring = smem + warp * (ST * C::SB);
    if (tid == 0) abort_flag = 0;
    if (lane == 0) {
#pragma unroll
        for (int s = 0; s < ST; ++s) mbar_init(&full[warp][s], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    const int* table = a.page_table + (size_t)seq * a.cols;
    int issued = 0, istage = 0, pages = 0;                     // a lane's page: of this warp's unit (issued & ~31) + lane
    int earlier = 0;                                           // units that a first walk had asked for
    auto issue = [&]() {
        if ((issued & 31) == 0) {
            pages = 0;
            if (issued + lane < n_mine) {
                const int block = tile_of(issued + lane) / (BRAID_PAGE_SIZE / C::US);
                const int p = block < a.cols ? table[block] : -1;
                if (p < 0 || p >= a.num_pages) atomicExch(a.error_flag, 1);      // never followed: page 0 is read instead
                else pages = p;
            }
        }
        const int page = __shfl_sync(0xffffffffu, pages, issued & 31);
        if (lane == 0) {
            const int t = tile_of(issued);
            mbar_expect_tx(&full[warp][istage], C::SB);
            bulk_load(ring + istage * C::SB, a.cache + ((size_t)page * a.nkh + kvh) * kv4_page_bytes(HD) + (t % (BRAID_PAGE_SIZE / C::US)) * C::SB,
                      C::SB, &full[warp][istage]);
        }
        ++issued;
        if (++istage == ST) istage = 0;
    };
    // units that hold only tokens cached before this step may be asked for at once
    if (a.settled) {
        while (issued < min(ST, n_mine) && (tile_of(issued) + 1) * C::US <= kv_before) issue();
        pdl_wait();
    }
    while (issued < min(ST, n_mine)) issue();

    // ---- queries: column r, numbers 32 w + 8 j .. + 7 of the head
    uint32_t q[W][PARTS][4];
    constexpr int GH = W > 4 ? 2 : 1;
    constexpr int QP = PARTS > 1 ? 3 : 2;                      // 16 bits of it (off by 2^-17, below the probabilities' 2^-12), or all
    uint32_t qb[QP][GH];                                       // the sum of group j's (and 4 + j's) numbers beside a zero, in parts
    int q_exp;                                                 // of column r: the queries are scaled by 2^q_exp
    const int col = r, tl = col / hpc, hl = col - tl * hpc;
    const bool in = tl < n_tok && hl < n_heads;
    const T* src = (const T*)a.q + (size_t)(q_start + (in ? tok0 + tl : 0)) * a.q_stride + (size_t)(head0 + (in ? hl : 0)) * HD + 8 * j;
    const bool wide = !(((uintptr_t)a.q | (uintptr_t)(a.q_stride * sizeof(T))) & 15);
    float x[W][8], most = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        if (wide) {
            constexpr int VW = 16 / sizeof(T);
#pragma unroll
            for (int i = 0; i < 8; i += VW) load_run<T, VW>(src + 32 * w + i, x[w] + i);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[w][i] = to_f32(src[32 * w + i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (!in) x[w][i] = 0.f;
            most = fmaxf(most, fabsf(x[w][i]));
        }
    }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    q_exp = 120 - exponent(most);                      // the column's largest number becomes one of 2^120
    float sums[GH];
#pragma unroll
    for (int h = 0; h < GH; ++h) sums[h] = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += x[w][i];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if ((w & 3) == j) sums[w >> 2] = sum;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[w][i] = scaled(x[w][i], q_exp - (i & 2 ? 4 : 0));       // numbers of odd n meet 16 times their code
#pragma unroll
        for (int p = 0; p < PARTS; ++p)
#pragma unroll
            for (int n = 0; n < 4; ++n) q[w][p][n] = split_pair(x[w][2 * n], x[w][2 * n + 1]);
    }
#pragma unroll
    for (int h = 0; h < GH; ++h) {
        float none = 0.f, sum = scaled(sums[h], q_exp - KV4_UNIT);
#pragma unroll
        for (int p = 0; p < QP; ++p) qb[p][h] = split_pair(none, sum);
    }
    // ---- this lane's columns of scores: 2 j + c
    int pos[2], lo[2];
    float sc[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int col = 2 * j + c, tl = col / hpc, hl = col - tl * hpc;
        const bool in = tl < n_tok && hl < n_heads;
        pos[c] = in ? pos_min + tl : -1;                       // -1: the column sees nothing
        lo[c] = a.window > 0 ? pos[c] - a.window + 1 : 0;
        sc[c] = scaled((in && a.head_scale ? a.scale * a.head_scale[head0 + hl] : a.scale) * (a.softcap > 0.f ? 1.f / a.softcap : LOG2E),
                       KV4_UNIT - __shfl_sync(0xffffffffu, q_exp, 8 * j + 4 * c));
    }

    // a factor that is positive commutes with the maximum, and leaves -infinity as it is
    bool late = !(a.softcap > 0.f) && !a.bias_slope;
    late = late && sc[0] > 0.f && sc[1] > 0.f;
    late = __all_sync(0xffffffffu, late);
    float lf[2];
    lf[0] = late ? sc[0] : 1.f;
    lf[1] = late ? sc[1] : 1.f;
    float o[2 * W][4], zs[2][W], m[2], l[2];
    bool ok = true;
    bool walked = PARTS == 1;
    uint32_t signs = 0;                                        // FAST: of the scaled probabilities; one is negative where its step's exponent passed 255
    int st = 0, step_exp[W];                                   // FAST: the steps of a group are scaled by 2^step_exp
    uint32_t phase = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) step_exp[w] = 0;
    // FAST takes the scaled probabilities as float16 numbers: they are rounded by 2^-11 (a code counts up to 15 steps, which with the 2^-8 of
    // bfloat16 made errors of 0.0046 of the result), and pass the type's range where a group's later steps are much larger than its
    // first ones (2^7 times, at a probability of 1): the results are then not finite, or, where the scaled step has passed float32's range too, its
    // sum of exponents has run into the sign bit, which steps and probabilities never have (`signs`).  At the other end, steps of down to 2^-23 of the first
    // ones keep all 11 bits at a probability of 1, and what lies below is rounded to multiples of 2^-24: where the first unit's
    // large values have next to no probability, that is all of the result (`low`, below).  Either way the warp walks once more in bfloat16, codes less
    // 8 and nothing scaled.
    auto walk = [&](auto FAST) {
    constexpr bool fast = decltype(FAST)::value;
#pragma unroll
    for (int i = 0; i < 2 * W; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        m[c] = -INFINITY;
        l[c] = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) zs[c][w] = 0.f;
    }
    for (int k = 0; k < n_mine; ++k) {
        ok = __all_sync(0xffffffffu, mbar_wait(&full[warp][st], phase, &abort_flag));
        if (!ok) break;
        const uint8_t* base = ring + st * C::SB;
        if (++st == ST) { st = 0; phase ^= 1u; }
        const int key0 = tile_of(k) * C::US;
        if (fast && k == 0) {
            // a group's scale: its largest step in the first unit, times a probability of 1, becomes one of 2^9
            float most[GH];
#pragma unroll
            for (int h = 0; h < GH; ++h) most[h] = 0.f;
#pragma unroll
            for (int rec = 0; rec < SR; ++rec)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int key = key0 + 16 * rec + 8 * h + r;
                    const uint32_t* g = reinterpret_cast<const uint32_t*>(base + rec * kv4_record_bytes(HD) + kv4_value_groups(HD)) + (8 * h + r) * W;
                    if (key <= pos_max && (key >= k_lo || key < a.keep_first))
#pragma unroll
                        for (int i = 0; i < GH; ++i)
                            if (4 * i + j < W) most[i] = fmaxf(most[i], kv4_step(g[4 * i + j]));
                }
            bool in = true;
#pragma unroll
            for (int i = 0; i < GH; ++i) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) most[i] = fmaxf(most[i], __shfl_xor_sync(0xffffffffu, most[i], x));
                const int e = most[i] == 0.f ? KV4_NO_STEP : 9 - exponent(most[i]);
                in &= e >= 0 && (e <= 100 || most[i] == 0.f);
#pragma unroll
                for (int w = 4 * i; w < W && w < 4 * i + 4; ++w) step_exp[w] = __shfl_sync(0xffffffffu, e, w & 3);
            }
            if (!__all_sync(0xffffffffu, in)) { walked = false; return; }
        }

        // ---- scores of the unit's tokens: rows 16 rec + r, + 8; s[rec][0, 1]: columns of row r, [2, 3]: of row r + 8
        float s[SR][4];
#pragma unroll
        for (int rec = 0; rec < SR; ++rec) {
            const uint8_t* rb = base + rec * kv4_record_bytes(HD);
            uint32_t ka[W], kb[W], ga[W], gb[W];
            lds_words<W>(rb + r * (HD / 2) + j * (4 * W), ka);
            lds_words<W>(rb + (r + 8) * (HD / 2) + j * (4 * W), kb);
            const uint8_t* groups = rb + kv4_key_groups(HD) + r * (4 * W);
            lds_words<W>(groups, ga);
            lds_words<W>(groups + 32 * W, gb);
            // what the lowest values add to the scores: a product with the queries' sums, whose operand the groups' words are as they lie
            uint32_t wa[2] = {0u, 0u}, wb[2] = {0u, 0u};
            if (W >= 4 || j < W) {
                wa[0] = reinterpret_cast<const uint32_t*>(groups)[j];
                wb[0] = reinterpret_cast<const uint32_t*>(groups + 32 * W)[j];
            }
            if (W == 8 || 4 + j < W) {
                wa[1] = reinterpret_cast<const uint32_t*>(groups)[4 + j];
                wb[1] = reinterpret_cast<const uint32_t*>(groups + 32 * W)[4 + j];
            }
            mma16816_zero(s[rec], wa[0], wb[0], wa[1], wb[1], qb[0][0], GH > 1 ? qb[0][GH - 1] : 0u);
#pragma unroll
            for (int p = 1; p < QP; ++p) mma16816(s[rec], wa[0], wb[0], wa[1], wb[1], qb[p][0], GH > 1 ? qb[p][GH - 1] : 0u);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const uint32_t a0 = codes<true, 0>(ka[w]), a1 = codes<true, 0>(kb[w]), a2 = codes<true, 1>(ka[w]), a3 = codes<true, 1>(kb[w]);
                const uint32_t b0 = codes<true, 2>(ka[w]), b1 = codes<true, 2>(kb[w]), b2 = codes<true, 3>(ka[w]), b3 = codes<true, 3>(kb[w]);
                const float sa = kv4_step(ga[w]), sb = kv4_step(gb[w]);
                float raw[4];
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    if (p == 0) mma16816_zero(raw, a0, a1, a2, a3, q[w][p][0], q[w][p][1]);
                    else mma16816(raw, a0, a1, a2, a3, q[w][p][0], q[w][p][1]);
                    mma16816(raw, b0, b1, b2, b3, q[w][p][2], q[w][p][3]);
                }
                s[rec][0] = fmaf(sa, raw[0], s[rec][0]);
                s[rec][1] = fmaf(sa, raw[1], s[rec][1]);
                s[rec][2] = fmaf(sb, raw[2], s[rec][2]);
                s[rec][3] = fmaf(sb, raw[3], s[rec][3]);
            }
        }
        // ---- factors, cap, bias; mask.  Plain scores are left as they are: their factor is applied where the exponential is taken
        if (!late)
#pragma unroll
            for (int rec = 0; rec < SR; ++rec)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[rec][e] *= sc[e & 1];
        if (a.softcap > 0.f) softcap_scores<SR * 4>(&s[0][0], 1.f, a.softcap * LOG2E);
        if (a.bias_slope) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int col = 2 * j + c, hl = col % hpc;
                const float r1 = hl < n_heads ? a.bias_slope[head0 + hl] : 0.f, r2 = hl < n_heads ? a.bias_rate[head0 + hl] : 0.f;
#pragma unroll
                for (int rec = 0; rec < SR; ++rec)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {          // (keys after the query are masked below)
                        const float d = (float)(pos[c] - (key0 + 16 * rec + 8 * h + r));
                        s[rec][2 * h + c] -= r1 * LOG2E * log1pf(r2 * fmaxf(d, 0.f));
                    }
            }
        }
        // (columns that are no query see as much as the others, and nobody reads them)
        const bool edge = !(key0 + C::US - 1 <= pos_min && (a.window == 0 || key0 >= pos_max - a.window + 1));
        if (edge) {
#pragma unroll
            for (int rec = 0; rec < SR; ++rec)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = key0 + 16 * rec + 8 * (e >> 1) + r, c = e & 1;
                    if (!(key <= pos[c] && (key >= lo[c] || key < a.keep_first))) s[rec][e] = -INFINITY;
                }
        }
        // ---- running maximum
        float top[2];
        bool raise = false;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float x = fmaxf(s[0][c], s[0][2 + c]);
#pragma unroll
            for (int rec = 1; rec < SR; ++rec) x = fmaxf(x, fmaxf(s[rec][c], s[rec][2 + c]));
            x *= lf[c];
            top[c] = x;
            raise |= x > m[c] + KV4_RAISE;
        }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x = top[c];
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                x = fmaxf(x, m[c]);
                const float f = x == -INFINITY ? 1.f : exp2f(m[c] - x);      // exp2(-inf) = 0
                m[c] = x;
                l[c] *= f;
#pragma unroll
                for (int w = 0; w < W; ++w) zs[c][w] *= f;
#pragma unroll
                for (int i = 0; i < 2 * W; ++i) { o[i][c] *= f; o[i][2 + c] *= f; }
            }
        }
        // ---- probabilities and values.  On an edge (EDGE) what a column does not see does not count, whatever it holds: a value's
        // step or lowest number may be NaN
        auto values = [&](auto EDGE) {
#pragma unroll
        for (int rec = 0; rec < SR; ++rec) {
            const uint8_t* rb = base + rec * kv4_record_bytes(HD);
            uint32_t ga[W], gb[W];
            lds_words<W>(rb + kv4_value_groups(HD) + r * (4 * W), ga);
            lds_words<W>(rb + kv4_value_groups(HD) + (r + 8) * (4 * W), gb);
            // value codes of tokens 2 j, 2 j + 1, 2 j + 8, 2 j + 9, numbers 32 w + 4 r .. + 3: 16 bits a group
            const uint8_t* vc = rb + kv4_value_codes(HD) + 2 * j * (HD / 2) + r * (2 * W);
            uint32_t v01[W], v89[W];
            if constexpr (W % 2 == 0) {
                uint32_t x0[W / 2], x1[W / 2], x8[W / 2], x9[W / 2];
                lds_words<W / 2>(vc, x0);
                lds_words<W / 2>(vc + HD / 2, x1);
                lds_words<W / 2>(vc + 8 * (HD / 2), x8);
                lds_words<W / 2>(vc + 9 * (HD / 2), x9);
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    v01[w] = __byte_perm(x0[w / 2], x1[w / 2], w & 1 ? 0x7632 : 0x5410);
                    v89[w] = __byte_perm(x8[w / 2], x9[w / 2], w & 1 ? 0x7632 : 0x5410);
                }
            } else {
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const uint16_t* u = reinterpret_cast<const uint16_t*>(vc) + w;
                    v01[w] = u[0] | ((uint32_t)u[HD / 4] << 16);
                    v89[w] = u[8 * (HD / 4)] | ((uint32_t)u[9 * (HD / 4)] << 16);
                }
            }
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = e & 1;
                p[e] = exp2_ftz(fmaf(s[rec][e], lf[c], m[c] == -INFINITY ? 0.f : -m[c]));
                l[c] += p[e];
            }
#pragma unroll
            for (int w = 0; w < W; ++w) {
                // (a step of 0 becomes some number below the codes' reach; its codes are 0)
                const float sa = __uint_as_float(ga[w] * 65536u + (fast ? (uint32_t)step_exp[w] << 23 : 0u));
                const float sb = __uint_as_float(gb[w] * 65536u + (fast ? (uint32_t)step_exp[w] << 23 : 0u));
                const float za = fast ? kv4_lowest(ga[w]) : fmaf(8.f, sa, kv4_lowest(ga[w])), zb = fast ? kv4_lowest(gb[w]) : fmaf(8.f, sb, kv4_lowest(gb[w]));
                const uint32_t a0 = codes<fast, 0>(v01[w]), a1 = codes<fast, 1>(v01[w]), a2 = codes<fast, 0>(v89[w]), a3 = codes<fast, 1>(v89[w]);
                const uint32_t b0 = codes<fast, 2>(v01[w]), b1 = codes<fast, 3>(v01[w]), b2 = codes<fast, 2>(v89[w]), b3 = codes<fast, 3>(v89[w]);
                float x[4] = {p[0] * sa, p[1] * sa, p[2] * sb, p[3] * sb};
                if constexpr (EDGE.value) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool seen = s[rec][e] != -INFINITY;
                        if (!seen) x[e] = 0.f;
                        if (seen) zs[e & 1][w] = fmaf(p[e], e < 2 ? za : zb, zs[e & 1][w]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) zs[e & 1][w] = fmaf(p[e], e < 2 ? za : zb, zs[e & 1][w]);
                }
                if constexpr (fast) {
                    const uint32_t x0 = pack_half(x[0], x[1]), x1 = pack_half(x[2], x[3]);
                    signs |= x0 | x1;
                    const uint32_t p0 = transpose8x8(x0), p1 = transpose8x8(x1);
                    mma16816_f16(o[2 * w], a0, a1, a2, a3, p0, p1);
                    mma16816_f16(o[2 * w + 1], b0, b1, b2, b3, p0, p1);
                } else {
                    // The tensor cores cut sums off instead of rounding them, which over thousands of tokens is a bias: a record's products are
                    // summed there, the records here.  (21 sequences of 7 tokens behind up to 11,614, heads of 32: errors of
                    // 1.7e-5 of a float32 result before, 6.7e-7 so; 71 -> 78 us.)
                    float t0[4], t1[4];
#pragma unroll
                    for (int part = 0; part < PARTS; ++part) {
                        const uint32_t p0 = transpose8x8(split_pair(x[0], x[1])), p1 = transpose8x8(split_pair(x[2], x[3]));
                        if (part == 0) {
                            mma16816_zero(t0, a0, a1, a2, a3, p0, p1);
                            mma16816_zero(t1, b0, b1, b2, b3, p0, p1);
                        } else {
                            mma16816(t0, a0, a1, a2, a3, p0, p1);
                            mma16816(t1, b0, b1, b2, b3, p0, p1);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) { o[2 * w][i] += t0[i]; o[2 * w + 1][i] += t1[i]; }
                }
            }
        }
        };
        if (edge || !fast) values(std::true_type{});
        else values(std::false_type{});
        __syncwarp();                                          // every lane has read the unit
        if (issued < n_mine) issue();
    }
    };
    if constexpr (PARTS == 1) walk(std::true_type{});
    bool low = false;
    if constexpr (PARTS == 1) {
        // Roundings of small products p step (to half of 2^-24) are at most 15 2^-25 a token of a result's number: less than 2^-11 of the
        // group's largest number, or that is too small.  (Numbers of odd n count codes 16 times.  A group that had no range in the first unit, and has zeros
        // for results, had none that counts: p step below 2^-126.)
        const float least = (float)(n_mine * C::US) * (15.f * 0x1p-38f);
        auto largest = [&](int w, int c) { return fmaxf(fmaxf(o[2 * w][c], o[2 * w + 1][c]), 0x1p-4f * fmaxf(o[2 * w][2 + c], o[2 * w + 1][2 + c])); };
        float v = INFINITY;
#pragma unroll
        for (int w = 0; w < W; ++w) v = fminf(v, fminf(largest(w, 0), largest(w, 1)));
        if (__any_sync(0xffffffffu, v < least)) {              // (of this lane's numbers; of all of a group's?)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const uint32_t mine = 0x11111111u << j;        // the lanes that have this column
                const bool sees = __ballot_sync(0xffffffffu, l[c] > 0.f) & mine;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const uint32_t enough = __ballot_sync(0xffffffffu, largest(w, c) >= least), some = __ballot_sync(0xffffffffu, largest(w, c) != 0.f);
                    low |= sees && !(enough & mine) && (step_exp[w] != KV4_NO_STEP || (some & mine));
                }
            }
        }
    }
    {
        float t = walked && !(signs & 0x80008000u) && !low ? 0.f : INFINITY;
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) t = fmaf(0.f, o[i][0], fmaf(0.f, o[i][1], fmaf(0.f, o[i][2], fmaf(0.f, o[i][3], t))));
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            t = fmaf(0.f, l[c], t);
#pragma unroll
            for (int w = 0; w < W; ++w) t = fmaf(0.f, zs[c][w], t);
        }
        if (__any_sync(0xffffffffu, ok && t != 0.f)) {
            if constexpr (PARTS == 1) for (; st != istage; phase ^= (st == ST - 1), st = st == ST - 1 ? 0 : st + 1)        // (units asked for and not walked)
                ok = __all_sync(0xffffffffu, mbar_wait(&full[warp][st], phase, &abort_flag)) && ok;
            if (PARTS != 1 || ok) {
                if constexpr (PARTS == 1) {
                    earlier = issued;
                    issued = 0;
                    while (issued < min(ST, n_mine)) issue();
                }
                walk(std::false_type{});
                walked = false;
            }
        }
    }
    if (!ok) {
        // a copy did not arrive in time: wait for the others (bounded too), so that none lands after the CTA has ended
        if (lane == 0) atomicExch(a.error_flag, 1);
        for (int s = 0; s < ST; ++s)
            if (earlier + issued > s) for (uint32_t i = 0; i < (1u << 20) && !mbar_try_wait(&full[warp][s], kv4_last_parity(earlier + issued, s, ST)); ++i) {}
    }

    // ---- the CTA's warps merge
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
            l[c] += __shfl_xor_sync(0xffffffffu, l[c], x);
#pragma unroll
            for (int w = 0; w < W; ++w) zs[c][w] += __shfl_xor_sync(0xffffffffu, zs[c][w], x);
        }
    __syncthreads();                                           // every warp is done with its ring
    float* mo = reinterpret_cast<float*>(smem);                // [warp][column][HD]
    float* ml = mo + NW * C::BM * HD;                          // [warp][column][2]
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int col = 2 * j + c;
        float* dst = mo + (warp * C::BM + col) * HD + 4 * r;
#pragma unroll
        for (int w = 0; w < W; ++w)
        {
            // FAST: codes counted in steps of 2^-24, those of odd n in steps 16 times that
            const int even = walked ? 24 - step_exp[w] : 0, odd = walked ? even - 4 : 0;
            *reinterpret_cast<float4*>(dst + 32 * w) = make_float4(
                fmaf(o[2 * w][c], pow2(even), zs[c][w]), fmaf(o[2 * w][2 + c], pow2(odd), zs[c][w]),
                fmaf(o[2 * w + 1][c], pow2(even), zs[c][w]), fmaf(o[2 * w + 1][2 + c], pow2(odd), zs[c][w]));
        }
        if (r == 0) { ml[(warp * C::BM + col) * 2] = m[c]; ml[(warp * C::BM + col) * 2 + 1] = l[c]; }
    }
    __syncthreads();
    const bool out_wide = !(((uintptr_t)a.out | (uintptr_t)(a.out_stride * sizeof(T))) & (4 * sizeof(T) - 1));
    // a column's numbers d .. d + 3 from what `n` slices of this CTA's (or the cluster's) warps left
    auto merge = [&](int col, int d, int n, float& M, float& L, float4& x) {
        M = -INFINITY;
        L = 0.f;
        x = make_float4(0.f, 0.f, 0.f, 0.f);
        const uint32_t at_ml = smem_u32(ml + col * 2), at_o = smem_u32(mo + col * HD + d);
        for (int i = 0; i < n; ++i)
#pragma unroll
            for (int w = 0; w < NW; ++w) M = fmaxf(M, ld_cluster2(at_ml + w * (C::BM * 8), i, a.cluster).x);
        const float ref = M == -INFINITY ? 0.f : M;
        for (int i = 0; i < n; ++i) {
            float2 sl[NW];
            float4 y[NW];
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                sl[w] = ld_cluster2(at_ml + w * (C::BM * 8), i, a.cluster);
                y[w] = ld_cluster4(at_o + w * (C::BM * HD * 4), i, a.cluster);
            }
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                // a slice without a finite score has weight 0, which leaves nothing of its zeros and all of a NaN (weight 1 if none has one)
                const float f = M == -INFINITY ? 1.f : exp2f(sl[w].x - ref);
                L = fmaf(sl[w].y, f, L);
                x.x = fmaf(y[w].x, f, x.x); x.y = fmaf(y[w].y, f, x.y); x.z = fmaf(y[w].z, f, x.z); x.w = fmaf(y[w].w, f, x.w);
            }
        }
    };
    if (a.cluster) cluster_barrier();                          // every CTA's results are in its shared memory
    const int first = a.cluster ? split * (NW * 32) + tid : tid, turn = a.cluster ? a.n_splits * (NW * 32) : NW * 32;
    for (int i = first; i < C::BM * (HD / 4); i += turn) {
        const int col = i / (HD / 4), d = (i - col * (HD / 4)) * 4;
        const int tl = col / hpc, hl = col - tl * hpc;
        if (!(tl < n_tok && hl < n_heads)) continue;
        const int head = head0 + hl;
        const size_t row = (size_t)(q_start + tok0 + tl);
        float M, L;
        float4 x;
        merge(col, d, a.cluster ? a.n_splits : 1, M, L, x);
        if (a.n_splits > 1 && !a.cluster) {
            const size_t prow = a.q_to > 0 ? (size_t)seq * a.q_to + tok0 + tl : row, at = (prow * a.nqh + head) * a.n_splits + split;
            *reinterpret_cast<float4*>(a.partial + at * HD + d) = x;
            if (d == 0) *reinterpret_cast<float2*>(a.partial + (size_t)a.partial_rows * a.nqh * a.n_splits * HD + at * 2) = make_float2(M, L);
            continue;
        }
        const float inv = kv4_finish(a, M, L, (int)row, head, (T*)nullptr);
        T* dst = (T*)a.out + row * a.out_stride + (size_t)head * HD + d;
        __align__(16) T y[4] = {from_f32<T>(x.x * inv), from_f32<T>(x.y * inv), from_f32<T>(x.z * inv), from_f32<T>(x.w * inv)};
        if (!out_wide) {
#pragma unroll
            for (int e = 0; e < 4; ++e) dst[e] = y[e];
        } else if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(y);
        else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(y);
    }
    if (a.cluster) cluster_barrier();                          // no CTA ends before the others have read its results
}

// The slices of a (row, head) made one: sum_s O_s 2^(m_s - M) / sum_s l_s 2^(m_s - M).  A CTA a (row, head): HD / 4 threads take four numbers
// each of every G-th slice (so that all loads of up to 8 G slices are on their way together), and the first of them join the shares.
template <typename T>
__global__ void __launch_bounds__(256)
attn_kv4_merge_kernel(const Kv4Args a) {
    constexpr int HD = BRAID_HD, Q = HD / 4, G = 256 / Q;
    pdl_trigger();
    pdl_wait();
    __shared__ float4 so[G][Q];
    __shared__ float2 sm[G];
    const int rh = blockIdx.x, head = rh % a.nqh, row = kv4_merged_row(a, rh / a.nqh);
    if (row < 0) return;
    const int g = threadIdx.x / Q, q = threadIdx.x - g * Q;
    const bool works = g < G;
    const float* po = a.partial + (size_t)rh * a.n_splits * HD + q * 4;
    const float2* pm = reinterpret_cast<const float2*>(a.partial + (size_t)a.partial_rows * a.nqh * a.n_splits * HD) + (size_t)rh * a.n_splits;
    float M = -INFINITY, L = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    auto join = [&](float m, float l, const float4& y) {       // a share without a finite score has weight 0: nothing of zeros, all of a NaN
        const float Mn = fmaxf(M, m), ref = Mn == -INFINITY ? 0.f : Mn, c = Mn == -INFINITY ? 1.f : exp2f(M - ref), f = Mn == -INFINITY ? 1.f : exp2f(m - ref);
        L = fmaf(L, c, l * f);
        x.x = fmaf(x.x, c, y.x * f); x.y = fmaf(x.y, c, y.y * f); x.z = fmaf(x.z, c, y.z * f); x.w = fmaf(x.w, c, y.w * f);
        M = Mn;
    };
    constexpr int B = 8;
    if (works)
        for (int s0 = g; s0 < a.n_splits; s0 += B * G) {
            float2 ml[B];
            float4 y[B];
#pragma unroll
            for (int i = 0; i < B; ++i) {
                const bool in = s0 + i * G < a.n_splits;
                ml[i] = in ? pm[s0 + i * G] : make_float2(-INFINITY, 0.f);
                y[i] = in ? *reinterpret_cast<const float4*>(po + (size_t)(s0 + i * G) * HD) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int i = 0; i < B; ++i)
                if (s0 + i * G < a.n_splits) join(ml[i].x, ml[i].y, y[i]);
        }
    if (works) {
        so[g][q] = x;
        if (q == 0) sm[g] = make_float2(M, L);
    }
    __syncthreads();
    if (threadIdx.x >= Q) return;
    for (int i = 1; i < G; ++i) join(sm[i].x, sm[i].y, so[i][q]);
    const float inv = kv4_finish(a, M, L, row, head, (T*)nullptr);
    T* dst = (T*)a.out + (size_t)row * a.out_stride + (size_t)head * HD + q * 4;
    const float y[4] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv};
#pragma unroll
    for (int e = 0; e < 4; ++e) dst[e] = from_f32<T>(y[e]);
}

// The same for up to 8 slices, a warp a (row, head): prompts have thousands of those, and a CTA for each was bound by its start (a step of 700
// tokens of 32 heads of 128 behind 16,500 in 3 slices, all of it: 275 us with a CTA each, 190 so).
template <typename T>
__global__ void __launch_bounds__(256)
attn_kv4_merge_few_kernel(const Kv4Args a) {
    constexpr int HD = BRAID_HD, W = HD / 32, V = W % 4 == 0 ? 4 : W % 2 == 0 ? 2 : 1, B = 8;
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long rh = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (rh >= (long long)a.partial_rows * a.nqh) return;
    const int head = (int)(rh % a.nqh), row = kv4_merged_row(a, (int)(rh / a.nqh)), n = a.n_splits;
    if (row < 0) return;
    const float2* pm = reinterpret_cast<const float2*>(a.partial + (size_t)a.partial_rows * a.nqh * n * HD) + (size_t)rh * n;
    const float* po = a.partial + (size_t)rh * n * HD + lane * V;
    const float2 ml = lane < n ? pm[lane] : make_float2(-INFINITY, 0.f);
    float y[B][W];                                             // numbers 32 V i + V lane + 0 .. V - 1 in y[][V i ...]
#pragma unroll
    for (int s = 0; s < B; ++s)
#pragma unroll
        for (int i = 0; i < W; i += V) {
            if (s >= n) break;
            const float* src = po + (size_t)s * HD + 32 * i;
            if constexpr (V == 4) *reinterpret_cast<float4*>(&y[s][i]) = *reinterpret_cast<const float4*>(src);
            else if constexpr (V == 2) *reinterpret_cast<float2*>(&y[s][i]) = *reinterpret_cast<const float2*>(src);
            else y[s][i] = *src;
        }
    float M = ml.x;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    M = __shfl_sync(0xffffffffu, M, 0);
    // a share without a finite score has weight 0: nothing of zeros, all of a NaN
    const float weight = M == -INFINITY ? 1.f : exp2f(ml.x - M);
    float L = 0.f, x[W];
#pragma unroll
    for (int i = 0; i < W; ++i) x[i] = 0.f;
#pragma unroll
    for (int s = 0; s < B; ++s) {
        const float w = __shfl_sync(0xffffffffu, weight, s), l = __shfl_sync(0xffffffffu, ml.y, s);
        if (s >= n) break;
        L = fmaf(l, w, L);
#pragma unroll
        for (int i = 0; i < W; ++i) x[i] = fmaf(y[s][i], w, x[i]);
    }
    const float inv = kv4_finish(a, M, L, row, head, (T*)nullptr);
    T* dst = (T*)a.out + (size_t)row * a.out_stride + (size_t)head * HD + lane * V;
#pragma unroll
    for (int i = 0; i < W; i += V)
#pragma unroll
        for (int e = 0; e < V; ++e) dst[32 * i + e] = from_f32<T>(x[i + e] * inv);
}

// ------------------------------------------------------------------ host side
// Four warps a CTA.  A unit is SR records of 16 tokens: four of them give a warp enough independent products to work on (one request of
// 128k, heads of 128: 53 us with two records a unit and 12 warps an SM, 45 with four and 8 (42 in all by now), which may take 255 registers then; 54 with
// 12 warps of four records in parts that come and go by themselves); two where the registers hold no more: float32, heads above 128.
// More queries than 8 columns hold are more CTAs: 16 columns a CTA, which share the codes' way to the operands but leave room for two records, took
// longer (us, 16 / 8 columns: 6 sequences of 5 tokens of 4 heads in a window of 4,096, 32 / 27; 64 of 5 behind 4,000, 214 / 179; heads of 64, 141 / 102).
#define KV4_NW 4
constexpr int kv4_sr(int parts) { return BRAID_HD <= 128 && parts == 1 ? 4 : 2; }
constexpr int kv4_st(int parts) { return kv4_sr(parts) == 4 || BRAID_HD > 128 ? 2 : 3; }
template <int PARTS> using Kv4C = Kv4Cfg<PARTS, KV4_NW, kv4_sr(PARTS), kv4_st(PARTS)>;

template <int PARTS>
static const void* kv4_kernel() { return (const void*)attn_kv4_kernel<PARTS, KV4_NW, kv4_sr(PARTS), kv4_st(PARTS)>; }

template <int PARTS>
static int launch_kv4(const Kv4Args& a, cudaStream_t s) {
    using C = Kv4C<PARTS>;
    static bool configured = false;
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(kv4_kernel<PARTS>(), cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) { braid_set_error("attn_kv4: cannot reserve %d bytes of shared memory: %s", C::SMEM, cudaGetErrorString(e)); return (int)e; }
        configured = true;
    }
    const int g = a.nqh / a.nkh, hpc = g < C::BM ? g : C::BM, tpc = C::BM / hpc, hchunks = (g + hpc - 1) / hpc;
    const long long gz = (long long)((a.max_q_len + tpc - 1) / tpc) * a.n_splits;
    const long long parts = a.cluster ? 1 : (gz + 65534) / 65535;
    if (gz > (a.cluster ? 65535 : 0x7fffffffLL - 65535) || (long long)a.nkh * hchunks * parts > 0x7fffffffLL || a.n_seqs > 65535)
        BRAID_REFUSE("attn_kv4: the step exceeds the grid limits (%lld tiles, %d heads, %d sequences)", gz, a.nkh * hchunks, a.n_seqs);
    if (gz == 0) return BRAID_OK;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.nkh * hchunks * parts), a.n_seqs, (unsigned)((gz + parts - 1) / parts));
    cfg.blockDim = dim3(KV4_NW * 32);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = braid_pdl_enabled();
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = a.n_splits;
    cfg.attrs = attr;
    cfg.numAttrs = a.cluster ? 2 : 1;
    cudaLaunchKernelEx(&cfg, attn_kv4_kernel<PARTS, KV4_NW, kv4_sr(PARTS), kv4_st(PARTS)>, a);
    BRAID_LAUNCH_CHECK();
}

extern "C" int braid_attn_kv4_head_dim(void) { return BRAID_HD; }
extern "C" int braid_attn_kv4_last_parity(int uses, int stage, int stages) { return (int)kv4_last_parity(uses, stage, stages); }
extern "C" int braid_attn_kv4_args_bytes(void) { return (int)sizeof(Kv4Args); }

// CTAs that the device holds at once.
extern "C" int braid_attn_kv4_slots(int f32) {
    int dev = 0, sms = 0, per_sm = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const void* f = f32 ? kv4_kernel<3>() : kv4_kernel<1>();
    const int bytes = f32 ? Kv4C<3>::SMEM : Kv4C<1>::SMEM;
    cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, f, KV4_NW * 32, bytes);
    if (e != cudaSuccess || per_sm <= 0 || sms <= 0) return 148 * 2;
    return per_sm * sms;
}

// Clusters of `size` CTAs that the device holds at once (0: none).
extern "C" int braid_attn_kv4_clusters(int f32, int size) {
    const void* f = f32 ? kv4_kernel<3>() : kv4_kernel<1>();
    const int bytes = f32 ? Kv4C<3>::SMEM : Kv4C<1>::SMEM;
    cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1, 1, size);
    cfg.blockDim = dim3(KV4_NW * 32);
    cfg.dynamicSmemBytes = bytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = size;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, f, &cfg) != cudaSuccess) { cudaGetLastError(); return 0; }
    return n;
}

// The slices' shares made one: also those of attn_kv4_prompt_kernel (attn_kv4_tc.cu).
extern "C" int braid_attn_kv4_merge(const Kv4Args* args, void* stream) {
    Kv4Args a = *args;
    a.partial_rows = a.q_to > 0 ? a.n_seqs * a.q_to : a.rows;
    const long long ctas = (long long)a.partial_rows * a.nqh;
    if (ctas <= 0 || a.n_splits < 1) return BRAID_OK;
    if (ctas > 0x7fffffffLL) BRAID_REFUSE("attn_kv4: the rows exceed the grid limit");
    if (!a.partial) BRAID_REFUSE("attn_kv4: slices that are no cluster need the partial buffer");
    if (a.head_sinks) a.has_sink = 1;
    const bool few = a.n_splits <= 8;
    const dim3 grid((unsigned)(few ? (ctas + 7) / 8 : ctas));
    if (a.f32) braid_launch(few ? attn_kv4_merge_few_kernel<float> : attn_kv4_merge_kernel<float>, grid, dim3(256), 0, (cudaStream_t)stream, a);
    else braid_launch(few ? attn_kv4_merge_few_kernel<__nv_bfloat16> : attn_kv4_merge_kernel<__nv_bfloat16>, grid, dim3(256), 0, (cudaStream_t)stream, a);
    BRAID_LAUNCH_CHECK();
}

// `args`: a Kv4Args, filled in by the caller (csrc/api.py has its layout).
extern "C" int braid_attn_kv4(const Kv4Args* args, void* stream) {
    Kv4Args a = *args;
    if (a.rows <= 0 || a.n_seqs <= 0) return BRAID_OK;
    if (a.head_sinks) a.has_sink = 1;
    if (a.window <= 0) a.window = a.keep_first = 0;
    if (!a.error_flag) BRAID_REFUSE("attn_kv4: error_flag is required");
    if (a.num_pages <= 0 || a.cols <= 0) BRAID_REFUSE("attn_kv4: the cache has no pages (pages=%d, table columns=%d)", a.num_pages, a.cols);
    if (a.nqh <= 0 || a.nkh <= 0 || a.nqh % a.nkh) BRAID_REFUSE("attn_kv4: %d query heads do not divide into %d kv heads", a.nqh, a.nkh);
    if ((uintptr_t)a.cache & 15) BRAID_REFUSE("attn_kv4: the cache must start on 16 bytes");
    if (a.keep_first < 0 || a.max_q_len < 0) BRAID_REFUSE("attn_kv4: keep_first=%d, max_q_len=%d must not be negative", a.keep_first, a.max_q_len);
    if (!a.bias_slope != !a.bias_rate) BRAID_REFUSE("attn_kv4: a distance bias has a slope and a rate a head");
    if (a.softcap > 0.f && a.bias_slope) BRAID_REFUSE("attn_kv4: a cap on the scores and a distance bias are not combined");
    if (a.q_to > 0 && (a.q_to < a.max_q_len || (long long)a.n_seqs * a.q_to > 0x7fffffffLL))
        BRAID_REFUSE("attn_kv4: sequences of up to %d tokens do not go with a longest one of %d, or are too many", a.q_to, a.max_q_len);
    a.partial_rows = a.q_to > 0 ? a.n_seqs * a.q_to : a.rows;
    if (a.n_splits < 1) a.n_splits = 1;
    if (a.n_splits <= 1 || a.n_splits > 8) a.cluster = 0;
    if (a.n_splits > 1 && !a.cluster && !a.partial) BRAID_REFUSE("attn_kv4: slices that are no cluster need the partial buffer");
    cudaStream_t s = (cudaStream_t)stream;
    const int rc = a.f32 ? launch_kv4<3>(a, s) : launch_kv4<1>(a, s);
    return rc || a.n_splits == 1 || a.cluster ? rc : braid_attn_kv4_merge(&a, stream);
}
