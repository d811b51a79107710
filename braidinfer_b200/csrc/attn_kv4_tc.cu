// Attention of prompts over a cache held in 4 bits, on the 5th-generation tensor cores (tcgen05): over the pages that kv4_expand_kernel
// (kv4.cu) has read back as float16 numbers, block c of sequence i as page i * cols + c.  Compiled for one head size:
// -DBRAID_HD=<32, 64, ... 256>.  The sizes computed with are 64, 128 and 256; a head's further numbers are zero (in the pages, and behind the
// queries' map).
//
// A CTA takes two groups of 128 columns of queries (tokens x the query heads of a kv head) and walks the keys that they see, 128 at a time:
//   S = Q K^T  (tensor memory, float32),   p = 2^(scale log2(e) S - m),   O += p V  (p in tensor memory)
// with the running maximum m of a row raised only when a tile exceeds it by more than 8 powers of two.  Warp 0 brings pages into two rings by
// TMA, warp 1 issues S, warp 3 P V, and 16 warps are the softmax: TWO threads share a row, each with half of a tile's keys (a page) and half of
// the result's columns, in two warps that meet at a barrier of their own once a tile.  That barrier carries the question whether any row's
// maximum has to be raised (barrier.red.or), so that the two exchange numbers only then.
//
// Heads above 128: a result of 128 rows fills as much tensor memory as two of the others.  There the two groups are the same 128 rows, each with half
// of the result's columns; both compute all scores and probabilities.  (The products of a tile are then 3,072 cycles, 1,024 of them twice.)
//
// All operands are float16 numbers: their 11 bits hold what the codes say, where bfloat16's 8 made errors of 0.0031 to 0.0035 of the result
// instead of 0.0017, which is the rounding of the result.  For their range, kv4_expand_kernel scales the keys and the values of a page and kv head
// by a power of two each, and a row's queries are scaled here; the scores' factor and the probabilities' exponent take that back.  The
// values of a sequence share one exponent in O, so a page whose values are far smaller than the largest (2^16 times) marks its sequence
// for the plain kernel, which computes it again.
//
// What bounds it: the exponentials of a tile take the SM 2,048 cycles, and so do its products.  So the two groups have ONE place for their
// scores: S of one is computed while the other's exponentials run, which keeps the groups half a turn apart without a barrier between them.
// A tile takes some 3,000 cycles, and a CTA some 14,000 beside its tiles (its start, the queries' way and conversion, the first tile's chain, the
// result).  Prompts of 1,800, 1,346 and 689 tokens / 700 tokens behind 16,500 (88 of 148 SMs), 32 heads of 128 over 8, us with
// the reading back, in bfloat16: 83 / 344 by attn_tc.cu (a thread a row, tiles of 64 keys, two CTAs an SM); 89 / 331 the same with two threads a
// row; 90 / 332 with both groups in a CTA and scores of their own (96 / 376 with barriers that let their exponentials take turns); 104 / 393 with
// tiles of 128 keys whose probabilities lie over the scores, where all of a group's steps wait for one another; 78 / 237 so, and 78 / 224 with
// the context in 3 slices.  In float16 86 / 231 (more registers for the softmax by setmaxnreg, 112 and 32: 3 and 13 % slower), 80 / 226
// with queries asked for before tensor memory is taken and the result written 32 bytes a thread.
#include "kv4.cuh"
#include "attn_tc.cuh"
#include "softcap.cuh"
#include <cuda_fp16.h>
#include <float.h>

#ifndef BRAID_HD
#error "compile with -DBRAID_HD=<head_dim>"
#endif


#define FA_BM 128
#define FA_BN 128                                // keys per tile: two pages
#define FA_PAGE BRAID_PAGE_SIZE
static_assert(FA_PAGE == 64, "a key tile of this kernel is two pages of 64 positions");
#define FA_SOFTMAX 4                             // warps before: TMA, S, one that only waits for the end, P V
#define FA_THREADS ((FA_SOFTMAX + 16) * 32)      // two groups of 8 softmax warps
#define FA_WIDE (BRAID_HD > 128)                 // the groups are the same rows
#define FA_HD (BRAID_HD <= 64 ? 64 : BRAID_HD <= 128 ? 128 : 256)              // the head size computed with
#define FA_OD (FA_WIDE ? 128 : FA_HD)            // result columns of a group
#define FA_QTILES (FA_WIDE ? 1 : 2)              // tiles of 128 rows a CTA
#define FA_HB (FA_HD / 64)                       // 64-element blocks of it
#define FA_QBLOCK_BYTES (128 * 128)              // [128 rows][64 elements] of 16 bits, 128-byte rows
#define FA_PBLOCK_BYTES (64 * 128)               // [64 positions][64 elements]: what a copy brings
#define FA_KBLOCK_BYTES (2 * FA_PBLOCK_BYTES)    // two pages on end
#define FA_Q_BYTES (FA_HB * FA_QBLOCK_BYTES)
#define FA_KV_BYTES (FA_HB * FA_KBLOCK_BYTES)    // one K or one V tile
#define FA_KST (FA_WIDE ? 1 : 2)                                 // stages of the key ring
#define FA_VST (FA_WIDE ? 1 : 2)                                 // stages of the value ring
#define FA_BAR_BYTES 256
#define FA_SMEM (FA_QTILES * FA_Q_BYTES + (FA_KST + FA_VST) * FA_KV_BYTES + FA_BAR_BYTES)
// tensor memory: O of the first 128 rows [0, 128), of the others [128, 256); the scores of both in turn [256, 384); P of either [384, 448), [448, 512)
#define FA_TMEM_COLS 512
#define FA_TMEM_S 256
#define FA_TMEM_P 384

// The two warps of a pair (64 threads): whether any of them says yes, and a plain meeting.  These barriers leave a warp's lanes free to part,
// and the accesses to tensor memory behind them want them together: hence the __syncwarp.
__device__ __forceinline__ bool pair_any(int id, bool yes) {
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(any) : "r"((uint32_t)yes), "r"(id) : "memory");
    __syncwarp();
    return any != 0;
}
__device__ __forceinline__ void pair_sync(int id) {
    asm volatile("barrier.cta.sync %0, 64;" ::"r"(id) : "memory");
    __syncwarp();
}
// 16 consecutive columns of this thread's lane written (no wait).
__device__ __forceinline__ void tmem_st16_nowait(uint32_t taddr, const uint32_t* w) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 :: "r"(taddr), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]), "r"(w[8]),
                    "r"(w[9]), "r"(w[10]), "r"(w[11]), "r"(w[12]), "r"(w[13]), "r"(w[14]), "r"(w[15])
                 : "memory");
}

// Two numbers at a time.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
        "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tadd.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
// 32 bytes on end, on 32: a whole sector of the cache, where 16 a thread are halves of two.
__device__ __forceinline__ void store32(void* p, const uint32_t* w) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
                 "r"(w[6]), "r"(w[7]) : "memory");
}
// An instruction descriptor with float16 operands instead of bfloat16 ones (bits 7 .. 9 of A, 10 .. 12 of B).
__host__ __device__ constexpr uint32_t fa_idesc_f16(uint32_t idesc) { return idesc & ~((7u << 7) | (7u << 10)); }

struct Kv4PromptArgs {
    const void* q;
    const void* pages;           // block c of sequence i: page i * cols + c, [2][nkh][64][FA_HD] float16, scaled
    __nv_bfloat16* out;
    const int* q_start;
    const int* q_len;
    const int* kv_before;
    int* error_flag;
    const float* head_sinks;     // [nqh] float32 natural-log scores: a sink a head (learned) instead of the one score; or null
    const __nv_bfloat16* head_gate;  // [rows, gate_stride]: head h's result is multiplied by sigmoid(head_gate[row, h]); or null
    const float* bias_slope;     // BIAS: [nqh] float32 r1 and r2 of the distance bias r1 ln(1 + r2 (p - j))
    const float* bias_rate;
    const int* scales;           // [pages, nkh, 2] exponents of the pages' keys and values, [n_seqs, nkh] of a sequence's largest values (kv4.cu)
    const int* top;
    int* repair;                 // [0] and [1 + seq0 + sequence] become 1 where pages' values differ too much
    long long q_stride, out_stride, gate_stride;
    float* partial;              // n_splits > 1: what attn_kv4_merge_kernel (attn_kv4.cu) reads
    int rows, n_seqs, max_q_len, nqh, nkh, cols, window, has_sink;
    float scale, sink, out_scale, softcap;
    // filled in here: in units of log2(e); CAP: scale / cap, the tanh's argument
    float scale_log2, sink_log2, cap_log2;
    int n_splits;
    int q_from;                  // only sequences that bring at least so many tokens
    int tiles;                   // > 0: the grid has so many token tiles of whatever sequences, in order; 0: as many for every sequence
    int seq0;
};

#define FA_PLAIN 0
#define FA_BIAS 1
#define FA_CAP 2
template <int FORM>
__global__ void __launch_bounds__(FA_THREADS, 1)
attn_kv4_prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kv, const Kv4PromptArgs a) {
    constexpr int HD = FA_HD;
    constexpr bool BIAS = FORM == FA_BIAS, CAP = FORM == FA_CAP;
    pdl_trigger();
    // the swizzled tiles want 1024-byte alignment; the start of dynamic shared memory is checked instead of rounded up
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {
        if (threadIdx.x == 0) atomicExch(a.error_flag, 1);
        return;
    }
    uint8_t* sQ = smem;
    uint8_t* sK = sQ + FA_QTILES * FA_Q_BYTES;     // [FA_KST]
    uint8_t* sV = sK + FA_KST * FA_KV_BYTES;       // [FA_VST]
    uint64_t* bars = (uint64_t*)(sV + FA_VST * FA_KV_BYTES);
    uint64_t* q_full = bars;                       // [1]
    uint64_t* q_ready = q_full + 1;                // [2] the queries of either group are float16
    uint64_t* k_full = q_ready + 2;                // [FA_KST]
    uint64_t* k_empty = k_full + FA_KST;           // [FA_KST]
    uint64_t* v_full = k_empty + FA_KST;           // [FA_VST]
    uint64_t* v_empty = v_full + FA_VST;           // [FA_VST]
    uint64_t* s_full = v_empty + FA_VST;           // [2] of the first, of the second group; the others alike
    uint64_t* s_free = s_full + 2;                 // [2] the scores are in registers
    uint64_t* p_ready = s_free + 2;                // [2]
    uint64_t* pv_done = p_ready + 2;               // [2]
    uint32_t* tmem_slot = (uint32_t*)(pv_done + 2);
    static_assert((3 + 2 * FA_KST + 2 * FA_VST + 8) * 8 + 8 <= FA_BAR_BYTES, "the barriers outgrow their bytes");
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    __shared__ float share[2][2][2][FA_BM];        // what the two threads of a row tell one another: [group][turn][half][row]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = a.nqh / a.nkh;
    const int hpc = g < FA_BM ? g : FA_BM;
    const int tpc = FA_BM / hpc;
    const int hchunks = (g + hpc - 1) / hpc;
    // CTAs start in the order x, y, z: all kv heads and sequences of the last token tile first, then
    // the tile before, ...: late tokens see the most keys, so the longest CTAs start first and the
    // short ones fill the gaps at the end
    // (more than 65,535 tiles are in parts along x)
    const int heads = a.nkh * hchunks, part = blockIdx.x / heads, hx = blockIdx.x - part * heads;
    const int kvh = hx / hchunks, hchunk = hx - kvh * hchunks;
    const int unit = (int)(gridDim.x / heads - part) * (int)gridDim.z - 1 - (int)blockIdx.z, split = unit % a.n_splits;
    int seq = blockIdx.y, tile = unit / a.n_splits;
    if (threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_kv) : "memory");
    }
    pdl_wait();
    if (a.tiles > 0) {
        // the grid's tile number `tile`: whose it is, and which of its tiles
        __shared__ int found[2];
        int before = 0;                           // tiles of the sequences before this round's
        if (threadIdx.x == 0) found[0] = -1;
        for (int s0 = 0; s0 < a.n_seqs && before <= tile; s0 += FA_THREADS) {
            const int s = s0 + threadIdx.x, n = s < a.n_seqs ? max(a.q_len[s], 0) : 0;
            const int mine = n >= a.q_from ? (n + FA_QTILES * tpc - 1) / (FA_QTILES * tpc) : 0;
            int upto = mine;                      // tiles of this warp's sequences up to this one
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            __shared__ int sums[FA_THREADS / 32];
            __syncthreads();
            if (lane == 31) sums[warp] = upto;
            __syncthreads();
            int all = 0, base = before;
            for (int w = 0; w < FA_THREADS / 32; ++w) {
                if (w < warp) base += sums[w];
                all += sums[w];
            }
            if (mine > 0 && tile >= base + upto - mine && tile < base + upto) {
                found[0] = s;
                found[1] = tile - (base + upto - mine);
            }
            before += all;
        }
        __syncthreads();
        seq = found[0];
        tile = found[1];
        if (seq < 0) return;
    }
    const int q_len = a.q_len[seq], q_start = a.q_start[seq], kv_before = a.kv_before[seq];
    const int tok0 = tile * (FA_QTILES * tpc);
    if (tok0 >= q_len || q_len < a.q_from) return;             // uniform over the CTA

    const int ng = FA_WIDE || q_len - tok0 > tpc ? 2 : 1;    // groups that hold tokens
    const int pos_min = kv_before + tok0, pos_max = kv_before + min(tok0 + FA_QTILES * tpc, q_len) - 1;
    const int k_lo = (a.window > 0 && pos_min - a.window + 1 > 0) ? pos_min - a.window + 1 : 0;
    int page_lo = k_lo / FA_PAGE, page_hi = pos_max / FA_PAGE + 1;
    if (a.n_splits > 1) {                         // slices of whole tiles
        const int per = ((page_hi - page_lo + 1) / 2 + a.n_splits - 1) / a.n_splits * 2;
        page_lo = min(page_hi, page_lo + split * per);
        page_hi = min(page_hi, page_lo + per);
    }
    const int n_tiles = (page_hi - page_lo + 1) / 2;
    const int head0 = kvh * g + hchunk * hpc;
    const int n_heads = min(hpc, g - hchunk * hpc);

    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        for (int s = 0; s < FA_KST; ++s) { mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 1); }
        for (int s = 0; s < FA_VST; ++s) { mbar_init(&v_full[s], 1); mbar_init(&v_empty[s], 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(&q_ready[s], 8); mbar_init(&s_full[s], 1); mbar_init(&s_free[s], 8); mbar_init(&p_ready[s], 8); mbar_init(&pv_done[s], 1); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        if (n_tiles > 0) {                        // (the queries are on their way while tensor memory is taken)
            mbar_expect_tx(q_full, (uint32_t)((FA_WIDE ? 1 : ng) * hpc * tpc * 128 * FA_HB));      // the box is hpc x tpc rows of 128 bytes
            for (int gr = 0; gr < (FA_WIDE ? 1 : ng); ++gr)
#pragma unroll
                for (int hb = 0; hb < FA_HB; ++hb)
                    tma_load_3d(&map_q, q_full, sQ + gr * FA_Q_BYTES + hb * FA_QBLOCK_BYTES, hb * 64, head0, q_start + tok0 + gr * tpc);
        }
    }
    if (warp == 1) tmem_alloc(tmem_slot, FA_TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    if (warp == 0) {
        if (lane == 0 && n_tiles > 0) {
            // key and value tiles go out independently, each as soon as its stage is free
            int jk = 0, jv = 0;
            uint32_t idle = 0;
            uint64_t idle_since = 0;
            while (jk < n_tiles || jv < n_tiles) {
                bool moved = false;
                const bool k_turn = jk < n_tiles && mbar_try_wait(&k_empty[jk % FA_KST], (uint32_t)((jk / FA_KST) & 1) ^ 1u);
                const bool v_turn = !k_turn && jv < n_tiles && mbar_try_wait(&v_empty[jv % FA_VST], (uint32_t)((jv / FA_VST) & 1) ^ 1u);
                if (k_turn || v_turn) {
                    const int j = k_turn ? jk : jv;
                    const int st = k_turn ? jk % FA_KST : jv % FA_VST;
                    uint64_t* bar = k_turn ? &k_full[st] : &v_full[st];
                    uint8_t* dst = (k_turn ? sK : sV) + st * FA_KV_BYTES;
                    mbar_expect_tx(bar, FA_KV_BYTES);
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        // behind an odd number of pages the last one again: masked, and multiplied by 0
                        int c = min(page_lo + 2 * j + b, page_hi - 1);
                        if (c >= a.cols) {                          // more keys than the caller said
                            atomicExch(a.error_flag, 1);
                            c = 0;
                        }
                        const int row = (((seq * a.cols + c) * 2 + (k_turn ? 0 : 1)) * a.nkh + kvh) * FA_PAGE;
#pragma unroll
                        for (int hb = 0; hb < FA_HB; ++hb)
                            tma_load_2d(&map_kv, bar, dst + hb * FA_KBLOCK_BYTES + b * FA_PBLOCK_BYTES, hb * 64, row);
                    }
                    if (k_turn) ++jk; else ++jv;
                    moved = true;
                }
                if (moved) { idle = 0; idle_since = 0; continue; }
                if (++idle >= TC_SPIN_LIMIT) { *abort_flag = 1; break; }
                if ((idle & 1023u) == 1023u) {              // the same bound as mbar_wait: time on the device's clock
                    if (*abort_flag) break;
                    const uint64_t now = global_timer_ns();
                    if (idle_since == 0) idle_since = now;
                    else if (now - idle_since > TC_WAIT_LIMIT_NS) { *abort_flag = 1; break; }
                }
            }
        }
    } else if (warp == 1) {
        // S of either group in turn, in one place: the next goes there when the one before is in registers
        if (lane == 0 && n_tiles > 0) {
            constexpr uint32_t idesc_qk = fa_idesc_f16(umma_idesc_bf16(FA_BM, FA_BN));
            // operand descriptors differ only in their start address (bits 0..13 of the low word, in 16-byte units)
            const uint64_t dq = umma_desc_sw128(smem_u32(sQ)), dk = umma_desc_sw128(smem_u32(sK));
            const uint32_t q_lo = (uint32_t)dq, k_lo = (uint32_t)dk, kq_hi = (uint32_t)(dq >> 32), ts = tmem_base + FA_TMEM_S;
            bool ok = mbar_wait(&q_ready[0], 0, abort_flag) && (ng == 1 || mbar_wait(&q_ready[1], 0, abort_flag));
            for (int j = 0; j < n_tiles && ok; ++j) {
                const int kst = j % FA_KST;
                ok = mbar_wait(&k_full[kst], (uint32_t)((j / FA_KST) & 1), abort_flag);
#pragma unroll
                for (int group = 0; group < 2; ++group) {
                    if (group >= ng || !ok) break;
                    // the one before: the first group's of this tile, or the last group's of the tile before
                    if (group) ok = mbar_wait(&s_free[0], (uint32_t)(j & 1), abort_flag);
                    else if (j > 0) ok = mbar_wait(&s_free[ng - 1], (uint32_t)((j - 1) & 1), abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t qs_lo = q_lo + (uint32_t)((FA_WIDE ? 0 : group * FA_Q_BYTES) >> 4), ks_lo = k_lo + (uint32_t)((kst * FA_KV_BYTES) >> 4);
#pragma unroll
                    for (int ks = 0; ks < BRAID_HD / 16; ++ks) {
                        const uint32_t qoff = ((ks >> 2) * FA_QBLOCK_BYTES + (ks & 3) * 32) >> 4, koff = ((ks >> 2) * FA_KBLOCK_BYTES + (ks & 3) * 32) >> 4;
                        umma_ss_lohi(ts, qs_lo + qoff, kq_hi, ks_lo + koff, kq_hi, idesc_qk, ks > 0 ? 1u : 0u);
                    }
                    umma_commit(&s_full[group]);
                }
                if (ok) umma_commit(&k_empty[kst]);
            }
        }
    } else if (warp == 3) {
        if (lane == 0 && n_tiles > 0) {
            constexpr uint32_t idesc_pv = fa_idesc_f16(umma_idesc_bf16_b_mn(FA_BM, FA_OD));
            const uint64_t dv = umma_desc_sw128_mn(smem_u32(sV), FA_KBLOCK_BYTES);
            const uint32_t v_lo = (uint32_t)dv, v_hi = (uint32_t)(dv >> 32);
            bool ok = true;
            for (int j = 0; j < n_tiles && ok; ++j) {
                const int vst = j % FA_VST;
                const uint32_t vs_lo = v_lo + (uint32_t)((vst * FA_KV_BYTES) >> 4);
                ok = mbar_wait(&v_full[vst], (uint32_t)((j / FA_VST) & 1), abort_flag);
                for (int group = 0; group < ng && ok; ++group) {
                    ok = mbar_wait(&p_ready[group], (uint32_t)(j & 1), abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t vg_lo = vs_lo + (uint32_t)((FA_WIDE ? group * 2 * FA_KBLOCK_BYTES : 0) >> 4);
                    const uint32_t to = tmem_base + group * 128, tp = tmem_base + FA_TMEM_P + group * 64;
#pragma unroll
                    for (int ks = 0; ks < FA_BN / 16; ++ks)
                        umma_ts_lohi(to, tp + ks * 8, vg_lo + (uint32_t)((ks * 16 * 128) >> 4), v_hi, idesc_pv, (ks > 0 || j > 0) ? 1u : 0u);
                    umma_commit(&pv_done[group]);
                }
                if (ok) umma_commit(&v_empty[vst]);
            }
        }
    } else if (warp >= FA_SOFTMAX && (warp - FA_SOFTMAX) >> 3 < ng) {
        const int group = (warp - FA_SOFTMAX) >> 3;            // the first or the second 128 rows, or 128 columns of the result
        const int tokg = tok0 + (FA_WIDE ? 0 : group * tpc), n_tok = min(tpc, q_len - tokg);
        const int first = kv_before + tokg, last = first + n_tok - 1;             // the group's positions
        const int quarter = warp & 3;                          // tensor-memory lanes 32 * quarter ...
        const int half = ((warp - FA_SOFTMAX) >> 2) & 1;                // this thread's half of a tile's keys
        const int pair = 1 + group * 4 + quarter;              // the barrier of the two warps that share their rows
        const int r = quarter * 32 + lane;                     // this thread's row
        const int tl = r / hpc, hl = r - tl * hpc;
        const bool valid = tl < n_tok && hl < n_heads;
        const int pos = valid ? first + tl : -1;
        const int lo = (a.window > 0) ? pos - a.window + 1 : 0;
        const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
        const uint32_t tmem_o = tmem_base + group * 128;
        float m = -INFINITY, l = 0.f;
        float r1 = 0.f, r2 = 0.f;                             // the row's distance bias
        if (BIAS && valid) { r1 = a.bias_slope[head0 + hl]; r2 = a.bias_rate[head0 + hl]; }
        bool ok = true;
        // The queries become float16 numbers, a row's largest one of 2^8 .. 2^9: each of a row's threads takes a half of the 128 bytes or
        // of the 128-byte blocks (in any order within: the tile's swizzle moves 16 bytes within them).
        float row_factor = a.scale_log2;                      // of the scores: 2^(the row's exponent) in it, and below 2^(the page's)
        if (n_tiles > 0) {
            constexpr int CHUNKS = FA_OD / 16;                // of 8 numbers
            uint8_t* src = sQ + (FA_WIDE ? 2 * group * FA_QBLOCK_BYTES : group * FA_Q_BYTES) + (HD > 64 ? half * FA_QBLOCK_BYTES : 0) + r * 128;
            const int chunk0 = HD > 64 ? 0 : half * CHUNKS;
            const bool came = mbar_wait(q_full, 0, abort_flag);
            ok = __all_sync(0xffffffffu, came) && ok;
            uint4 x[CHUNKS];
            uint32_t top2 = 0u;                                // the largest of even and of odd numbers (a NaN is none)
#pragma unroll
            for (int i = 0; i < CHUNKS; ++i) {
                x[i] = *reinterpret_cast<const uint4*>(src + (chunk0 + ((i + lane) & (CHUNKS - 1))) * 16);
                const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t size = w[e] & 0x7fff7fffu;
                    const __nv_bfloat162 t = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&top2), *reinterpret_cast<const __nv_bfloat162*>(&size));
                    top2 = *reinterpret_cast<const uint32_t*>(&t);
                }
            }
            float most = fmaxf(__uint_as_float(top2 << 16), __uint_as_float(top2 & 0xffff0000u));
            share[group][1][half][r] = most;
            if (FA_WIDE) {                                     // four threads have a row's numbers
                asm volatile("barrier.cta.sync %0, 128;" ::"r"(9 + quarter) : "memory");
                __syncwarp();
                most = fmaxf(most, fmaxf(share[1 - group][1][half][r], share[1 - group][1][1 - half][r]));
            } else {
                pair_sync(pair);
            }
            most = fmaxf(most, share[group][1][1 - half][r]);
            const int qe = most > 0.f ? min(max(kv4_exponent(most) - 8, -126), 119) : 0;
            row_factor *= kv4_pow2(qe);
            const float f = kv4_pow2(-qe);
#pragma unroll
            for (int i = 0; i < CHUNKS; ++i) {
                uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const __half2 y = __floats2half2_rn(__uint_as_float(w[e] << 16) * f, __uint_as_float(w[e] & 0xffff0000u) * f);
                    w[e] = *reinterpret_cast<const uint32_t*>(&y);
                }
                *reinterpret_cast<uint4*>(src + (chunk0 + ((i + lane) & (CHUNKS - 1))) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_ready[group]);
        }
        const int top = a.top[(size_t)seq * a.nkh + kvh];     // the exponent that all of the result has
        bool apart = false;
        auto exps_of = [&](int j) {                           // this thread's half of a tile's keys is a page
            const int page = min(min(page_lo + 2 * j + half, page_hi - 1), a.cols - 1);
            return *reinterpret_cast<const int2*>(a.scales + (((size_t)seq * a.cols + page) * a.nkh + kvh) * 2);
        };
        int2 next_exps = make_int2(0, 0);
        if (n_tiles > 0) next_exps = exps_of(0);
        for (int j = 0; j < n_tiles; ++j) {
            const int2 exps = next_exps;
            if (j + 1 < n_tiles) next_exps = exps_of(j + 1);  // (a trip to L2, a tile ahead)
            // (a warp whose wait ran out goes on to meet its partner at every barrier below, so that neither waits for the other for good)
            const bool came = mbar_wait(&s_full[group], (uint32_t)(j & 1), abort_flag);
            ok = __all_sync(0xffffffffu, came) && ok;
            tc_fence_after();
            float sv[64];
            tmem_ld32x2(tmem_base + FA_TMEM_S + half * 64 + lane_addr, sv);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_free[group]);           // (one arrival a warp)
            // (finite, for products that are 0)
            const float factor_s = fmaxf(fminf(exps.x ? row_factor * kv4_pow2(exps.x - KV4_EXPONENT) : row_factor, FLT_MAX), -FLT_MAX);
            // with the bias or the cap the scores are scaled there
            const float sc = BIAS || CAP ? 1.f : factor_s;
            // The probabilities' exponent: values are scaled by their page's own, and the result has the sequence's largest.  2^7 makes a
            // probability, up to 2^8 against a maximum that was not raised, one of up to 2^15, so that those down to 2^-21 keep 11 bits.
            const int below = exps.y ? exps.y - top : 0;
            apart |= below < -16;
            const int pe = max(below, -40) + 7;
            const int key0 = page_lo * FA_PAGE + j * FA_BN + half * 64;
            const bool all_visible = (key0 + 63 <= first) && (a.window == 0 || key0 >= last - a.window + 1);
            if (BIAS) {                                       // keys after the query (a negative distance) are masked below
                const float d0 = (float)(pos - key0);
#pragma unroll
                for (int i = 0; i < 64; ++i)
                    sv[i] = fmaf(sv[i], factor_s, -r1 * __log2f(fmaf(r2, d0 - (float)i, 1.f)));
            }
            if (CAP) softcap_scores<64>(sv, factor_s, a.cap_log2);
            if (!all_visible) {
#pragma unroll
                for (int i = 0; i < 64; ++i)
                    if (!(key0 + i <= pos && key0 + i >= lo)) sv[i] = -INFINITY;
            }
            float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
            for (int i = 0; i < 64; i += 4) {
                mx0 = fmaxf(mx0, sv[i]); mx1 = fmaxf(mx1, sv[i + 1]);
                mx2 = fmaxf(mx2, sv[i + 2]); mx3 = fmaxf(mx3, sv[i + 3]);
            }
            float mx = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * sc;     // scale > 0 commutes with the maximum
            if (!valid) mx = -INFINITY;
            // raise m only when the tile towers over it; -inf + 8 = -inf, so the first finite maximum always does
            const bool any = pair_any(pair, mx > m + FA_RAISE);
            float factor = 1.f;
            if (any) {
                share[group][j & 1][half][r] = mx;
                pair_sync(pair);
                mx = fmaxf(mx, share[group][j & 1][1 - half][r]);
                if (mx > m + FA_RAISE) {
                    factor = fast_exp2(m - mx);                // exp2(-inf) = 0: nothing was summed yet
                    m = mx;
                }
            }
            // a row that is no query (past the tile's tokens or heads) sums nothing: exp2(-inf) = 0
            const float ms = !valid ? INFINITY : ((m == -INFINITY) ? 0.f : m);
            if (j > 0) {
                // the group's product before this one has read its probabilities and is in O (waited for at every turn: a parity only tells
                // apart a barrier that is at most one phase off)
                const bool done = mbar_wait(&pv_done[group], (uint32_t)((j - 1) & 1), abort_flag);
                ok = __all_sync(0xffffffffu, done) && ok;
                tc_fence_after();
            }
            // probabilities times 2^pe, rounded to float16
            const float shift = (float)pe - ms;
            const float2 sc2 = make_float2(sc, sc), shift2 = make_float2(shift, shift);
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t pk[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 t = fma2(make_float2(sv[c * 32 + 2 * i], sv[c * 32 + 2 * i + 1]), sc2, shift2);
                    const float p0 = fast_exp2(t.x), p1 = fast_exp2(t.y);
                    sum = add2(sum, make_float2(p0, p1));
                    const __half2 b = __floats2half2_rn(p0, p1);
                    pk[i] = *reinterpret_cast<const uint32_t*>(&b);
                }
                __syncwarp();
                tmem_st16_nowait(tmem_base + FA_TMEM_P + group * 64 + half * 32 + c * 16 + lane_addr, pk);
            }
            l = fmaf(sum.x + sum.y, kv4_pow2(-pe), l * factor);
            __syncwarp();
            if (any && j > 0) {                                // (the same for every lane)
                // a half of the row's columns
#pragma unroll
                for (int h = 0; h < FA_OD / 64; ++h) {
                    float ov[32];
                    tmem_ld32(tmem_o + half * (FA_OD / 2) + h * 32 + lane_addr, ov);
#pragma unroll
                    for (int i = 0; i < 32; ++i) ov[i] *= factor;
                    __syncwarp();
                    tmem_st32_nowait(tmem_o + half * (FA_OD / 2) + h * 32 + lane_addr, reinterpret_cast<const uint32_t*>(ov));
                }
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[group]);
        }
        if (n_tiles > 0) {
            pair_sync(pair);                                   // the last exchange has been read
            share[group][0][half][r] = l;
            pair_sync(pair);
            l += share[group][0][1 - half][r];
            const bool done = mbar_wait(&pv_done[group], (uint32_t)((n_tiles - 1) & 1), abort_flag);
            ok = __all_sync(0xffffffffu, done) && ok;
            tc_fence_after();
        }
        if (apart) {
            a.repair[1 + a.seq0 + seq] = 1;
            a.repair[0] = 1;
        }
        const float o_factor = top ? kv4_pow2(top - KV4_EXPONENT - 7) : 1.f;
        const size_t row = (size_t)(q_start + tokg + tl);
        const int head = head0 + hl;
        float inv = o_factor;
        if (a.n_splits == 1 && valid) {
            // the sink joins the sum where the row is finished: l counts in units of 2^m; a sink far above every
            // score makes the sum infinite and the row zero, which is the limit
            const float sk = a.head_sinks ? a.head_sinks[head] * 1.4426950408889634f : a.sink_log2;
            inv *= a.out_scale / (a.has_sink ? l + exp2f(sk - m) : l);
            if (a.head_gate) inv *= 1.f / (1.f + __expf(-__bfloat162float(a.head_gate[row * a.gate_stride + head])));
        }
        const bool wide = !(((uintptr_t)a.out | (uintptr_t)a.out_stride * 2) & 31);       // rows of the result start on 32 bytes
        const size_t at = (row * a.nqh + head) * a.n_splits + split;
        if (a.n_splits > 1 && valid && half == 0 && !(FA_WIDE && group))
            *reinterpret_cast<float2*>(a.partial + (size_t)a.rows * a.nqh * a.n_splits * BRAID_HD + at * 2) = make_float2(m, l);
#pragma unroll
        for (int h = 0; h < FA_OD / 64; ++h) {                 // a half of the row's columns
            const int ct = half * (FA_OD / 2) + h * 32, c0 = ct + (FA_WIDE ? group * 128 : 0);
            if (c0 >= BRAID_HD) break;
            float ov[32];
            __syncwarp();
            if (n_tiles > 0) {
                tmem_ld32(tmem_o + ct + lane_addr, ov);
            } else {                                           // a slice without a key
#pragma unroll
                for (int i = 0; i < 32; ++i) ov[i] = 0.f;
            }
            if (ok && valid && a.n_splits > 1) {
                float* dst = a.partial + at * BRAID_HD + c0;
#pragma unroll
                for (int c = 0; c < 32; c += 8) {
                    uint32_t w[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(ov[c + i] * inv);
                    store32(dst + c, w);
                }
            } else if (ok && valid) {
                __nv_bfloat16* dst = a.out + row * a.out_stride + (size_t)head * BRAID_HD + c0;
#pragma unroll
                for (int c = 0; c < 32; c += 16) {
                    uint32_t w[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        __nv_bfloat162 b = __floats2bfloat162_rn(ov[c + 2 * i] * inv, ov[c + 2 * i + 1] * inv);
                        w[i] = *reinterpret_cast<uint32_t*>(&b);
                    }
                    if (wide) {
                        store32(dst + c, w);
                    } else {
                        *reinterpret_cast<uint4*>(dst + c) = make_uint4(w[0], w[1], w[2], w[3]);
                        *reinterpret_cast<uint4*>(dst + c + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag) atomicExch(a.error_flag, 1);
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, FA_TMEM_COLS);
    }
}

// ------------------------------------------------------------------ host side
extern "C" int braid_attn_kv4_prompt_args_bytes(void) { return (int)sizeof(Kv4PromptArgs); }

// `args`: a Kv4PromptArgs, filled in by the caller but for its last numbers (csrc/api.py has its layout).
extern "C" int braid_attn_kv4_prompt(const Kv4PromptArgs* args, void* stream) {
    Kv4PromptArgs a = *args;
    if (a.rows <= 0 || a.n_seqs <= 0 || a.max_q_len <= 0) return BRAID_OK;
    if (a.head_sinks) a.has_sink = 1;
    if (a.nqh <= 0 || a.nkh <= 0 || a.nqh % a.nkh) BRAID_REFUSE("attn_kv4: %d query heads do not divide into %d kv heads", a.nqh, a.nkh);
    if ((a.q_stride % 8) || (a.out_stride % 8) || (((uintptr_t)a.q | (uintptr_t)a.out | (uintptr_t)a.pages) & 15))
        BRAID_REFUSE("attn_kv4: prompts' queries, results and pages must be 16-byte aligned");
    if (!a.error_flag || !a.scales || !a.top || !a.repair) BRAID_REFUSE("attn_kv4: the error flag, the pages' exponents and the flags are required");
    if (!a.bias_slope != !a.bias_rate) BRAID_REFUSE("attn_kv4: a distance bias has a slope and a rate a head");
    if (a.softcap > 0.f && a.bias_slope) BRAID_REFUSE("attn_kv4: a cap on the scores and a distance bias are not combined");
    // without a bias or a cap the maximum is taken, and keys are masked, before the factor
    if (!(a.softcap > 0.f) && !a.bias_slope && !(a.scale > 0.f)) BRAID_REFUSE("attn_kv4: the factor on plain scores must be positive, not %g", (double)a.scale);
    TcEncodeTiledFn fn = tc_encode_tiled_fn();
    if (!fn) BRAID_REFUSE("attn_kv4: the driver does not export cuTensorMapEncodeTiled");
    const int g = a.nqh / a.nkh;
    const int hpc = g < FA_BM ? g : FA_BM, tpc = FA_BM / hpc, hchunks = (g + hpc - 1) / hpc;
    if (a.n_splits < 1) a.n_splits = 1;
    if (a.n_splits > 1 && (!a.partial || (uintptr_t)a.partial & 31)) BRAID_REFUSE("attn_kv4: slices need the partial buffer, on 32 bytes");
    // A CTA for every tile that a sequence may have, or, where the rows are too few for that, for every tile that the step may have: those look up
    // whose tile they are.  (A CTA that finds nothing to do still takes an SM for some us.  512 tokens beside 63 single ones, attention as a whole: 387
    // us by sequence, 282 by step; 900 beside 100 sequences of up to 50: 246, 162; 3,000, 100, 200 and 1,500: 118, 114.)
    const long long every = (a.max_q_len + FA_QTILES * tpc - 1) / (FA_QTILES * tpc);
    const long long most = a.rows / (FA_QTILES * tpc) + (a.q_from > 1 ? (a.rows / a.q_from < a.n_seqs ? a.rows / a.q_from : a.n_seqs) : a.n_seqs);
    a.tiles = 2 * most <= every * a.n_seqs ? (int)most : 0;
    const long long gx = (a.tiles ? most : every) * a.n_splits, parts = (gx + 65534) / 65535;
    if (gx > 0x7fffffffLL - 65535 || (long long)a.nkh * hchunks * parts > 0x7fffffffLL || a.n_seqs > 65535)
        BRAID_REFUSE("attn_kv4: the step exceeds the grid limits (%lld token tiles, %d sequences)", gx, a.n_seqs);
    if ((long long)a.n_seqs * a.cols * 2 * a.nkh * FA_PAGE > 0x7fffffffLL) BRAID_REFUSE("attn_kv4: the pages' rows pass 32 bits");
    CUtensorMap mq, mkv;
    {
        cuuint64_t dims[3] = {(cuuint64_t)BRAID_HD, (cuuint64_t)a.nqh, (cuuint64_t)a.rows};
        cuuint64_t strides[2] = {(cuuint64_t)BRAID_HD * 2, (cuuint64_t)a.q_stride * 2};
        cuuint32_t box[3] = {64, (cuuint32_t)hpc, (cuuint32_t)tpc};
        cuuint32_t estr[3] = {1, 1, 1};
        CUresult r = fn(&mq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(a.q), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) BRAID_REFUSE("attn_kv4: cuTensorMapEncodeTiled(q) failed with %d", (int)r);
    }
    {
        cuuint64_t dims[2] = {(cuuint64_t)FA_HD, (cuuint64_t)a.n_seqs * a.cols * 2 * a.nkh * FA_PAGE};
        cuuint64_t strides[1] = {(cuuint64_t)FA_HD * 2};
        cuuint32_t box[2] = {64, FA_PAGE};
        cuuint32_t estr[2] = {1, 1};
        CUresult r = fn(&mkv, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(a.pages), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) BRAID_REFUSE("attn_kv4: cuTensorMapEncodeTiled(pages) failed with %d", (int)r);
    }
    static bool configured = false;
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(attn_kv4_prompt_kernel<FA_PLAIN>, cudaFuncAttributeMaxDynamicSharedMemorySize, FA_SMEM);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(attn_kv4_prompt_kernel<FA_BIAS>, cudaFuncAttributeMaxDynamicSharedMemorySize, FA_SMEM);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(attn_kv4_prompt_kernel<FA_CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, FA_SMEM);
        if (e != cudaSuccess) { braid_set_error("attn_kv4: cannot reserve %d bytes of shared memory: %s", FA_SMEM, cudaGetErrorString(e)); return (int)e; }
        configured = true;
    }
    const float log2e = 1.4426950408889634f;
    a.scale_log2 = a.softcap > 0.f ? a.scale / a.softcap : a.scale * log2e;
    a.sink_log2 = a.sink * log2e;
    a.cap_log2 = a.softcap * log2e;
    braid_launch(a.softcap > 0.f ? attn_kv4_prompt_kernel<FA_CAP> : a.bias_slope ? attn_kv4_prompt_kernel<FA_BIAS> : attn_kv4_prompt_kernel<FA_PLAIN>,
                 dim3((unsigned)(a.nkh * hchunks * parts), a.tiles ? 1 : a.n_seqs, (unsigned)((gx + parts - 1) / parts)), dim3(FA_THREADS), FA_SMEM, (cudaStream_t)stream, mq, mkv, a);
    BRAID_LAUNCH_CHECK();
}
