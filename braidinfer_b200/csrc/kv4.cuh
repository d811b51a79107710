// The pages of a cache held in 4 bits.
//
// Per token and kv head, groups of 32 neighbouring numbers of the head share a step and a lowest value (both bfloat16);
// a number is lowest + step * code, code 0 .. 15.  With x the number rounded to bfloat16, lo and hi the group's lowest and
// highest: step = bfloat16((hi - lo) / 15), code = round((x - lo) / step), ties to even, kept within 0 .. 15 (0 where the
// step is 0).  A group whose range is not finite has step and lowest value NaN.
//
// Storage [page][kv head][record 0..3], a record holding 16 tokens:
//   key codes    [16][HD / 2 bytes]   32-bit word j * W + w (W = HD / 32): numbers 32 w + 8 j + 2 n + b in bits 16 b + 4 n
//   value codes  [16][HD / 2 bytes]   16-bit word i * W + w: numbers 32 w + 4 i + n in bits 4 n
//   key groups   [16][W] 32-bit words: step in the lower half, lowest value in the upper
//   value groups [16][W]
// so a record is 20 HD bytes, contiguous.  The order of the codes is that of the registers in which the tensor cores take
// them (attn_kv4.cu): lane 4 r + j of a warp reads the W neighbouring words of token r that it multiplies, and one mask and one "or"
// make two codes a pair of bfloat16 numbers.
#pragma once
#include "common.cuh"
#include "page.h"

#define KV4_GROUP 32
#define KV4_REC 16                                            // tokens a record
__host__ __device__ constexpr int kv4_record_bytes(int hd) { return 20 * hd; }
__host__ __device__ constexpr int kv4_page_bytes(int hd) { return BRAID_PAGE_SIZE / KV4_REC * kv4_record_bytes(hd); }
// offsets within a record
__host__ __device__ constexpr int kv4_value_codes(int hd) { return 8 * hd; }
__host__ __device__ constexpr int kv4_key_groups(int hd) { return 16 * hd; }
__host__ __device__ constexpr int kv4_value_groups(int hd) { return 18 * hd; }

__device__ __forceinline__ float kv4_step(uint32_t group) { return __uint_as_float(group << 16); }
__device__ __forceinline__ float kv4_lowest(uint32_t group) { return __uint_as_float(group & 0xffff0000u); }

// Powers of two of float32's normal numbers, and the exponent of a number that is 0 or one of those (0: -127).
#define KV4_EXPONENT 200                                      // added to exponents that are kept, so that 0 can say "all zero"
__device__ __forceinline__ float kv4_pow2(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ int kv4_exponent(float x) { return (int)((__float_as_uint(x) >> 23) & 255u) - 127; }
