// seq_attn.h — what the attention kernels over the caches of a batch share.
#pragma once

#include "kv_cache.h"

namespace uaii_hip {

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f2_t __attribute__((ext_vector_type(2)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef float f4u_t __attribute__((ext_vector_type(4), aligned(4)));  // rows of a caller's buffer start at any float
typedef float f16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;

// Global memory at p + off, p being the same in all lanes: the address in scalar registers.
// (Through the address space: a generic pointer's loads would count as LDS reads too, and
// each wait for LDS would wait for them.)
#define UAII_GLOBAL __attribute__((address_space(1)))
typedef const UAII_GLOBAL uint8_t* gptr_t;
__device__ inline gptr_t uniform_at(const uint8_t* p, int64_t off) {
  const uint64_t x = (uint64_t)p + (uint64_t)off;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
  return reinterpret_cast<gptr_t>((uint64_t)hi << 32 | lo);
}
template <typename T>
__device__ inline T load_at(gptr_t p, uint32_t off) {
  return *reinterpret_cast<const UAII_GLOBAL T*>(p + off);
}

__device__ inline float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127

// Power of two that brings the largest magnitude `top` of a row into [2^14, 2^15), as an
// exponent: an f16 below 2^-14 would lose significant bits.
__device__ inline int row_exponent(float top) {
  if (!(top > 0.0f)) return 0;
  return min(100, max(-113, 15 - ((int)((__float_as_uint(top) >> 23) & 0xff) - 126)));
}

// Two f32 as f16 pairs hi + lo, about 22 significant bits together.
__device__ inline void split2(float a, float b, h2_t& hi, h2_t& lo) {
  float minus = -1.0f;  // not known to be -1: the remainder is then one mixed-precision FMA, no conversion and subtraction
  asm("" : "+s"(minus));
  hi = __builtin_convertvector((f2_t{a, b}), h2_t);
  lo = __builtin_convertvector((f2_t{fmaf((float)hi.x, minus, a), fmaf((float)hi.y, minus, b)}), h2_t);
}

// The 8-bit values of a word, (byte - 128) 2^-9 in f16: the byte as an f16 subnormal
// (byte 2^-24) times 2^15, less 2^-2, one fused operation a pair and exact.
__device__ inline h2_t q8_pair(uint32_t bytes_0_and_2) {
  const h2_t up = {(_Float16)32768.0f, (_Float16)32768.0f}, off = {(_Float16)-0.25f, (_Float16)-0.25f};
  return __builtin_elementwise_fma(__builtin_bit_cast(h2_t, bytes_0_and_2), up, off);
}
constexpr float kQ8Unit = 512.0f;  // 2^9: what a product of such values is multiplied by

// tanh in f32, off by at most 2^-23 relative: up to kTanhNear an odd polynomial of degree
// 11 (the smallest relative error over that range, 2^-26, by weighted least squares), further
// out (1 - t) / (1 + t) with t = exp(-2 |x|). Scores stand mostly in the first part, and it
// needs neither an exponential nor a quotient.
constexpr float kTanhNear = 0.7f;
__device__ inline float tanh_near(float x) {
  const float u = x * x;
  return x * fmaf(u, fmaf(u, fmaf(u, fmaf(u, fmaf(u, -0.00508831f, 0.02002442f), -0.05352599f), 0.13328414f), -0.3333313f), 0.99999999f);
}
__device__ inline float tanh_far(float x) {
  const float t = __builtin_amdgcn_exp2f(-2.0f * kLog2e * fabsf(x));
  return copysignf((1.0f - t) * __builtin_amdgcn_rcpf(1.0f + t), x);
}

// Attention partials of a row: [hd] sums of p v, then the running maximum (base 2) and
// sum of p; 4 floats for those two keep rows 16-byte aligned.
__host__ __device__ inline int64_t part_stride(int hd) { return hd + 4; }

// Weight of a partial with running maximum m and sum l; a sum that is NaN stays in.
__device__ inline float weight_of(float m, float l, float M) {
  if (l != l) return 1.0f;
  return m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M);
}

// ---- many rows over one cache (rows_block.h) -------------------------------------------

// Rows of one kv head are its G query heads' rows of query 0, of query 1, and so on:
// row r is query r / G, head r % G. The keys are positions of one cache: kc, vc of `a`, or
// its prefix.
struct RowsAttnArgs {
  SeqAttnArgs a;
  int64_t R;      // rows of a kv head
  int G;
  int nr, splits;  // row waves of a block and key splits (rows_attn_shape); with more than one split, and for a prefix, partials are written
  bool prefix;    // keys 0 .. n_prefix - 1 of kp, vp, for one query a sequence
  float* part;    // [splits][n_kv][R][part_stride]
};

// The fewest row waves there is a kernel for: LDS and registers do not hold f32 rows' pairs
// for a lone wave.
constexpr int rows_least(int type, int hd) { return type != KV_F32 || hd <= 64 ? 1 : hd <= 128 ? 2 : 4; }

void rows_attn_shape(RowsAttnArgs* r);  // nr and splits from the rest
int64_t rows_attn_blocks(const RowsAttnArgs& r);
hipError_t launch_rows_attn(const RowsAttnArgs& r, hipStream_t s);  // a prompt's

}  // namespace uaii_hip
