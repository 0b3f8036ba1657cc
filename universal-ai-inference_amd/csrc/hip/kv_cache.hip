// kv_cache.hip — K and V rows into the caches of a batch, and back.
//
// Replaces KvCache::append_layer (include/uaii/runtime/kv_cache.hpp:80-120) for several
// sequences at once; 8-bit caches have no counterpart in the reference.
//
// An 8-bit row x[hd] of one head is stored as d = f32(max |x| / 127) and the steps
// q = x / d rounded to the nearest whole number, ties to even. The quotient's rounding is
// that of the exact quotient: q0 = rint(x * (1 / d)) is at most one step off, and the
// residual x - q0 d, which one FMA gives exactly (both are multiples of the smaller last
// place and the difference is under 2 d), says which way. A row with an infinity or a NaN
// gets a NaN scale and reads back as NaN.
//
// Both kernels move 4 (f32 side) + 1 to 4 (cache side) bytes a value and are bound by
// that. A group of lanes takes a head's row, four values a lane, and the rows of one head
// at consecutive positions follow each other over the groups, so that the cache side is
// one contiguous stream and the f32 side runs of 4 hd bytes; two rows' loads of a group
// are in flight together.
#include "kv_cache.h"

#include <algorithm>
#include <type_traits>

namespace uaii_hip {
namespace {

// Rows of a caller's buffer start at any float.
typedef float f4u_t __attribute__((ext_vector_type(4), aligned(4)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef _Float16 h4_t __attribute__((ext_vector_type(4)));

constexpr int UNROLL = 2;

struct Place {
  int64_t src;    // floats from the f32 side's start
  int64_t value;  // values from the sequence's cache start
  int64_t row;    // rows of hd values from there (the scale's index)
  int64_t seq;
  bool in;
};

__device__ inline Place place_of(const KvRowsArgs& a, uint32_t unit, uint32_t units) {
  Place p;
  p.in = unit < units;
  unit = p.in ? unit : units - 1;
  const uint32_t rows = (uint32_t)a.rows, sh = unit / rows, i = unit - sh * rows;
  const uint32_t s = sh / (uint32_t)a.n_kv, h = sh - s * (uint32_t)a.n_kv;
  const int64_t at = a.p0 + (a.past ? (int64_t)a.past[s] : 0) + i;
  p.in = p.in && at >= 0 && at < a.max_seq;
  p.seq = s;
  p.src = ((int64_t)s * rows + i) * a.ld + (int64_t)h * a.hd;
  p.row = (int64_t)h * a.max_seq + (p.in ? at : 0);
  p.value = p.row * a.hd;
  return p;
}

// Largest of the GS lanes of a group, on DPP moves within 16 lanes.
template <int GS>
__device__ inline uint32_t group_max(uint32_t v) {
  auto dpp = [&](auto ctrl) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xF, 0xF, false); };
  v = max(v, dpp(std::integral_constant<int, 0xB1>{}));                          // quad_perm [1,0,3,2]
  v = max(v, dpp(std::integral_constant<int, 0x4E>{}));                          // quad_perm [2,3,0,1]
  if constexpr (GS >= 8) v = max(v, dpp(std::integral_constant<int, 0x141>{}));  // row_half_mirror
  if constexpr (GS >= 16) v = max(v, dpp(std::integral_constant<int, 0x140>{}));  // row_mirror
  if constexpr (GS >= 32) v = max(v, (uint32_t)__shfl_xor((int)v, 16, 64));
  if constexpr (GS >= 64) v = max(v, (uint32_t)__shfl_xor((int)v, 32, 64));
  return v;
}

__device__ inline uint32_t q8_byte(float x, float d, float rd) {
  float q = rintf(x * rd);
  const float r = fmaf(-q, d, x), half = 0.5f * d;
  const bool odd = ((int)q & 1) != 0;
  if (r > half || (r == half && odd)) q += 1.0f;
  else if (r < -half || (r == -half && odd)) q -= 1.0f;
  q = fminf(fmaxf(q, -127.0f), 127.0f);
  return (uint32_t)((int)q + 128);
}

template <int TYPE, int GS>
__global__ void __launch_bounds__(256) k_kv_write(KvRowsArgs a, uint32_t units) {
  const float* src = blockIdx.y ? a.v : a.k;
  uint8_t* cache = blockIdx.y ? a.vc : a.kc;
  const int64_t seq_bytes = kv_seq_bytes(TYPE, a.n_kv, a.max_seq, a.hd);
  const int l = threadIdx.x % GS;
  const int off = min(4 * l, a.hd - 4);  // lanes behind a narrow row repeat its end
  const bool lane = 4 * l < a.hd;
  const uint32_t per = 256 / GS;
  const uint32_t u0 = blockIdx.x * (per * UNROLL) + threadIdx.x / GS;
  Place p[UNROLL];
  f4_t x[UNROLL];
#pragma unroll
  for (int j = 0; j < UNROLL; ++j) {
    p[j] = place_of(a, u0 + per * j, units);
    x[j] = *reinterpret_cast<const f4u_t*>(src + p[j].src + off);
  }
#pragma unroll
  for (int j = 0; j < UNROLL; ++j) {
    uint8_t* base = cache + p[j].seq * seq_bytes;
    const bool put = p[j].in && lane;
    if constexpr (TYPE == KV_F32) {
      if (put) *reinterpret_cast<f4_t*>(reinterpret_cast<float*>(base) + p[j].value + off) = x[j];
    } else if constexpr (TYPE == KV_F16) {
      h4_t h;
#pragma unroll
      for (int e = 0; e < 4; ++e) h[e] = (_Float16)x[j][e];
      if (put) *reinterpret_cast<h4_t*>(reinterpret_cast<_Float16*>(base) + p[j].value + off) = h;
    } else {
      // as bits, a larger magnitude is a larger integer: infinities and NaNs come out on top
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(x[j][e]) & 0x7fffffffu);
      top = group_max<GS>(top);
      const bool finite = top < 0x7f800000u;
      const float amax = finite ? __uint_as_float(top) : 0.0f;
      const float d = fminf(amax / 127.0f, 0x1.0204060p+121f);  // 127 d stays finite
      // near the bottom of the range 1 / d overflows: quotients of rows times 2^64
      const float up = amax < 0x1p-100f ? 0x1p64f : 1.0f;
      const float ds = d * up, rd = d > 0.0f ? 1.0f / ds : 0.0f;
      uint32_t w = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t b = finite && d > 0.0f ? q8_byte(x[j][e] * up, ds, rd) : 128u;
        w |= b << (8 * e);
      }
      if (put) *reinterpret_cast<uint32_t*>(base + p[j].value + off) = w;
      if (p[j].in && l == 0)
        reinterpret_cast<float*>(base + (int64_t)a.n_kv * a.max_seq * a.hd)[p[j].row] = finite ? d : __uint_as_float(0x7fc00000u);
    }
  }
}

template <int TYPE, int GS>
__global__ void __launch_bounds__(256) k_kv_read(KvRowsArgs a, float* __restrict__ out, uint32_t units) {
  const int64_t seq_bytes = kv_seq_bytes(TYPE, a.n_kv, a.max_seq, a.hd);
  const int l = threadIdx.x % GS;
  const int off = min(4 * l, a.hd - 4);
  const bool lane = 4 * l < a.hd;
  const uint32_t per = 256 / GS;
  const uint32_t u0 = blockIdx.x * (per * UNROLL) + threadIdx.x / GS;
  Place p[UNROLL];
  f4_t x[UNROLL];
  // places outside the cache read row 0 of their head, which is in it
#pragma unroll
  for (int j = 0; j < UNROLL; ++j) {
    p[j] = place_of(a, u0 + per * j, units);
    const uint8_t* base = a.kc + p[j].seq * seq_bytes;
    if constexpr (TYPE == KV_F32) {
      x[j] = *reinterpret_cast<const f4_t*>(reinterpret_cast<const float*>(base) + p[j].value + off);
    } else if constexpr (TYPE == KV_F16) {
      const h4_t h = *reinterpret_cast<const h4_t*>(reinterpret_cast<const _Float16*>(base) + p[j].value + off);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j][e] = (float)h[e];
    } else {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(base + p[j].value + off);
      const float d = reinterpret_cast<const float*>(base + (int64_t)a.n_kv * a.max_seq * a.hd)[p[j].row];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j][e] = (float)((int)((w >> (8 * e)) & 255u) - 128) * d;
    }
  }
#pragma unroll
  for (int j = 0; j < UNROLL; ++j)
    if (p[j].in && lane) *reinterpret_cast<f4u_t*>(out + p[j].src + off) = x[j];
}

template <int TYPE>
hipError_t go(const KvRowsArgs& a, float* out, hipStream_t s) {
  const uint32_t units = (uint32_t)(a.n_seq * a.n_kv * a.rows);
  auto launch = [&](auto write, auto read, int gs) {
    const uint32_t per = 256 / gs * UNROLL;
    const dim3 grid((units + per - 1) / per, out ? 1 : 2);
    if (out) UAII_LAUNCH(read, grid, dim3(256), 0, s, a, out, units);
    else UAII_LAUNCH(write, grid, dim3(256), 0, s, a, units);
    return hipGetLastError();
  };
  if (a.hd <= 16) return launch((k_kv_write<TYPE, 4>), (k_kv_read<TYPE, 4>), 4);
  if (a.hd <= 32) return launch((k_kv_write<TYPE, 8>), (k_kv_read<TYPE, 8>), 8);
  if (a.hd <= 64) return launch((k_kv_write<TYPE, 16>), (k_kv_read<TYPE, 16>), 16);
  if (a.hd <= 128) return launch((k_kv_write<TYPE, 32>), (k_kv_read<TYPE, 32>), 32);
  return launch((k_kv_write<TYPE, 64>), (k_kv_read<TYPE, 64>), 64);
}

hipError_t dispatch(const KvRowsArgs& a, float* out, hipStream_t s) {
  if (a.n_seq == 0 || a.rows == 0) return hipSuccess;
  if (a.n_seq * a.n_kv > INT32_MAX / a.rows || a.hd % 16 || a.hd < 16 || a.hd > 256) return hipErrorInvalidValue;
  switch (a.type) {
    case KV_F32: return go<KV_F32>(a, out, s);
    case KV_F16: return go<KV_F16>(a, out, s);
    case KV_Q8: return go<KV_Q8>(a, out, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t launch_kv_write(const KvRowsArgs& a, hipStream_t s) { return dispatch(a, nullptr, s); }
hipError_t launch_kv_read(const KvRowsArgs& a, float* out, hipStream_t s) { return dispatch(a, out, s); }

}  // namespace uaii_hip
