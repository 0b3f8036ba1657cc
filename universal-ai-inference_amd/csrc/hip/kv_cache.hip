// kv_cache.hip — K and V rows into the caches of a batch, and back.
//
// Replaces KvCache::append_layer (include/uaii/runtime/kv_cache.hpp:80-120) for several
// sequences at once; 8-bit caches have no counterpart in the reference.
//
// An 8-bit row x[hd] of one head is stored as d = f32(max |x| / 127) and the steps
// q = x / d rounded to the nearest whole number, ties to even. The quotient's rounding is
// that of the exact quotient: q0 = rint(x * (1 / d)) is at most one step off, and the
// residual x - q0 d, which one FMA gives exactly (both are multiples of the smaller last
// place and the difference is under 2 d), says which way. Where all residuals of a wave
// are under half a step, which is nearly always, q0 stands as it is; only the others take
// the whole way (q8_any). A row with an infinity or a NaN gets a NaN scale and reads back
// as NaN.
//
// Both kernels move 4 (f32 side) + 1 to 4 (cache side) bytes a value. A group of lanes
// takes a head's row, eight values a lane, and the rows of one head at consecutive
// positions follow each other over the groups, so that the cache side is one contiguous
// stream and the f32 side runs of 4 hd bytes; two rows' loads of a group are in flight
// together. What bounds writing to KV_Q8 is the vector instructions: with four values a
// lane, a division for each place and the whole way for each value they took 14.3 us for
// 4001 rows of 8 heads of 128 in K and V, of which the 41 MB need 8.6; now 9.1.
// Reading that K or V back (21 MB, 4.3 us) takes 5.8 us, of which 2 are the launch's.
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

// Division of numbers below 2^31 by one of them: floor(n / d) is n m / 2^(31 + shift) for
// m = ceil(2^(31 + shift) / d), 2^shift being the power of two at d or next above it.
struct Divisor {
  uint32_t d, m, shift;
  explicit Divisor(uint32_t by) : d(by), shift(0) {
    while ((1u << shift) < d) ++shift;
    m = (uint32_t)((((uint64_t)1 << (31 + shift)) + d - 1) / d);
  }
  __device__ uint32_t of(uint32_t n) const { return __umulhi(2 * n, m) >> shift; }
};

struct Grid {
  uint32_t units;  // rows of heads
  Divisor rows, heads;
};

struct Place {
  int64_t src;    // floats from the f32 side's start
  int64_t value;  // values from the sequence's cache start
  int64_t row;    // rows of hd values from there (the scale's index)
  uint32_t seq;
  bool in;
};

__device__ inline Place place_of(const KvRowsArgs& a, const Grid& g, uint32_t unit) {
  Place p;
  p.in = unit < g.units;
  unit = p.in ? unit : g.units - 1;
  const uint32_t sh = g.rows.of(unit), i = unit - sh * g.rows.d;
  const uint32_t s = g.heads.of(sh), h = sh - s * g.heads.d;
  const int64_t at = a.p0 + (a.past ? (int64_t)a.past[s] : 0) + i;
  p.in = p.in && at >= 0 && at < a.max_seq;
  p.seq = s;
  p.src = (s * g.rows.d + i) * a.ld + h * (uint32_t)a.hd;
  p.row = (int64_t)((uint64_t)h * (uint32_t)a.max_seq) + (p.in ? at : 0);
  p.value = p.row * (uint32_t)a.hd;
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

// Any row: the scale, and the bytes of the lane's values.
__device__ inline float q8_any(bool finite, float amax, const f4_t (&x)[2], uint32_t (&w)[2]) {
  const float d = fminf(amax / 127.0f, 0x1.0204060p+121f);  // 127 d stays finite
  // near the bottom of the range 1 / d overflows: quotients of rows times 2^64
  const float up = amax < 0x1p-100f ? 0x1p64f : 1.0f;
  const float ds = d * up, rd = d > 0.0f ? 1.0f / ds : 0.0f;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    w[c] = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t b = finite && d > 0.0f ? q8_byte(x[c][e] * up, ds, rd) : 128u;
      w[c] |= b << (8 * e);
    }
  }
  return finite ? d : __uint_as_float(0x7fc00000u);
}

// A lane has eight values of a row: four, and four 4 GS further on.
template <int TYPE, int GS>
__global__ void __launch_bounds__(256) k_kv_write(KvRowsArgs a, Grid g) {
  const float* src = blockIdx.y ? a.v : a.k;
  uint8_t* cache = blockIdx.y ? a.vc : a.kc;
  const int64_t seq_bytes = kv_seq_bytes(TYPE, a.n_kv, a.max_seq, a.hd);
  const int l = threadIdx.x % GS;
  const int off[2] = {min(4 * l, a.hd - 4), min(4 * l + 4 * GS, a.hd - 4)};  // those behind the row's end repeat it
  const bool lane[2] = {4 * l < a.hd, 4 * l + 4 * GS < a.hd};
  const uint32_t per = 256 / GS;
  const uint32_t u0 = blockIdx.x * (per * UNROLL) + threadIdx.x / GS;
  Place p[UNROLL];
  f4_t x[UNROLL][2];
#pragma unroll
  for (int j = 0; j < UNROLL; ++j) {
    p[j] = place_of(a, g, u0 + per * j);
#pragma unroll
    for (int c = 0; c < 2; ++c) x[j][c] = *reinterpret_cast<const f4u_t*>(src + p[j].src + off[c]);
  }
#pragma unroll
  for (int j = 0; j < UNROLL; ++j) {
    uint8_t* base = cache + p[j].seq * seq_bytes;
    if constexpr (TYPE == KV_F32) {
#pragma unroll
      for (int c = 0; c < 2; ++c)
        if (p[j].in && lane[c]) *reinterpret_cast<f4_t*>(reinterpret_cast<float*>(base) + p[j].value + off[c]) = x[j][c];
    } else if constexpr (TYPE == KV_F16) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        h4_t h;
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = (_Float16)x[j][c][e];
        if (p[j].in && lane[c]) *reinterpret_cast<h4_t*>(reinterpret_cast<_Float16*>(base) + p[j].value + off[c]) = h;
      }
    } else {
      // as bits, a larger magnitude is a larger integer: infinities and NaNs come out on top
      uint32_t top = 0;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(x[j][c][e]) & 0x7fffffffu);
      top = group_max<GS>(top);
      const bool finite = top < 0x7f800000u;
      const float amax = finite ? __uint_as_float(top) : 0.0f;
      // amax / 127: the product with f32(1 / 127), which is off by 2^-28 of it, and one step by
      // the exact remainder give the nearest number (Markstein)
      constexpr float r127 = 1.0f / 127.0f;
      const float d0 = amax * r127, d1 = fmaf(fmaf(-127.0f, d0, amax), r127, d0);
      float d = d1;
      const float rd = __builtin_amdgcn_rcpf(d), half = 0.5f * d;
      // x / d + 128 rounded to a whole number by adding it to one whose last place is 1
      constexpr float kWhole = 0x1.8p23f + 128.0f;
      float off_by = 0.0f;
      uint32_t t[2][4], w[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = fmaf(x[j][c][e], rd, kWhole);
          off_by = fmaxf(off_by, fabsf(fmaf(kWhole - y, d, x[j][c][e])));
          t[c][e] = __float_as_uint(y);
        }
        w[c] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(t[c][3], t[c][2], 0x0c0c0400), __builtin_amdgcn_perm(t[c][1], t[c][0], 0x0c0c0400), 0x05040100);
      }
      // under half a step off is right; ties, quotients that are off and the ends of the range are looked at
      if (__any(!(amax >= 0x1p-100f && amax < 0x1p127f && off_by < half))) d = q8_any(finite, amax, x[j], w);
#pragma unroll
      for (int c = 0; c < 2; ++c)
        if (p[j].in && lane[c]) *reinterpret_cast<uint32_t*>(base + p[j].value + off[c]) = w[c];
      if (p[j].in && l == 0) reinterpret_cast<float*>(base + (int64_t)a.n_kv * a.max_seq * a.hd)[p[j].row] = d;
    }
  }
}

template <int TYPE, int GS>
__global__ void __launch_bounds__(256) k_kv_read(KvRowsArgs a, float* __restrict__ out, Grid g) {
  const int64_t seq_bytes = kv_seq_bytes(TYPE, a.n_kv, a.max_seq, a.hd);
  const int l = threadIdx.x % GS;
  const int off[2] = {min(4 * l, a.hd - 4), min(4 * l + 4 * GS, a.hd - 4)};
  const bool lane[2] = {4 * l < a.hd, 4 * l + 4 * GS < a.hd};
  const uint32_t per = 256 / GS;
  const uint32_t u0 = blockIdx.x * (per * UNROLL) + threadIdx.x / GS;
  Place p[UNROLL];
  f4_t x[UNROLL][2];
  // places outside the cache read row 0 of their head, which is in it
#pragma unroll
  for (int j = 0; j < UNROLL; ++j) {
    p[j] = place_of(a, g, u0 + per * j);
    const uint8_t* base = a.kc + p[j].seq * seq_bytes;
    float d = 0.0f;
    if constexpr (TYPE == KV_Q8) d = reinterpret_cast<const float*>(base + (int64_t)a.n_kv * a.max_seq * a.hd)[p[j].row];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if constexpr (TYPE == KV_F32) {
        x[j][c] = *reinterpret_cast<const f4_t*>(reinterpret_cast<const float*>(base) + p[j].value + off[c]);
      } else if constexpr (TYPE == KV_F16) {
        const h4_t h = *reinterpret_cast<const h4_t*>(reinterpret_cast<const _Float16*>(base) + p[j].value + off[c]);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[j][c][e] = (float)h[e];
      } else {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(base + p[j].value + off[c]);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[j][c][e] = (float)((int)((w >> (8 * e)) & 255u) - 128) * d;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < UNROLL; ++j)
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (p[j].in && lane[c]) *reinterpret_cast<f4u_t*>(out + p[j].src + off[c]) = x[j][c];
}

template <int TYPE>
hipError_t go(const KvRowsArgs& a, float* out, hipStream_t s) {
  const Grid g{(uint32_t)(a.n_seq * a.n_kv * a.rows), Divisor((uint32_t)a.rows), Divisor((uint32_t)a.n_kv)};
  auto launch = [&](auto write, auto read, int gs) {
    const uint32_t per = 256 / gs * UNROLL;
    const dim3 grid((g.units + per - 1) / per, out ? 1 : 2);
    if (out) UAII_LAUNCH(read, grid, dim3(256), 0, s, a, out, g);
    else UAII_LAUNCH(write, grid, dim3(256), 0, s, a, g);
    return hipGetLastError();
  };
  if (a.hd <= 32) return launch((k_kv_write<TYPE, 4>), (k_kv_read<TYPE, 4>), 4);
  if (a.hd <= 64) return launch((k_kv_write<TYPE, 8>), (k_kv_read<TYPE, 8>), 8);
  if (a.hd <= 128) return launch((k_kv_write<TYPE, 16>), (k_kv_read<TYPE, 16>), 16);
  return launch((k_kv_write<TYPE, 32>), (k_kv_read<TYPE, 32>), 32);
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
