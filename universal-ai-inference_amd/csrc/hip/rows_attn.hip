// rows_attn.hip — attention of many rows over one cache on the matrix cores: the rows of a
// prompt, or the queries of a batch over the prefix that its sequences share.
#include "seq_attn.h"

#include <algorithm>

namespace uaii_hip {
namespace {

__device__ inline f16_t mfma(h8_t a, h8_t b, f16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// Four f16 of the transposed 4 x 16 piece that a group of 16 lanes names (8 bytes each).
__device__ inline h4_t lds_tr4(const _Float16* p) {
  typedef short s4_t __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s4_t* lds4;
  return __builtin_bit_cast(h4_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p));
}

__device__ inline void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the next tile's loads stay in flight
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

__device__ inline int wave_min_i(int v) {
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ inline int wave_max_i(int v) {
  for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
  return v;
}

template <int TYPE, int NW>
constexpr int tile_keys() {
  return TYPE == KV_F32 || NW < 4 ? 32 : 64;
}

template <int TYPE, int HD, int NW>
__global__ void __launch_bounds__(64 * NW, HD == 256 ? 1 : 2) k_rows_attn(RowsAttnArgs r) {
  constexpr int NT = 64 * NW, TK = tile_keys<TYPE, NW>();
  constexpr int PL = TYPE == KV_F32 ? 2 : 1;            // f16 planes of a tile (hi, lo)
  constexpr bool SC = TYPE != KV_F16;                   // a factor for each key
  constexpr int KP = HD + 8;                            // tile row (halfs)
  constexpr int NC = HD / 16, ND = HD / 32;             // dim chunks of S, dim tiles of O
  constexpr int PE = TYPE == KV_Q8 ? 16 : 8;            // dims of a staged piece
  constexpr int PR = HD / PE;                           // pieces of a key's row
  constexpr int PIECES = TK * PR / NT;
  constexpr int PW = TYPE == KV_F32 ? 2 : 1;            // 16-byte words of a piece
  __shared__ __attribute__((aligned(16))) _Float16 ks[2][PL][TK * KP];
  __shared__ __attribute__((aligned(16))) _Float16 vs[2][PL][TK * KP];
  __shared__ __attribute__((aligned(16))) float ksc[2][SC ? TK : 4], vsc[2][SC ? TK : 4];
  // non-finite values of a tile: a bit a dim, and whether a wave's pieces have one
  __shared__ uint8_t nonfinite[2][SC && PL == 1 ? 1 : TK][HD / 8];
  __shared__ int bad[2][NW], rng[NW][4];

  const SeqAttnArgs& a = r.a;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
  const int kvh = (int)(blockIdx.x % (unsigned)a.n_kv);
  const int sx = (int)(blockIdx.x / (unsigned)a.n_kv);
  const int split = sx % r.splits;
  const int nx = (int)((r.R + 32 * NW - 1) / (32 * NW));
  const int64_t row_at = (int64_t)(nx - 1 - sx / r.splits) * (32 * NW) + 32 * wave + col;  // the longest first
  const bool valid = row_at < r.R;
  const int64_t row = valid ? row_at : r.R - 1;
  const int query = (int)(row / r.G), head = kvh * r.G + (int)(row % r.G);

  // positions [lo, hi) of the keys that the row sees, and its own
  int pos, lo = 0, hi;
  if (r.prefix) {
    const int n = (int)min((int64_t)max(a.n_keys[query], 0), a.max_seq);
    pos = a.n_prefix + n - 1;
    hi = a.n_prefix;
  } else {
    pos = a.p0 + query;
    hi = max(pos + 1, a.bidir);
    if (a.first) lo = max(0, a.first[query]);
  }
  if (a.window) lo = max(lo, pos - a.window + 1);
  if (lo >= hi) lo = INT32_MAX, hi = 0;
  const int wlo = wave_min_i(lo), wlo_max = wave_max_i(lo), whi_min = wave_min_i(hi), whi = wave_max_i(hi);
  int blo = wlo, bhi = whi, blo_max = wlo_max, bhi_min = whi_min;
  if constexpr (NW > 1) {
    if (lane == 0) rng[wave][0] = wlo, rng[wave][1] = wlo_max, rng[wave][2] = whi_min, rng[wave][3] = whi;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      blo = min(blo, rng[w][0]), blo_max = max(blo_max, rng[w][1]);
      bhi_min = min(bhi_min, rng[w][2]), bhi = max(bhi, rng[w][3]);
    }
  }
  blo = __builtin_amdgcn_readfirstlane(blo), bhi = __builtin_amdgcn_readfirstlane(bhi);
  // this split's tiles
  const int tiles = bhi > blo ? (bhi - blo + TK - 1) / TK : 0;
  const int tile0 = (int)((int64_t)tiles * split / r.splits), tile1 = (int)((int64_t)tiles * (split + 1) / r.splits);
  const int k0 = blo + tile0 * TK, k1 = min(bhi, blo + tile1 * TK);

  // q * scale * 2^e as f16 hi + lo: the lane has dims 16 c + 8 h .. + 7 of its row
  h8_t qhi[NC], qlo[NC];
  float unit;  // of a raw product
  {
    const float* qp = a.q + (int64_t)query * a.ldq + (int64_t)head * a.hd;
    float qv[NC][8], top = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int d = 16 * c + 8 * h;
      const f4_t x0 = *reinterpret_cast<const f4u_t*>(qp + min(d, a.hd - 8)), x1 = *reinterpret_cast<const f4u_t*>(qp + min(d, a.hd - 8) + 4);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        qv[c][k] = d < a.hd ? (k < 4 ? x0[k] : x1[k - 4]) * a.scale : 0.0f;
        top = fmaxf(top, fabsf(qv[c][k]));
      }
    }
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const int e = row_exponent(top);
    const float up = pow2i(e);
    unit = pow2i(-e) * (TYPE == KV_Q8 ? kQ8Unit : 1.0f);
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        h2_t x, y;
        split2(qv[c][k] * up, qv[c][k + 1] * up, x, y);
        qhi[c][k] = x.x, qhi[c][k + 1] = x.y, qlo[c][k] = y.x, qlo[c][k + 1] = y.y;
      }
  }
  const bool capped = a.cap > 0.0f, sloped = a.slopes != nullptr;
  const float to_cap = capped ? unit / a.cap : 0.0f;
  const float mul = (capped ? a.cap : unit) * kLog2e;  // scores in base 2
  const float slope = sloped ? a.slopes[head] * kLog2e : 0.0f;

  // The lane's row: probabilities are 2^(y - m + 10) / D. m follows the maximum in steps (a
  // score may pass it by 2^4), D is a power of two over the values' factors so far.
  f16_t o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = f16_t{};
  float m = -INFINITY, l = 0.0f, D = SC ? 0x1p-60f : 1.0f, lgD = SC ? -60.0f : 0.0f;

  const int64_t seq = r.prefix ? a.pre_seq : a.max_seq;
  const uint8_t* kbase = r.prefix ? a.kp : a.kc;
  const uint8_t* vbase = r.prefix ? a.vp : a.vc;
  constexpr int ES = TYPE == KV_F32 ? 4 : TYPE == KV_F16 ? 2 : 1;
  const int64_t first = (int64_t)kvh * seq;
  const float* kscale = reinterpret_cast<const float*>(kbase + (int64_t)a.n_kv * seq * a.hd) + first;  // KV_Q8
  const float* vscale = reinterpret_cast<const float*>(vbase + (int64_t)a.n_kv * seq * a.hd) + first;
  kbase += first * a.hd * ES;
  vbase += first * a.hd * ES;

  u4_t kreg[PIECES][PW], vreg[PIECES][PW];
  float screg = 0.0f;
  // keys behind the last one repeat it, dims behind the last piece that piece: both are in
  // the cache, and masked or met by zeros of q
  auto load_tile = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < PIECES; ++u) {
      const int c = threadIdx.x + NT * u, key = min(t + c / PR, k1 - 1), d = min(c % PR * PE, a.hd - PE);
      const int64_t off = ((int64_t)key * a.hd + d) * ES;
#pragma unroll
      for (int w = 0; w < PW; ++w) {
        kreg[u][w] = *reinterpret_cast<const u4_t*>(kbase + off + 16 * w);
        vreg[u][w] = *reinterpret_cast<const u4_t*>(vbase + off + 16 * w);
      }
    }
    if constexpr (TYPE == KV_Q8) {
      if ((int)threadIdx.x < 2 * TK) screg = ((int)threadIdx.x < TK ? kscale : vscale)[min(t + (int)threadIdx.x % TK, k1 - 1)];
    }
  };
  // f32 pieces: rows scaled to their largest finite magnitude, as hi + lo
  auto store_f32 = [&](const u4_t (&x)[PW], _Float16* hi_at, _Float16* lo_at, float* factor) __attribute__((always_inline)) {
    if constexpr (TYPE == KV_F32) {
      float v[8], top = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[k] = __uint_as_float(x[k / 4][k % 4]);
        const float mag = fabsf(v[k]);
        top = fmaxf(top, mag <= 3.4028235e38f ? mag : 0.0f);
      }
#pragma unroll
      for (int s = 1; s < PR; s <<= 1) top = fmaxf(top, __shfl_xor(top, s, 64));
      const int e = row_exponent(top);
      const float up = pow2i(e);
      h8_t hi8, lo8;
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        h2_t p, q;
        split2(v[k] * up, v[k + 1] * up, p, q);
        hi8[k] = p.x, hi8[k + 1] = p.y, lo8[k] = q.x, lo8[k + 1] = q.y;
      }
      *reinterpret_cast<h8_t*>(hi_at) = hi8;
      *reinterpret_cast<h8_t*>(lo_at) = lo8;
      if (factor) *factor = pow2i(-e);
    }
  };
  auto store_tile = [&](int t, int buf) __attribute__((always_inline)) {
    // Where some row does not see some key, a probability of 0 must not meet a value that is
    // not finite: such values are stored as 0 and marked.
    if constexpr (TYPE != KV_Q8) {
      bool any = false;
      if (t < blo_max || t + TK > bhi_min) {
        uint32_t top = 0;
#pragma unroll
        for (int u = 0; u < PIECES; ++u)
#pragma unroll
          for (int w = 0; w < 4 * PW; ++w) {
            const uint32_t x = vreg[u][w / 4][w % 4];
            top = TYPE == KV_F16 ? max(top, max(x & 0x7fffu, x >> 16 & 0x7fffu)) : max(top, (x & 0x7fffffffu) >> 16);
          }
        any = __any(top >= (TYPE == KV_F16 ? 0x7c00u : 0x7f80u));
        if (any) {
#pragma unroll
          for (int u = 0; u < PIECES; ++u) {
            const int c = threadIdx.x + NT * u;
            uint32_t bits = 0;
#pragma unroll
            for (int w = 0; w < 4 * PW; ++w) {
              uint32_t x = vreg[u][w / 4][w % 4];
              if constexpr (TYPE == KV_F16) {
                const bool x0 = (x & 0x7c00u) == 0x7c00u, x1 = (x & 0x7c000000u) == 0x7c000000u;
                bits |= (x0 ? 1u : 0u) << (2 * w) | (x1 ? 2u : 0u) << (2 * w);
                x &= (x0 ? 0u : 0xffffu) | (x1 ? 0u : 0xffff0000u);
              } else {
                const bool out = (x & 0x7f800000u) == 0x7f800000u;
                bits |= (out ? 1u : 0u) << w;
                x = out ? 0u : x;
              }
              vreg[u][w / 4][w % 4] = x;
            }
            nonfinite[buf][c / PR][c % PR] = (uint8_t)bits;
          }
        }
      }
      if (lane == 0) bad[buf][wave] = any;
    }
#pragma unroll
    for (int u = 0; u < PIECES; ++u) {
      const int c = threadIdx.x + NT * u, key = c / PR, at = key * KP + c % PR * PE;
      if constexpr (TYPE == KV_F16) {
        *reinterpret_cast<u4_t*>(&ks[buf][0][at]) = kreg[u][0];
        *reinterpret_cast<u4_t*>(&vs[buf][0][at]) = vreg[u][0];
      } else if constexpr (TYPE == KV_Q8) {
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const u4_t x = kv ? vreg[u][0] : kreg[u][0];
          h8_t y[2];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const h2_t p = q8_pair(__builtin_amdgcn_perm(0, x[w], 0x0c010c00)), q = q8_pair(__builtin_amdgcn_perm(0, x[w], 0x0c030c02));
            h8_t& to = y[w / 2];
            to[4 * (w % 2)] = p.x, to[4 * (w % 2) + 1] = p.y, to[4 * (w % 2) + 2] = q.x, to[4 * (w % 2) + 3] = q.y;
          }
          _Float16* to = kv ? &vs[buf][0][at] : &ks[buf][0][at];
          *reinterpret_cast<h8_t*>(to) = y[0];
          *reinterpret_cast<h8_t*>(to + 8) = y[1];
        }
      } else {
        store_f32(kreg[u], &ks[buf][0][at], &ks[buf][PL - 1][at], c % PR == 0 ? &ksc[buf][key] : nullptr);
        store_f32(vreg[u], &vs[buf][0][at], &vs[buf][PL - 1][at], c % PR == 0 ? &vsc[buf][key] : nullptr);
      }
    }
    if constexpr (TYPE == KV_Q8) {
      if ((int)threadIdx.x < TK) ksc[buf][threadIdx.x] = screg;
      else if ((int)threadIdx.x < 2 * TK) vsc[buf][threadIdx.x - TK] = screg;
    }
  };

  auto compute = [&](int kt, int buf, int sub, bool marked) __attribute__((always_inline)) {
    // S^T = K . Q^T: element i is key kt + 8 (i / 4) + 4 h + i % 4 of the lane's row
    f16_t s = f16_t{};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int at = (32 * sub + col) * KP + 16 * c + 8 * h;
      const h8_t kf = *reinterpret_cast<const h8_t*>(&ks[buf][0][at]);
      s = mfma(kf, qhi[c], s);
      s = mfma(kf, qlo[c], s);
      if constexpr (PL == 2) s = mfma(*reinterpret_cast<const h8_t*>(&ks[buf][1][at]), qhi[c], s);
    }
    if constexpr (SC) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f4_t f = *reinterpret_cast<const f4_t*>(&ksc[buf][32 * sub + 8 * q + 4 * h]);
#pragma unroll
        for (int k = 0; k < 4; ++k) s[4 * q + k] *= f[k];
      }
    }
    float y_of = mul;  // times s: the score
    if (capped) {
      float far = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] *= to_cap;
        far = fmaxf(far, fabsf(s[i]));
      }
      if (__any(!(far < 0.9f))) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = fabsf(s[i]) < 0.9f ? tanh_near(s[i]) : tanh_far(s[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = tanh_near(s[i]);
      }
    }
    const int key0 = kt + 4 * h;
    if (sloped) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = key0 + 8 * (i / 4) + i % 4;
        s[i] = fmaf(s[i], mul, -slope * (float)abs(pos - key));
      }
      y_of = 1.0f;
    }
    const bool partly = kt < wlo_max || kt + 32 > whi_min;  // wave-uniform
    uint32_t seen = 0xffffu;
    if (partly) {
      seen = 0;
      const int l0 = lo - key0, h0 = hi - key0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int k = 8 * (i / 4) + i % 4;
        const bool in = k >= l0 && k < h0;
        s[i] = in ? s[i] : -INFINITY;
        seen |= (in ? 1u : 0u) << i;
      }
    }
    float top = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
    top *= y_of;
    if (__any(top > m + 4.0f)) {
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float mnew = fmaxf(m, top);
      const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mnew);
      m = mnew;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] *= alpha;
    }
    if constexpr (SC) {
      const float f = vsc[buf][32 * sub + col];
      if (__any(f > D && f < INFINITY)) {
        const float t = wave_max(f < INFINITY ? f : 0.0f);
        const int e = min(126, (int)((__float_as_uint(t) >> 23) & 0xff) - 126);
        const float Dnew = pow2i(e), beta = D / Dnew;
        D = Dnew;
        lgD = (float)e;
        l *= beta;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] *= beta;
      }
    }
    const float ref = (m == -INFINITY ? 0.0f : m) + lgD - 10.0f;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], y_of, -ref));
      sum += s[i];
    }
    l += sum;
    if constexpr (SC) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f4_t f = *reinterpret_cast<const f4_t*>(&vsc[buf][32 * sub + 8 * q + 4 * h]);
#pragma unroll
        for (int k = 0; k < 4; ++k) s[4 * q + k] *= f[k];
      }
      if (partly) {  // a factor of a key that the row does not see may be NaN
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = seen >> i & 1 ? s[i] : 0.0f;
      }
    }
    // O^T += V^T . P^T, 16 keys a step: elements 8 c .. 8 c + 7 of P are the step's keys
    // 8 (t / 4) + 4 h + t % 4, and V's are read transposed in that order
    h8_t phi[2], plo[2];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int t = 0; t < 8; t += 2) {
        h2_t x, y;
        split2(s[8 * c + t], s[8 * c + t + 1], x, y);
        phi[c][t] = x.x, phi[c][t + 1] = x.y, plo[c][t] = y.x, plo[c][t + 1] = y.y;
      }
    auto v_at = [&](int plane, int c, int d) __attribute__((always_inline)) {
      const _Float16* p = &vs[buf][plane][(32 * sub + 16 * c + 4 * h + ((lane & 15) >> 2)) * KP + 32 * d + 16 * (lane >> 4 & 1) + 4 * (lane & 3)];
      const h4_t x = lds_tr4(p), y = lds_tr4(p + 8 * KP);
      return h8_t{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    };
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const h8_t vf = v_at(0, c, d);
        o[d] = mfma(vf, phi[c], o[d]);
        o[d] = mfma(vf, plo[c], o[d]);
        if constexpr (PL == 2) o[d] = mfma(v_at(1, c, d), phi[c], o[d]);
      }
    if (marked) {  // rows that see a value that is not finite
      const uint32_t other = (uint32_t)__shfl_xor((int)seen, 32, 64);
      for (int k = 0; k < 32; ++k) {
        const uint32_t half = (k >> 2 & 1) == h ? seen : other;
        const bool in = half >> (4 * (k >> 3) + (k & 3)) & 1;
        const uint8_t* marks = nonfinite[buf][32 * sub + k];
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int piece = 4 * d + q, c = (32 * sub + k) * PR + piece;
            const uint32_t bits = bad[buf][c % NT / 64] ? marks[piece] >> (4 * h) : 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (in && (bits >> e & 1)) o[d][4 * q + e] = __uint_as_float(0x7fc00000u);
          }
      }
    }
  };

  const bool busy = __any(valid);
  if (k0 < k1) {
    load_tile(k0);
    store_tile(k0, 0);
    lds_barrier();
    int buf = 0;
    for (int t = k0; t < k1; t += TK) {
      const bool more = t + TK < k1;  // block-uniform
      if (more) load_tile(t + TK);
      bool marked = false;
      if constexpr (TYPE != KV_Q8) {
#pragma unroll
        for (int w = 0; w < NW; ++w) marked |= __builtin_amdgcn_readfirstlane(bad[buf][w]) != 0;
      }
#pragma unroll
      for (int sub = 0; sub < TK / 32; ++sub) {
        const int kt = t + 32 * sub;
        if (busy && kt < whi && kt + 32 > wlo && kt < k1) compute(kt, buf, sub, marked);
      }
      if (more) store_tile(t + TK, buf ^ 1);
      lds_barrier();
      buf ^= 1;
    }
  }

  l += __shfl_xor(l, 32, 64);
  if (!valid) return;
  if (r.splits == 1 && !r.prefix) {
    const float inv = l == 0.0f ? 0.0f : (TYPE == KV_Q8 ? kQ8Unit : 1.0f) / l;
    float* out = a.out + (int64_t)query * a.ldo + (int64_t)head * a.hd;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int at = 32 * d + 8 * q + 4 * h;
        if (at < a.hd)
          *reinterpret_cast<f4u_t*>(out + at) = f4_t{o[d][4 * q] * inv, o[d][4 * q + 1] * inv, o[d][4 * q + 2] * inv, o[d][4 * q + 3] * inv};
      }
  } else {
    const float f = D * 0x1p-10f, fo = TYPE == KV_Q8 ? f * kQ8Unit : f;
    float* out = r.part + (((int64_t)split * a.n_kv + kvh) * r.R + row) * part_stride(a.hd);
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int at = 32 * d + 8 * q + 4 * h;
        if (at < a.hd)
          *reinterpret_cast<f4_t*>(out + at) = f4_t{o[d][4 * q] * fo, o[d][4 * q + 1] * fo, o[d][4 * q + 2] * fo, o[d][4 * q + 3] * fo};
      }
    if (h == 0) out[a.hd] = m, out[a.hd + 1] = l * f;
  }
}

// Waves of a block: each takes 32 rows.
int waves_of(int type, int64_t R) { return type == KV_F32 || R > 64 ? 4 : R > 32 ? 2 : 1; }

template <int TYPE, int HD, int NW>
hipError_t go(const RowsAttnArgs& r, hipStream_t s) {
  const int64_t blocks = (r.R + 32 * NW - 1) / (32 * NW) * r.a.n_kv * r.splits;
  if (blocks > INT32_MAX) return hipErrorInvalidValue;
  UAII_LAUNCH((k_rows_attn<TYPE, HD, NW>), dim3((unsigned)blocks), dim3(64 * NW), 0, s, r);
  return hipGetLastError();
}

template <int TYPE, int HD>
hipError_t by_waves(const RowsAttnArgs& r, hipStream_t s) {
  if constexpr (TYPE != KV_F32) {
    const int nw = waves_of(TYPE, r.R);
    if (nw == 1) return go<TYPE, HD, 1>(r, s);
    if (nw == 2) return go<TYPE, HD, 2>(r, s);
  }
  return go<TYPE, HD, 4>(r, s);
}

template <int TYPE>
hipError_t by_width(const RowsAttnArgs& r, hipStream_t s) {
  if (r.a.hd <= 64) return by_waves<TYPE, 64>(r, s);
  if (r.a.hd <= 128) return by_waves<TYPE, 128>(r, s);
  return by_waves<TYPE, 256>(r, s);
}

}  // namespace

int rows_attn_splits(const RowsAttnArgs& r, int64_t keys) {
  const int nw = waves_of(r.a.type, r.R);
  const int64_t blocks = (r.R + 32 * nw - 1) / (32 * nw) * r.a.n_kv;
  const int64_t full = (int64_t)device_cus() * (r.a.hd > 128 ? 4 : 8) / nw;
  const int64_t most = std::min<int64_t>(128, keys / 128);
  return (int)std::max<int64_t>(1, std::min<int64_t>(most, r.prefix ? full / blocks : (full + blocks - 1) / blocks));
}

hipError_t launch_rows_attn(const RowsAttnArgs& r, hipStream_t s) {
  if (r.R <= 0 || r.splits < 1 || r.a.hd % 16 || r.a.hd < 16 || r.a.hd > 256 || ((r.splits > 1 || r.prefix) && !r.part))
    return hipErrorInvalidValue;
  switch (r.a.type) {
    case KV_F32: return by_width<KV_F32>(r, s);
    case KV_F16: return by_width<KV_F16>(r, s);
    case KV_Q8: return by_width<KV_Q8>(r, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace uaii_hip
