// batch_block.h — what a block does in attention of one query for each sequence of a batch over
// the sequence's own keys (batch_attn.hip).
//
// Memory bounds it: each key and value is read once, by a block that has all query heads of
// its kv head (by fours in 16-byte loads, straight into the registers that the matrix ops
// take them from; LDS holds q alone). Four waves take 16 or 32 keys in turn; the next tile's
// keys are loaded into the registers of this one's as soon as its scores stand, its values
// when its sums do. With up to 8 query heads the low halves of q and of the probabilities
// take the columns that the high ones leave, half the matrix ops. KV_Q8, 32 chats of up to
// 8000 keys, 32/8 heads of 128 (285 MB): 59.7 us, 4774 GB/s, what a copy of 1 GiB reaches;
// f16, 12 windows of 1024 keys of 16/8 heads of 256 (99 MB): 30.5, 3240 GB/s, one and a half
// units of keys for each block that the device holds.
#pragma once

#include "seq_attn.h"

namespace uaii_hip {
namespace {

constexpr int UNIT = 128;  // keys

struct BatchArgs {
  SeqAttnArgs a;
  int G, groups;       // query heads of a kv head, and its row groups of RC
  float* slots;        // [2 blocks][RC][part_stride]: a block's first and last run
  float* whole;        // [n_seq * n_kv * groups][RC][part_stride], with a prefix only
  int2* info;          // for each (sequence, kv head, group): its first block, and how many follow
  int pre_splits, blocks;
  int fold;            // keys of a prefix that each sequence reads with its own
  int parts;           // > 1: a block for each of so many units of every head, used or not; 1: one for all of a head's
};

__device__ inline f4_t mfma32(h8_t a, h8_t b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ inline f4_t mfma16(h4_t a, h4_t b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0); }
__device__ inline f4_t mfma4(float a, float b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// What a sequence reads: with a prefix that is read with it (`fold` keys), the visible ones of
// that, padded to whole tiles, and behind them its own. Both are one run of places:
// 0 .. pre - 1 are prefix keys plo + place, padded .. end - 1 its own keys lo + place - padded.
struct Span {
  int plo, pre, padded, lo, end;
  __device__ int units() const { return (end + UNIT - 1) / UNIT; }
};

__device__ inline Span span_of(const SeqAttnArgs& a, int fold, int64_t s) {
  Span p;
  const int n = (int)min((int64_t)max(a.n_keys[s], 0), a.max_seq);
  p.lo = a.window ? max(0, n - a.window) : 0;
  p.plo = a.window ? min(fold, max(0, fold + n - a.window)) : 0;
  p.pre = fold - p.plo;
  p.padded = (p.pre + 31) & ~31;
  p.end = p.padded + n - p.lo;
  return p;
}

template <int N>
__device__ inline void load_words(gptr_t p, uint32_t off, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    w[0] = load_at<uint32_t>(p, off);
  } else if constexpr (N == 2) {
    typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
    const u2_t x = load_at<u2_t>(p, off);
    w[0] = x[0], w[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const u4_t x = load_at<u4_t>(p, off + 4 * i);
      w[i] = x[0], w[i + 1] = x[1], w[i + 2] = x[2], w[i + 3] = x[3];
    }
  }
}

// Rows of a group: the matrix op has 16 columns. With up to 8 rows (PACK) the f16 types put
// the high halves of q, and of the probabilities, into columns 0-7 and the low halves
// beside them into 8-15, half the matrix ops.
constexpr int rows_of(bool pack) { return pack ? 8 : 16; }

// LDS of a block.
template <int TYPE, int HD, bool PACK>
struct BatchLds {
  static constexpr int NW = 4, RC = rows_of(PACK), NC = HD / 32;
  static constexpr int QH = TYPE == KV_F32 ? HD / 8 : PACK ? NC : 2 * NC;  // fragments of q, 1 KB each (f32: 256 B each, by fours)
  static constexpr int WS = HD + 4;                                        // row of the waves' outputs
  __attribute__((aligned(16))) uint32_t qf[TYPE == KV_F32 ? HD / 4 * 64 : QH * 256];
  __attribute__((aligned(16))) float wo[NW][RC][WS];
  __attribute__((aligned(16))) float sc[NW][64];
  float wm[NW][16], wl[NW][16], qtop[16];
  int scan[NW], found[2];
};

template <int TYPE, int HD, bool PACK>
__device__ __forceinline__ void batch_block(const BatchArgs& b, unsigned block, BatchLds<TYPE, HD, PACK>& mem) {
  constexpr int NW = 4;
  constexpr int ES = TYPE == KV_F32 ? 4 : TYPE == KV_F16 ? 2 : 1;
  constexpr int NS = TYPE == KV_F32 || HD == 256 ? 1 : 2;  // 16-key subtiles of a tile
  constexpr int KT = 16 * NS;
  constexpr int RC = rows_of(PACK);
  constexpr int E = HD / 16;                // value dims of a lane
  constexpr int KW = HD / 4 * ES / 4;       // words of a lane's part of a key
  constexpr int VW = E * ES / 4;            // words of its part of a value row
  constexpr int NC = HD / 32;               // 32-dim chunks of a score
  constexpr bool SC = TYPE == KV_Q8;
  auto& qf = mem.qf;
  auto& wo = mem.wo;
  auto& sc = mem.sc;
  auto& wm = mem.wm;
  auto& wl = mem.wl;
  auto& qtop = mem.qtop;
  auto& scan = mem.scan;
  auto& found = mem.found;

  const SeqAttnArgs& a = b.a;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int H = a.n_kv * b.groups;
  const int n_seq = (int)a.rows;

  // ---- this block's units [u, u1) of the batch's, and the sequence that holds the first
  int s, base, u, u1;  // base: the first unit of sequence s
  int total = 0, blocks = 0;
  if (b.parts > 0) {
    // block by block, and those behind a head's last unit have nothing to do
    const int hx = (int)block / b.parts, uu = (int)block % b.parts;
    s = hx / H;
    const int n = span_of(a, b.fold, s).units();
    if (uu >= n) {
      if (b.parts == 1 && b.pre_splits == 0) {  // no join follows: a sequence with no keys
        const int kvh = hx % H / b.groups, r0 = hx % b.groups * RC, rows = min(RC, b.G - r0);
        float* out = a.out + (int64_t)s * a.ldo + (int64_t)(kvh * b.G + r0) * a.hd;
        for (int x = tid; x < rows * a.hd; x += 256) out[x] = 0.0f;
      }
      return;
    }
    base = 0;
    u = hx % H * n + uu;
    u1 = u + (b.parts == 1 ? n : 1);
  } else {
    if (n_seq <= 64) {
      // a lane for each sequence, in every wave
      const int n = lane < n_seq ? span_of(a, b.fold, lane).units() : 0;
      int incl = n;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(incl, o, 64);
        incl += lane >= o ? x : 0;
      }
      total = __builtin_amdgcn_readlane(incl, 63) * H;
      const int at = (int)((int64_t)total * block / max(1, min(b.blocks, total)));
      s = __builtin_ctzll(__ballot(at < incl * H) | 1ull << 63);
      base = (__builtin_amdgcn_readlane(incl, s) - __builtin_amdgcn_readlane(n, s)) * H;
    } else {
      const int per = (n_seq + 255) / 256, s0 = min(n_seq, tid * per), s1 = min(n_seq, s0 + per);
      int mine = 0;
      for (int i = s0; i < s1; ++i) mine += span_of(a, b.fold, i).units();
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(incl, o, 64);
        incl += lane >= o ? x : 0;
      }
      if (lane == 63) scan[wave] = incl;
      __syncthreads();
      int below = 0;
      total = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        below += w < wave ? scan[w] : 0;
        total += scan[w];
      }
      total *= H;
      const int at = (int)((int64_t)total * block / max(1, min(b.blocks, total)));
      int before = below + incl - mine;  // units of a head's worth of the sequences before s0
      if (before * H <= at && at < (before + mine) * H) {
        int i = s0;
        for (;; ++i) {
          const int n = span_of(a, b.fold, i).units();
          if (at < (before + n) * H) break;
          before += n;
        }
        found[0] = i;
        found[1] = before;
      }
      __syncthreads();
      s = __builtin_amdgcn_readfirstlane(found[0]), base = __builtin_amdgcn_readfirstlane(found[1]) * H;
    }
    blocks = min(b.blocks, total);  // each has a unit at least
    if ((int)block >= blocks) return;
    u = (int)((int64_t)total * block / blocks);
    u1 = (int)((int64_t)total * (block + 1) / blocks);
  }

  const bool capped = a.cap > 0.0f, sloped = a.slopes != nullptr;
  const int crow = PACK ? col & 7 : col;  // the lane's row of the group
  const bool low = PACK && col >= 8;      // it works on the low halves

  while (u < u1) {
    Span sp = span_of(a, b.fold, s);
    int units = sp.units();
    while (units == 0) {  // sequences with no keys
      if (++s >= n_seq) return;
      sp = span_of(a, b.fold, s);
      units = sp.units();
    }
    const int hx = (u - base) / units, uu = (u - base) % units, ue = min(units, uu + u1 - u);
    const int kvh = hx / b.groups, head0 = kvh * b.G + hx % b.groups * RC;
    const int rows = min(RC, b.G - hx % b.groups * RC);
    const int k0 = UNIT * uu, k1 = min(sp.end, UNIT * ue);  // places

    // the sources: the prefix's cache and the sequence's, from the kv head's first row on, so
    // that a place's row is the place in both
    struct Source {
      const uint8_t *k, *v;
      const float *kscale, *vscale;  // KV_Q8
    };
    const uint32_t row_bytes = (uint32_t)a.hd * ES;
    auto source = [&](const uint8_t* k, const uint8_t* v, int64_t seq, int64_t first) __attribute__((always_inline)) {
      const int64_t row = kvh * seq + first, scales = (int64_t)a.n_kv * seq * a.hd;
      return Source{k + row * row_bytes, v + row * row_bytes, reinterpret_cast<const float*>(k + scales) + row,
                    reinterpret_cast<const float*>(v + scales) + row};
    };
    const Source shared = source(a.kp, a.vp, a.pre_seq, sp.plo);
    const Source own = source(a.kc + (int64_t)s * a.seq_bytes, a.vc + (int64_t)s * a.seq_bytes, a.max_seq, (int64_t)sp.lo - sp.padded);
    // places of tile t's source that are keys end here
    auto limit = [&](int t) __attribute__((always_inline)) { return t < sp.padded ? min(sp.pre, k1) : k1; };

    uint32_t kw[NS][KW], vw[NS][4][VW];  // a tile: the lane's parts of its keys and of its values
    float fw;                            // KV_Q8: a key's factor in the lower lanes, a value's in the upper
    // keys behind the last repeat it and are masked; dims behind the row's end repeat its
    // last piece, which meets zeros of q or goes to outputs that are not stored
    auto load_keys = [&](int t) __attribute__((always_inline)) {
      const bool pre = t < sp.padded;
      const int from = min(t, limit(t) - 1), last = limit(t) - 1 - from;  // a tile of padding repeats the last key too
      const gptr_t kt = uniform_at(pre ? shared.k : own.k, (int64_t)from * row_bytes);
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const uint32_t kr = (uint32_t)min(16 * i + col, last) * row_bytes;
#pragma unroll
        for (int w = 0; w < KW; w += 4) {
          constexpr int P = 16 / ES;
          const u4_t y = load_at<u4_t>(kt, kr + (uint32_t)min(g * (HD / 4) + w / 4 * P, a.hd - P) * ES);
          kw[i][w] = y[0], kw[i][w + 1] = y[1], kw[i][w + 2] = y[2], kw[i][w + 3] = y[3];
        }
      }
      if constexpr (SC) {
        const float* kf = pre ? shared.kscale : own.kscale;
        const float* vf = pre ? shared.vscale : own.vscale;
        fw = (lane < 32 ? kf : vf)[from + min(lane & 31, last)];
      }
    };
    auto load_values = [&](int t) __attribute__((always_inline)) {
      const int from = min(t, limit(t) - 1), last = limit(t) - 1 - from;
      const gptr_t vt = uniform_at(t < sp.padded ? shared.v : own.v, (int64_t)from * row_bytes);
      const uint32_t d = (uint32_t)min(col * E, a.hd - E) * ES;
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) load_words<VW>(vt, (uint32_t)min(16 * i + 4 * g + r, last) * row_bytes + d, vw[i][r]);
    };

    // q's part of a thread (row tid / 16, E dims), ahead of the first tile, so that nothing
    // waits for the tile with it
    const int qr = tid >> 4, qd = (tid & 15) * E;
    float qv[E];
    if (qr < rows) {
      const float* at = a.q + (int64_t)s * a.ldq + (int64_t)(head0 + qr) * a.hd + min(qd, a.hd - E);
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        const f4_t x = *reinterpret_cast<const f4u_t*>(at + e);
        qv[e] = x[0], qv[e + 1] = x[1], qv[e + 2] = x[2], qv[e + 3] = x[3];
      }
    }
    const int step = NW * KT, mine = k0 + wave * KT;
    if (mine < k1) load_keys(mine), load_values(mine);

    // ---- q as fragments in LDS, f16 halves scaled to the row's largest magnitude
    {
      float top = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        qv[e] = qr < rows && qd < a.hd ? qv[e] * a.scale : 0.0f;
        top = fmaxf(top, fabsf(qv[e]));
      }
      top = fmaxf(top, dpp_mov<0xB1>(top));   // quad_perm [1,0,3,2]
      top = fmaxf(top, dpp_mov<0x4E>(top));   // quad_perm [2,3,0,1]
      top = fmaxf(top, dpp_mov<0x141>(top));  // row_half_mirror
      top = fmaxf(top, dpp_mov<0x140>(top));  // row_mirror
      if ((tid & 15) == 0) qtop[qr] = top;
      const float up = TYPE == KV_F32 ? 1.0f : pow2i(row_exponent(top));
      if (qr < RC) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
          const int d = qd + e, part = d / (HD / 4), at = d % (HD / 4);  // lanes 16 part .. + 15 hold it
          if constexpr (TYPE == KV_F32) {
            reinterpret_cast<f4_t*>(qf)[at / 4 * 64 + 16 * part + qr] = f4_t{qv[e], qv[e + 1], qv[e + 2], qv[e + 3]};
          } else {
            // bytes of a word pair up as 0 and 2, 1 and 3
            constexpr int B = TYPE == KV_Q8 ? 2 : 1, C = TYPE == KV_Q8 ? 1 : 2;
            h2_t h0, h1, l0, l1;
            split2(qv[e] * up, qv[e + B] * up, h0, l0);
            split2(qv[e + C] * up, qv[e + 3] * up, h1, l1);
            h4_t* to = reinterpret_cast<h4_t*>(qf) + (at / 8 * 64 + 16 * part + qr) * 2 + at / 4 % 2;
            to[0] = h4_t{h0.x, h0.y, h1.x, h1.y};
            to[PACK ? 16 : NC * 128] = h4_t{l0.x, l0.y, l1.x, l1.y};
          }
        }
      }
    }
    __syncthreads();
    const float unit = TYPE == KV_F32 ? 1.0f : pow2i(-row_exponent(qtop[crow])) * (SC ? kQ8Unit : 1.0f);
    const float to_cap = capped ? fminf(unit / a.cap, 0x1p127f) : 0.0f;  // finite: a score of 0 stays 0
    const float mul = (capped ? a.cap : unit) * kLog2e;  // scores in base 2
    const float slope = sloped && crow < rows ? a.slopes[head0 + crow] * kLog2e : 0.0f;

    f4_t o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
    // as in rows_attn.hip: probabilities are 2^(y - m + 10) / D
    float m = -INFINITY, l = 0.0f, D = SC ? 0x1p-60f : 1.0f, lgD = SC ? -60.0f : 0.0f;

    // A tile's keys are used up before its softmax and its values behind it: the next tile's
    // are loaded into the same registers from there on, and are on their way through the other
    // half of the work.
    for (int t = mine; t < k1; t += step) {
      f4_t y[NS];
      if constexpr (SC) {
        sc[wave][lane] = fw;
        const float f = lane >= 32 ? fw : 0.0f;
        if (__any(f > D && f < INFINITY)) {
          const float top = wave_max_dpp(f < INFINITY ? f : 0.0f);
          const int e = min(126, (int)((__float_as_uint(top) >> 23) & 0xff) - 126);
          const float Dnew = pow2i(e), beta = D / Dnew;
          D = Dnew;
          lgD = (float)e;
          l *= beta;
#pragma unroll
          for (int k = 0; k < E; ++k) o[k] *= beta;
        }
      }
#pragma unroll
      for (int i = 0; i < NS; ++i) y[i] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
      if constexpr (TYPE == KV_F32) {
#pragma unroll
        for (int w = 0; w < KW; w += 4) {
          const f4_t q = reinterpret_cast<const f4_t*>(qf)[w / 4 * 64 + lane];
#pragma unroll
          for (int k = 0; k < 4; ++k) y[0] = mfma4(__uint_as_float(kw[0][w + k]), q[k], y[0]);
        }
      } else {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const h8_t q0 = reinterpret_cast<const h8_t*>(qf)[c * 64 + lane];
          h8_t q1;
          if constexpr (!PACK) q1 = reinterpret_cast<const h8_t*>(qf)[(NC + c) * 64 + lane];
#pragma unroll
          for (int i = 0; i < NS; ++i) {
            h8_t kf;
            if constexpr (TYPE == KV_F16) {
              kf = __builtin_bit_cast(h8_t, (u4_t{kw[i][4 * c], kw[i][4 * c + 1], kw[i][4 * c + 2], kw[i][4 * c + 3]}));
            } else {
#pragma unroll
              for (int w = 0; w < 2; ++w) {
                const uint32_t z = kw[i][2 * c + w];
                const h2_t p = q8_pair(z & 0x00ff00ffu), q = q8_pair(__builtin_amdgcn_perm(0, z, 0x0c030c01));
                kf[4 * w] = p.x, kf[4 * w + 1] = p.y, kf[4 * w + 2] = q.x, kf[4 * w + 3] = q.y;
              }
            }
            y[i] = mfma32(kf, q0, y[i]);
            if constexpr (!PACK) y[i] = mfma32(kf, q1, y[i]);
          }
        }
        if constexpr (PACK) {
#pragma unroll
          for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) y[i][r] += dpp_mov<0x128>(y[i][r]);  // row_ror 8: the other half's column
        }
      }
      const int next = t + step < k1 ? t + step : t;  // the last turn loads its own tile again
      load_keys(next);
      // element r of y[i]: key t + 16 i + 4 g + r
      f4_t vf[NS];
      if constexpr (SC) {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          y[i] *= *reinterpret_cast<const f4_t*>(&sc[wave][16 * i + 4 * g]);
          vf[i] = *reinterpret_cast<const f4_t*>(&sc[wave][32 + 16 * i + 4 * g]);
        }
        __builtin_amdgcn_wave_barrier();
      }
      float y_of = mul;
      if (capped) {
        float out = 0.0f;
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            y[i][r] *= to_cap;
            out = fmaxf(out, fabsf(y[i][r]));
          }
        const bool some_far = __any(!(out < kTanhNear));
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float near = tanh_near(y[i][r]);
            y[i][r] = some_far && !(fabsf(y[i][r]) < kTanhNear) ? tanh_far(y[i][r]) : near;
          }
      }
      if (sloped) {
        // positions between the tile's first key and the query (own keys: the query is the last of them)
        const int far = sp.end - 1 - t + (t < sp.padded ? sp.pre - sp.padded + sp.lo : 0);
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) y[i][r] = fmaf(y[i][r], mul, -slope * (float)(far - 16 * i - 4 * g - r));
        y_of = 1.0f;
      }
      if (t + KT > limit(t)) {
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) y[i][r] = t + 16 * i + 4 * g + r < limit(t) ? y[i][r] : -INFINITY;
      }
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, y[i][r]);
      top *= y_of;
      if (__any(top > m + 4.0f)) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float mnew = fmaxf(m, top);
        const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mnew);
        m = mnew;
        l *= alpha;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] *= alpha;
      }
      const float ref = (m == -INFINITY ? 0.0f : m) + lgD - 10.0f;
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          y[i][r] = __builtin_amdgcn_exp2f(fmaf(y[i][r], y_of, -ref));
          l += y[i][r];
        }
      if constexpr (SC) {
#pragma unroll
        for (int i = 0; i < NS; ++i) y[i] *= vf[i];
      }
      // O^T += V^T . P^T: the lane's probabilities are the operand as they lie, the keys
      // 4 g + r of a subtile being its k index; a value's dims are E col + e
      if constexpr (TYPE == KV_F32) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] = mfma4(__uint_as_float(vw[0][r][e]), y[0][r], o[e]);
      } else {
        h4_t p0[NS], p1[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
          for (int r = 0; r < 4; r += 2) {
            h2_t hi, lo;
            split2(y[i][r], y[i][r + 1], hi, lo);
            if constexpr (PACK) {
              const uint32_t z = low ? __builtin_bit_cast(uint32_t, lo) : __builtin_bit_cast(uint32_t, hi);
              hi = __builtin_bit_cast(h2_t, z);
            }
            p0[i][r] = hi.x, p0[i][r + 1] = hi.y;
            p1[i][r] = lo.x, p1[i][r + 1] = lo.y;
          }
#pragma unroll
        for (int e = 0; e < E; ++e) {
          h4_t vv[NS];
#pragma unroll
          for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int r = 0; r < 4; r += 2) {
              h2_t z;
              if constexpr (TYPE == KV_F16) {
                z = __builtin_bit_cast(h2_t, __builtin_amdgcn_perm(vw[i][r + 1][e / 2], vw[i][r][e / 2], e & 1 ? 0x07060302 : 0x05040100));
              } else {
                z = q8_pair(__builtin_amdgcn_perm(vw[i][r + 1][e / 4], vw[i][r][e / 4], 0x0c040c00 + (e & 3) * 0x00010001));
              }
              vv[i][r] = z.x, vv[i][r + 1] = z.y;
            }
          if constexpr (NS == 2) {
            const h8_t v8 = __builtin_shufflevector(vv[0], vv[NS - 1], 0, 1, 2, 3, 4, 5, 6, 7);
            o[e] = mfma32(v8, __builtin_shufflevector(p0[0], p0[NS - 1], 0, 1, 2, 3, 4, 5, 6, 7), o[e]);
            if constexpr (!PACK) o[e] = mfma32(v8, __builtin_shufflevector(p1[0], p1[NS - 1], 0, 1, 2, 3, 4, 5, 6, 7), o[e]);
          } else {
            o[e] = mfma16(vv[0], p0[0], o[e]);
            if constexpr (!PACK) o[e] = mfma16(vv[0], p1[0], o[e]);
          }
        }
      }
      load_values(next);
    }

    // ---- the waves' results together
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    const float back = D * 0x1p-10f, back_o = SC ? back * kQ8Unit : back;
    if constexpr (PACK) {
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[e][r] += dpp_mov<0x128>(o[e][r]);
    }
    if (!low) {
      if (g == 0) wm[wave][crow] = m, wl[wave][crow] = l * back;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < E; e += 4)
          *reinterpret_cast<f4_t*>(&wo[wave][crow][(4 * g + r) * E + e]) = f4_t{o[e][r], o[e + 1][r], o[e + 2][r], o[e + 3][r]} * back_o;
    }
    __syncthreads();
    const bool complete = uu == 0 && ue == units;
    if (b.parts == 0 && uu == 0 && tid == 0) {
      // block of unit v: the last one whose first unit, total b / blocks, is not behind it
      const int last = complete ? (int)block : (int)(((int64_t)(u + units) * blocks - 1) / total);
      b.info[(int64_t)s * H + hx] = make_int2((int)block, last - (int)block);
    }
    const int64_t stride = part_stride(a.hd);
    const bool direct = complete && b.pre_splits == 0;
    float* part = b.parts > 0 ? b.slots + (int64_t)block * RC * stride
                  : complete ? b.whole + ((int64_t)s * H + hx) * RC * stride
                             : b.slots + (2 * (int64_t)block + (uu == 0)) * RC * stride;
    for (int x = tid; x < rows * (a.hd / 4); x += 256) {
      const int r = x / (a.hd / 4), d = x % (a.hd / 4) * 4;
      float M = -INFINITY, den = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w) M = fmaxf(M, wm[w][r]);
      f4_t acc = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = weight_of(wm[w][r], wl[w][r], M);
        acc += f * *reinterpret_cast<const f4_t*>(&wo[w][r][d]);
        den += f * wl[w][r];
      }
      if (direct) {
        const float inv = den == 0.0f ? 0.0f : 1.0f / den;
        *reinterpret_cast<f4u_t*>(a.out + (int64_t)s * a.ldo + (int64_t)(head0 + r) * a.hd + d) = acc * inv;
      } else {
        *reinterpret_cast<f4_t*>(part + r * stride + d) = acc;
        if (d == 0) part[r * stride + a.hd] = M, part[r * stride + a.hd + 1] = den;
      }
    }
    __syncthreads();

    u += ue - uu;
    if (ue == units && hx == H - 1) {
      ++s;
      base = u;
    }
  }
}

}  // namespace
}  // namespace uaii_hip
