// rows_block.h — what a block does in attention of many rows over one cache on the matrix
// cores: the rows of a prompt (rows_attn.hip), or the queries of a batch over the prefix that
// its sequences share (batch_attn.hip).
//
// One pass over the keys with the running maximum and sum of the softmax. A wave has 32 rows
// (16 with rows of 256) and takes 32 keys a turn: S^T = K . Q^T puts a row's scores into the
// lanes that hold its sums, so that maximum, sum and probabilities stay in registers, and the
// probabilities are the operand of O^T += V^T . P^T as they lie; V is read from LDS
// transposed. The next tile's loads stand between the matrix ops of the scores, its way into
// LDS between those of the sums.
//
// Precision: a cache's values enter the f16 matrix ops as they are (f16), as whole numbers
// 2^-9 (KV_Q8, a key's factor on its score, a value's on its probability) or as f16 pairs
// hi + lo (f32, scaled by a power of two for each row); q and the probabilities are pairs.
// So a product takes two matrix ops (f32: three) where plain f16 would take one, and results
// stand within 2e-7 to 7e-7 of 64-bit ones, like f32 sums. Scores and probabilities are in
// base 2; the maximum follows in steps of 2^4, 2^10 keeps small probabilities above f16's
// subnormals, and D, a power of two over the values' factors so far, keeps p times factor
// below f16's end.
//
// What bounds it: matrix ops and vector ops share a SIMD's two waves. f16 rows of 128 (4096
// rows of 32/8 heads in three documents, 162 us): 427 TFLOP/s of the formula, 855 of matrix
// ops where a large f16 library product reaches 1178; the matrix cores are busy 38 % of all
// SIMD cycles, the vector units 34 %, and the rest is the longest blocks' end, where CUs have
// run out of others, and each block's way to its first tile (5 us, of which a block beside it
// hides a part). KV_Q8 with softcap and window (1003 rows over 1500 keys, 73 us): 29 vector
// ops a score (7 for tanh, 6.5 for the bytes' way to f16), busy 51 %, the matrix cores 26 %.
#pragma once

#include "seq_attn.h"

#include <type_traits>

namespace uaii_hip {
namespace {

__device__ inline f16_t mfma(h8_t a, h8_t b, f16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ inline f4_t mfma(h8_t a, h8_t b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

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

// Largest and smallest of the 64 lanes, in a scalar register.
__device__ inline int wave_max_i(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false));   // quad_perm [1,0,3,2]
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false));   // quad_perm [2,3,0,1]
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false));  // row_half_mirror
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, false));  // row_mirror
  return max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
             max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}
__device__ inline int wave_min_i(int v) { return -wave_max_i(-v); }  // of values above INT32_MIN

// A block has 4 waves: NR of them take MR rows each, and the NK = 4 / NR groups of such waves
// take the tiles of the block's keys in turn, each in an LDS region of its own.
//
// MR is 32, on the 32x32 matrix ops, where a fragment of keys or values read from LDS serves
// twice as many rows; the rows' queries and sums take HD registers of a lane, which at
// head_dim 256 leaves none: 16 rows there, on the 16x16 ops.
constexpr int row_tile(int hd) { return hd > 128 ? 16 : 32; }
template <int TYPE, int HD, int NR>
constexpr int tile_keys() {
  return TYPE == KV_Q8 && HD == 64 && NR == 4 ? 64 : 32;  // a piece for each thread
}

// LDS of a block.
template <int TYPE, int HD, int NR>
struct RowsLds {
  static constexpr int NK = 4 / NR, TK = tile_keys<TYPE, HD, NR>(), MR = row_tile(HD), GL = 64 / MR;
  static constexpr int PL = TYPE == KV_F32 ? 2 : 1, ND = HD / MR, NQ = MR / (4 * GL), NC = HD / (8 * GL);
  static constexpr bool SC = TYPE != KV_F16, QL = NR == 1;
  static constexpr int NB = NR == 1 ? 1 : 2;         // buffers of a region; a lone wave needs one
  static constexpr int KP = HD + 8, VP = HD + 16;    // rows of a tile (halfs): see v_at
  struct Tile {
    __attribute__((aligned(16))) _Float16 k[PL][TK * KP];
    __attribute__((aligned(16))) _Float16 v[PL][TK * VP];
    __attribute__((aligned(16))) float kf[SC ? TK : 4], vf[SC ? TK : 4];
  };
  // values of a tile that are not finite: a bit a dim (KV_Q8: one for the row), and whether a
  // wave's pieces have one (KV_Q8: whether the tile has); of this tile and the next
  struct Marks {
    uint8_t at[TK][TYPE == KV_Q8 ? 1 : HD / 8];
    int any[TYPE == KV_Q8 ? 1 : NR];
  };
  struct Merge {  // of the groups behind the first
    f4_t o[NK > 1 ? NK - 1 : 1][NR][ND * NQ][64];
    float ml[NK > 1 ? NK - 1 : 1][NR][2][64], D[NK > 1 ? NK - 1 : 1][NR];
  };
  static constexpr size_t kTiles = sizeof(Tile) * NB * NK, kMerge = NK > 1 ? sizeof(Merge) : 0;
  __attribute__((aligned(16))) char tiles[kTiles > kMerge ? kTiles : kMerge];
  __attribute__((aligned(16))) h8_t qs[QL ? 2 * NC * 64 : 1];
  Marks marks[NK][2];
  float qtop[QL ? NK : 1][MR];
  int rng[NR][4];
};

// A block's work. PREFIX: the keys are 0 .. n_prefix - 1 of kp, vp, for one query a sequence, and
// partials are written; else the rows are a prompt's.
template <int TYPE, int HD, int NR, bool PREFIX>
__device__ __forceinline__ void rows_block(const RowsAttnArgs& r, unsigned block, RowsLds<TYPE, HD, NR>& mem) {
  constexpr int NK = 4 / NR, NT = 64 * NR, TK = tile_keys<TYPE, HD, NR>(), SUBS = TK / 32;
  constexpr int MR = row_tile(HD), GL = 64 / MR;        // lane groups: lanes of a row
  constexpr int NE = 32 / GL, KS = MR == 32 ? 8 : 16;   // scores of a lane for 32 keys: element i is key KS (i / 4) + 4 h + i % 4
  constexpr bool QL = NR == 1;                          // q's fragments in LDS: the waves share their rows
  constexpr int PL = TYPE == KV_F32 ? 2 : 1;            // f16 planes of a tile (hi, lo)
  constexpr bool SC = TYPE != KV_F16;                   // a factor for each key
  constexpr int KP = RowsLds<TYPE, HD, NR>::KP, VP = RowsLds<TYPE, HD, NR>::VP;
  constexpr int CD = 8 * GL, NC = HD / CD, ND = HD / MR;  // dim chunks of S, dim tiles of O
  constexpr int NQ = MR / (4 * GL);                     // runs of 4 dims that a lane has of an O tile: MR d + KS q + 4 h
  using Acc = std::conditional_t<MR == 32, f16_t, f4_t>;
  constexpr int PE = TYPE == KV_Q8 ? 16 : 8;            // dims of a staged piece
  constexpr int PR = HD / PE;                           // pieces of a key's row
  constexpr int PIECES = TK * PR / NT;
  constexpr int PW = TYPE == KV_F32 ? 2 : 1;            // 16-byte words of a piece
  using Lds = RowsLds<TYPE, HD, NR>;
  using Tile = typename Lds::Tile;
  using Marks = typename Lds::Marks;
  using Merge = typename Lds::Merge;
  constexpr int NB = Lds::NB;
  auto& lds = mem.tiles;
  auto& marks = mem.marks;
  auto& qs = mem.qs;
  auto& qtop = mem.qtop;
  auto& rng = mem.rng;

  const SeqAttnArgs& a = r.a;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rw = wave % NR, kg = wave / NR, tid = threadIdx.x - NT * kg;
  const int lane = threadIdx.x & 63, col = lane % MR, h = lane / MR;
  Tile* tiles = reinterpret_cast<Tile*>(lds) + NB * kg;
  const int kvh = (int)(block % (unsigned)a.n_kv);
  const int sx = (int)(block / (unsigned)a.n_kv);
  const int split = sx % r.splits;
  const uint32_t R = (uint32_t)r.R, nx = (R + MR * NR - 1) / (MR * NR);
  const uint32_t row_at = (nx - 1 - (uint32_t)(sx / r.splits)) * (MR * NR) + MR * rw + col;  // the longest first
  const bool valid = row_at < R;
  const uint32_t row = valid ? row_at : R - 1;
  const int query = (int)(row / (uint32_t)r.G), head = kvh * r.G + (int)(row - (uint32_t)query * r.G);

  // q, before anything that the way to the first tile waits for
  constexpr int LC = QL ? NC / NK : NC;  // chunks that the wave loads: all, or its share where LDS holds q
  auto chunk = [&](int i) { return QL ? i * NK + kg : i; };
  f4_t qv[LC][2];
#pragma unroll
  for (int i = 0; i < LC; ++i) {
    const float* at = a.q + (int64_t)query * a.ldq + (int64_t)head * a.hd + min(CD * chunk(i) + 8 * h, a.hd - 8);
    qv[i][0] = *reinterpret_cast<const f4u_t*>(at), qv[i][1] = *reinterpret_cast<const f4u_t*>(at + 4);
  }

  // positions [lo, hi) of the keys that the row sees, and its own
  int pos, lo = 0, hi;
  if (PREFIX) {
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
  int wlo = 0, wlo_max = 0, whi_min = a.n_prefix, whi = a.n_prefix;  // over the wave's rows
  int blo = 0, bhi = a.n_prefix, blo_max = 0, bhi_min = a.n_prefix;  // and the block's
  if (!PREFIX || a.window) {
    wlo = wave_min_i(lo), wlo_max = wave_max_i(lo), whi_min = wave_min_i(hi), whi = wave_max_i(hi);
    blo = wlo, bhi = whi, blo_max = wlo_max, bhi_min = whi_min;
    if constexpr (NR > 1) {
      if (lane == 0 && kg == 0) rng[rw][0] = wlo, rng[rw][1] = wlo_max, rng[rw][2] = whi_min, rng[rw][3] = whi;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NR; ++w) {
        blo = min(blo, __builtin_amdgcn_readfirstlane(rng[w][0])), blo_max = max(blo_max, __builtin_amdgcn_readfirstlane(rng[w][1]));
        bhi_min = min(bhi_min, __builtin_amdgcn_readfirstlane(rng[w][2])), bhi = max(bhi, __builtin_amdgcn_readfirstlane(rng[w][3]));
      }
    }
  }
  if (blo >= bhi) blo = bhi = 0;  // no row sees a key: no tiles, and none behind the end of int for a later group
  // this split's tiles
  const int n_tiles = (bhi - blo + TK - 1) / TK;
  const int tile0 = (int)((int64_t)n_tiles * split / r.splits), tile1 = (int)((int64_t)n_tiles * (split + 1) / r.splits);
  const int k0 = blo + tile0 * TK, k1 = min(bhi, blo + tile1 * TK);

  const int64_t seq = PREFIX ? a.pre_seq : a.max_seq;
  const uint8_t* kbase = PREFIX ? a.kp : a.kc;
  const uint8_t* vbase = PREFIX ? a.vp : a.vc;
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
  const uint32_t row_bytes = (uint32_t)a.hd * ES;
  // (`slot` hides tid from the loop: its few additions again each turn, not their results in
  // registers that the products need)
  auto load_tile = [&](int t) __attribute__((always_inline)) {
    uint32_t slot = tid;
    asm volatile("" : "+v"(slot));
    const gptr_t kt = uniform_at(kbase, (int64_t)t * row_bytes);
    const gptr_t vt = uniform_at(vbase, (int64_t)t * row_bytes);
    const int last = __builtin_amdgcn_readfirstlane(k1 - 1 - t);
#pragma unroll
    for (int u = 0; u < PIECES; ++u) {
      const uint32_t c = slot + NT * u;
      const uint32_t off = min(c / PR, (uint32_t)last) * row_bytes + min(c % PR * PE, (uint32_t)(a.hd - PE)) * ES;
#pragma unroll
      for (int w = 0; w < PW; ++w) {
        kreg[u][w] = load_at<u4_t>(kt, off + 16 * w);
        vreg[u][w] = load_at<u4_t>(vt, off + 16 * w);
      }
    }
    if constexpr (TYPE == KV_Q8) {
      if (slot < 2 * TK) screg = (slot < TK ? kscale : vscale)[t + (int)min(slot % TK, (uint32_t)last)];
    }
  };
  const int mine = k0 + kg * TK;  // the group's first tile

  auto row_max = [](float v) __attribute__((always_inline)) {  // over a row's lanes
    if constexpr (MR == 16) v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
  };
  // q * scale * 2^e as f16 hi + lo: the lane has dims CD c + 8 h .. + 7 of its row
  h8_t qhi[QL ? 1 : NC], qlo[QL ? 1 : NC];
  float unit;  // of a raw product
  {
    float top = 0.0f;
    // behind q, so that nothing waits for the tile with it
    if (mine < k1) load_tile(mine);
#pragma unroll
    for (int i = 0; i < LC; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float x = CD * chunk(i) + 8 * h < a.hd ? qv[i][k / 4][k % 4] * a.scale : 0.0f;
        qv[i][k / 4][k % 4] = x;
        top = fmaxf(top, fabsf(x));
      }
    top = row_max(top);
    if constexpr (QL) {
      qtop[kg][col] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NK; ++w) top = fmaxf(top, qtop[w][col]);
    }
    const int e = row_exponent(top);
    const float up = pow2i(e);
    unit = pow2i(-e) * (TYPE == KV_Q8 ? kQ8Unit : 1.0f);
#pragma unroll
    for (int i = 0; i < LC; ++i) {
      h8_t hi8, lo8;
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        h2_t x, y;
        split2(qv[i][k / 4][k % 4] * up, qv[i][k / 4][k % 4 + 1] * up, x, y);
        hi8[k] = x.x, hi8[k + 1] = x.y, lo8[k] = y.x, lo8[k + 1] = y.y;
      }
      if constexpr (QL) qs[64 * chunk(i) + lane] = hi8, qs[64 * (NC + chunk(i)) + lane] = lo8;
      else qhi[i] = hi8, qlo[i] = lo8;
    }
    if constexpr (QL) __syncthreads();
  }
  const bool capped = a.cap > 0.0f, sloped = a.slopes != nullptr;
  const float to_cap = capped ? fminf(unit / a.cap, 0x1p127f) : 0.0f;  // finite: a score of 0 stays 0
  const float mul = (capped ? a.cap : unit) * kLog2e;  // scores in base 2
  const float slope = sloped ? a.slopes[head] * kLog2e : 0.0f;

  // The lane's row: probabilities are 2^(y - m + 10) / D. m follows the maximum in steps (a
  // score may pass it by 2^4), D is a power of two over the values' factors so far.
  Acc o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = Acc{};
  float m = -INFINITY, l = 0.0f, D = SC ? 0x1p-60f : 1.0f, lgD = SC ? -60.0f : 0.0f;

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
      top = fmaxf(top, dpp_mov<0xB1>(top));   // quad_perm [1,0,3,2]
      top = fmaxf(top, dpp_mov<0x4E>(top));   // quad_perm [2,3,0,1]
      top = fmaxf(top, dpp_mov<0x141>(top));  // row_half_mirror
      if constexpr (PR >= 16) top = fmaxf(top, dpp_mov<0x140>(top));  // row_mirror
      if constexpr (PR >= 32) top = fmaxf(top, __shfl_xor(top, 16, 64));
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
  // Where some row does not see some key, a probability of 0 must not meet a value that is not
  // finite: such values (KV_Q8: factors) are stored as 0 and marked.
  auto partly = [&](int t) __attribute__((always_inline)) { return t < blo_max || t + TK > bhi_min; };
  auto mark = [&](Marks& to) __attribute__((always_inline)) {
    if constexpr (TYPE == KV_Q8) {
      constexpr int VWAVE = TK == 64 ? 1 : 0;  // the wave that holds the values' factors
      if (rw == VWAVE) {
        const bool factor = tid >= TK, out = factor && !(fabsf(screg) < INFINITY);
        const bool any = __any(out);
        if (factor) to.at[tid - TK][0] = out;
        screg = out ? 0.0f : screg;
        if (lane == 0) to.any[0] = any;
      }
    } else {
      uint32_t top = 0;
#pragma unroll
      for (int u = 0; u < PIECES; ++u)
#pragma unroll
        for (int w = 0; w < 4 * PW; ++w) {
          const uint32_t x = vreg[u][w / 4][w % 4];
          top = TYPE == KV_F16 ? max(top, max(x & 0x7fffu, x >> 16 & 0x7fffu)) : max(top, (x & 0x7fffffffu) >> 16);
        }
      const bool any = __any(top >= (TYPE == KV_F16 ? 0x7c00u : 0x7f80u));
      if (any) {
#pragma unroll
        for (int u = 0; u < PIECES; ++u) {
          const uint32_t c = tid + NT * u;
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
          to.at[c / PR][c % PR] = (uint8_t)bits;
        }
      }
      if (lane == 0) to.any[rw] = any;
    }
  };
  auto store_tile = [&](Tile& to) __attribute__((always_inline)) {
    uint32_t slot = tid;
    asm volatile("" : "+v"(slot));
#pragma unroll
    for (int u = 0; u < PIECES; ++u) {
      const uint32_t c = slot + NT * u, key = c / PR, d = c % PR * PE;
      _Float16 *kt = &to.k[0][key * KP + d], *vt = &to.v[0][key * VP + d];
      if constexpr (TYPE == KV_F16) {
        *reinterpret_cast<u4_t*>(kt) = kreg[u][0];
        *reinterpret_cast<u4_t*>(vt) = vreg[u][0];
      } else if constexpr (TYPE == KV_Q8) {
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const u4_t x = kv ? vreg[u][0] : kreg[u][0];
          h8_t y[2];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const h2_t p = q8_pair(__builtin_amdgcn_perm(0, x[w], 0x0c010c00)), q = q8_pair(__builtin_amdgcn_perm(0, x[w], 0x0c030c02));
            h8_t& z = y[w / 2];
            z[4 * (w % 2)] = p.x, z[4 * (w % 2) + 1] = p.y, z[4 * (w % 2) + 2] = q.x, z[4 * (w % 2) + 3] = q.y;
          }
          h8_t* at = reinterpret_cast<h8_t*>(kv ? vt : kt);
          at[0] = y[0], at[1] = y[1];
        }
      } else {
        store_f32(kreg[u], kt, &to.k[PL - 1][key * KP + d], d == 0 ? &to.kf[key] : nullptr);
        store_f32(vreg[u], vt, &to.v[PL - 1][key * VP + d], d == 0 ? &to.vf[key] : nullptr);
      }
    }
    if constexpr (TYPE == KV_Q8) {
      if (slot < 2 * TK) *(slot < TK ? &to.kf[slot] : &to.vf[slot - TK]) = screg;
    }
  };

  // S^T = K . Q^T of 32 keys
  // (`loads`: global loads beside them, of the next tile)
  auto products = [&](const Tile& x, int sub, float (&s)[NE], auto loads) __attribute__((always_inline)) {
    constexpr int KT = 32 / MR;  // key tiles
    Acc acc[KT];
#pragma unroll
    for (int i = 0; i < KT; ++i) acc[i] = Acc{};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      h8_t q0, q1;
      if constexpr (QL) q0 = qs[64 * c + lane], q1 = qs[64 * (NC + c) + lane];
      else q0 = qhi[c], q1 = qlo[c];
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        const int at = (32 * sub + MR * i + col) * KP + CD * c + 8 * h;
        const h8_t kf = *reinterpret_cast<const h8_t*>(&x.k[0][at]);
        acc[i] = mfma(kf, q0, acc[i]);
        acc[i] = mfma(kf, q1, acc[i]);
        if constexpr (PL == 2) acc[i] = mfma(*reinterpret_cast<const h8_t*>(&x.k[1][at]), q0, acc[i]);
      }
    }
    // The order: fragments are read AHEAD steps before their matrix ops, and the loads stand
    // between the ops, where the wave would only wait (issued together they hold it up: a load
    // of 64 x 16 bytes takes the CU's vector memory path 16 cycles, and four waves share it).
    constexpr int OPS = PL == 2 ? 3 : 2, READS = PL, Q = QL ? 2 : 0, STEPS = NC * KT, AHEAD = STEPS > 4 ? 3 : 1;
    constexpr int LOADS = (decltype(loads)::value + STEPS - 1) / STEPS;
    __builtin_amdgcn_sched_group_barrier(0x100, (READS + Q) * AHEAD, 0);
#pragma unroll
    for (int i = 0; i < STEPS - AHEAD; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x8, OPS, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, READS + Q, 0);
      if constexpr (LOADS > 0) __builtin_amdgcn_sched_group_barrier(0x20, LOADS, 0);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x8, OPS, 0);
      if constexpr (LOADS > 0) __builtin_amdgcn_sched_group_barrier(0x20, LOADS, 0);
    }
#pragma unroll
    for (int i = 0; i < NE; ++i) s[i] = acc[i / (NE / KT)][i % (NE / KT)];
  };
  // the factors of a lane's keys
  auto times = [&](float (&s)[NE], const float* f) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < NE / 4; ++q) {
      const f4_t x = *reinterpret_cast<const f4_t*>(f + KS * q + 4 * h);
#pragma unroll
      for (int k = 0; k < 4; ++k) s[4 * q + k] *= x[k];
    }
  };
  // One tile, and beside it, where there is a `next` one, that one's way to its place (`to`, `note`).
  auto compute = [&](auto more, int t, const Tile& x, const Marks& known, bool marked, int next, Tile& to, Marks& note) __attribute__((always_inline)) {
    constexpr bool NEXT = decltype(more)::value;
#pragma unroll
    for (int sub = 0; sub < SUBS; ++sub) {
      const int kt = t + 32 * sub, key0 = kt + 4 * h;
      float s[NE];
      if constexpr (NEXT) {
        if (sub == 0) load_tile(next);
      }
      if (NEXT && sub == 0) {
        products(x, sub, s, std::integral_constant<int, 2 * PIECES * PW + (TYPE == KV_Q8)>{});
      } else {
        products(x, sub, s, std::integral_constant<int, 0>{});
      }
      if constexpr (SC) times(s, x.kf + 32 * sub);
      float y_of = mul;  // times s: the score
      if (capped) {
        float far = 0.0f;
#pragma unroll
        for (int i = 0; i < NE; ++i) {
          s[i] *= to_cap;
          far = fmaxf(far, fabsf(s[i]));
        }
        if (__any(!(far < kTanhNear))) {
#pragma unroll
          for (int i = 0; i < NE; ++i) {
            const float near = tanh_near(s[i]), out = tanh_far(s[i]);
            s[i] = fabsf(s[i]) < kTanhNear ? near : out;
          }
        } else {
#pragma unroll
          for (int i = 0; i < NE; ++i) s[i] = tanh_near(s[i]);
        }
      }
      if (sloped) {
        const float away = (float)(pos - key0);
#pragma unroll
        for (int i = 0; i < NE; ++i) s[i] = fmaf(-slope, fabsf(away - (float)(KS * (i / 4) + i % 4)), s[i] * mul);
        y_of = 1.0f;
      }
      uint32_t seen = (1u << NE) - 1;
      if (kt < wlo_max || kt + 32 > whi_min) {  // some row of the wave does not see some key
        seen = 0;
        const int l0 = lo - key0, h0 = hi - key0;
#pragma unroll
        for (int i = 0; i < NE; ++i) {
          const int k = KS * (i / 4) + i % 4;
          const bool in = k >= l0 && k < h0;
          s[i] = in ? s[i] : -INFINITY;
          seen |= (in ? 1u : 0u) << i;
        }
      }
      float top = s[0];
#pragma unroll
      for (int i = 1; i < NE; ++i) top = fmaxf(top, s[i]);
      top *= y_of;
      if (__any(top > m + 4.0f)) {
        top = row_max(top);
        const float mnew = fmaxf(m, top);
        const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mnew);
        m = mnew;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] *= alpha;
      }
      if constexpr (SC) {
        const float f = x.vf[32 * sub + (lane & 31)];
        if (__any(f > D && f < INFINITY)) {
          const float big = wave_max_dpp(f < INFINITY ? f : 0.0f);
          const int e = min(126, (int)((__float_as_uint(big) >> 23) & 0xff) - 126);  // the next power of two
          const float Dnew = pow2i(e), beta = D / Dnew;
          D = Dnew;
          lgD = (float)e;
          l *= beta;
#pragma unroll
          for (int d = 0; d < ND; ++d) o[d] *= beta;
        }
      }
      if constexpr (NEXT) {
        if (sub + 1 == SUBS && partly(next)) mark(note);
      }
      const float ref = (m == -INFINITY ? 0.0f : m) + lgD - 10.0f;
      f4_t sum = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], y_of, -ref));
        sum[i % 4] += s[i];
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      if constexpr (SC) times(s, x.vf + 32 * sub);
      // O^T += V^T . P^T: elements 8 c .. 8 c + 7 of P are the keys of a step (16, or 32 with
      // 16 rows), in the order in which V is read, transposed: the 16 lanes of a read take 4
      // keys x 32 bytes, which rows 8 words past a multiple of 64 keep in banks of their own
      auto v_at = [&](int plane, int c, int d) __attribute__((always_inline)) {
        const int key = 32 * sub + 16 * c + 4 * h + ((lane & 15) >> 2), dim = MR * d + 4 * (lane & 3) + (MR == 32 ? 16 * (lane >> 4 & 1) : 0);
        const _Float16* p = &x.v[plane][key * VP + dim];
        const h4_t y = lds_tr4(p), z = lds_tr4(p + KS * VP);
        return h8_t{y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w};
      };
#pragma unroll
      for (int c = 0; c < NE / 8; ++c) {
        h8_t phi, plo;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          h2_t y, z;
          split2(s[8 * c + e], s[8 * c + e + 1], y, z);
          phi[e] = y.x, phi[e + 1] = y.y, plo[e] = z.x, plo[e + 1] = z.y;
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const h8_t vf = v_at(0, c, d);
          o[d] = mfma(vf, phi, o[d]);
          o[d] = mfma(vf, plo, o[d]);
          if constexpr (PL == 2) o[d] = mfma(v_at(1, c, d), phi, o[d]);
        }
      }
      if constexpr (NEXT) {
        if (sub + 1 == SUBS) store_tile(to);
      }
      {
        constexpr int OPS = PL == 2 ? 3 : 2, READS = 2 * PL, STEPS = NE / 8 * ND, AHEAD = STEPS > 4 ? 3 : 2;
        constexpr int WRITES = (2 * PIECES * (TYPE == KV_F16 ? 1 : 2) + (TYPE == KV_Q8) + AHEAD - 1) / AHEAD;
        __builtin_amdgcn_sched_group_barrier(0x100, READS * AHEAD, 1);
#pragma unroll
        for (int i = 0; i < STEPS - AHEAD; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x8, OPS, 1);
          __builtin_amdgcn_sched_group_barrier(0x100, READS, 1);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x8, OPS, 1);
          if (NEXT && sub + 1 == SUBS) __builtin_amdgcn_sched_group_barrier(0x200, WRITES, 1);
        }
      }
      if (marked) {  // rows that see a value that is not finite
        for (int k = 0; k < 32; ++k) {
          // the key's bit is with the lanes of its group
          const uint32_t bits_of_group = (uint32_t)__shfl((int)seen, col + MR * (k / 4 % GL), 64);
          const bool in = bits_of_group >> (k / KS * 4 + k % 4) & 1;
          const uint8_t* bad = known.at[32 * sub + k];
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
              const int piece = (MR * d + KS * q + 4 * h) / 8, c = TYPE == KV_Q8 ? 0 : (32 * sub + k) * PR + piece;
              const uint32_t bits = TYPE == KV_Q8 ? bad[0] * 15u : known.any[c % NT / 64] ? bad[piece] >> (4 * (h & 1)) : 0u;
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (in && (bits >> e & 1)) o[d][4 * q + e] = __uint_as_float(0x7fc00000u);
            }
        }
      }
    }
  };

  const bool busy = __any(valid);
  const int rounds = (tile1 - tile0 + NK - 1) / NK;
  if (mine < k1) {
    if (partly(mine)) mark(marks[kg][0]);
    store_tile(tiles[0]);
  }
  if constexpr (NR > 1) lds_barrier();
  auto marked = [&](int t, const Marks& known) __attribute__((always_inline)) {
    bool any = false;
    if (partly(t)) {
#pragma unroll
      for (int w = 0; w < (TYPE == KV_Q8 ? 1 : NR); ++w) any |= __builtin_amdgcn_readfirstlane(known.any[w]) != 0;
    }
    return any;
  };
  // a tile that the wave's rows meet
  auto met = [&](int t) __attribute__((always_inline)) { return busy && t < whi && t + TK > wlo; };
  int t = mine;
  for (int i = 0; i + 1 < rounds; ++i) {  // a group that has no tile in the last round stages this one again
    const int next = t + NK * TK < k1 ? t + NK * TK : t;
    Tile& to = tiles[NB == 2 ? (i + 1) & 1 : 0];
    Marks& note = marks[kg][(i + 1) & 1];
    if (met(t)) {
      compute(std::true_type{}, t, tiles[NB == 2 ? i & 1 : 0], marks[kg][i & 1], marked(t, marks[kg][i & 1]), next, to, note);
    } else {
      load_tile(next);
      if (partly(next)) mark(note);
      store_tile(to);
    }
    t += NK * TK;
    if constexpr (NR > 1) lds_barrier();
  }
  if (rounds > 0 && t < k1 && met(t)) {
    const int i = rounds - 1;
    compute(std::false_type{}, t, tiles[NB == 2 ? i & 1 : 0], marks[kg][i & 1], marked(t, marks[kg][i & 1]), t, tiles[0], marks[kg][0]);
  }
  if constexpr (MR == 16) l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);

  if constexpr (NK > 1) {
    Merge& g = *reinterpret_cast<Merge*>(lds);
    __syncthreads();
    if (kg > 0) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int q = 0; q < NQ; ++q) g.o[kg - 1][rw][NQ * d + q][lane] = f4_t{o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]};
      g.ml[kg - 1][rw][0][lane] = m, g.ml[kg - 1][rw][1][lane] = l;
      if (lane == 0) g.D[kg - 1][rw] = D;
    }
    __syncthreads();
    if (kg > 0) return;
    float M = m, Dm = D;
#pragma unroll
    for (int k = 0; k < NK - 1; ++k) M = fmaxf(M, g.ml[k][rw][0][lane]), Dm = fmaxf(Dm, g.D[k][rw]);
    const float keep = weight_of(m, l, M) * (D / Dm);
    l *= keep;
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] *= keep;
#pragma unroll
    for (int k = 0; k < NK - 1; ++k) {
      const float lk = g.ml[k][rw][1][lane], f = weight_of(g.ml[k][rw][0][lane], lk, M) * (g.D[k][rw] / Dm);
      l += f * lk;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          const f4_t y = g.o[k][rw][NQ * d + q][lane];
#pragma unroll
          for (int e = 0; e < 4; ++e) o[d][4 * q + e] += f * y[e];
        }
    }
    m = M, D = Dm;
  }
  if (!valid) return;
  if (r.splits == 1 && !PREFIX) {
    const float inv = l == 0.0f ? 0.0f : (TYPE == KV_Q8 ? kQ8Unit : 1.0f) / l;
    float* out = a.out + (int64_t)query * a.ldo + (int64_t)head * a.hd;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        const int at = MR * d + KS * q + 4 * h;
        if (at < a.hd)
          *reinterpret_cast<f4u_t*>(out + at) = f4_t{o[d][4 * q] * inv, o[d][4 * q + 1] * inv, o[d][4 * q + 2] * inv, o[d][4 * q + 3] * inv};
      }
  } else {
    const float f = D * 0x1p-10f, fo = TYPE == KV_Q8 ? f * kQ8Unit : f;
    float* out = r.part + (((int64_t)split * a.n_kv + kvh) * r.R + row) * part_stride(a.hd);
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        const int at = MR * d + KS * q + 4 * h;
        if (at < a.hd)
          *reinterpret_cast<f4_t*>(out + at) = f4_t{o[d][4 * q] * fo, o[d][4 * q + 1] * fo, o[d][4 * q + 2] * fo, o[d][4 * q + 3] * fo};
      }
    if (h == 0) out[a.hd] = m, out[a.hd + 1] = l * f;
  }
}

}  // namespace
}  // namespace uaii_hip
