// rows_attn.hip — attention of a prompt's rows over one cache: the kernel, and the shape of a
// launch.
#include "rows_block.h"

#include <algorithm>

namespace uaii_hip {
namespace {

template <int TYPE, int HD, int NR>
__global__ void __launch_bounds__(256, 2) k_rows_attn(RowsAttnArgs r) {
  __shared__ RowsLds<TYPE, HD, NR> lds;
  rows_block<TYPE, HD, NR, false>(r, blockIdx.x, lds);
}

// Whether a CU holds one block, not two, by its LDS.
bool one_held(const RowsAttnArgs& r, int nr) {
  const bool f32 = r.a.type == KV_F32;
  return r.a.hd > 128 ? nr < 4 || f32 : r.a.hd > 64 ? nr == 1 || (f32 && nr == 2) : f32 && nr == 1;
}

int64_t row_blocks(const RowsAttnArgs& r, int nr) {
  const int rows = row_tile(r.a.hd) * nr;
  return (r.R + rows - 1) / rows * r.a.n_kv;
}

template <int TYPE, int HD, int NR>
hipError_t go(const RowsAttnArgs& r, hipStream_t s) {
  const int64_t blocks = row_blocks(r, NR) * r.splits;
  if (blocks > INT32_MAX) return hipErrorInvalidValue;
  UAII_LAUNCH((k_rows_attn<TYPE, HD, NR>), dim3((unsigned)blocks), dim3(256), 0, s, r);
  return hipGetLastError();
}

template <int TYPE, int HD>
hipError_t by_waves(const RowsAttnArgs& r, hipStream_t s) {
  const int nr = r.nr;
  if constexpr (rows_least(TYPE, HD) <= 1) {
    if (nr == 1) return go<TYPE, HD, 1>(r, s);
  }
  if constexpr (rows_least(TYPE, HD) <= 2) {
    if (nr == 2) return go<TYPE, HD, 2>(r, s);
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

// Row waves and key splits by an estimate of the launch's time, in cycles of a wave. Measured
// on f16 caches of head_dim 128: a block's way to its first tile and from its last one 10 k; a
// turn (32 keys) 3.5 k where each wave stages its own tiles, 2.8 k where two share one, 2.4 k
// where four do (1.6 times the first two with rows of 256); 1.35 times that with two blocks
// on a CU. A split writes its rows' sums and the join reads them, 12 bytes a cycle and CU,
// and takes its 50 of the join's way. (4012 rows of 8 heads over a window of 1500, KV_Q8:
// two row waves 73 us, four and two splits 88; 10400 rows of one head of 256 over 1300: four
// row waves and three splits 41 us, two row waves 70; 24 rows of one such head over 30000:
// 128 splits 17, 64 21; 1024 rows of 8 f32 heads of 128 over 1256: four row waves and eight
// splits 46, two and two 60.)
//
// Over a prefix there is one block a CU, and only one that leaves another the room for a
// block of the sequences' own keys: with blocks of one row wave, which take all of a CU
// (f16, 32/8 heads of 128), 20 sequences and a prefix of 2500 took 29 us, with others 24;
// with two blocks of rows a CU 48 sequences and a prefix of 6000 took 43 us, with one 30.
void rows_attn_shape(RowsAttnArgs* r) {
  const SeqAttnArgs& a = r->a;
  int64_t most = a.n_prefix, mean = most;  // keys of a row
  if (!r->prefix) {
    most = std::max<int64_t>((int64_t)a.p0 + a.rows, a.bidir);
    mean = std::max<int64_t>(a.p0 + (a.rows + 1) / 2, a.bidir);
    if (a.window) most = std::min<int64_t>(most, (int64_t)a.window + row_tile(a.hd) * 4 / r->G), mean = std::min(mean, most);
  }
  const int least = rows_least(a.type, a.hd);
  const double row_bytes = (double)r->R * a.n_kv * part_stride(a.hd) * 8 / device_cus();
  double best = 0;
  for (int nr = 4; nr >= least; nr /= 2) {
    const int nk = 4 / nr;
    const bool one = one_held(*r, nr);
    if (r->prefix && one && nr < 4) break;
    const int64_t blocks = row_blocks(*r, nr), full = (int64_t)device_cus() * (one || r->prefix ? 1 : 2);
    const double turn = (nr == 4 ? 2400 : nr == 2 ? 2800 : 3500) * (a.hd > 128 && nr < 4 ? 1.6 : a.hd > 64 ? 1.0 : 0.65) * (a.type == KV_F32 ? 1.5 : 1.0);
    for (int64_t splits : {(int64_t)1, full / 2 / blocks, full / blocks}) {
      splits = std::min<int64_t>({splits, 128, (most + 127) / 128});
      if (splits < 1) continue;
      const int64_t all = blocks * splits, waits = (all + full - 1) / full;
      const double turns = std::max(1.0, (waits > 1 ? mean : most) / 32.0 / nk / splits);
      const double shared = full > device_cus() && all > device_cus() ? 1.35 : 1.0;
      double cost = (waits > 1 ? (double)all / full + 0.3 : 1.0) * (10e3 + turns * turn * shared);
      if (splits > 1 || r->prefix) cost += splits * (row_bytes / 12 + 50) + 4e3;
      if (best == 0 || cost < best) best = cost, r->nr = nr, r->splits = (int)splits;
    }
  }
}

int64_t rows_attn_blocks(const RowsAttnArgs& r) { return row_blocks(r, r.nr) * r.splits; }

hipError_t launch_rows_attn(const RowsAttnArgs& r, hipStream_t s) {
  if (r.R <= 0 || r.splits < 1 || (r.nr != 1 && r.nr != 2 && r.nr != 4) || r.a.hd % 16 || r.a.hd < 16 || r.a.hd > 256 || r.prefix || (r.splits > 1 && !r.part))
    return hipErrorInvalidValue;
  switch (r.a.type) {
    case KV_F32: return by_width<KV_F32>(r, s);
    case KV_F16: return by_width<KV_F16>(r, s);
    case KV_Q8: return by_width<KV_Q8>(r, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace uaii_hip
