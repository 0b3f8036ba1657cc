// batch_attn.hip — attention of one query for each sequence of a batch over a prefix that all
// share and the sequence's own keys, and the join of partial results.
//
// Lengths are on the device, so the host cannot cut the work to them. Each (sequence, kv
// head) is cut into units of 128 keys and the units of the whole batch, in order, are
// dealt out evenly to a grid that just fills the device: a block works through the runs of
// units that fall to it, writes a finished head's rows to the output at once, and leaves
// the partial results of its first and last run, where a head goes on in another block,
// to the join. A short capacity takes a block for each head, and a batch of few units in all
// one for each unit that its capacity allows: no block has to look for its share (7 sequences of up to 3000 KV_Q8 keys, 8/4 heads of
// 192: 14 us, with shares of 64 keys 20; but with four blocks for each that the device holds,
// 48 sequences of up to 400 keys and their prefix took 52 where shares took 45).
//
// A prefix that is not short is read once for all queries, by blocks of rows beside the
// others in the same launch.
#include "batch_block.h"
#include "rows_block.h"

#include <algorithm>
#include <atomic>

namespace uaii_hip {
namespace {

template <int TYPE, int HD, bool PACK>
__global__ void __launch_bounds__(256, HD == 256 && (TYPE == KV_F32 || !PACK) ? 1 : 2) k_batch_attn(BatchArgs b) {
  __shared__ BatchLds<TYPE, HD, PACK> lds;
  batch_block(b, blockIdx.x, lds);
}

// All queries over the prefix, and beside that the sequences' own keys: the one is bound by
// the matrix cores, the other by memory. (48 users, f16, 32/8 heads of 128, a prefix of 6000
// and up to 400 keys each: 26 us, as two launches 24 and 17; KV_Q8, 5 answers over 30011
// keys, 20/4 heads of 64: 12.6 us, 13.5 and 6.4.)
template <int TYPE, int HD, int NR>
__global__ void __launch_bounds__(256, HD == 256 && TYPE == KV_F32 ? 1 : 2) k_prefix_attn(RowsAttnArgs r, BatchArgs b, unsigned row_blocks) {
  __shared__ union {
    RowsLds<TYPE, HD, NR> rows;
    BatchLds<TYPE, HD, TYPE != KV_F32> own;
  } lds;
  if (blockIdx.x < row_blocks) rows_block<TYPE, HD, NR, true>(r, blockIdx.x, lds.rows);
  else batch_block(b, blockIdx.x - row_blocks, lds.own);
}

// Partial results of a row into its output: a block of W waves for each (row, query head),
// eight partials of a wave at a time: up to 8 in one wave, up to 32 in four, and sixteen waves
// for more, so that most joins are one round trip to memory: 4.7 us for 1024 rows of two or
// three partials, 5.5 for 100 rows of 65, of which 2 are the launch; 9.1 for 10400 rows of
// 256 with three (43 MB, 4700 GB/s).
struct JoinArgs {
  SeqAttnArgs a;
  int G, rc, groups, parts, fold;
  const float* slots;
  const float* whole;
  const int2* info;      // with parts 0
  bool batch;            // rows have own keys
  const float* part;     // [splits][n_kv][rows * G][part_stride]
  int splits;
};

template <int W>
__global__ void __launch_bounds__(64 * W) k_attn_join(JoinArgs j) {
  __shared__ float wm[W], wl[W];
  __shared__ __attribute__((aligned(16))) float wo[W][256];
  const SeqAttnArgs& a = j.a;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = (int)(blockIdx.x / (unsigned)a.n_heads), head = (int)(blockIdx.x % (unsigned)a.n_heads);
  const int kvh = head / j.G, gr = head % j.G, H = a.n_kv * j.groups;
  const int64_t stride = part_stride(a.hd);
  // the row's own partials: those of blocks b0 .. b1, or one in `whole`
  int own = 0;
  int64_t ahead = 0, step = 0;  // floats from the first to the second, and from there on
  const float* at = nullptr;
  if (j.batch) {
    const Span sp = span_of(a, j.fold, row);
    const int units = sp.units();
    if (units > 0) {
      const int hx = kvh * j.groups + gr / j.rc;
      if (j.parts > 0) {
        own = j.parts == 1 ? 1 : units;
        at = j.slots + ((int64_t)row * H + hx) * j.parts * j.rc * stride;
        ahead = step = j.rc * stride;
      } else {
        const int2 at_blocks = j.info[(int64_t)row * H + hx];
        own = at_blocks.y + 1;
        at = own == 1 ? j.whole + ((int64_t)row * H + hx) * j.rc * stride : j.slots + (2 * (int64_t)at_blocks.x + 1) * j.rc * stride;
        ahead = j.rc * stride, step = 2 * ahead;  // the last run of the first block, the first runs of those behind it
      }
      if (own == 1 && j.splits == 0) return;  // written
      at += gr % j.rc * stride;
    }
  }
  const int64_t R = a.rows * j.G;
  const float* pre = j.part + ((int64_t)kvh * R + (int64_t)row * j.G + gr) * stride;
  auto part_of = [&](int i) -> const float* {
    if (i >= own) return pre + (int64_t)(i - own) * a.n_kv * R * stride;
    return i == 0 ? at : at + ahead + (i - 1) * step;
  };
  const int n = own + j.splits, d = min(4 * lane, a.hd - 4);
  float m = -INFINITY, l = 0.0f;
  f4_t o = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
  constexpr int U = 8;
  for (int i0 = wave; i0 < n; i0 += U * W) {
    float mi[U], li[U];
    f4_t oi[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const float* p = part_of(min(i0 + k * W, n - 1));
      mi[k] = p[a.hd], li[k] = p[a.hd + 1];
      oi[k] = *reinterpret_cast<const f4_t*>(p + d);
    }
    float M = m;
#pragma unroll
    for (int k = 0; k < U; ++k) M = i0 + k * W < n ? fmaxf(M, mi[k]) : M;
    const float keep = weight_of(m, l, M);
    l *= keep;
    o *= keep;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (i0 + k * W >= n) continue;
      const float f = weight_of(mi[k], li[k], M);
      l += f * li[k];
      o += f * oi[k];
    }
    m = M;
  }
  if (lane == 0) wm[wave] = m, wl[wave] = l;
  *reinterpret_cast<f4_t*>(&wo[wave][4 * lane]) = o;
  __syncthreads();
  if (wave != 0 || 4 * lane >= a.hd) return;
  float M = -INFINITY, den = 0.0f;
#pragma unroll
  for (int w = 0; w < W; ++w) M = fmaxf(M, wm[w]);
  f4_t acc = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const float f = weight_of(wm[w], wl[w], M);
    den += f * wl[w];
    acc += f * *reinterpret_cast<const f4_t*>(&wo[w][4 * lane]);
  }
  const float inv = den == 0.0f ? 0.0f : 1.0f / den;
  *reinterpret_cast<f4u_t*>(a.out + (int64_t)row * a.ldo + (int64_t)head * a.hd + 4 * lane) = acc * inv;
}

// Calls f with the kernel of the call's type, width and row packing.
template <typename F>
auto with_kernel(int type, int hd, bool pack, F f) {
  const int w = hd <= 64 ? 0 : hd <= 128 ? 1 : 2;
  if (type == KV_F32) return w == 0 ? f(&k_batch_attn<KV_F32, 64, false>) : w == 1 ? f(&k_batch_attn<KV_F32, 128, false>) : f(&k_batch_attn<KV_F32, 256, false>);
  if (type == KV_F16) {
    if (pack) return w == 0 ? f(&k_batch_attn<KV_F16, 64, true>) : w == 1 ? f(&k_batch_attn<KV_F16, 128, true>) : f(&k_batch_attn<KV_F16, 256, true>);
    return w == 0 ? f(&k_batch_attn<KV_F16, 64, false>) : w == 1 ? f(&k_batch_attn<KV_F16, 128, false>) : f(&k_batch_attn<KV_F16, 256, false>);
  }
  if (pack) return w == 0 ? f(&k_batch_attn<KV_Q8, 64, true>) : w == 1 ? f(&k_batch_attn<KV_Q8, 128, true>) : f(&k_batch_attn<KV_Q8, 256, true>);
  return w == 0 ? f(&k_batch_attn<KV_Q8, 64, false>) : w == 1 ? f(&k_batch_attn<KV_Q8, 128, false>) : f(&k_batch_attn<KV_Q8, 256, false>);
}

// And of its type, width and row waves.
template <int TYPE, int HD, typename F>
auto with_waves(int nr, F f) {
  if constexpr (rows_least(TYPE, HD) <= 1) {
    if (nr == 1) return f(&k_prefix_attn<TYPE, HD, 1>);
  }
  if constexpr (rows_least(TYPE, HD) <= 2) {
    if (nr == 2) return f(&k_prefix_attn<TYPE, HD, 2>);
  }
  return f(&k_prefix_attn<TYPE, HD, 4>);
}
template <typename F>
auto with_prefix_kernel(int type, int hd, int nr, F f) {
  const int w = hd <= 64 ? 0 : hd <= 128 ? 1 : 2;
  if (type == KV_F32) return w == 0 ? with_waves<KV_F32, 64>(nr, f) : w == 1 ? with_waves<KV_F32, 128>(nr, f) : with_waves<KV_F32, 256>(nr, f);
  if (type == KV_F16) return w == 0 ? with_waves<KV_F16, 64>(nr, f) : w == 1 ? with_waves<KV_F16, 128>(nr, f) : with_waves<KV_F16, 256>(nr, f);
  return w == 0 ? with_waves<KV_Q8, 64>(nr, f) : w == 1 ? with_waves<KV_Q8, 128>(nr, f) : with_waves<KV_Q8, 256>(nr, f);
}

// Blocks of such a kernel that the device holds at once (asked once for each); nr 0: without a prefix.
int resident_blocks(int type, int hd, bool pack, int nr) {
  static std::atomic<int> known[3][3][5];
  std::atomic<int>& k = known[type][hd <= 64 ? 0 : hd <= 128 ? 1 : 2][nr == 0 ? pack : nr == 4 ? 4 : 1 + nr];
  int n = k.load(std::memory_order_relaxed);
  if (n == 0) {
    auto held = [](auto kernel) {
      int per_cu = 0;
      if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, kernel, 256, 0) != hipSuccess || per_cu < 1) {
        (void)hipGetLastError();
        per_cu = 1;
      }
      return per_cu;
    };
    n = (nr == 0 ? with_kernel(type, hd, pack, held) : with_prefix_kernel(type, hd, nr, held)) * device_cus();
    k.store(n, std::memory_order_relaxed);
  }
  return n;
}

struct Plan {
  int G, groups, rc, blocks, parts, splits, fold;
  int64_t row_blocks;  // over the prefix
  bool pack, too_many;  // too_many: units, for 32-bit numbers
  RowsAttnArgs rows;
  size_t part, slots, whole, info;  // bytes of the scratch's parts
  size_t bytes() const { return part + slots + whole + info; }
};

size_t pad256(size_t n) { return (n + 255) / 256 * 256; }

Plan plan_of(const SeqAttnArgs& a) {
  Plan p{};
  p.G = a.n_heads / a.n_kv;
  const size_t row = (size_t)part_stride(a.hd) * 4;
  p.rows.a = a;
  p.rows.G = p.G;
  p.rows.R = a.rows * p.G;
  if (!a.n_keys) {
    rows_attn_shape(&p.rows);
    p.splits = p.rows.splits > 1 ? p.rows.splits : 0;
  } else {
    const bool narrow = a.type != KV_F32 && p.G <= 8;
    auto units_of = [&](bool pack, int fold) {  // the most there can be, and what goes with them
      p.pack = pack;
      p.rc = rows_of(pack);
      p.groups = (p.G + p.rc - 1) / p.rc;
      const int64_t seen = a.window ? std::min<int64_t>(a.window, a.max_seq + fold) : a.max_seq + fold;
      return a.rows * a.n_kv * p.groups * ((seen + (fold ? 31 : 0) + UNIT - 1) / UNIT);
    };
    // Short capacities take one block a head and no join: up to four units, or eight where the
    // heads alone are blocks for half of the CUs and rows are not wide. (us, one block a head
    // and a block a unit, all of the capacity used; KV_Q8, 8 heads of 64, one sequence: 256
    // keys 6.3, 9.2, 512 keys 7.7, 9.3; with 40 keys in it 5.5, 7.6. f16, 8 heads of 128, one
    // sequence of 768 11.2, 10.1; 16 sequences of 512 10.2, 13.4, of 1024 15.7, 22.9, of 2048
    // 25.4, 27.0 (KV_Q8 16.7, 14.7); 12 windows of 1024, 8 heads of 256 39.8, 33.2.)
    auto one_block = [&](int64_t units) {
      const int64_t heads = a.rows * a.n_kv * p.groups;
      return units <= (a.hd <= 128 && heads >= device_cus() / 2 ? 8 : 4) * heads;
    };
    // Each sequence reads the prefix with its own keys where that is at most half a unit more;
    // where one block a head still does, if the blocks do not read it too often; and where
    // every unit still has a block of its own, all on the device at once. Else one read serves
    // all. (us, read by each and by all, 50 keys each; f16, 8 heads of 128: 4 sequences, prefix
    // of 60 6.1, 10.4, of 500 10.3, 12.0; 32, of 120 7.1, 13.1, of 500 10.3, 14.2; 100, of 60
    // 13.4, 18.1, of 250 23.8, 24.1, of 500 31.4, 26.2; 8 with 100, of 6000 25.0, 17.6. KV_Q8, 4
    // heads of 64: 4, of 500 11.0, 9.7; 32, of 250 8.0, 10.0; 8 with 200, of 1000 11.6, 11.5.)
    int64_t resident = resident_blocks(a.type, a.hd, narrow, 0);
    const int64_t folded = units_of(narrow, a.n_prefix);
    if (a.n_prefix <= UNIT / 2 || (one_block(folded) && a.rows * a.n_kv * p.groups * a.n_prefix <= 192 << 10) || folded <= resident) p.fold = a.n_prefix;
    const bool shared = a.n_prefix > p.fold;
    const int64_t units = units_of(narrow || (shared && a.type != KV_F32), p.fold);  // the kernel with a prefix has packed rows only
    if (shared) {
      p.rows.prefix = true;
      rows_attn_shape(&p.rows);
      p.splits = p.rows.splits;
      p.row_blocks = rows_attn_blocks(p.rows);
      resident = std::max<int64_t>(device_cus(), resident_blocks(a.type, a.hd, p.pack, p.rows.nr) - p.row_blocks);
    }
    const int64_t heads = a.rows * a.n_kv * p.groups;
    p.too_many = units > INT32_MAX;
    if (one_block(units) && !p.too_many) p.parts = 1;
    else if (units <= 2 * resident) p.parts = (int)(units / heads);
    p.blocks = (int)(p.parts ? heads * p.parts : std::min(units, resident));
    if (p.parts != 1 || shared) p.slots = pad256((p.parts ? 1 : 2) * (size_t)p.blocks * p.rc * row);
    p.info = p.parts ? 0 : pad256((size_t)heads * sizeof(int2));
    if (shared) p.whole = p.parts ? 0 : pad256((size_t)heads * p.rc * row);
  }
  p.part = pad256((size_t)p.splits * a.n_kv * p.rows.R * row);
  return p;
}

}  // namespace

size_t seq_attn_scratch(const SeqAttnArgs& a) { return plan_of(a).bytes(); }

hipError_t launch_seq_attn(const SeqAttnArgs& a, char* scratch, hipStream_t s) {
  Plan p = plan_of(a);
  if (a.rows <= 0 || p.too_many || (p.bytes() > 0 && !scratch)) return hipErrorInvalidValue;
  JoinArgs j{};
  j.a = a;
  j.G = p.G;
  j.groups = j.rc = 1;
  j.splits = p.splits;
  j.part = p.rows.part = reinterpret_cast<float*>(scratch);
  hipError_t e = hipSuccess;
  if (!a.n_keys) {
    e = launch_rows_attn(p.rows, s);
    if (e != hipSuccess || p.splits == 0) return e;
  }
  if (a.n_keys) {
    BatchArgs b{};
    b.a = a;
    b.G = p.G;
    b.groups = p.groups;
    b.slots = reinterpret_cast<float*>(scratch + p.part);
    b.whole = reinterpret_cast<float*>(scratch + p.part + p.slots);
    b.info = reinterpret_cast<int2*>(scratch + p.part + p.slots + p.whole);
    b.pre_splits = p.splits;
    b.blocks = p.blocks;
    b.parts = p.parts;
    b.fold = p.fold;
    if (p.row_blocks > 0) {
      const int64_t all = p.row_blocks + b.blocks;
      if (all > INT32_MAX) return hipErrorInvalidValue;
      e = with_prefix_kernel(a.type, a.hd, p.rows.nr, [&](auto kernel) {
        UAII_LAUNCH(kernel, dim3((unsigned)all), dim3(256), 0, s, p.rows, b, (unsigned)p.row_blocks);
        return hipGetLastError();
      });
    } else {
      e = with_kernel(a.type, a.hd, p.pack, [&](auto kernel) {
        UAII_LAUNCH(kernel, dim3((unsigned)b.blocks), dim3(256), 0, s, b);
        return hipGetLastError();
      });
    }
    if (e != hipSuccess || (p.parts == 1 && p.splits == 0)) return e;  // each row is written
    j.rc = p.rc;
    j.groups = p.groups;
    j.parts = p.parts;
    j.fold = p.fold;
    j.slots = b.slots;
    j.whole = b.whole;
    j.info = b.info;
    j.batch = true;
  }
  // about how many partials a row has: a wave takes eight in one round trip
  const int64_t parts = p.splits + (a.n_keys ? std::max<int64_t>(1, p.blocks / (a.rows * a.n_kv * p.groups)) : 0);
  const dim3 grid((unsigned)(a.rows * a.n_heads));
  if (parts <= 8) UAII_LAUNCH(k_attn_join<1>, grid, dim3(64), 0, s, j);
  else if (parts <= 32) UAII_LAUNCH(k_attn_join<4>, grid, dim3(256), 0, s, j);
  else UAII_LAUNCH(k_attn_join<16>, grid, dim3(1024), 0, s, j);
  return hipGetLastError();
}

}  // namespace uaii_hip
