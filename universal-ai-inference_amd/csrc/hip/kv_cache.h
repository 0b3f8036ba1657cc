// kv_cache.h — caches of a batch: their layout and the arguments of the kernels that
// write, read back and attend over them (kv_cache.hip, batch_attn.hip, rows_attn.hip).
#pragma once

#include "common.h"

namespace uaii_hip {

enum KvType : int { KV_F32 = 0, KV_F16 = 1, KV_Q8 = 2 };

// One sequence's K (or V): [n_kv][max_seq][hd] values and, for KV_Q8, [n_kv][max_seq] f32
// scales behind them. KV_Q8 stores a value as the byte q + 128, q * scale being the value:
// with the offset a byte needs no sign extension on its way to f16, and a cache of zeros
// reads as zeros. One scale for a head's row: a score is then one integer product times
// one factor, and a value's factor joins its probability; scales of 32 values cost 3 %
// more bytes and a factor for each chunk of a product.
__host__ __device__ inline int64_t kv_seq_bytes(int type, int64_t n_kv, int64_t max_seq, int64_t hd) {
  const int64_t n = n_kv * max_seq;
  if (type == KV_Q8) return (n * (hd + 4) + 15) / 16 * 16;
  return n * hd * (type == KV_F16 ? 2 : 4);
}

struct KvRowsArgs {
  const float* k;  // [n_seq * rows][ld]
  const float* v;
  int64_t ld;
  uint8_t* kc;
  uint8_t* vc;
  int type;
  int64_t n_seq, rows;
  int n_kv, hd;
  int64_t max_seq;
  int64_t p0;           // row i of sequence s: position p0 + past[s] + i
  const int32_t* past;  // or null
};

hipError_t launch_kv_write(const KvRowsArgs& a, hipStream_t s);
// One cache (kc) back into `out` [n_seq * rows][ld]; k, v and vc are not used.
hipError_t launch_kv_read(const KvRowsArgs& a, float* out, hipStream_t s);

// Attention over such caches. A row is a query; its keys are a prefix that all rows share
// (positions 0 .. n_prefix - 1) and, behind it, those of its own sequence.
struct SeqAttnArgs {
  const float* q;  // [rows][ldq]
  int64_t ldq;
  float* out;  // [rows][ldo]
  int64_t ldo;
  int64_t rows;
  int n_heads, n_kv, hd;
  float scale, cap;     // cap 0: none
  const float* slopes;  // [n_heads] or null
  int window;           // 0: none
  int type;
  // batch: row s over sequence s's own keys
  const uint8_t* kc;
  const uint8_t* vc;
  int64_t max_seq, seq_bytes;
  const int32_t* n_keys;
  const uint8_t* kp;
  const uint8_t* vp;
  int64_t pre_seq;
  int n_prefix;
  // prompt (n_keys null): row i at position p0 + i over the cache (kc, vc)
  int p0, bidir;
  const int32_t* first;
};

// Device scratch of the call, and its launches.
size_t seq_attn_scratch(const SeqAttnArgs& a);
hipError_t launch_seq_attn(const SeqAttnArgs& a, char* scratch, hipStream_t s);

}  // namespace uaii_hip
