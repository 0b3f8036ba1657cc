// batch_layer.cpp — the entry points of include/uaii_hip.h for the caches of a batch:
// checks of arguments, then the launchers of kv_cache.hip, batch_attn.hip and
// rows_attn.hip.
#include "uaii_hip.h"

#include "hip/kv_cache.h"
#include "scratch.h"

#include <cmath>
#include <cstdint>

using namespace uaii_hip;

namespace {

constexpr int kErrArg = -1;  // invalid argument
constexpr int64_t kMaxPositions = (int64_t)1 << 30;  // positions and steps past them are 32-bit in the kernels
constexpr float kMaxCap = 1e20f;  // scores over a larger one could pass the lower end of f32

hipStream_t S(void* s) { return static_cast<hipStream_t>(s); }

bool layout_ok(int kv_type, int n_kv_heads, int head_dim, int64_t max_seq) {
  return (kv_type == KV_F32 || kv_type == KV_F16 || kv_type == KV_Q8) && n_kv_heads > 0 && n_kv_heads <= 65535 &&
         head_dim >= 16 && head_dim <= 256 && head_dim % 16 == 0 && max_seq > 0 && max_seq <= kMaxPositions;
}

bool aligned16(const void* p) { return p && (uintptr_t)p % 16 == 0; }
bool aligned4(const void* p) { return p && (uintptr_t)p % 4 == 0; }

// [rows][ld] floats of which `width` a row are used. Rows of one pitch may lie between each
// other, as the columns of one wide buffer do.
bool overlap(const float* a, int64_t lda, const float* b, int64_t ldb, int64_t rows, int64_t width) {
  const uintptr_t a0 = (uintptr_t)a, a1 = a0 + (uintptr_t)((rows - 1) * lda + width) * 4;
  const uintptr_t b0 = (uintptr_t)b, b1 = b0 + (uintptr_t)((rows - 1) * ldb + width) * 4;
  if (a1 <= b0 || b1 <= a0) return false;
  const uintptr_t pitch = (uintptr_t)lda * 4, used = (uintptr_t)width * 4, from = (a0 > b0 ? a0 - b0 : b0 - a0) % pitch;
  return lda != ldb || from < used || pitch - from < used;
}

// The rows of uaii_hip_kv_append_batch and uaii_hip_kv_read.
bool rows_ok(int kv_type, int64_t n_seq, int64_t rows, int n_kv_heads, int head_dim, int64_t max_seq, int64_t p0,
             const int32_t* past, int64_t ld) {
  if (!layout_ok(kv_type, n_kv_heads, head_dim, max_seq) || n_seq < 0 || rows < 0 || p0 < 0 || p0 > max_seq ||
      (past && !aligned4(past)))
    return false;
  if (n_seq == 0 || rows == 0) return true;
  return ld >= (int64_t)n_kv_heads * head_dim && rows <= INT32_MAX && n_seq <= INT32_MAX / rows &&
         n_seq * rows <= INT32_MAX / n_kv_heads && (past || p0 + rows <= max_seq);
}

KvRowsArgs rows_args(int kv_type, int64_t n_seq, int64_t rows, int n_kv_heads, int head_dim, int64_t max_seq,
                     int64_t p0, const int32_t* past, int64_t ld) {
  KvRowsArgs a{};
  a.ld = ld;
  a.type = kv_type;
  a.n_seq = n_seq;
  a.rows = rows;
  a.n_kv = n_kv_heads;
  a.hd = head_dim;
  a.max_seq = max_seq;
  a.p0 = p0;
  a.past = past;
  return a;
}

// What both attentions check and take over; false: refused.
bool attn_args(const float* q, int64_t ldq, int64_t rows, const void* kcache, const void* vcache, int kv_type,
               int64_t max_seq, int n_heads, int n_kv_heads, int head_dim, const uaii_hip_score_options* o, float* out,
               int64_t ldo, SeqAttnArgs* a) {
  if (!layout_ok(kv_type, n_kv_heads, head_dim, max_seq) || n_heads <= 0 || n_heads > 65535 || n_heads % n_kv_heads ||
      rows < 0 || rows > INT32_MAX / n_heads)
    return false;
  const int64_t width = (int64_t)n_heads * head_dim;
  if (rows > 0 && (!aligned4(q) || !aligned4(out) || !aligned16(kcache) || !aligned16(vcache) || ldq < width ||
                   ldo < width || overlap(q, ldq, out, ldo, rows, width)))
    return false;
  a->q = q;
  a->ldq = ldq;
  a->out = out;
  a->ldo = ldo;
  a->rows = rows;
  a->n_heads = n_heads;
  a->n_kv = n_kv_heads;
  a->hd = head_dim;
  a->type = kv_type;
  a->kc = static_cast<const uint8_t*>(kcache);
  a->vc = static_cast<const uint8_t*>(vcache);
  a->max_seq = max_seq;
  a->seq_bytes = kv_seq_bytes(kv_type, n_kv_heads, max_seq, head_dim);
  if (o) {
    if (o->struct_size < sizeof(*o) || !std::isfinite(o->scale) || !(o->softcap >= 0.0f && o->softcap <= kMaxCap) ||
        o->window < 0 || (o->slopes && !aligned4(o->slopes)))
      return false;
    a->scale = o->scale;
    a->cap = o->softcap;
    a->slopes = o->slopes;
    a->window = o->window > INT32_MAX ? 0 : (int)o->window;  // wider than any cache: none
  }
  if (a->scale == 0.0f) a->scale = 1.0f / std::sqrt((float)head_dim);
  return true;
}

int attend(const SeqAttnArgs& a, void* stream) {
  uaii::Scratch scratch(S(stream));
  const size_t bytes = seq_attn_scratch(a);
  if (bytes > 0) {
    const hipError_t e = scratch.reserve(bytes);
    if (e != hipSuccess) return (int)e;
  }
  return (int)launch_seq_attn(a, scratch.data(), S(stream));
}

}  // namespace

extern "C" {

int64_t uaii_hip_kv_cache_bytes(int kv_type, int n_kv_heads, int64_t max_seq, int head_dim) {
  return layout_ok(kv_type, n_kv_heads, head_dim, max_seq) ? kv_seq_bytes(kv_type, n_kv_heads, max_seq, head_dim) : -1;
}

int uaii_hip_kv_append_batch(const float* k, const float* v, int64_t ld, void* kcache, void* vcache, int kv_type,
                             int64_t n_seq, int64_t rows, int n_kv_heads, int head_dim, int64_t max_seq, int64_t p0,
                             const int32_t* past, void* stream) {
  if (!rows_ok(kv_type, n_seq, rows, n_kv_heads, head_dim, max_seq, p0, past, ld)) return kErrArg;
  if (n_seq == 0 || rows == 0) return 0;
  if (!aligned4(k) || !aligned4(v) || !aligned16(kcache) || !aligned16(vcache)) return kErrArg;
  KvRowsArgs a = rows_args(kv_type, n_seq, rows, n_kv_heads, head_dim, max_seq, p0, past, ld);
  a.k = k;
  a.v = v;
  a.kc = static_cast<uint8_t*>(kcache);
  a.vc = static_cast<uint8_t*>(vcache);
  return (int)launch_kv_write(a, S(stream));
}

int uaii_hip_kv_read(const void* cache, int kv_type, int64_t n_seq, int64_t rows, int n_kv_heads, int head_dim,
                     int64_t max_seq, int64_t p0, const int32_t* past, float* out, int64_t ld, void* stream) {
  if (!rows_ok(kv_type, n_seq, rows, n_kv_heads, head_dim, max_seq, p0, past, ld)) return kErrArg;
  if (n_seq == 0 || rows == 0) return 0;
  if (!aligned16(cache) || !aligned4(out)) return kErrArg;
  KvRowsArgs a = rows_args(kv_type, n_seq, rows, n_kv_heads, head_dim, max_seq, p0, past, ld);
  a.kc = static_cast<uint8_t*>(const_cast<void*>(cache));  // only read
  return (int)launch_kv_read(a, out, S(stream));
}

void uaii_hip_score_options_init(uaii_hip_score_options* options) {
  if (!options) return;
  *options = uaii_hip_score_options{};
  options->struct_size = sizeof(*options);
}

int uaii_hip_attention_batch(const float* q, int64_t ldq, int64_t n_seq, const void* kcache, const void* vcache,
                             int kv_type, int64_t max_seq, const int32_t* n_keys, const void* kprefix,
                             const void* vprefix, int64_t prefix_seq, int64_t n_prefix, int n_heads, int n_kv_heads,
                             int head_dim, const uaii_hip_score_options* options, float* out, int64_t ldo,
                             void* stream) {
  SeqAttnArgs a{};
  if (!attn_args(q, ldq, n_seq, kcache, vcache, kv_type, max_seq, n_heads, n_kv_heads, head_dim, options, out, ldo, &a))
    return kErrArg;
  if (n_prefix < 0 || n_prefix > kMaxPositions - max_seq) return kErrArg;
  if (n_prefix > 0 && (!aligned16(kprefix) || !aligned16(vprefix) || prefix_seq < n_prefix || prefix_seq > kMaxPositions))
    return kErrArg;
  if (n_seq == 0) return 0;
  if (!aligned4(n_keys)) return kErrArg;
  a.n_keys = n_keys;
  a.kp = static_cast<const uint8_t*>(kprefix);
  a.vp = static_cast<const uint8_t*>(vprefix);
  a.pre_seq = prefix_seq;
  a.n_prefix = (int)n_prefix;
  return attend(a, stream);
}

int uaii_hip_attention_prompt(const float* q, int64_t ldq, int64_t m, const void* kcache, const void* vcache,
                              int kv_type, int64_t max_seq, int64_t p0, int64_t bidirectional,
                              const int32_t* first_key, int n_heads, int n_kv_heads, int head_dim,
                              const uaii_hip_score_options* options, float* out, int64_t ldo, void* stream) {
  SeqAttnArgs a{};
  if (!attn_args(q, ldq, m, kcache, vcache, kv_type, max_seq, n_heads, n_kv_heads, head_dim, options, out, ldo, &a))
    return kErrArg;
  if (p0 < 0 || p0 > max_seq || m > max_seq - p0 || bidirectional < 0 || bidirectional > p0 + m ||
      (first_key && !aligned4(first_key)))
    return kErrArg;
  if (m == 0) return 0;
  a.p0 = (int)p0;
  a.bidir = (int)bidirectional;
  a.first = first_key;
  return attend(a, stream);
}

}  // extern "C"
