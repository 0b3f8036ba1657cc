// batch_attn.hip — attention over the caches of a batch, one block a (row, query head).
#include "kv_cache.h"

namespace uaii_hip {
namespace {

__device__ inline float cache_value(const uint8_t* base, int type, int n_kv, int64_t max_seq, int hd, int h, int64_t j, int d) {
  const int64_t row = (int64_t)h * max_seq + j;
  if (type == KV_F32) return reinterpret_cast<const float*>(base)[row * hd + d];
  if (type == KV_F16) return (float)reinterpret_cast<const _Float16*>(base)[row * hd + d];
  const float s = reinterpret_cast<const float*>(base + (int64_t)n_kv * max_seq * hd)[row];
  return (float)((int)base[row * hd + d] - 128) * s;
}

__global__ void __launch_bounds__(256) k_seq_attn(SeqAttnArgs a) {
  __shared__ float q_s[256], p_s[256], red[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r = blockIdx.x;
  const int h = blockIdx.y, kh = h / (a.n_heads / a.n_kv);
  const bool batch = a.n_keys != nullptr;
  const int pre = batch ? a.n_prefix : 0;
  int pos, hi, lo = 0;
  if (batch) {
    const int n = (int)min((int64_t)max(a.n_keys[r], 0), a.max_seq);
    pos = pre + n - 1;
    hi = pre + n;
  } else {
    pos = a.p0 + (int)r;
    hi = max(pos + 1, a.bidir);
    if (a.first) lo = max(0, a.first[r]);
  }
  if (a.window) lo = max(lo, pos - a.window + 1);
  const uint8_t* kc = a.kc + (batch ? r * a.seq_bytes : 0);
  const uint8_t* vc = a.vc + (batch ? r * a.seq_bytes : 0);
  if (tid < a.hd) q_s[tid] = a.q[r * a.ldq + (int64_t)h * a.hd + tid] * a.scale;
  __syncthreads();
  float m = -INFINITY, l = 0.0f, o = 0.0f;
  for (int64_t t0 = lo; t0 < hi; t0 += 256) {
    const int64_t j = t0 + tid;
    float s = -INFINITY;
    if (j < hi) {
      float dot = 0.0f;
      for (int d = 0; d < a.hd; ++d)
        dot += q_s[d] * (j < pre ? cache_value(a.kp, a.type, a.n_kv, a.pre_seq, a.hd, kh, j, d)
                                 : cache_value(kc, a.type, a.n_kv, a.max_seq, a.hd, kh, j - pre, d));
      s = a.cap > 0.0f ? a.cap * tanhf(dot / a.cap) : dot;
      if (a.slopes) s -= a.slopes[h] * (float)abs((int)(pos - j));
    }
    float mx = wave_max(s);
    if (lane == 0) red[wave] = mx;
    __syncthreads();
    const float mnew = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float p = s == -INFINITY ? 0.0f : expf(s - mnew);
    p_s[tid] = p;
    const float sum = wave_sum(p);
    __syncthreads();
    if (lane == 0) red[wave] = sum;
    __syncthreads();
    const float alpha = m == -INFINITY ? 0.0f : expf(m - mnew);
    l = l * alpha + (red[0] + red[1] + red[2] + red[3]);
    m = mnew;
    o *= alpha;
    if (tid < a.hd) {
      const int n = (int)min((int64_t)256, hi - t0);
      for (int i = 0; i < n; ++i) {
        const int64_t jj = t0 + i;
        o += p_s[i] * (jj < pre ? cache_value(a.vp, a.type, a.n_kv, a.pre_seq, a.hd, kh, jj, tid)
                                : cache_value(vc, a.type, a.n_kv, a.max_seq, a.hd, kh, jj - pre, tid));
      }
    }
    __syncthreads();
  }
  if (tid < a.hd) a.out[r * a.ldo + (int64_t)h * a.hd + tid] = lo < hi ? o / l : 0.0f;
}

}  // namespace

hipError_t launch_seq_attn(const SeqAttnArgs& a, hipStream_t s) {
  if (a.rows == 0) return hipSuccess;
  UAII_LAUNCH(k_seq_attn, dim3((unsigned)a.rows, (unsigned)a.n_heads), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace uaii_hip
