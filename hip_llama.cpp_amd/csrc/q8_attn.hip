// q8_attn.hip — causal attention over the int8 K/V cache (include/thaDNN/thaDNN_q8_kv.hpp).
#include "q8_kv.hpp"

namespace tl {

struct Q8AttnArgs {
  Q8KVLayer l;
  Q8KVCall call;
  const float* q;
  float* out;
  long long q_stride, out_stride;
  int n_heads, mul;  // query heads, and how many of them share a K/V head
};

// One wave per (sequence, row, query head): lanes take keys for the scores, dimensions for the values.
__global__ void __launch_bounds__(64) k_q8_attn(Q8AttnArgs a) {
  keep_implicit_args();  // common.hpp
  __shared__ float qs[kQ8KVMaxHead];
  __shared__ float ps[64];
  const Q8KVLayer& l = a.l;
  unsigned u = blockIdx.x;
  const int hq = u % a.n_heads;
  u /= a.n_heads;
  const int i = u % a.call.n_tokens, b = u / a.call.n_tokens;
  const int n = a.call.n_d ? a.call.n_d[b] : a.call.n_tokens;
  if (i >= n) return;
  const long long p = (long long)a.call.pos_d[b] + i;
  const int T = p < 0 || p >= l.seq_len ? 0 : (int)p + 1;
  const int lane = threadIdx.x, h = hq / a.mul;
  const long long row = (long long)b * a.call.n_tokens + i;
  const float* q = a.q + row * a.q_stride + (long long)hq * l.head_size;
  for (int d = lane; d < l.head_size; d += 64) qs[d] = q[d];
  __syncthreads();
  const int8_t* k = l.k + b * l.seq_codes + h * l.head_codes;
  const int8_t* v = l.v + b * l.seq_codes + h * l.head_codes;
  const float* ks = l.ks + b * l.seq_scales + h * l.head_scales;
  const float* vs = l.vs + b * l.seq_scales + h * l.head_scales;
  const float root = sqrtf((float)l.head_size);

  float m = -INFINITY, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int t0 = 0; t0 < T; t0 += 64) {
    const int t = t0 + lane;
    float x = -INFINITY;
    if (t < T) {
      const int8_t* kt = k + (long long)t * l.lanes;
      float dot = 0.f;
      for (int d = 0; d < l.head_size; ++d) dot = fmaf(qs[d], (float)kt[d], dot);
      x = dot * ks[t >> l.block_log2] / root;
    }
    const float top = fmaxf(m, wave_max(x));
    const float base = top == -INFINITY ? 0.f : top;  // only NaN scores so far
    const float f = expf(m - base);
    const float e = t < T ? expf(x - base) : 0.f;
    sum = sum * f + wave_sum(e);
    m = top;
    __syncthreads();
    ps[lane] = t < T ? e * vs[t >> l.block_log2] : 0.f;
    __syncthreads();
    const int keys = min(64, T - t0);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = lane + 64 * r;
      if (d >= l.head_size) break;
      float acc = o[r] * f;
      for (int s = 0; s < keys; ++s) {
        const long long slot = t0 + s;
        acc = fmaf(ps[s], (float)v[(slot >> 4) * (16LL * l.lanes) + d * 16 + (slot & 15)], acc);
      }
      o[r] = acc;
    }
  }
  float* out = a.out + row * a.out_stride + (long long)hq * l.head_size;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (lane + 64 * r < l.head_size) out[lane + 64 * r] = T ? o[r] / sum : 0.f;
}

}  // namespace tl

extern "C" size_t thaDNN_q8_attention_workspace(const Q8KVCache* c, int n_batches, int n_tokens, int n_heads) {
  return 0;
}

extern "C" thablasStatus_t thaDNN_q8_attention_batch(thablasHandle_t* handle, const Q8KVCache* c, int layer,
                                                     int n_batches, int n_tokens, const int* pos_d, const int* n_d,
                                                     int n_heads, const float* q, float* out, int q_stride,
                                                     int out_stride, void* work, size_t work_bytes) {
  tl::Q8AttnArgs a = {};
  const thablasStatus_t ok = tl::q8kv_layer(handle, c, layer, n_batches, n_tokens, pos_d, n_d, a.l);
  if (ok != THABLAS_STATUS_SUCCESS) return ok;
  if (n_heads <= 0 || n_heads % c->n_kv_heads) return THABLAS_STATUS_INVALID_VALUE;
  const long long row = (long long)n_heads * c->head_size;
  if (q_stride < row || out_stride < row || (((uintptr_t)q | (uintptr_t)out) & 3)) return THABLAS_STATUS_INVALID_VALUE;
  if (n_batches == 0 || n_tokens == 0) return THABLAS_STATUS_SUCCESS;
  if (!q || !out) return THABLAS_STATUS_INVALID_VALUE;
  a.call = {pos_d, n_d, n_batches, n_tokens};
  a.q = q;
  a.out = out;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.n_heads = n_heads;
  a.mul = n_heads / c->n_kv_heads;
  const unsigned __int128 grid = (unsigned __int128)n_batches * n_tokens * n_heads;
  if (grid > 0x7fffffff) return THABLAS_STATUS_NOT_SUPPORTED;
  tl::Q8KVDevice dev(handle->current_gpu_id);
  if (!dev.ok) return THABLAS_STATUS_INVALID_VALUE;
  hipLaunchKernelGGL(tl::k_q8_attn, dim3((unsigned)grid), dim3(64), 0, handle->calc_stream, a);
  return tl::q8kv_status(hipGetLastError());
}
