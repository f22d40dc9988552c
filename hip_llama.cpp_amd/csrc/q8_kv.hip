// q8_kv.hip — the int8 K/V cache: rows quantised as they are written, and read back
// (include/thaDNN/thaDNN_q8_kv.hpp).
//
// Both kernels give a thread four dimensions of sixteen tokens: a float4 of each row, a dword of each key's
// codes, and the four 16-byte runs in which the value codes of those dimensions lie side by side, so neither
// layout needs an exchange between lanes.
#include "q8_kv.hpp"

using tl::f4;

extern "C" size_t thallama_q8_kv_bytes(int n_batches, int n_layers, int n_kv_heads, int head_size, int seq_len,
                                       int block) {
  if (!tl::q8kv_sizes_ok(n_batches, n_layers, n_kv_heads, head_size, seq_len) || !tl::q8kv_supported(head_size, block))
    return 0;
  const size_t codes = tl::q8kv_codes(n_batches, n_layers, n_kv_heads, head_size, seq_len, block);
  const size_t heads = (size_t)n_batches * n_layers * n_kv_heads;  // codes bounds it
  const size_t scales = tl::q8kv_part((unsigned __int128)heads * (tl::q8kv_slots(seq_len, block) / block) * sizeof(float));
  return codes ? 2 * codes + 2 * scales : 0;
}

extern "C" int thallama_q8_kv_map(Q8KVCache* c, void* mem, int n_batches, int n_layers, int n_kv_heads, int head_size,
                                  int seq_len, int block) {
  const size_t all = thallama_q8_kv_bytes(n_batches, n_layers, n_kv_heads, head_size, seq_len, block);
  if (!c || !mem || ((uintptr_t)mem & 255) || !all) return -1;
  const size_t codes = tl::q8kv_codes(n_batches, n_layers, n_kv_heads, head_size, seq_len, block);
  char* p = static_cast<char*>(mem);
  c->k = reinterpret_cast<int8_t*>(p);
  c->v = reinterpret_cast<int8_t*>(p + codes);
  c->ks = reinterpret_cast<float*>(p + 2 * codes);
  c->vs = reinterpret_cast<float*>(p + 2 * codes + (all - 2 * codes) / 2);
  c->n_batches = n_batches;
  c->n_layers = n_layers;
  c->n_kv_heads = n_kv_heads;
  c->head_size = head_size;
  c->seq_len = seq_len;
  c->block = block;
  return 0;
}

namespace tl {

// Dimensions d .. d + 3 of a row; those from head_size on read as 0.
template <bool VEC>
TL_DEVICE f4 row4_load(const float* row, int d, int head_size) {
  if constexpr (VEC) return *reinterpret_cast<const f4*>(row + d);
  f4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (d + e < head_size) x[e] = row[d + e];
  return x;
}
template <bool VEC>
TL_DEVICE void row4_store(float* row, int d, int head_size, f4 x) {
  if constexpr (VEC) {
    *reinterpret_cast<f4*>(row + d) = x;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (d + e < head_size) row[d + e] = x[e];
  }
}

TL_DEVICE int byte_of(int x, int i) { return (int)(signed char)(x >> (8 * i)); }

// The code of x under `scale`: 0 where the scale is 0 or NaN.
TL_DEVICE int kv_code(float x, float scale) { return scale > 0.f ? q8_code(x, scale) : 0; }

struct StoreArgs {
  Q8KVLayer l;
  Q8KVCall call;
  const float* x[2];  // keys, values
  long long stride;
  int spanned;  // blocks that n_tokens rows may touch
};

// One workgroup quantises what the call writes of one (keys or values, sequence, head, block of tokens):
// thread (g, d4) the tokens 16g .. 16g + 15 of the block in dimensions 4*d4 .. + 3.
template <bool VEC>
__global__ void __launch_bounds__(512) k_q8kv_store(StoreArgs a) {
  keep_implicit_args();  // common.hpp: rocprofv3 --pmc needs the hidden kernargs
  __shared__ unsigned red[8];
  const Q8KVLayer& l = a.l;
  unsigned u = blockIdx.x;
  const int jb = u % a.spanned;
  u /= a.spanned;
  const int h = u % l.heads;
  u /= l.heads;
  const int which = u & 1, b = u >> 1;

  long long row0;
  int first, last;
  q8kv_span(a.call, l.seq_len, b, row0, first, last);
  if (first >= last) return;
  const int j = (first >> l.block_log2) + jb;
  const int start = j << l.block_log2;  // of the block; below first only in the first one
  if (jb && start >= last) return;
  const int quads = l.lanes / 4;
  const int g = threadIdx.x / quads, d = (threadIdx.x - g * quads) * 4;
  const int t0 = start + 16 * g;
  const bool mine = (16 * g) >> l.block_log2 == 0;
  const long long head = b * l.seq_codes + h * l.head_codes;
  float* scale_p = (which ? l.vs : l.ks) + b * l.seq_scales + h * l.head_scales + j;

  // the rows: zeros where the call has none, and in dimensions from head_size on
  f4 x[16];
  const float* src = a.x[which] + (long long)h * l.head_size;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int t = t0 + i;
    const bool in = mine && t >= first && t < last && d < l.head_size;
    x[i] = in ? row4_load<VEC>(src + ((long long)b * a.call.n_tokens + (t - row0)) * a.stride, d, l.head_size)
              : f4{0.f, 0.f, 0.f, 0.f};
  }
  // |x| compared as integers: NaN above infinity above every number
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(x[i][e]) & 0x7fffffffu);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
  for (unsigned w = 0; w < blockDim.x / 64; ++w) top = max(top, red[w]);

  float scale = __fdiv_rn(__uint_as_float(top), 127.0f);
  if (scale < 1.17549435e-38f) scale = 0.f;
  if (top >= 0x7f800000u) scale = __builtin_nanf("");
  const bool earlier = start < first;
  float was = 0.f;
  if (earlier) {
    was = *scale_p;
    if (!(scale > was) && scale == scale) scale = was;  // a NaN on either side stays
  }
  const bool again = earlier && !(scale == was);
  __syncthreads();  // every thread has read the old scale
  if (threadIdx.x == 0) *scale_p = scale;
  if (!mine || t0 >= last || (t0 + 16 <= first && !again)) return;

  if (which == 0) {
    int* dst = reinterpret_cast<int*>(l.k + head + (long long)t0 * l.lanes + d);
    const int step = l.lanes / 4;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int t = t0 + i;
      if (t >= last || (t < first && !again)) continue;
      int c[4];
      if (t < first) {
        const int old = dst[(long long)i * step];
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = kv_code(__fmul_rn((float)byte_of(old, e), was), scale);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = kv_code(x[i][e], scale);
      }
      dst[(long long)i * step] = (c[0] & 255) | (c[1] & 255) << 8 | (c[2] & 255) << 16 | c[3] << 24;
    }
  } else {
    typedef int i4 __attribute__((ext_vector_type(4)));
    i4* dst = reinterpret_cast<i4*>(l.v + head + (long long)t0 * l.lanes + (long long)d * 16);
    const bool whole = t0 >= first && t0 + 16 <= last;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      i4 w = {0, 0, 0, 0};
      if (!whole) w = dst[e];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int t = t0 + i;
        const int old = byte_of(w[i / 4], i % 4);
        int c = old;
        if (t >= first && t < last) c = kv_code(x[i][e], scale);
        else if (t < first && again) c = kv_code(__fmul_rn((float)old, was), scale);
        w[i / 4] = (w[i / 4] & ~(255 << (8 * (i % 4)))) | (c & 255) << (8 * (i % 4));
      }
      dst[e] = w;
    }
  }
}

struct LoadArgs {
  Q8KVLayer l;
  Q8KVCall call;
  float* x[2];
  long long stride;
  int groups;   // groups of 16 slots that n_tokens rows may touch
  int columns;  // workgroups across a row
  int from;     // 0: keys and values, or keys alone; 1: values alone
};

// Thread: dimensions d .. d + 3 of one head in the 16 tokens of one group of slots.
template <bool VEC>
__global__ void __launch_bounds__(256) k_q8kv_load(LoadArgs a, int both) {
  keep_implicit_args();  // common.hpp
  const Q8KVLayer& l = a.l;
  unsigned u = blockIdx.x;
  const int col = u % a.columns;
  u /= a.columns;
  const int jg = u % a.groups;
  u /= a.groups;
  const int which = both ? (int)(u & 1) : a.from, b = both ? u >> 1 : u;

  long long row0;
  int first, last;
  q8kv_span(a.call, l.seq_len, b, row0, first, last);
  const int t0 = ((first >> 4) + jg) << 4;
  if (first >= last || t0 >= last) return;
  const int quads = l.lanes / 4;
  const int at = col * 256 + threadIdx.x;
  const int h = at / quads, d = (at - h * quads) * 4;
  if (h >= l.heads || d >= l.head_size) return;

  const float scale = (which ? l.vs : l.ks)[b * l.seq_scales + h * l.head_scales + (t0 >> l.block_log2)];
  const long long head = b * l.seq_codes + h * l.head_codes + (long long)t0 * l.lanes;
  float* dst = a.x[which] + ((long long)b * a.call.n_tokens + (t0 - row0)) * a.stride + (long long)h * l.head_size;
  int w[16];  // keys: a dword of each token; values: four dwords of each dimension
  if (which == 0) {
    const int* src = reinterpret_cast<const int*>(l.k + head + d);
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = t0 + i >= first && t0 + i < last ? src[(long long)i * (l.lanes / 4)] : 0;
  } else {
    typedef int i4 __attribute__((ext_vector_type(4)));
    const i4* src = reinterpret_cast<const i4*>(l.v + head + d * 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const i4 q = src[e];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[4 * e + i] = q[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if (t0 + i < first || t0 + i >= last) continue;
    f4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      x[e] = __fmul_rn((float)(which == 0 ? byte_of(w[i], e) : byte_of(w[4 * e + i / 4], i % 4)), scale);
    row4_store<VEC>(dst + i * a.stride, d, l.head_size, x);
  }
}

}  // namespace tl

extern "C" thablasStatus_t thaDNN_q8_kv_store_batch(thablasHandle_t* handle, const Q8KVCache* c, int layer,
                                                    int n_batches, int n_tokens, const int* pos_d, const int* n_d,
                                                    const float* k, const float* v, int kv_stride) {
  tl::StoreArgs a = {};
  const thablasStatus_t ok = tl::q8kv_layer(handle, c, layer, n_batches, n_tokens, pos_d, n_d, a.l);
  if (ok != THABLAS_STATUS_SUCCESS) return ok;
  if (((uintptr_t)k | (uintptr_t)v) & 3 || kv_stride < (long long)c->n_kv_heads * c->head_size) return THABLAS_STATUS_INVALID_VALUE;
  if (n_batches == 0 || n_tokens == 0) return THABLAS_STATUS_SUCCESS;
  if (!k || !v) return THABLAS_STATUS_INVALID_VALUE;
  a.call = {pos_d, n_d, n_batches, n_tokens};
  a.x[0] = k;
  a.x[1] = v;
  a.stride = kv_stride;
  const long long spanned = ((long long)n_tokens + c->block - 2) / c->block + 1;
  const long long most = (c->seq_len + (long long)c->block - 1) / c->block;
  a.spanned = (int)(spanned < most ? spanned : most);
  const unsigned __int128 grid = (unsigned __int128)2 * n_batches * c->n_kv_heads * a.spanned;
  if (grid > 0x7fffffff) return THABLAS_STATUS_NOT_SUPPORTED;
  const int threads = ((c->block / 16) * (a.l.lanes / 4) + 63) / 64 * 64;
  tl::Q8KVDevice dev(handle->current_gpu_id);
  if (!dev.ok) return THABLAS_STATUS_INVALID_VALUE;
  auto kernel = tl::q8kv_vec4(c->head_size, kv_stride, k, v) ? tl::k_q8kv_store<true> : tl::k_q8kv_store<false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(threads), 0, handle->calc_stream, a);
  return tl::q8kv_status(hipGetLastError());
}

extern "C" thablasStatus_t thaDNN_q8_kv_load_batch(thablasHandle_t* handle, const Q8KVCache* c, int layer,
                                                   int n_batches, int n_tokens, const int* pos_d, const int* n_d,
                                                   float* k, float* v, int kv_stride) {
  tl::LoadArgs a = {};
  const thablasStatus_t ok = tl::q8kv_layer(handle, c, layer, n_batches, n_tokens, pos_d, n_d, a.l);
  if (ok != THABLAS_STATUS_SUCCESS) return ok;
  if (((uintptr_t)k | (uintptr_t)v) & 3 || kv_stride < (long long)c->n_kv_heads * c->head_size) return THABLAS_STATUS_INVALID_VALUE;
  if (n_batches == 0 || n_tokens == 0 || (!k && !v)) return THABLAS_STATUS_SUCCESS;
  a.call = {pos_d, n_d, n_batches, n_tokens};
  a.x[0] = k;
  a.x[1] = v;
  a.stride = kv_stride;
  a.from = k ? 0 : 1;
  const long long groups = ((long long)n_tokens + 14) / 16 + 1, most = ((long long)c->seq_len + 15) / 16;
  a.groups = (int)(groups < most ? groups : most);
  const long long columns = ((long long)c->n_kv_heads * (a.l.lanes / 4) + 255) / 256;
  a.columns = (int)columns;
  const int both = k && v;
  const unsigned __int128 grid = (unsigned __int128)(both ? 2 : 1) * n_batches * a.groups * columns;
  if (grid > 0x7fffffff) return THABLAS_STATUS_NOT_SUPPORTED;
  tl::Q8KVDevice dev(handle->current_gpu_id);
  if (!dev.ok) return THABLAS_STATUS_INVALID_VALUE;
  auto kernel = tl::q8kv_vec4(c->head_size, kv_stride, k, v) ? tl::k_q8kv_load<true> : tl::k_q8kv_load<false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), 0, handle->calc_stream, a, both);
  return tl::q8kv_status(hipGetLastError());
}
