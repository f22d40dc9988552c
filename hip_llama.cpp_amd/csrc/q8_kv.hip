// q8_kv.hip — the int8 K/V cache: rows quantised as they are written, and read back
// (include/thaDNN/thaDNN_q8_kv.hpp).
//
// Both kernels give a thread four dimensions of sixteen or eight tokens: a float4 of each row, a dword of each key's
// codes, and the four runs in which the value codes of those dimensions lie side by side, so neither layout needs
// an exchange between lanes.
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

// Dimensions d .. d + 3 of a row; those from head_size on read as 0.  A call passes over its rows once: nontemporal, which
// is what carries the large calls (8 x 2048 rows of 4096 and their codes, MI355X: stored in 157 us without, 120 with, read
// back in 134 and 129 by 16 tokens a thread; one row each of sixteen sequences' blocks read back in 8.2 and 6.2).
template <bool VEC>
TL_DEVICE f4 row4_load(const float* row, int d, int head_size) {
  if constexpr (VEC) return __builtin_nontemporal_load(reinterpret_cast<const f4*>(row + d));
  f4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (d + e < head_size) x[e] = row[d + e];
  return x;
}
template <bool VEC>
TL_DEVICE void row4_store(float* row, int d, int head_size, f4 x) {
  if constexpr (VEC) {
    __builtin_nontemporal_store(x, reinterpret_cast<f4*>(row + d));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (d + e < head_size) row[d + e] = x[e];
  }
}

typedef int i2 __attribute__((ext_vector_type(2)));
typedef int i4 __attribute__((ext_vector_type(4)));

TL_DEVICE int byte_of(int x, int i) { return (int)(signed char)(x >> (8 * i)); }
// The low bytes of four integers in one word.
TL_DEVICE int pack4(int a, int b, int c, int d) {
  const unsigned lo = __builtin_amdgcn_perm((unsigned)b, (unsigned)a, 0x0c0c0400u);
  const unsigned hi = __builtin_amdgcn_perm((unsigned)d, (unsigned)c, 0x04000c0cu);
  return (int)(lo | hi);
}

// Codes under one scale: round(x / scale), half away from zero, the quotient rounded to fp32 as if it were divided.
// With both brought by the scale's power of two to where nothing over- or underflows (a quotient that loses bits
// there is a code of 0), r = RN(1 / s), y = RN(x r), the remainder x - y s is exact and RN(y + r (x - y s)) is RN(x / s)
// (Markstein; common.hpp q8_div_fast).  |x / s| <= 127 (1 + 2^-23), where truncating y + copysign(pred(0.5), y)
// rounds half away.  A scale of 0 or NaN has codes of 0.
struct KvCoder {
  float s, r;
  int e;
  TL_DEVICE explicit KvCoder(float scale) {
    const bool ok = scale > 0.f;
    e = ok ? -__builtin_amdgcn_frexp_expf(scale) : 0;
    s = ok ? __builtin_ldexpf(scale, e) : 0.f;
    r = ok ? __fdiv_rn(1.f, s) : 0.f;
  }
  TL_DEVICE int operator()(float x) const {
    x = __builtin_ldexpf(x, e);
    const float y = __fmul_rn(x, r);
    const float q = __builtin_fmaf(__builtin_fmaf(-y, s, x), r, y);
    return (int)__fadd_rn(q, __builtin_copysignf(0.49999997f, q));
  }
};

struct StoreArgs {
  Q8KVLayer l;
  Q8KVCall call;
  const float* x[2];  // keys, values
  long long stride;
  int spanned;  // blocks that n_tokens rows may touch
  int threads;  // of a head: block / 16 * lanes / 4
  int heads;    // of a workgroup: several where one has less than a wave of threads
  int groups;   // of heads
};

// A workgroup quantises what the call writes of one (keys or values, sequence, block of tokens) and one or a few
// heads: thread (head, g, d4) the tokens 16g .. 16g + 15 of the block in dimensions 4*d4 .. + 3, held in registers
// between the maximum and the codes.  A group of one new token has code of its own: a decode step's store waits for
// instructions as for anything else (sixteen rows of 32 heads of 128: 5.5 us, with the general code alone 7.3).  Prompts
// are bound by memory: 8 x 2048 such rows 120 us, 5.6 TB/s of rows in and codes out.
template <bool VEC>
__global__ void __launch_bounds__(512) k_q8kv_store(StoreArgs a) {
  keep_implicit_args();  // common.hpp: rocprofv3 --pmc needs the hidden kernargs
  __shared__ unsigned red[16];
  const Q8KVLayer& l = a.l;
  unsigned u = blockIdx.x;
  const int jb = u % a.spanned;
  u /= a.spanned;
  const int hg = u % a.groups;
  u /= a.groups;
  const int which = u & 1, b = u >> 1;

  long long row0;
  int first, last;
  q8kv_span(a.call, l.seq_len, b, row0, first, last);
  if (first >= last) return;
  const int j = (first >> l.block_log2) + jb;
  const int start = j << l.block_log2, end = start + (1 << l.block_log2);
  if (start >= last) return;
  const int unit = threadIdx.x / a.threads, within = threadIdx.x - unit * a.threads;
  const int quads = l.lanes / 4;
  const int g = within / quads, d = (within - g * quads) * 4;
  const int t0 = start + 16 * g;
  const int h = hg * a.heads + unit;
  const bool mine = unit < a.heads && h < l.heads;
  const bool full = first <= start && end <= last;
  const long long head = b * l.seq_codes + (mine ? h : 0) * l.head_codes;
  float* scale_p = (which ? l.vs : l.ks) + b * l.seq_scales + (mine ? h : 0) * l.head_scales + j;
  const float* src = a.x[which] + (long long)h * l.head_size + ((long long)b * a.call.n_tokens + (t0 - row0)) * a.stride;
  const bool earlier = start < first;
  const float was = earlier ? *scale_p : 0.f;

  // |x| compared as integers: NaN above infinity above every number
  auto largest = [](unsigned top, f4 x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
    return top;
  };
  const int lo = max(first - t0, 0), hi = min(last - t0, 16);  // the group's new tokens
  const bool one = hi - lo == 1;
  f4 x[16];
  x[0] = f4{0.f, 0.f, 0.f, 0.f};
  unsigned top = 0;
  const bool live = mine && d < l.head_size;
  if (one) {
    if (live) x[0] = row4_load<VEC>(src + lo * a.stride, d, l.head_size);
    top = largest(top, x[0]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = live && i >= lo && i < hi ? row4_load<VEC>(src + i * a.stride, d, l.head_size) : f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 16; ++i) top = largest(top, x[i]);
  }
  if (a.heads == 1) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();  // also: every thread has read the old scale
    for (unsigned w = 0; w < blockDim.x / 64; ++w) top = max(top, red[w]);
  } else {
    if (threadIdx.x < 16) red[threadIdx.x] = 0;
    __syncthreads();
    if (mine) atomicMax(&red[unit], top);
    __syncthreads();
    top = mine ? red[unit] : 0;
  }

  float scale = __fdiv_rn(__uint_as_float(top), 127.0f);
  if (scale < 1.17549435e-38f) scale = 0.f;
  if (top >= 0x7f800000u) scale = __builtin_nanf("");
  if (earlier && !(scale > was) && scale == scale) scale = was;  // a NaN on either side stays
  const bool again = earlier && !(scale == was);                 // earlier tokens change their codes
  if (!mine) return;
  if (within == 0) *scale_p = scale;

  const KvCoder code(scale);
  int* kd = reinterpret_cast<int*>(l.k + head + (long long)t0 * l.lanes + d);
  i4* vd = reinterpret_cast<i4*>(l.v + head + (long long)t0 * l.lanes + (long long)d * 16);
  const int step = l.lanes / 4;
  if (full) {
    if (which == 0) {
#pragma unroll
      for (int i = 0; i < 16; ++i) kd[i * step] = pack4(code(x[i][0]), code(x[i][1]), code(x[i][2]), code(x[i][3]));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        i4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack4(code(x[4 * i][e]), code(x[4 * i + 1][e]), code(x[4 * i + 2][e]), code(x[4 * i + 3][e]));
        vd[e] = w;
      }
    }
    return;
  }
  // codes of the tokens lo <= q .. q + 3 < hi
  auto put = [&](int q, int lo, int hi, f4 y0, f4 y1, f4 y2, f4 y3) {
    const f4 y[4] = {y0, y1, y2, y3};
    if (which == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (q + i >= lo && q + i < hi) kd[(q + i) * step] = pack4(code(y[i][0]), code(y[i][1]), code(y[i][2]), code(y[i][3]));
      return;
    }
    int8_t* at = reinterpret_cast<int8_t*>(vd) + q;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int w = pack4(code(y[0][e]), code(y[1][e]), code(y[2][e]), code(y[3][e]));
      if (q >= lo && q + 4 <= hi) {
        *reinterpret_cast<int*>(at + 16 * e) = w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (q + i >= lo && q + i < hi) at[16 * e + i] = (int8_t)byte_of(w, i);
      }
    }
  };
  if (one) {  // a decode step's token
    const int c[4] = {code(x[0][0]), code(x[0][1]), code(x[0][2]), code(x[0][3])};
    if (which == 0) {
      kd[lo * step] = pack4(c[0], c[1], c[2], c[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) reinterpret_cast<int8_t*>(vd)[16 * e + lo] = (int8_t)c[e];
    }
  } else {
#pragma unroll
    for (int q = 0; q < 16; q += 4)
      if (q < hi && q + 4 > lo) put(q, lo, hi, x[q], x[q + 1], x[q + 2], x[q + 3]);
  }
  if (!again) return;
#pragma unroll 1
  for (int q = 0; q < min(lo, 16); q += 4) {
    const int8_t* at = which ? reinterpret_cast<const int8_t*>(vd) + q : reinterpret_cast<const int8_t*>(kd + q * step);
    int w[4];
    f4 y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const int*>(at + i * (which ? 16 : l.lanes));
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) y[i][e] = __fmul_rn((float)(which ? byte_of(w[e], i) : byte_of(w[i], e)), was);
    put(q, 0, lo, y[0], y[1], y[2], y[3]);
  }
}

struct LoadArgs {
  Q8KVLayer l;
  Q8KVCall call;
  float* x[2];
  long long stride;
  int groups;   // groups of 8 slots that n_tokens rows may touch
  int columns;  // workgroups across a row
  int from;     // 0: keys and values, or keys alone; 1: values alone
};

// Thread: dimensions d .. d + 3 of one head in the 8 tokens of one group of slots.  Bound by memory: 8 x 2048 rows of
// 4096 117 us, 5.7 TB/s of codes in and rows out (with 16 tokens 140, with 4 121).
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
  const int t0 = ((first >> 3) + jg) << 3;
  if (first >= last || t0 >= last) return;
  const int quads = l.lanes / 4;
  const int at = col * 256 + threadIdx.x;
  const int h = at / quads, d = (at - h * quads) * 4;
  if (h >= l.heads || d >= l.head_size) return;
  const float scale = (which ? l.vs : l.ks)[b * l.seq_scales + h * l.head_scales + (t0 >> l.block_log2)];
  float* dst = a.x[which] + ((long long)b * a.call.n_tokens + (t0 - row0)) * a.stride + (long long)h * l.head_size;
  int w[8];
  if (which == 0) {
    const int* src = reinterpret_cast<const int*>(l.k + b * l.seq_codes + h * l.head_codes + (long long)t0 * l.lanes + d);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = src[(long long)i * (l.lanes / 4)];
  } else {
    const int8_t* src = l.v + b * l.seq_codes + h * l.head_codes + (long long)(t0 & ~15) * l.lanes + (t0 & 8) + d * 16;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const i2 q = *reinterpret_cast<const i2*>(src + 16 * e);
      w[2 * e] = q.x;
      w[2 * e + 1] = q.y;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (t0 + i < first || t0 + i >= last) continue;
    f4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      x[e] = __fmul_rn((float)(which == 0 ? byte_of(w[i], e) : byte_of(w[2 * e + i / 4], i % 4)), scale);
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
  a.threads = (c->block / 16) * (a.l.lanes / 4);
  a.heads = a.threads < 64 ? 64 / a.threads : 1;
  a.groups = (c->n_kv_heads + a.heads - 1) / a.heads;
  const unsigned __int128 grid = (unsigned __int128)2 * n_batches * a.groups * a.spanned;
  const int threads = (a.threads * a.heads + 63) / 64 * 64;
  if (!tl::q8kv_grid_ok(grid, threads)) return THABLAS_STATUS_NOT_SUPPORTED;
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
  const long long groups = ((long long)n_tokens + 6) / 8 + 1, most = ((long long)c->seq_len + 7) / 8;
  a.groups = (int)(groups < most ? groups : most);
  const long long columns = ((long long)c->n_kv_heads * (a.l.lanes / 4) + 255) / 256;
  a.columns = (int)columns;
  const int both = k && v;
  const unsigned __int128 grid = (unsigned __int128)(both ? 2 : 1) * n_batches * a.groups * columns;
  if (!tl::q8kv_grid_ok(grid, 256)) return THABLAS_STATUS_NOT_SUPPORTED;
  tl::Q8KVDevice dev(handle->current_gpu_id);
  if (!dev.ok) return THABLAS_STATUS_INVALID_VALUE;
  auto kernel = tl::q8kv_vec4(c->head_size, kv_stride, k, v) ? tl::k_q8kv_load<true> : tl::k_q8kv_load<false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), 0, handle->calc_stream, a, both);
  return tl::q8kv_status(hipGetLastError());
}
