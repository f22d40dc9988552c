// q8_kv.hpp — what the int8 K/V cache's kernels share: its layout, the checks of a call's arguments and the
// span of a sequence (include/thaDNN/thaDNN_q8_kv.hpp).
#pragma once
#include "../../include/thaDNN/thaDNN_q8_kv.hpp"
#include "common.hpp"

namespace tl {

constexpr int kQ8KVMaxHead = 256;
constexpr int kQ8KVMaxSeq = 1 << 30;

// One layer of the cache as a kernel sees it.
struct Q8KVLayer {
  int8_t* k;
  int8_t* v;
  float* ks;
  float* vs;
  long long seq_codes;    // codes from a sequence to the next (all layers)
  long long seq_scales;   // scales likewise
  long long head_codes;   // slots * lanes
  long long head_scales;  // slots / block
  int heads, head_size, lanes, seq_len, block_log2;
};

// What one call does: rows of n_batches sequences at device-side positions.
struct Q8KVCall {
  const int* pos_d;
  const int* n_d;
  int n_batches, n_tokens;
};

// The position of sequence b's row 0 and the number of its rows, asked for at once by scalar loads.
TL_DEVICE void q8kv_start(const Q8KVCall& call, int b, long long& row0, int& n) {
  typedef const __attribute__((address_space(4))) int* scalar;
  const int* count = call.n_d ? call.n_d : call.pos_d;
  const int p = ((scalar)(uintptr_t)call.pos_d)[b], c = ((scalar)(uintptr_t)count)[b];
  row0 = p;
  n = call.n_d ? min(max(c, 0), call.n_tokens) : call.n_tokens;
}
// Positions [first, last) of sequence b's rows, clipped to the cache.
TL_DEVICE void q8kv_span(const Q8KVCall& call, int seq_len, int b, long long& row0, int& first, int& last) {
  int n;
  q8kv_start(call, b, row0, n);
  first = (int)max(row0, 0LL);
  last = (int)max(0LL, min(row0 + n, (long long)seq_len));
}

inline int q8kv_lanes(int head_size) { return (head_size + 15) / 16 * 16; }
inline long long q8kv_slots(int seq_len, int block) {
  const int unit = block > 64 ? block : 64;
  return ((long long)seq_len + unit - 1) / unit * unit;
}
inline bool q8kv_sizes_ok(int n_batches, int n_layers, int n_kv_heads, int head_size, int seq_len) {
  // a row of K/V fits an int, and so does every slot with a stride over all waves of a call
  return n_batches > 0 && n_layers > 0 && n_kv_heads > 0 && head_size > 0 && seq_len > 0 && seq_len <= kQ8KVMaxSeq &&
         (long long)n_kv_heads * head_size <= 0x7fffffffLL;
}
inline size_t q8kv_part(unsigned __int128 bytes) {  // a part of the cache's allocation; too large: 0
  bytes = (bytes + 255) / 256 * 256;
  return bytes >> 60 ? 0 : (size_t)bytes;
}
inline size_t q8kv_codes(int n_batches, int n_layers, int n_kv_heads, int head_size, int seq_len, int block) {
  return q8kv_part((unsigned __int128)n_batches * n_layers * n_kv_heads * q8kv_slots(seq_len, block) * q8kv_lanes(head_size));
}
inline bool q8kv_supported(int head_size, int block) {
  return head_size <= kQ8KVMaxHead && (block == 16 || block == 32 || block == 64 || block == 128);
}

// The checks every operator makes; THABLAS_STATUS_SUCCESS and `l` filled, or the status to return.
inline thablasStatus_t q8kv_layer(const thablasHandle_t* handle, const Q8KVCache* c, int layer, int n_batches,
                                  int n_tokens, const int* pos_d, const int* n_d, Q8KVLayer& l) {
  if (!handle) return THABLAS_STATUS_HANDLE_IS_NULLPTR;
  if (handle->current_gpu_id < 0 || !c || layer < 0 || n_batches < 0 || n_tokens < 0) return THABLAS_STATUS_INVALID_VALUE;
  if (!q8kv_sizes_ok(c->n_batches, c->n_layers, c->n_kv_heads, c->head_size, c->seq_len) || c->block <= 0)
    return THABLAS_STATUS_INVALID_VALUE;
  if (layer >= c->n_layers || n_batches > c->n_batches) return THABLAS_STATUS_INVALID_VALUE;
  if (!q8kv_supported(c->head_size, c->block)) return THABLAS_STATUS_NOT_SUPPORTED;
  if (!q8kv_codes(c->n_batches, c->n_layers, c->n_kv_heads, c->head_size, c->seq_len, c->block)) return THABLAS_STATUS_INVALID_VALUE;
  if (n_batches && n_tokens && (!pos_d || !c->k || !c->v || !c->ks || !c->vs)) return THABLAS_STATUS_INVALID_VALUE;
  if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return THABLAS_STATUS_INVALID_VALUE;
  if (((uintptr_t)c->ks | (uintptr_t)c->vs | (uintptr_t)pos_d | (uintptr_t)n_d) & 3) return THABLAS_STATUS_INVALID_VALUE;
  const long long slots = q8kv_slots(c->seq_len, c->block);
  l.heads = c->n_kv_heads;
  l.head_size = c->head_size;
  l.lanes = q8kv_lanes(c->head_size);
  l.seq_len = c->seq_len;
  l.block_log2 = __builtin_ctz((unsigned)c->block);
  l.head_codes = slots * l.lanes;
  l.head_scales = slots >> l.block_log2;
  l.seq_codes = l.head_codes * l.heads * c->n_layers;
  l.seq_scales = l.head_scales * l.heads * c->n_layers;
  const long long lc = l.head_codes * l.heads * layer, ls = l.head_scales * l.heads * layer;
  l.k = c->k + lc;
  l.v = c->v + lc;
  l.ks = c->ks + ls;
  l.vs = c->vs + ls;
  return THABLAS_STATUS_SUCCESS;
}

// A launch takes fewer than 2^32 threads.
inline bool q8kv_grid_ok(unsigned __int128 grid, int threads) { return grid * threads <= 0xffffffffu; }

// Rows of `row` floats, `stride` apart, at p: float4 accesses hold if everything is a multiple of 16 bytes.
inline bool q8kv_vec4(int head_size, int stride, const void* p, const void* q) {
  return head_size % 4 == 0 && stride % 4 == 0 && (((uintptr_t)p | (uintptr_t)q) & 15) == 0;
}

// Launches go to the handle's device, whichever is current.
struct Q8KVDevice {
  int before = -1;
  bool ok = true;
  explicit Q8KVDevice(int dev) {
    int cur = 0;
    if (hipGetDevice(&cur) != hipSuccess) {
      (void)hipGetLastError();
      ok = false;
      return;
    }
    if (cur == dev) return;
    ok = hipSetDevice(dev) == hipSuccess;
    if (ok) before = cur;
    else (void)hipGetLastError();  // this call's status reports it
  }
  ~Q8KVDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
  Q8KVDevice(const Q8KVDevice&) = delete;
  Q8KVDevice& operator=(const Q8KVDevice&) = delete;
};

inline thablasStatus_t q8kv_status(hipError_t e) {
  return e == hipSuccess ? THABLAS_STATUS_SUCCESS : THABLAS_STATUS_EXECUTION_FAILED;
}

}  // namespace tl
