// thaDNN_q8_kv.hpp — the K/V cache held in int8, and the attention that reads it.  Additions beside the
// fp32 cache and its three-kernel attention (thaDNN_mha.hpp): the reference has no 8-bit cache.
//
// A cache holds int8 codes with one fp32 scale for each block of `block` tokens of a (sequence, layer,
// K/V head).  Codes and scales are runq's (runq.c:145-171):
//   scale = max |x| / 127 over the block's values, code = round(x / scale), half away from zero,
// both quotients rounded to fp32; a value reads back as code * scale.  A scale below the smallest normal
// float is 0, and so are its codes.  A block that holds a value that is not finite has a scale of NaN: it
// reads back as NaN until a store that begins at its first token makes it anew.
#pragma once
#include <stddef.h>
#include <stdint.h>
#include "../thaBLAS.hpp"
#ifdef __cplusplus
extern "C" {
#endif

// Host struct of DEVICE pointers.  With slots = seq_len rounded up to a multiple of max(64, block) and
// lanes = head_size rounded up to a multiple of 16:
//   k   [n_batches][n_layers][n_kv_heads][slots][lanes]          a key's codes side by side
//   v   [n_batches][n_layers][n_kv_heads][slots/16][lanes][16]   16 tokens of one dimension side by side
//   ks, vs [n_batches][n_layers][n_kv_heads][slots/block]
// k and v are 16-byte aligned.  No call needs what the buffers hold at first.
typedef struct {
  int8_t* k;
  int8_t* v;
  float* ks;
  float* vs;
  int n_batches, n_layers, n_kv_heads;
  int head_size;  // 1 .. 256
  int seq_len;    // positions 0 .. seq_len - 1; at most 2^30
  int block;      // tokens of a scale: 16, 32, 64 or 128
} Q8KVCache;

// Bytes of one allocation that holds all four parts; 0 for sizes that no cache has.
size_t thallama_q8_kv_bytes(int n_batches, int n_layers, int n_kv_heads, int head_size, int seq_len, int block);
// Points *c into mem, a device allocation of thallama_q8_kv_bytes(...) bytes, aligned to 256.  0 on success, -1 for bad arguments.
int thallama_q8_kv_map(Q8KVCache* c, void* mem, int n_batches, int n_layers, int n_kv_heads, int head_size, int seq_len, int block);

// The three operators work on one layer of sequences 0 .. n_batches - 1, each with up to n_tokens rows:
// row i < n_d[b] of sequence b is at position pos_d[b] + i.  pos_d and n_d are DEVICE int arrays (read when
// the kernels run, so a captured graph follows what they hold then); n_d may be NULL: n_tokens rows each.
// Row i of sequence b begins at (b*n_tokens + i) * stride floats; strides are in floats.  Counts outside
// 0 .. n_tokens are taken as the nearest one of these.  No access leaves the cache or the rows, whatever
// pos_d and n_d hold.  All work is enqueued on handle->calc_stream of device handle->current_gpu_id.
// Statuses: HANDLE_IS_NULLPTR; INVALID_VALUE for null or misaligned pointers, negative or inconsistent
// sizes; NOT_SUPPORTED for a head size or block outside the ranges above, or more work than one launch holds.

// Quantises rows k, v [n_batches][n_tokens][n_kv_heads * head_size] into the cache.  Rows at positions outside
// 0 .. seq_len - 1 are dropped.  In a block that holds tokens below pos_d[b] the scale only grows, and when it
// does, those tokens' codes are made again from the values they stand for; tokens from pos_d[b] on are taken
// as not yet written.  (The codes of a block so depend on how its tokens were divided into calls, within half a
// step for each growth.)  What lies behind the last written token is left as it was.
thablasStatus_t thaDNN_q8_kv_store_batch(thablasHandle_t* handle, const Q8KVCache* c, int layer, int n_batches,
                                         int n_tokens, const int* pos_d, const int* n_d, const float* k,
                                         const float* v, int kv_stride);

// Reads rows back to fp32.  Rows from n_d[b] on, and rows at positions outside 0 .. seq_len - 1, are left as
// they were.  k or v may be NULL: that one is not read.
thablasStatus_t thaDNN_q8_kv_load_batch(thablasHandle_t* handle, const Q8KVCache* c, int layer, int n_batches,
                                        int n_tokens, const int* pos_d, const int* n_d, float* k, float* v,
                                        int kv_stride);

// Bytes of workspace that thaDNN_q8_attention_batch may use for the cache's sequences, whatever their number and rows
// (0 for arguments that the call refuses).
size_t thaDNN_q8_attention_workspace(const Q8KVCache* c, int n_batches, int n_tokens, int n_heads);

// Causal attention of n_heads query heads over the cache, query head h with K/V head h / (n_heads / n_kv_heads):
//   out_i[h] = sum_{t <= p} softmax_t(q_i[h] . k_t / sqrtf(head_size)) v_t,   p = pos_d[b] + i
// in fp32's accuracy: q is taken to 2^-24 of its row's largest component, and to 2^-47 where that is past some 34 times the
// others; a weight times its value block's scale to 2^-24 of the largest such product among up to 256 keys around it, and to
// 2^-48 of it where the row's sums are under 6 to 16 times that product (so that a key of most of the weight and of small
// values costs the others no accuracy); or to 2^-64 of the largest scale, if that is more.
// A decode step is n_tokens = 1 after its token's store, a prompt's chunk n_tokens > 1.
// A row at a position outside 0 .. seq_len - 1 sees no key: zeros.  Rows from n_d[b] on are left as they were.
// q and out are [n_batches][n_tokens][n_heads * head_size] and do not overlap.  work (16-byte aligned) is zeroed once,
// before its first call, and then left to these calls, of any shape: each leaves it ready for the next.  The zeroing is
// done before that call's kernel runs: by thallama_memset, which waits for it, or by hipMemsetAsync on
// handle->calc_stream, outside any capture (a plain hipMemset is not ordered before that stream).  work belongs to a call
// until its kernel has run: calls that may run at once, captured ones among them, have one each.  A call during which
// pos_d or n_d change leaves it to be zeroed again.
thablasStatus_t thaDNN_q8_attention_batch(thablasHandle_t* handle, const Q8KVCache* c, int layer, int n_batches,
                                          int n_tokens, const int* pos_d, const int* n_d, int n_heads,
                                          const float* q, float* out, int q_stride, int out_stride, void* work,
                                          size_t work_bytes);

#ifdef __cplusplus
}
#endif
