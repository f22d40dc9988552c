// q8_attn.hip — causal attention over the int8 K/V cache (include/thaDNN/thaDNN_q8_kv.hpp).
//
//   out = sum_t 2^(x_t - m) v_t / sum_t 2^(x_t - m),   x_t = log2(e) / sqrt(head_size) q . k_t,  k_t = sk c_t,  v_t = sv c_t
//
// Both products run on the int8 matrix cores with the cache's codes as they are, and still have fp32's accuracy.
// The fp32 factor on the other side is held as a 24-bit integer n = d2 2^16 + d1 2^8 + d0 of three signed bytes
// (balanced digits: the bytes of n + 0x808080, each less 128), so
//   sum n c = 2^16 sum d2 c + (2^8 sum d1 c + sum d0 c),
// three exact int8 products with int32 sums.  For the scores n = q / 2^e 0x7f7f7f, with 2^e the power of two over a
// row's largest |q|: off by 2^-24 of that, as an fp32 number is.  For the values it is the softmax weight times the
// value block's scale, w_t = 2^(x_t - m) sv_t, which is what has to be small beside the row's largest w: with
// sv = f 2^e, 1/2 <= f < 1, the running maximum is taken of x_t + e_t, u_t = 2^(x_t + e_t - M) is at most 1 and
// n_t = u_t f_t 0x7f7f7f.  The sum of the weights adds u_t 2^(E - e_t), E the largest e so far; value scales under
// 2^(E - 40) count as that e with a smaller f, so that u_t cannot vanish where its weight does not.
//
// One i8 product does 16x16x64 in the time in which fp32's does 16x16x8 on eight times the registers; the cache
// is read as it is, without a conversion.
//
// Layout.  S^T = K Q^T and O^T = V^T W^T: a lane holds one query row (column lane & 15) throughout, and with the
// group g = lane >> 4 the sixteen keys 16g .. 16g + 15 of a tile of 64.  The score product's row m of its j-th
// 16-key step is key 16 (m >> 2) + 4 j + (m & 3), so that the lane's four results of step j are keys 16g + 4j .. + 3
// and the four steps together the sixteen bytes that the value product's second operand wants from that lane; the
// cache's value layout (16 tokens of a dimension side by side) is its first operand.  Nothing crosses lanes but
// the row maximum.
#include "q8_kv.hpp"

namespace tl {

typedef int i4 __attribute__((ext_vector_type(4)));

constexpr float kDigits = 8355711.f;  // 0x7f7f7f, the largest n whose balanced digits fit three signed bytes
constexpr float kNone = -1e30f;       // a maximum over nothing

struct Q8AttnArgs {
  Q8KVLayer l;
  Q8KVCall call;
  const float* q;
  float* out;
  float* part;  // nsplit > 1: [unit][split][row of the tile][head_size + 4] (sums, then M, sum of weights, E)
  long long q_stride, out_stride;
  int n_heads, mul;  // query heads, and how many of them share a K/V head
  int tiles;         // row tiles of a (sequence, K/V head)
  int nsplit;        // workgroups that share a row tile's keys
  int lrows;         // rows of a tile that any sequence can have
  int vec;           // rows are 16-byte aligned
  float c0;          // log2(e) / sqrt(head_size) / kDigits
};

// ---- lanes l, l ^ 16, l ^ 32, l ^ 48 hold one query row
TL_DEVICE float rows_max(float v) {
  v2u r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
}
TL_DEVICE float rows_sum(float v) {
  v2u r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r.x) + __uint_as_float(r.y);
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r.x) + __uint_as_float(r.y);
}
TL_DEVICE unsigned rows_umax(unsigned v) {
  v2u r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  v = max(r.x, r.y);
  r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return max(r.x, r.y);
}

// Balanced digits of four 24-bit integers (in the low bytes of t) as bytes 0 .. 3 of three words, lowest digit first.
TL_DEVICE void digits4(const unsigned (&n)[4], int& p0, int& p1, int& p2) {
  unsigned t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = (n[i] + 0x808080u) ^ 0x808080u;
  const unsigned a = __builtin_amdgcn_perm(t[1], t[0], 0x05010400u), b = __builtin_amdgcn_perm(t[3], t[2], 0x05010400u);
  const unsigned c = __builtin_amdgcn_perm(t[1], t[0], 0x0c0c0602u), d = __builtin_amdgcn_perm(t[3], t[2], 0x06020c0cu);
  p0 = (int)__builtin_amdgcn_perm(b, a, 0x05040100u);
  p1 = (int)__builtin_amdgcn_perm(b, a, 0x07060302u);
  p2 = (int)(c | d);
}

TL_DEVICE i4 mfma(i4 a, i4 b, i4 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }

// A wave's state for QT tiles of 16 query rows.  KS = steps of 64 dimensions.
template <int KS, int QT>
struct AttnWave {
  static constexpr int DT = 4 * KS;  // value tiles of 16 dimensions
  i4 q[QT][3][KS];                   // query digits, lowest first
  int qe[QT];                        // their power of two
  float qn[QT];                      // 1, or NaN for a query that is not finite
  int seen[QT];                      // keys that the row sees
  float M[QT], sum[QT];
  f4 o[QT][DT];
  int E;
};

template <int KS, int QT>
TL_DEVICE void attn_begin(AttnWave<KS, QT>& s, const Q8AttnArgs& a, int b, int h, int r0, int rows, long long pos) {
  const int lane = threadIdx.x & 63, kg = lane >> 4;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = r0 + 16 * t + (lane & 15);
    const bool in = r < rows;
    const int i = in ? r / a.mul : 0;
    const long long p = pos + i;
    s.seen[t] = in && p >= 0 && p < a.l.seq_len ? (int)p + 1 : 0;
    const float* src = a.q + ((long long)b * a.call.n_tokens + i) * a.q_stride +
                       (long long)(h * a.mul + (in ? r - i * a.mul : 0)) * a.l.head_size;
    float x[KS][16];
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int d = 64 * k + 16 * kg;
      if (a.vec) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          f4 v = {0.f, 0.f, 0.f, 0.f};
          if (in && d + e < a.l.head_size) v = *reinterpret_cast<const f4*>(src + d + e);
#pragma unroll
          for (int c = 0; c < 4; ++c) x[k][e + c] = v[c];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) x[k][e] = in && d + e < a.l.head_size ? src[d + e] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(x[k][e]) & 0x7fffffffu);
    }
    top = rows_umax(top);
    s.qn[t] = top < 0x7f800000u ? 1.f : __builtin_nanf("");
    s.qe[t] = top < 0x7f800000u ? __builtin_amdgcn_frexp_expf(__uint_as_float(top)) : 0;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        unsigned n[4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
          n[c] = (unsigned)(int)rintf(__builtin_ldexpf(x[k][4 * e + c], -s.qe[t]) * kDigits);
        int p0, p1, p2;
        digits4(n, p0, p1, p2);
        s.q[t][0][k][e] = p0;
        s.q[t][1][k][e] = p1;
        s.q[t][2][k][e] = p2;
      }
    s.M[t] = kNone;
    s.sum[t] = 0.f;
#pragma unroll
    for (int d = 0; d < 4 * KS; ++d) s.o[t][d] = f4{0.f, 0.f, 0.f, 0.f};
  }
  s.E = -126;
}

// NT tiles of 64 keys from t0 on.
template <int KS, int QT, int NT>
TL_DEVICE void attn_keys(AttnWave<KS, QT>& s, const Q8AttnArgs& a, const int8_t* k, const int8_t* v, const float* ks,
                         const float* vs, int t0, int T) {
  constexpr int DT = 4 * KS;
  const int lane = threadIdx.x & 63, row = lane & 15, g = lane >> 4;
  const int lanes = a.l.lanes;

  // scales of this lane's sixteen keys in each tile; those of keys that nobody sees are 0
  float sk[NT], f[NT], lift[NT];
  int e[NT];
  int top = s.E;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int t = t0 + 64 * n + 16 * g;
    const bool in = t < T;
    const int j = min(t, T - 1) >> a.l.block_log2;
    sk[n] = in ? ks[j] : 0.f;
    f[n] = in ? vs[j] : 0.f;
    e[n] = f[n] > 0.f ? __builtin_amdgcn_frexp_expf(f[n]) : -126;
    top = max(top, e[n]);
  }
  {
    v2u r = __builtin_amdgcn_permlane32_swap((unsigned)top, (unsigned)top, false, false);
    top = max((int)r.x, (int)r.y);
    r = __builtin_amdgcn_permlane16_swap((unsigned)top, (unsigned)top, false, false);
    top = max((int)r.x, (int)r.y);
  }
  const int grow = top - s.E;
  s.E = top;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    e[n] = max(e[n], top - 40);
    lift[n] = f[n] == f[n] ? __builtin_ldexpf(1.f, top - e[n]) : f[n];  // a NaN scale makes the sum NaN
    f[n] = __builtin_ldexpf(f[n], -e[n]) * kDigits;
  }

  // scores
  i4 p[QT][NT][3];
  float alpha[QT];
  f4 x[QT][NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float c1[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) c1[t] = __builtin_ldexpf(a.c0 * sk[n], s.qe[t]) * s.qn[t];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int8_t* kp = k + (long long)(t0 + 64 * n + 16 * (row >> 2) + 4 * j + (row & 3)) * lanes;
      i4 key[KS];
#pragma unroll
      for (int c = 0; c < KS; ++c) {
        const int d = 64 * c + 16 * g;
        key[c] = *reinterpret_cast<const i4*>(kp + (d < lanes ? d : 0));  // the query's digits are 0 from lanes on
      }
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        i4 hi = {0, 0, 0, 0}, lo = {0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < KS; ++c) {
          hi = mfma(key[c], s.q[t][2][c], hi);
          lo = mfma(key[c], s.q[t][1][c], lo);
        }
        lo <<= 8;
#pragma unroll
        for (int c = 0; c < KS; ++c) lo = mfma(key[c], s.q[t][0][c], lo);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[t][n][j][i] = fmaf((float)hi[i], 65536.f * c1[t], fmaf((float)lo[i], c1[t], (float)e[n]));
      }
    }
  }

  // weights
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    float m = kNone;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int first = t0 + 64 * n + 16 * g;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (first + 4 * j + i >= s.seen[t]) x[t][n][j][i] = -INFINITY;
          m = fmaxf(m, x[t][n][j][i]);
        }
    }
    m = fmaxf(rows_max(m), s.M[t]);
    alpha[t] = __builtin_amdgcn_exp2f(s.M[t] - m);
    s.M[t] = m;
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int first = t0 + 64 * n + 16 * g;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float u = __builtin_amdgcn_exp2f(x[t][n][j][i] - m);
          sum = first + 4 * j + i >= s.seen[t] ? sum : fmaf(u, lift[n], sum);  // 0 x NaN of a block behind the row
          w[i] = __float_as_uint(fmaf(u, f[n], 8388608.f));  // its low bytes: the nearest integer
        }
        int p0, p1, p2;
        digits4(w, p0, p1, p2);
        p[t][n][0][j] = p0;
        p[t][n][1][j] = p1;
        p[t][n][2][j] = p2;
      }
    }
    s.sum[t] = fmaf(__builtin_ldexpf(s.sum[t], grow), alpha[t], sum);
  }

  // values
  const int8_t* vp = v + (long long)((t0 >> 4) + g) * (16 * lanes) + 16 * row;
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    if (16 * d >= lanes) continue;
    i4 val[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) val[n] = *reinterpret_cast<const i4*>(vp + (long long)(64 * n) * lanes + 256 * d);
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      i4 hi = {0, 0, 0, 0}, lo = {0, 0, 0, 0};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        hi = mfma(val[n], p[t][n][2], hi);
        lo = mfma(val[n], p[t][n][1], lo);
      }
      lo <<= 8;
#pragma unroll
      for (int n = 0; n < NT; ++n) lo = mfma(val[n], p[t][n][0], lo);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s.o[t][d][i] = fmaf(s.o[t][d][i], alpha[t], fmaf((float)hi[i], 65536.f, (float)lo[i]));
    }
  }
}

// What a wave, a workgroup or a split knows of a row: sum_t 2^(x_t) v_t = 2^M o and sum_t 2^(x_t) = 2^(M - E) sum.
struct RowPart {
  float M, sum, E;
};
TL_DEVICE void row_join(float M, float E, const RowPart& r, float& wo, float& ws) {
  wo = __builtin_amdgcn_exp2f(r.M - M);
  ws = r.sum == 0.f ? 0.f : __builtin_amdgcn_exp2f((r.M - M) + (E - r.E)) * r.sum;
}

// One workgroup: QT tiles of 16 query rows of one (sequence, K/V head), and of their keys the share of split
// blockIdx's low part; its waves take runs of 64-key tiles.
template <int KS, int QT>
__global__ void __launch_bounds__(256) k_q8_attn(Q8AttnArgs a) {
  keep_implicit_args();  // common.hpp: rocprofv3 --pmc needs the hidden kernargs
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const Q8KVLayer& l = a.l;
  constexpr int R = 16 * QT;
  unsigned u = blockIdx.x;
  const int split = u % a.nsplit;
  u /= a.nsplit;
  const unsigned unit = u;
  const unsigned pairs = a.call.n_batches * l.heads;
  const int tile = a.tiles - 1 - u / pairs;  // the longest rows first
  u %= pairs;
  const int h = u % l.heads, b = u / l.heads;
  const int count = a.call.n_d ? min(max(a.call.n_d[b], 0), a.call.n_tokens) : a.call.n_tokens;
  const int rows = count * a.mul, r0 = tile * R;
  if (r0 >= rows) return;
  const long long pos = a.call.pos_d[b];
  const int nr = min(R, rows - r0);
  const int T = pos + r0 / a.mul >= l.seq_len ? 0 : (int)max(0LL, min(pos + (r0 + nr - 1) / a.mul + 1, (long long)l.seq_len));

  const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6, lane = threadIdx.x & 63;
  const int tiles = (T + 63) / 64, share = (tiles + a.nsplit - 1) / a.nsplit;
  const int lo = min(tiles, split * share), hi = min(tiles, lo + share);
  const int each = (hi - lo + waves - 1) / waves;
  const int from = __builtin_amdgcn_readfirstlane(min(hi, lo + wave * each));
  const int to = __builtin_amdgcn_readfirstlane(min(hi, from + each));

  AttnWave<KS, QT> s;
  attn_begin<KS, QT>(s, a, b, h, r0, rows, pos);
  const int8_t* k = l.k + b * l.seq_codes + h * l.head_codes;
  const int8_t* v = l.v + b * l.seq_codes + h * l.head_codes;
  const float* ks = l.ks + b * l.seq_scales + h * l.head_scales;
  const float* vs = l.vs + b * l.seq_scales + h * l.head_scales;
  int at = from;
  for (; at + 2 <= to; at += 2) attn_keys<KS, QT, 2>(s, a, k, v, ks, vs, 64 * at, T);
  if (at < to) attn_keys<KS, QT, 1>(s, a, k, v, ks, vs, 64 * at, T);

  // join the waves' rows
  const int hs = l.head_size, step = 64 * KS + 4;
  float* stat = lds + waves * a.lrows * step;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = 16 * t + (lane & 15);
    s.sum[t] = rows_sum(s.sum[t]);
    if (r >= nr) continue;
    float* dst = lds + (wave * a.lrows + r) * step + 4 * (lane >> 4);
#pragma unroll
    for (int d = 0; d < 4 * KS; ++d) *reinterpret_cast<f4*>(dst + 16 * d) = s.o[t][d];
    if (lane < 16) {
      stat[3 * (wave * a.lrows + r)] = s.M[t];
      stat[3 * (wave * a.lrows + r) + 1] = s.sum[t];
      stat[3 * (wave * a.lrows + r) + 2] = (float)s.E;
    }
  }
  __syncthreads();
  const int quads = (hs + 3) / 4;
  for (int it = threadIdx.x; it < nr * quads; it += blockDim.x) {
    const int r = it / quads, d = (it - r * quads) * 4;
    float M = kNone, E = -126.f;
    for (int w = 0; w < waves; ++w) {
      M = fmaxf(M, stat[3 * (w * a.lrows + r)]);
      E = fmaxf(E, stat[3 * (w * a.lrows + r) + 2]);
    }
    f4 o = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
    for (int w = 0; w < waves; ++w) {
      const float* st = stat + 3 * (w * a.lrows + r);
      float wo, ws;
      row_join(M, E, {st[0], st[1], st[2]}, wo, ws);
      const f4 x = *reinterpret_cast<const f4*>(lds + (w * a.lrows + r) * step + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], wo, o[e]);
      sum += ws;
    }
    if (a.nsplit > 1) {
      float* dst = a.part + (((long long)unit * a.nsplit + split) * R + r) * (hs + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (d + e < hs) dst[d + e] = o[e];
      if (d == 0) {
        dst[hs] = M;
        dst[hs + 1] = sum;
        dst[hs + 2] = E;
      }
      continue;
    }
    const int i = (r0 + r) / a.mul;
    float* dst = a.out + ((long long)b * a.call.n_tokens + i) * a.out_stride + (long long)(h * a.mul + r0 + r - i * a.mul) * hs + d;
    const float inv = 1.f / (sum * kDigits);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = M == kNone && sum == 0.f ? 0.f : __builtin_ldexpf(o[e] * inv, (int)E);
    if (a.vec) {
      *reinterpret_cast<f4*>(dst) = o;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (d + e < hs) dst[e] = o[e];
    }
  }
}

// Joins the splits of one (row tile, row): one wave each, lanes along the dimensions.
__global__ void __launch_bounds__(64) k_q8_attn_join(Q8AttnArgs a, int R) {
  keep_implicit_args();  // common.hpp
  const int lane = threadIdx.x, hs = a.l.head_size;
  const int r = blockIdx.x % R;
  const unsigned unit = blockIdx.x / R, pairs = a.call.n_batches * a.l.heads;
  const int tile = a.tiles - 1 - unit / pairs, h = unit % pairs % a.l.heads, b = unit % pairs / a.l.heads;
  const int count = a.call.n_d ? min(max(a.call.n_d[b], 0), a.call.n_tokens) : a.call.n_tokens;
  const int row = tile * R + r;
  if (row >= count * a.mul) return;
  const float* src = a.part + ((long long)unit * a.nsplit * R + r) * (hs + 4);
  const long long step = (long long)R * (hs + 4);
  float M = kNone, E = -126.f;
  for (int s = 0; s < a.nsplit; ++s) {
    M = fmaxf(M, src[s * step + hs]);
    E = fmaxf(E, src[s * step + hs + 2]);
  }
  const int i = row / a.mul;
  float* dst = a.out + ((long long)b * a.call.n_tokens + i) * a.out_stride + (long long)(h * a.mul + row - i * a.mul) * hs;
  for (int d = lane; d < hs; d += 64) {
    float o = 0.f, sum = 0.f;
    for (int s = 0; s < a.nsplit; ++s) {
      const float* st = src + s * step + hs;
      float wo, ws;
      row_join(M, E, {st[0], st[1], st[2]}, wo, ws);
      o = fmaf(src[s * step + d], wo, o);
      sum += ws;
    }
    dst[d] = M == kNone && sum == 0.f ? 0.f : __builtin_ldexpf(o / (sum * kDigits), (int)E);
  }
}

constexpr int kAttnBlocks = 512;  // workgroups that keep the card's 256 CUs busy

// How a call's rows and keys are divided.
struct AttnPlan {
  int qt, waves, nsplit;
  long long tiles, units;
};
static AttnPlan attn_plan(const Q8KVCache* c, int n_batches, int n_tokens, int n_heads) {
  AttnPlan p;
  const long long rows = (long long)n_tokens * (n_heads / c->n_kv_heads), pairs = (long long)n_batches * c->n_kv_heads;
  p.qt = rows > 16 && c->head_size <= 128 && pairs * ((rows + 31) / 32) >= kAttnBlocks ? 2 : 1;
  p.tiles = (rows + 16 * p.qt - 1) / (16 * p.qt);
  p.units = pairs * p.tiles;
  p.waves = 4;
  const long long most = (c->seq_len + 64LL * p.waves - 1) / (64 * p.waves);  // every wave has a tile to do
  p.nsplit = (int)max(1LL, min(most, min(64LL, kAttnBlocks / p.units)));
  return p;
}

template <int KS, int QT>
static hipError_t attn_launch(const Q8AttnArgs& a, const AttnPlan& p, hipStream_t s) {
  const size_t lds = (size_t)p.waves * a.lrows * (64 * KS + 4 + 3) * sizeof(float);
  if (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)k_q8_attn<KS, QT>, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((k_q8_attn<KS, QT>), dim3((unsigned)(p.units * p.nsplit)), dim3(64 * p.waves), lds, s, a);
  return hipGetLastError();
}

}  // namespace tl

static bool attn_sizes_ok(const Q8KVCache* c, int n_heads) {
  return n_heads > 0 && n_heads % c->n_kv_heads == 0;
}

extern "C" size_t thaDNN_q8_attention_workspace(const Q8KVCache* c, int n_batches, int n_tokens, int n_heads) {
  if (!c || n_batches <= 0 || n_tokens <= 0 || !tl::q8kv_sizes_ok(c->n_batches, c->n_layers, c->n_kv_heads, c->head_size, c->seq_len) ||
      !tl::q8kv_supported(c->head_size, c->block) || !attn_sizes_ok(c, n_heads))
    return 0;
  // a call of fewer rows may split its keys among more workgroups, but never has more than this many parts
  const long long rows = (long long)n_tokens * (n_heads / c->n_kv_heads), units = (long long)n_batches * c->n_kv_heads * ((rows + 15) / 16);
  const long long parts = units < tl::kAttnBlocks ? units * 64 : tl::kAttnBlocks;
  return (size_t)(parts < tl::kAttnBlocks ? parts : tl::kAttnBlocks) * 16 * (c->head_size + 4) * sizeof(float);
}

extern "C" thablasStatus_t thaDNN_q8_attention_batch(thablasHandle_t* handle, const Q8KVCache* c, int layer,
                                                     int n_batches, int n_tokens, const int* pos_d, const int* n_d,
                                                     int n_heads, const float* q, float* out, int q_stride,
                                                     int out_stride, void* work, size_t work_bytes) {
  tl::Q8AttnArgs a = {};
  const thablasStatus_t ok = tl::q8kv_layer(handle, c, layer, n_batches, n_tokens, pos_d, n_d, a.l);
  if (ok != THABLAS_STATUS_SUCCESS) return ok;
  if (!attn_sizes_ok(c, n_heads)) return THABLAS_STATUS_INVALID_VALUE;
  const long long row = (long long)n_heads * c->head_size;
  if (q_stride < row || out_stride < row || (((uintptr_t)q | (uintptr_t)out) & 3)) return THABLAS_STATUS_INVALID_VALUE;
  if (n_batches == 0 || n_tokens == 0) return THABLAS_STATUS_SUCCESS;
  if (!q || !out) return THABLAS_STATUS_INVALID_VALUE;
  const int mul = n_heads / c->n_kv_heads;
  const tl::AttnPlan p = tl::attn_plan(c, n_batches, n_tokens, n_heads);
  if ((long long)n_tokens * mul > 0x7fffffffLL - 64 || p.units * p.nsplit > 0x7fffffffLL / 16) return THABLAS_STATUS_NOT_SUPPORTED;
  const size_t need = p.nsplit > 1 ? (size_t)p.units * p.nsplit * 16 * p.qt * (c->head_size + 4) * sizeof(float) : 0;
  if (need && (!work || ((uintptr_t)work & 15) || work_bytes < need)) return THABLAS_STATUS_INVALID_VALUE;
  a.call = {pos_d, n_d, n_batches, n_tokens};
  a.q = q;
  a.out = out;
  a.part = static_cast<float*>(work);
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.n_heads = n_heads;
  a.mul = mul;
  a.tiles = (int)p.tiles;
  a.nsplit = p.nsplit;
  a.lrows = (int)min((long long)n_tokens * mul, 16LL * p.qt);
  a.vec = tl::q8kv_vec4(c->head_size, q_stride, q, out) && out_stride % 4 == 0;
  a.c0 = (float)(1.4426950408889634 / __builtin_sqrt((double)c->head_size) / tl::kDigits);
  tl::Q8KVDevice dev(handle->current_gpu_id);
  if (!dev.ok) return THABLAS_STATUS_INVALID_VALUE;
  const int ks = (a.l.lanes + 63) / 64;
  hipStream_t s = handle->calc_stream;
  hipError_t e;
  if (ks == 1) e = p.qt == 2 ? tl::attn_launch<1, 2>(a, p, s) : tl::attn_launch<1, 1>(a, p, s);
  else if (ks == 2) e = p.qt == 2 ? tl::attn_launch<2, 2>(a, p, s) : tl::attn_launch<2, 1>(a, p, s);
  else e = ks == 3 ? tl::attn_launch<3, 1>(a, p, s) : tl::attn_launch<4, 1>(a, p, s);
  if (e != hipSuccess) return THABLAS_STATUS_EXECUTION_FAILED;
  if (p.nsplit > 1)
    hipLaunchKernelGGL(tl::k_q8_attn_join, dim3((unsigned)(p.units * 16 * p.qt)), dim3(64), 0, s, a, 16 * p.qt);
  return tl::q8kv_status(hipGetLastError());
}
