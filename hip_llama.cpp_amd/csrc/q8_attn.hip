// q8_attn.hip — causal attention over the int8 K/V cache (include/thaDNN/thaDNN_q8_kv.hpp).
//
//   out = sum_t 2^(x_t - m) v_t / sum_t 2^(x_t - m),   x_t = log2(e) / sqrt(head_size) q . k_t,  k_t = sk c_t,  v_t = sv c_t
//
// Both products run on the int8 matrix cores with the cache's codes as they are, and still have fp32's accuracy.
// The fp32 factor on the other side is held as a 24-bit integer n = d2 2^16 + d1 2^8 + d0 of three signed bytes
// (balanced digits: those of n + 0x8080, the lower two less 0x80), so
//   sum n c = 2^16 sum d2 c + (2^8 sum d1 c + sum d0 c),
// three exact int8 products with int32 sums.  For the scores n = q / 2^e 0x7f7f7f, with 2^e the power of two over a
// row's largest |q|: off by 2^-24 of that, as an fp32 number is; rows whose largest is far above the others, which would be
// left few of these bits, take their keys again with three digits more.  For the values it is the softmax weight times the
// value block's scale, w_t = 2^(x_t - m) sv_t, which is what has to be small beside the row's largest w: with
// sv = f 2^e, 1/2 <= f < 1, and E the row's largest e so far, the running maximum M is taken of y_t = x_t + (e_t - E) (as
// exact as x_t itself, whatever the values' size), u_t = 2^(y_t - M) is at most 1 and n_t = u_t f_t 0x7f7f7f.  The sum of
// the weights adds u_t 2^(E - e_t); value scales under 2^(E - 40) count as that e with a smaller f, so that u_t cannot
// vanish where its weight does not; a row is so off by up to 2^-64 of 127 of the largest value scale in sight, too.  M is
// the maximum of one step's 64 to 256 keys, so that a large weight elsewhere costs the step's own no digits; the steps are
// summed in fp32, in units of a power that follows M only where it rises past 2^16 of it.  A large weight on a key of
// small values still costs its neighbours theirs (a model's first token, with nearly all of a row's weight and nothing in
// its values: the row would be 4e-5 to 1e-1 off): where a step leaves a row's sums small its weights get three more digits
// behind these.  Against 64 bits the shapes named at the kernels are 5e-7 to 7e-7 off (2-norm), an fp32 softmax over the
// same codes 2e-7 to 1.8e-6; with such a key in each row, or a large component in each query, both 2e-7 to 2e-6.
//
// The int8 cores' peak is 5 POP/s beside 157 TFLOP/s for fp32 inputs, so three products are still ten times as fast as
// one in fp32, and the cache is read as it is, without a conversion.
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
constexpr float kRound = 8421504.f;   // 2^23 + 0x8080: a sum with it is rounded to a whole number
constexpr float kNone = -3.4e38f;     // a maximum over nothing
constexpr float kLag = 16.f;          // log2 of how far a step's maximum may be past the sums' unit
constexpr int kUnit = 28;             // power of two in c0, so that its product with a key scale is a normal float
constexpr int kWaves = 4;             // of a workgroup
constexpr int kCountStep = 32;        // a cache line for each count of arrivals

struct Q8AttnArgs {
  Q8KVLayer l;
  Q8KVCall call;
  const float* q;
  float* out;
  unsigned* arrived;  // nsplit > 1: [unit] workgroups that have left their part; 0 between calls
  float* part;        // nsplit > 1: [unit][split][lrows][head_size rounded up to 4, + 4]
  long long q_stride, out_stride;
  int mul;           // query heads that share a K/V head
  int tiles;         // row tiles of a (sequence, K/V head)
  int nsplit;        // workgroups that share a row tile's keys
  int lrows;         // rows of a tile that any sequence can have
  int vec;           // rows are 16-byte aligned
  float c0;          // log2(e) / sqrt(head_size) / kDigits 2^kUnit: 2.9 .. 46
};

// A sum of weights beside values so large that it leaves fp32's range: what is divided by it is under 2^-64 of them either
// way, and an infinity would not come back from a factor of 0.  A NaN stays.
TL_DEVICE float sum_kept(float s) { return s > 0x1p120f ? 0x1p120f : s; }

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

// The digits of four integers n, given t = n + 0x8080 with anything above its 24 bits, as bytes 0 .. 3 of three words,
// lowest digit first: the added 0x80s carry, the low bytes less 0x80 are the two lower digits, the third is the top one.
TL_DEVICE void digits4(const unsigned (&t)[4], int& p0, int& p1, int& p2) {
  const unsigned a = __builtin_amdgcn_perm(t[1], t[0], 0x05010400u), b = __builtin_amdgcn_perm(t[3], t[2], 0x05010400u);
  const unsigned c = __builtin_amdgcn_perm(t[1], t[0], 0x0c0c0602u), d = __builtin_amdgcn_perm(t[3], t[2], 0x06020c0cu);
  p0 = (int)(__builtin_amdgcn_perm(b, a, 0x05040100u) ^ 0x80808080u);
  p1 = (int)(__builtin_amdgcn_perm(b, a, 0x07060302u) ^ 0x80808080u);
  p2 = (int)(c | d);
}

TL_DEVICE i4 mfma(i4 a, i4 b, i4 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }

// A wave's state: 16 query rows, this lane's being number lane & 15.  KS = steps of 64 dimensions.
template <int KS>
struct AttnRows {
  i4 q[3][KS];   // query digits, lowest first
  int qe;        // their power of two, less kUnit
  float qn;      // 1, or NaN for a query that is not finite
  int seen;      // keys that the row sees
  float M, sum;  // running maximum (of scores and value exponents, these less E), sum of weights
  f4 o[4 * KS];  // sums over the values: dimensions 16 d + 4 (lane >> 4) .. + 3
  int E;         // largest value exponent that the row has seen

  TL_DEVICE void none() {  // before the first key
    M = kNone;
    sum = 0.f;
    E = -126;
#pragma unroll
    for (int d = 0; d < 4 * KS; ++d) o[d] = f4{0.f, 0.f, 0.f, 0.f};
  }
};

struct AttnUnit {  // what a workgroup works on
  int b, h, r0, rows, nr, T;
  long long pos;
};
// Row tile `tile` of R rows of pair (b, h); false if the sequence has no such rows.
TL_DEVICE bool attn_unit(const Q8AttnArgs& a, unsigned pair, int tile, int R, AttnUnit& w) {
  w.h = pair % a.l.heads;
  w.b = pair / a.l.heads;
  int count;
  q8kv_start(a.call, w.b, w.pos, count);
  w.rows = count * a.mul;
  w.r0 = tile * R;
  if (w.r0 >= w.rows) return false;
  w.nr = min(R, w.rows - w.r0);
  const long long first = w.pos + w.r0 / a.mul, last = w.pos + (w.r0 + w.nr - 1) / a.mul;
  w.T = first >= a.l.seq_len ? 0 : (int)max(0LL, min(last + 1, (long long)a.l.seq_len));
  return true;
}

// This lane's part of row r0 + (lane & 15) of the `rows` of (b, h), and the keys that the row sees.  A row behind the
// last is the last one again; it sees what the tile sees and is never stored.  Every load is made, from inside the row, so that
// none is waited for before the next is asked for.
template <int KS>
TL_DEVICE int attn_query(float (&x)[KS][16], const Q8AttnArgs& a, int b, int h, int r0, int rows, long long pos, int T) {
  const int lane = threadIdx.x & 63, kg = lane >> 4, hs = a.l.head_size;
  const int r = min(r0 + (lane & 15), rows - 1);
  const int i = r / a.mul;
  const long long p = pos + i;
  const float* src = a.q + ((long long)b * a.call.n_tokens + i) * a.q_stride + (long long)(h * a.mul + r - i * a.mul) * hs;
  if (a.vec) {
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const f4 v = *reinterpret_cast<const f4*>(src + min(64 * k + 16 * kg + e, hs - 4));
#pragma unroll
        for (int c = 0; c < 4; ++c) x[k][e + c] = v[c];
      }
  } else {
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int e = 0; e < 16; ++e) x[k][e] = src[min(64 * k + 16 * kg + e, hs - 1)];
  }
  return r0 + (lane & 15) >= rows ? T : p >= 0 && p < a.l.seq_len ? (int)p + 1 : 0;
}

// 0 behind the head's end.
template <int KS>
TL_DEVICE void attn_clip(float (&x)[KS][16], int hs) {
  if (hs >= 64 * KS) return;
  const int left = hs - 16 * ((threadIdx.x & 63) >> 4);
#pragma unroll
  for (int k = 0; k < KS; ++k)
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (64 * k + e >= left) x[k][e] = 0.f;
}

// Three more digits of the query, for rows that need them: 1 / 0x7f7f7f of the others'.
template <int KS, bool WIDE>
struct AttnMore {
  i4 q[3][WIDE ? KS : 1];
};

// The query's digits.  True if they are too few for the row: where a few components are so much larger than the rest that
// these have few of the 24 bits.  Goes by the mean of some of each sixteen components, none taken for more than 2^-5 of the
// largest number, so that up to half of them may be large, and zeros, which need no bits, for as much: under 0.6 of that
// where the largest component is past some 34 times the width of the others' distribution.
template <int KS>
TL_DEVICE bool attn_begin(AttnRows<KS>& s, float (&x)[KS][16], int hs, int seen) {
  s.seen = seen;
  attn_clip<KS>(x, hs);
  unsigned top = 0;
#pragma unroll
  for (int k = 0; k < KS; ++k)
#pragma unroll
    for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(x[k][e]) & 0x7fffffffu);
  top = rows_umax(top);
  s.qn = top < 0x7f800000u ? 1.f : __builtin_nanf("");
  const int qe = top < 0x7f800000u ? __builtin_amdgcn_frexp_expf(__uint_as_float(top)) : 0;
  s.qe = qe - kUnit;
  constexpr float most = kDigits / 32.f;
  constexpr int kSome = KS == 1 ? 8 : 4;
  float size = 0.f;
#pragma unroll
  for (int k = 0; k < KS; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      unsigned n[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float y = __builtin_ldexpf(x[k][4 * e + c], -qe) * kDigits;
        if (4 * e < kSome) size += __uint_as_float(min((__float_as_uint(y) & 0x7fffffffu) - 1u, __float_as_uint(most)));
        n[c] = (unsigned)(int)rintf(y) + 0x8080u;
      }
      int p0, p1, p2;
      digits4(n, p0, p1, p2);
      s.q[0][k][e] = p0;
      s.q[1][k][e] = p1;
      s.q[2][k][e] = p2;
    }
  // with the zeros behind the head's end
  return rows_sum(size) < most * (4.f * KS * kSome - 0.4f * (float)((hs >> 4) * kSome + min(hs & 15, kSome))) && top - 1u < 0x7f7fffffu;
}

// Scales of this lane's sixteen keys in each of NT tiles of 64 from t0 on; behind the last key those of its block.
template <int NT>
struct AttnScales {
  float sk[NT], f[NT], lift[NT];
  int e[NT];
  TL_DEVICE void load(const Q8AttnArgs& a, const float* ks, const float* vs, int lane, int t0, int T) {
    const unsigned g16 = lane & 48, last = (unsigned)(T - 1);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const unsigned j = min(t0 + 64u * n + g16, last) >> a.l.block_log2;
      sk[n] = ks[j];
      f[n] = vs[j];
    }
  }
  // Exponents of the value scales, as far as the row sees their keys (`left` of them, counted from the lane's first tile
  // on): a row's exponent goes by what it sees.
  TL_DEVICE void exponents(bool edge, int left) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      e[n] = f[n] > 0.f ? __builtin_amdgcn_frexp_expf(f[n]) : -126;
      if (edge && 64 * n >= left) e[n] = -126;
    }
  }
  // Their factors, once the row's largest exponent E is known.
  TL_DEVICE void factors(int E) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      e[n] = max(e[n], E - 40);
      lift[n] = f[n] == f[n] ? __builtin_ldexpf(1.f, E - e[n]) : f[n];  // a NaN scale makes the sum NaN
      f[n] = __builtin_ldexpf(f[n], -e[n]) * kDigits;
    }
  }
};

// Scores x_t + (e_t - E) of NT tiles of 64 keys, -inf for those that the row does not see, whose factors become 0.
// key: (tile, 16-key step, 64-dimension step) -> sixteen codes.
template <int KS, int NT, bool WIDE, class Key>
TL_DEVICE void attn_scores(f4 (&x)[NT][4], AttnScales<NT>& c, const AttnRows<KS>& s, const AttnMore<KS, WIDE>& more, const Q8AttnArgs& a, bool edge, int left,
                           Key key) {
  // Each turn asks for the next one's operands, starts this one's products and finishes the last one's, so that neither
  // LDS nor the matrix pipe is waited for.
  {
    constexpr int Z = WIDE ? 6 : 3;
    i4 k[2][KS], acc[2][Z];
    auto digits = [&](int z, int d) { return z < 3 ? s.q[z % 3][d] : more.q[z % 3][WIDE ? d : 0]; };
    float c1 = 0.f, ce = 0.f;
#pragma unroll
    for (int d = 0; d < KS; ++d) k[0][d] = key(0, 0, d);
#pragma unroll
    for (int u = 0; u <= 4 * NT; ++u) {
      if (u + 1 < 4 * NT) {
#pragma unroll
        for (int d = 0; d < KS; ++d) k[(u + 1) & 1][d] = key((u + 1) / 4, (u + 1) & 3, d);
      }
      if (u < 4 * NT) {
#pragma unroll
        for (int z = 0; z < Z; ++z) acc[u & 1][z] = mfma(k[u & 1][0], digits(z, 0), i4{0, 0, 0, 0});
#pragma unroll
        for (int d = 1; d < KS; ++d)
#pragma unroll
          for (int z = 0; z < Z; ++z) acc[u & 1][z] = mfma(k[u & 1][d], digits(z, d), acc[u & 1][z]);
      }
      if (u > 0) {
        const int n = (u - 1) / 4, j = (u - 1) & 3;
        if (j == 0) {
          c1 = __builtin_ldexpf(a.c0 * c.sk[n], s.qe) * s.qn;
          ce = (float)(c.e[n] - s.E);
        }
        const i4(&r)[Z] = acc[(u - 1) & 1];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float y = fmaf((float)r[2][i], 65536.f * c1, fmaf((float)((r[1][i] << 8) + r[0][i]), c1, ce));
          if constexpr (WIDE) y = fmaf(fmaf((float)r[5][i], 65536.f, (float)((r[4][i] << 8) + r[3][i])), c1 * (1.f / kDigits), y);
          x[n][j][i] = y;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (!edge) return;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (64 * n + 4 * j + i >= left) x[n][j][i] = -INFINITY;
#pragma unroll
  for (int n = 0; n < NT; ++n)
    if (64 * n >= left) c.f[n] = c.lift[n] = 0.f;  // a block behind the row may hold NaN
}

// The largest score of the row.
template <int NT>
TL_DEVICE float attn_most(const f4 (&x)[NT][4]) {
  float m = kNone;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) m = fmaxf(m, x[n][j][i]);
  return rows_max(m);
}

// o += beta sum n_t v_t of NT tiles, n_t in the digits p.  val: (tile, 16-dimension step) -> sixteen codes; turns as above.
template <int KS, int NT, class Val>
TL_DEVICE void attn_values(f4 (&o)[4 * KS], const i4 (&p)[NT][3], float beta, Val val) {
  constexpr int DT = 4 * KS;
  i4 v[2][NT], acc[2][3];
#pragma unroll
  for (int n = 0; n < NT; ++n) v[0][n] = val(n, 0);
#pragma unroll
  for (int u = 0; u <= DT; ++u) {
    if (u + 1 < DT) {
#pragma unroll
      for (int n = 0; n < NT; ++n) v[(u + 1) & 1][n] = val(n, u + 1);
    }
    if (u < DT) {
#pragma unroll
      for (int z = 0; z < 3; ++z) acc[u & 1][z] = mfma(v[u & 1][0], p[0][z], i4{0, 0, 0, 0});
#pragma unroll
      for (int n = 1; n < NT; ++n)
#pragma unroll
        for (int z = 0; z < 3; ++z) acc[u & 1][z] = mfma(v[u & 1][n], p[n][z], acc[u & 1][z]);
    }
    if (u > 0) {
      const i4(&r)[3] = acc[(u - 1) & 1];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o[u - 1][i] = fmaf(fmaf((float)r[2][i], 65536.f, (float)((r[1][i] << 8) + r[0][i])), beta, o[u - 1][i]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The codes of a (sequence, K/V head), and the keys that a workgroup's rows see.
struct AttnHead {
  const int8_t *k, *v;
  const float *ks, *vs;
  int T;
  TL_DEVICE AttnHead(const Q8AttnArgs& a, const AttnUnit& w)
      : k(a.l.k + w.b * a.l.seq_codes + w.h * a.l.head_codes), v(a.l.v + w.b * a.l.seq_codes + w.h * a.l.head_codes),
        ks(a.l.ks + w.b * a.l.seq_scales + w.h * a.l.head_scales), vs(a.l.vs + w.b * a.l.seq_scales + w.h * a.l.head_scales), T(w.T) {}
  // This lane's operands of the tile at t0: key step j and dimension step d, values' dimension step d.  Behind the lanes
  // the first ones again: the query's digits are 0 there, and such values are no row's.
  TL_DEVICE const int8_t* key(const Q8AttnArgs& a, int lane, int t0, int j, int d) const {
    const int row = lane & 15, at = 64 * d + 16 * (lane >> 4);
    return k + (long long)(t0 + 16 * (row >> 2) + (row & 3)) * a.l.lanes + 4 * j * a.l.lanes + (at < a.l.lanes ? at : 0);
  }
  TL_DEVICE const int8_t* value(const Q8AttnArgs& a, int lane, int t0, int d) const {
    const int row = lane & 15, g = lane >> 4;
    return v + (long long)((t0 >> 4) + g) * (16 * a.l.lanes) + 16 * row + (16 * d < a.l.lanes ? 256 * d : 0);
  }
};

// One step of NT tiles of 64 keys from t0 on; key and val as above.  ready() runs between the two products.  The rows of
// the wave whose weights need further digits, as bits.
template <int KS, int NT, bool WIDE, class Key, class Val, class Ready>
TL_DEVICE unsigned attn_step(AttnRows<KS>& s, const AttnMore<KS, WIDE>& more, const Q8AttnArgs& a, AttnScales<NT>& c, int t0, bool edge, Key key, Val val,
                             Ready ready) {
  constexpr int DT = 4 * KS;
  const int g = (threadIdx.x & 63) >> 4;
  const int left = s.seen - t0 - 16 * g;  // keys of this lane's first tile and behind it that the row sees
  int top = s.E, grow = 0;
  c.exponents(edge, left);
#pragma unroll
  for (int n = 0; n < NT; ++n) top = max(top, c.e[n]);
  if (__any(top > s.E)) {  // rare behind the first step
    v2u r = __builtin_amdgcn_permlane32_swap((unsigned)top, (unsigned)top, false, false);
    top = max((int)r.x, (int)r.y);
    r = __builtin_amdgcn_permlane16_swap((unsigned)top, (unsigned)top, false, false);
    top = max((int)r.x, (int)r.y);
    grow = top - s.E;
    s.E = top;
    s.M -= (float)grow;  // kNone stays
  }
  c.factors(s.E);
  f4 x[NT][4];
  attn_scores<KS, NT>(x, c, s, more, a, edge, left, key);
  const float m = attn_most<NT>(x);  // of this step alone: it sets the size that the step's weights are rounded to
  // Rare behind the first step (four prompts of 2048 tokens, 32 heads of 128: 278 us; scaled in each step 282).
  const float M = m - kLag > s.M ? __builtin_ceilf(m) : s.M;  // whole, so that it moves by grow without a rounding
  if (__any(M != s.M || grow)) {
    const float alpha = __builtin_amdgcn_exp2f(s.M - M);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) s.o[d][i] *= alpha;
    s.sum = s.sum == 0.f ? 0.f : s.sum * __builtin_amdgcn_exp2f((s.M - M) + (float)grow);  // either alone may be out of range
    s.M = M;
  }
  const float beta = __builtin_amdgcn_exp2f(m - M);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[n][j][i] = __builtin_amdgcn_exp2f(x[n][j][i] - m);
  float sum = 0.f;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float part = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) part += (x[n][j][0] + x[n][j][1]) + (x[n][j][2] + x[n][j][3]);
    sum = fmaf(part, c.lift[n], sum);
  }
  s.sum = sum_kept(fmaf(sum, beta, s.sum));
  i4 p[NT][3];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      unsigned w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(fmaf(x[n][j][i], c.f[n], kRound));  // low bytes n + 0x8080, rounded to nearest
      int p0, p1, p2;
      digits4(w, p0, p1, p2);
      p[n][0][j] = p0;
      p[n][1][j] = p1;
      p[n][2][j] = p2;
    }

  ready();
  attn_values<KS, NT>(s.o, p, beta, val);

  // Too few digits?  Half a unit for each n_t of 64 to 256 keys, of codes up to 127 and about 30 in the mean, is some 50 to
  // 130 units beside the row's sums, which are about 2^28 where one key's ordinary codes are all that counts: few are under
  // 2^25.5 to 2^26 units.  (2^26 at heads of 128 costs calls of one round of workgroups an eighth, 352 tiles of 64 rows 24.4
  // us for 22.7, where blocks with a large token leave the others small codes.)  Looked at in the first 32 dimensions, or 16
  // of fewer; lanes whose four of these go past the head's end have no say.
  constexpr float kFew = KS == 1 ? 0x1p26f : 0x1.6ap25f;
  const float second = KS > 1 || a.l.head_size >= 32 ? 1.f : 0.f;
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) most = fmaxf(most, fmaxf(fabsf(s.o[0][i]), fabsf(s.o[1][i]) * second));
  unsigned long long few = __ballot((most < kFew * beta || (KS == 1 && 4 * g + 4 > a.l.head_size)) && m > kNone);
  few &= few >> 32;
  return (unsigned)(few & (few >> 16)) & 0xffffu;  // all four lanes of a row
}

// The least number of keys that one of the wave's rows sees.
TL_DEVICE int attn_least(int seen) {
  seen = min(seen, __builtin_amdgcn_mov_dpp(seen, 0xB1, 0xF, 0xF, false));   // common.hpp row16_max's steps
  seen = min(seen, __builtin_amdgcn_mov_dpp(seen, 0x4E, 0xF, 0xF, false));
  seen = min(seen, __builtin_amdgcn_mov_dpp(seen, 0x141, 0xF, 0xF, false));
  seen = min(seen, __builtin_amdgcn_mov_dpp(seen, 0x140, 0xF, 0xF, false));
  return __builtin_amdgcn_readfirstlane(seen);
}

// In which of a wave's steps, `step` keys apart and together T, the lane's row needs further digits for its weights: a bit
// for each, or for several where they are more than 32.  A row's own, so that no row depends on its neighbours in the tile.
struct AttnMarks {
  unsigned bits = 0;
  int shift;
  TL_DEVICE AttnMarks(int T, int step) : shift(max(0, __builtin_clz((unsigned)step) - __builtin_clz((unsigned)T | 1u) - 4)) {}
  TL_DEVICE void mark(int i, unsigned rows) { bits |= ((rows >> (threadIdx.x & 15)) & 1u) << (i >> shift); }
};

// What a step's weights have beyond their 24 bits: u_t f_t 0x7f7f7f - n_t, at most 1/2, in three more digits of 2^-24 each.
// A row needs it where one key has far more weight than others and next to nothing in its values (a model's first token),
// in the steps that hold such a key.  Its operands are read again when all keys are through, and taken tile by tile: in the
// loop itself the registers would be short.  With such a first key in every row: one row of 32 heads over 2048 keys 9.1 ->
// 9.9 us, eight to 32768 keys 65.8 -> 68.3, four prompts 278 -> 327.
template <int KS, int NT, bool WIDE>
TL_DEVICE void attn_further(AttnRows<KS>& s, const AttnMore<KS, WIDE>& more, const Q8AttnArgs& a, const AttnHead& h, int t0, bool edge, bool mine) {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // addresses are made here, not ahead and kept in registers
  const int left = s.seen - t0 - 16 * (lane >> 4), tiles = min(NT, (h.T - t0 + 63) / 64);
  f4 x[1][4];
  AttnScales<1> c;
  auto scores = [&](int n) {
    c.load(a, h.ks, h.vs, lane, t0 + 64 * n, h.T);
    c.exponents(edge, left - 64 * n);
    c.factors(s.E);
    attn_scores<KS, 1>(x, c, s, more, a, edge, left - 64 * n, [&](int, int j, int d) { return *reinterpret_cast<const i4*>(h.key(a, lane, t0 + 64 * n, j, d)); });
  };
  float m = kNone;  // the step's
#pragma unroll 1
  for (int n = 0; n < tiles; ++n) {
    scores(n);
    m = fmaxf(m, attn_most<1>(x));
  }
#pragma unroll 1
  for (int n = 0; n < tiles; ++n) {
    if (NT > 1) scores(n);
    i4 p[1][3];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      unsigned w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float u = __builtin_amdgcn_exp2f(x[0][j][i] - m);
        const float whole = fmaf(u, c.f[0], kRound) - kRound;
        w[i] = (unsigned)(int)rintf(fmaf(u, c.f[0], -whole) * (2.f * kDigits)) + 0x8080u;
      }
      int p0, p1, p2;
      digits4(w, p0, p1, p2);
      p[0][0][j] = p0;
      p[0][1][j] = p1;
      p[0][2][j] = p2;
    }
    attn_values<KS, 1>(s.o, p, mine ? __builtin_amdgcn_exp2f(m - s.M) * (0.5f / kDigits) : 0.f,
                       [&](int, int d) { return *reinterpret_cast<const i4*>(h.value(a, lane, t0 + 64 * n, d)); });
  }
}
// The marked ones of a wave's steps 0 .. last, that of number i from key from + i * step on.
template <int KS, int NT, bool WIDE>
TL_DEVICE void attn_marked(AttnRows<KS>& s, const AttnMore<KS, WIDE>& more, const Q8AttnArgs& a, const AttnHead& h, const AttnMarks& marks, int from, int step,
                           int last, int least) {
  if (__builtin_expect(!__any(marks.bits), 1)) return;
#pragma unroll 1
  for (int i = 0; i <= last; ++i) {
    const bool mine = (marks.bits >> (i >> marks.shift)) & 1u;
    if (__any(mine)) attn_further<KS, NT>(s, more, a, h, from + i * step, from + i * step + 64 * NT > least, mine);
  }
}

// These, from the query's values again.
template <int KS>
TL_DEVICE AttnMore<KS, true> attn_more(const AttnRows<KS>& s, const Q8AttnArgs& a, const AttnUnit& w, int r0, bool mine) {
  float x[KS][16];
  (void)attn_query<KS>(x, a, w.b, w.h, r0, w.rows, w.pos, w.T);
  attn_clip<KS>(x, a.l.head_size);
  AttnMore<KS, true> more;
#pragma unroll
  for (int k = 0; k < KS; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      unsigned n[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float y = __builtin_ldexpf(x[k][4 * e + c], -(s.qe + kUnit));
        n[c] = (unsigned)(int)rintf(fmaf(y, kDigits, -rintf(y * kDigits)) * kDigits) + 0x8080u;  // at most 3/4 is left: two roundings
      }
      int p0, p1, p2;
      digits4(n, p0, p1, p2);
      more.q[0][k][e] = mine ? p0 : 0;  // the others' rows stay as they are without
      more.q[1][k][e] = mine ? p1 : 0;
      more.q[2][k][e] = mine ? p2 : 0;
    }
  return more;
}

// A wave's keys, its steps of 64 from key `from` on `step` apart, with six digits of the queries that want them (`mine`).
// Rare, and plain: one row of 32 heads over 2048 keys 9.1 -> 15.4 us, four prompts 278 -> 1216 where every row wants them.
template <int KS>
TL_DEVICE void attn_wide(AttnRows<KS>& s, const Q8AttnArgs& a, const AttnUnit& w, const AttnHead& h, int r0, bool mine, int from, int step, int least) {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // as above
  const AttnMore<KS, true> more = attn_more<KS>(s, a, w, r0, mine);
  AttnMarks marks(h.T, step);
  s.none();
  int i = 0;
#pragma unroll 1
  for (int t0 = from; t0 < h.T; t0 += step, ++i) {
    AttnScales<1> c;
    c.load(a, h.ks, h.vs, lane, t0, h.T);
    marks.mark(i, attn_step<KS, 1>(s, more, a, c, t0, t0 + 64 > least, [&](int, int j, int d) { return *reinterpret_cast<const i4*>(h.key(a, lane, t0, j, d)); },
                                   [&](int, int d) { return *reinterpret_cast<const i4*>(h.value(a, lane, t0, d)); }, [] {}));
  }
  attn_marked<KS, 1>(s, more, a, h, marks, from, step, i - 1, least);
}

// A wave, a workgroup or a split knows of a row sum_t 2^(x_t) v_t = 2^(M + E) o and sum_t 2^(x_t) = 2^M sum.  Joins the
// first n of N such parts, st = (M, sum, E), to one.
template <int N>
TL_DEVICE void parts_join(const f4 (&x)[N], const f4 (&st)[N], int n, f4& o, float& M, float& sum, float& E) {
  float top = E;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) top = fmaxf(top, st[i].z);
  float m = M + (E - top);
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) m = fmaxf(m, st[i].x + (st[i].z - top));
  auto weight = [&](float M1, float sum1) { return sum1 == 0.f ? 0.f : __builtin_amdgcn_exp2f(M1 - m) * sum1; };
  sum = weight(M, sum);
  const float w = __builtin_amdgcn_exp2f(M + (E - top) - m);
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] *= w;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i >= n) continue;
    sum += weight(st[i].x, st[i].y);
    const float wi = __builtin_amdgcn_exp2f(st[i].x + (st[i].z - top) - m);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(x[i][e], wi, o[e]);
  }
  sum = sum_kept(sum);
  M = m;
  E = top;
}

// Where row r of the unit goes, and its sums' factor: 2^e inv.  A row without keys is zeros.
struct AttnOut {
  float* at;
  float inv;
  int e;
  TL_DEVICE AttnOut(const Q8AttnArgs& a, const AttnUnit& w, int r, float M, float sum, float E) {
    const int i = (w.r0 + r) / a.mul;
    at = a.out + ((long long)w.b * a.call.n_tokens + i) * a.out_stride + (long long)(w.h * a.mul + w.r0 + r - i * a.mul) * a.l.head_size;
    inv = M == kNone && sum == 0.f ? 0.f : 1.f / (sum * (kDigits * 0x1p-23f));
    e = (int)E - 23;
  }
  TL_DEVICE void store(const Q8AttnArgs& a, int d, f4 o) const {  // dimensions d .. d + 3
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] = __builtin_ldexpf(o[c] * inv, e);
    if (a.vec) {
      *reinterpret_cast<f4*>(at + d) = o;
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (d + c < a.l.head_size) at[d + c] = o[c];
    }
  }
};

// 16 bytes a lane from memory, at `from` + the lane's offset, to LDS, at `to` + 16 * lane; lds_wait: everybody's have
// arrived.  Written out, because with the builtin the compiler waits for every load under way before the next read of any
// LDS.
TL_DEVICE void lds_bring(const int8_t* from, unsigned offset, i4* to) {
  const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) void*)to);
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(from), "{m0}"(at) : "memory");
}
TL_DEVICE void lds_wait() {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  __syncthreads();
}

// A tile of 64 keys as one wave holds it.  ONCE: no other row tile reads these codes, and they need not stay in L2 (kept
// there, eight rows over 10923 to 32768 keys take 73.7 us for 65.8; not kept, 256 rows of 32 heads over 16640 keys,
// sixteen tiles a head, 228 for 167).
template <int KS, bool ONCE>
struct AttnTile {
  i4 k[4][KS], v[4 * KS];
  AttnScales<1> c;
  TL_DEVICE static i4 codes(const int8_t* p) {
    const i4* q = reinterpret_cast<const i4*>(p);
    return ONCE ? __builtin_nontemporal_load(q) : *q;
  }
  TL_DEVICE void load_keys(const Q8AttnArgs& a, const AttnHead& h, int t0) {
    c.load(a, h.ks, h.vs, threadIdx.x & 63, t0, h.T);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int d = 0; d < KS; ++d) k[j][d] = codes(h.key(a, threadIdx.x & 63, t0, j, d));
  }
  TL_DEVICE void load_values(const Q8AttnArgs& a, const AttnHead& h, int t0) {
#pragma unroll
    for (int d = 0; d < 4 * KS; ++d) v[d] = codes(h.value(a, threadIdx.x & 63, t0, d));
  }
};

// Few rows: one workgroup takes 16 query rows of one (sequence, K/V head) and, of their keys, every nsplit-th run of
// a 64-key tile for each of its waves.  A wave asks for its next keys as soon as the scores are done with these, and for
// its next values when the sums are.  The waves' results are joined in LDS; where several workgroups share a row tile,
// each leaves its result in the workspace and the last one to arrive joins them, in the order of the splits whoever it is.
//
// Long contexts are bound by memory: eight rows of 32 heads over 8 K/V heads of 128 at 10923 to 32768 keys 65.8 us,
// 5.4 TB/s of codes (the vector pipe 27% busy), sixteen rows of 32 heads at 683 to 2048 keys 34.6 us, 5.2 TB/s.  Short ones
// are bound by a chain of latencies: positions, keys, two products and the joins, 12 heads of 64 over 301 keys 6.1 us, 32
// of 128 over 2048 keys 9.1 (0.8 until the positions are there, 2.7 to the first codes, 2 for a tile, 0.9 to join the
// waves, 2.5 the workgroups).
template <int KS, bool ONCE>
__global__ void __launch_bounds__(256, KS == 1 ? 4 : KS < 4 ? 2 : 1) k_q8_attn_few(Q8AttnArgs a) {
  keep_implicit_args();  // common.hpp: rocprofv3 --pmc needs the hidden kernargs
  extern __shared__ __attribute__((aligned(16))) float lds[];
  __shared__ int last;
  const Q8KVLayer& l = a.l;
  unsigned u = blockIdx.x;
  const int split = u % a.nsplit;
  const unsigned unit = u / a.nsplit, pairs = a.call.n_batches * l.heads;
  AttnUnit w;
  if (!attn_unit(a, unit % pairs, a.tiles - 1 - unit / pairs, 16, w)) return;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  // few keys for so many workgroups: as many as have a tile for each wave, or one alone for up to two each
  const int tiles = (w.T + 63) / 64, nsplit = tiles <= 2 * kWaves ? 1 : min(a.nsplit, (tiles + kWaves - 1) / kWaves);
  if (split >= nsplit) return;
  const AttnHead h(a, w);
  const int row = lane & 15, g = lane >> 4;
  const int step = 64 * kWaves * nsplit;
  int t0 = 64 * (split * kWaves + wave);
  AttnRows<KS> s;
  s.none();
  if (t0 < w.T) {
    AttnTile<KS, ONCE> tile;
    bool more;
    {
      float x[KS][16];
      const int seen = attn_query<KS>(x, a, w.b, w.h, w.r0, w.rows, w.pos, w.T);
      tile.load_keys(a, h, t0);
      tile.load_values(a, h, t0);
      more = attn_begin<KS>(s, x, a.l.head_size, seen);
    }
    const int least = attn_least(s.seen);
    if (__builtin_expect(__any(more), 0)) {
      attn_wide<KS>(s, a, w, h, w.r0, more, t0, step, least);
    } else {
      const AttnMore<KS, false> none{};
      auto key = [&](int, int j, int d) { return tile.k[j][d]; };
      auto val = [&](int, int d) { return tile.v[d]; };
      const int from = t0;
      AttnMarks marks(w.T, step);
      int i = 0;
      for (; t0 + step < w.T; t0 += step, ++i) {
        AttnScales<1> c = tile.c;
        marks.mark(i, attn_step<KS, 1>(s, none, a, c, t0, t0 + 64 > least, key, val, [&] { tile.load_keys(a, h, t0 + step); }));
        tile.load_values(a, h, t0 + step);
      }
      marks.mark(i, attn_step<KS, 1>(s, none, a, tile.c, t0, t0 + 64 > least, key, val, [] {}));
      attn_marked<KS, 1>(s, none, a, h, marks, from, step, i, least);
    }
  }

  // join the waves' rows
  const int hs = l.head_size, wide = 64 * KS + 4;
  f4* stat = reinterpret_cast<f4*>(lds + kWaves * a.lrows * wide);
  s.sum = rows_sum(s.sum);
  if (row < w.nr) {
    float* dst = lds + (wave * a.lrows + row) * wide + 4 * g;
#pragma unroll
    for (int d = 0; d < 4 * KS; ++d) *reinterpret_cast<f4*>(dst + 16 * d) = s.o[d];
    if (lane < 16) stat[wave * a.lrows + row] = f4{s.M, s.sum, (float)s.E, 0.f};
  }
  __syncthreads();
  const int quads = (hs + 3) / 4;
  const __amdgpu_buffer_rsrc_t parts = rsrc_of(a.part);
  const unsigned part = 16u * (quads + 1);                // bytes of a row's part: sums, then M, sum of weights, E
  const unsigned mine = unit * a.nsplit * a.lrows * part;  // of the unit's first
  for (int it = threadIdx.x; it < w.nr * quads; it += blockDim.x) {
    const int r = it / quads, d = it - r * quads;
    f4 o = {0.f, 0.f, 0.f, 0.f};
    float M = kNone, E = -126.f, sum = 0.f;
    f4 x[kWaves], st[kWaves];
#pragma unroll
    for (int n = 0; n < kWaves; ++n) {
      st[n] = stat[n * a.lrows + r];
      x[n] = *reinterpret_cast<const f4*>(lds + (n * a.lrows + r) * wide + 4 * d);
    }
    parts_join(x, st, kWaves, o, M, sum, E);
    if (nsplit == 1) {
      AttnOut(a, w, r, M, sum, E).store(a, 4 * d, o);
      continue;
    }
    const unsigned at = mine + (split * a.lrows + r) * part;
    st4_sc1(parts, at + 16 * d, o);
    if (d == 0) st4_sc1(parts, at + 16 * quads, f4{M, sum, E, 0.f});
  }
  if (nsplit == 1) return;

  // Parts are written through and read past the caches of the XCDs (sc1); each wave's have arrived before the count.
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  __syncthreads();
  if (threadIdx.x == 0) {
    const unsigned before = __hip_atomic_fetch_add(&a.arrived[unit * kCountStep], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = before == (unsigned)nsplit - 1;
    if (last) __hip_atomic_store(&a.arrived[unit * kCountStep], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last) return;
  for (int it = threadIdx.x; it < w.nr * quads; it += blockDim.x) {
    const int r = it / quads, d = it - r * quads;
    const unsigned at = mine + r * part, stride = a.lrows * part;
    f4 o = {0.f, 0.f, 0.f, 0.f};
    float M = kNone, E = -126.f, sum = 0.f;
    for (int n0 = 0; n0 < nsplit; n0 += 8) {  // eight parts under way at once, each joined to what is before it
      f4 x[8], st[8];
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const unsigned p = at + min(n0 + n, nsplit - 1) * stride;
        st[n] = ld4_sc1(parts, p + 16 * quads);
        x[n] = ld4_sc1(parts, p + 16 * d);
      }
      parts_join(x, st, nsplit - n0, o, M, sum, E);
    }
    AttnOut(a, w, r, M, sum, E).store(a, 4 * d, o);
  }
}

// Many rows: each of four waves takes 16 query rows of one (sequence, K/V head), and all of them the same keys, which
// pass through LDS in chunks of NT tiles: the values' codes come in while the scores are computed, the next
// chunk's keys while the values are.  LDS holds the codes in the order in which the lanes want them, one KiB for
// each operand of a product, so that a load (16 bytes a lane, memory to LDS) and a read are both linear in the lane.
//
// Bound by vector instructions and by power: 64 keys x 16 rows at heads of 128 take a SIMD 2100 cycles, of which 363
// vector instructions and 48 products fill 1720, and the products, beside them, 768.  Four 2048-token prompts of 32 heads:
// 272 to 280 us by the card, 491 to 505 TFLOP/s of attention (three times that in int8 operations), the vector pipe 80%
// busy at the 1.92 GHz that the card holds under this load.  Two tiles a step leave room for three waves on a SIMD (2%
// faster than four tiles and two waves), heads of 64 fit three with four.
template <int KS, int NT>
__global__ void __launch_bounds__(256, KS < 3 ? 3 : 2) k_q8_attn_many(Q8AttnArgs a) {
  keep_implicit_args();  // common.hpp
  __shared__ __attribute__((aligned(1024))) i4 kbuf[NT * 4 * KS * 64];
  __shared__ __attribute__((aligned(1024))) i4 vbuf[NT * 4 * KS * 64];
  const Q8KVLayer& l = a.l;
  const unsigned pairs = a.call.n_batches * l.heads;
  AttnUnit w;
  if (!attn_unit(a, blockIdx.x % pairs, a.tiles - 1 - blockIdx.x / pairs, 64, w)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int row = lane & 15, g = lane >> 4;
  const AttnHead h(a, w);

  // wave i brings operands i, i + 4, ...; tiles behind the last key are not brought
  unsigned key_at[KS];
#pragma unroll
  for (int c = 0; c < KS; ++c)
    key_at[c] = (16 * (row >> 2) + 4 * wave + (row & 3)) * l.lanes + (64 * c + 16 * g < l.lanes ? 64 * c + 16 * g : 0);
  const unsigned value_at = g * 16 * l.lanes + 16 * row;
  auto keys_in = [&](int t0) {
#pragma unroll
    for (int f = 0; f < NT * KS; ++f) {
      const int n = f / KS, c = f % KS;  // operand (n, wave, c)
      if (t0 + 64 * n >= w.T) continue;
      lds_bring(h.k + (long long)(t0 + 64 * n) * l.lanes, key_at[c], &kbuf[((n * 4 + wave) * KS + c) * 64]);
    }
  };
  auto values_in = [&](int t0) {
#pragma unroll
    for (int f = 0; f < NT * KS; ++f) {
      const int n = f / KS, d = (f % KS) * 4 + wave;  // operand (n, d)
      if (t0 + 64 * n >= w.T || 16 * d >= l.lanes) continue;
      lds_bring(h.v + (long long)(t0 + 64 * n) * l.lanes + 256 * d, value_at, &vbuf[(n * 4 * KS + d) * 64]);
    }
  };

  if (w.T > 0) keys_in(0);
  AttnRows<KS> s;
  s.none();
  bool more;
  {
    float x[KS][16];
    const int seen = attn_query<KS>(x, a, w.b, w.h, w.r0 + 16 * wave, w.rows, w.pos, w.T);
    more = attn_begin<KS>(s, x, a.l.head_size, seen);
  }
  const AttnMore<KS, false> none{};
  const int least = attn_least(s.seen);
  const int most = -attn_least(-s.seen);
  AttnMarks marks(w.T, 64 * NT);
  for (int t0 = 0; t0 < w.T; t0 += 64 * NT) {
    AttnScales<NT> sc;
    sc.load(a, h.ks, h.vs, lane, t0, w.T);
    lds_wait();  // this chunk's keys are in, and every wave has left the last chunk's values
    values_in(t0);
    auto ready = [&] {
      lds_wait();  // the values are in, and every wave has left this chunk's keys
      if (t0 + 64 * NT < w.T) keys_in(t0 + 64 * NT);
    };
    if (t0 >= most) {  // the other waves' rows see further
      ready();
      continue;
    }
    marks.mark(t0 / (64 * NT),
               attn_step<KS, NT>(s, none, a, sc, t0, t0 + 64 * NT > least, [&](int n, int j, int c) { return kbuf[((n * 4 + j) * KS + c) * 64 + lane]; },
                                 [&](int n, int d) { return vbuf[(n * 4 * KS + d) * 64 + lane]; }, ready));
  }
  attn_marked<KS, NT>(s, none, a, h, marks, 0, 64 * NT, (w.T - 1) / (64 * NT), least);
  auto leave = [&](bool mine) {
    const float sum = rows_sum(s.sum);
    if (16 * wave + row >= w.nr || !mine) return;
    const AttnOut out(a, w, 16 * wave + row, s.M, sum, (float)s.E);
#pragma unroll
    for (int d = 0; d < 4 * KS; ++d)
      if (16 * d + 4 * g < l.head_size) out.store(a, 16 * d + 4 * g, s.o[d]);
  };
  leave(!more);
  if (__builtin_expect(__any(more), 0)) {
    attn_wide<KS>(s, a, w, h, w.r0 + 16 * wave, true, 0, 64, least);
    leave(more);
  }
}

constexpr int kAttnUnits = 256;  // row tiles that fill the card by themselves: one for each CU
constexpr int kMaxSplit = 128;

inline size_t attn_part(int head_size) { return 16 * ((head_size + 3) / 4 + 1); }  // bytes of a row's part

// How a call's rows and keys are divided.
struct AttnPlan {
  bool many;
  int nsplit;
  long long tiles, units;
};
static AttnPlan attn_plan(const Q8KVCache* c, int n_batches, int n_tokens, int n_heads) {
  AttnPlan p;
  const long long rows = (long long)n_tokens * (n_heads / c->n_kv_heads), pairs = (long long)n_batches * c->n_kv_heads;
  // Tiles of 64 rows that fill the card go to k_q8_attn_many: from 256 of them on (256, of 32 heads x 512 rows: 16.7 us,
  // k_q8_attn_few 19.8; 224: 17.0 and 18.0; 352: 22.7 and 28.7), at heads of up to 64, where the few rows' kernel fits
  // four waves on a SIMD, from 512 (264, of 12 heads x 1400 rows: 24.4 us and 16.6; 528, of two
  // sequences: 26.3 and 27.7).
  p.many = rows >= 64 && pairs * ((rows + 63) / 64) >= (c->head_size <= 64 ? 2 : 1) * kAttnUnits;
  p.tiles = p.many ? (rows + 63) / 64 : (rows + 15) / 16;
  p.units = pairs * p.tiles;
  // The keys of few tiles are divided until there is a workgroup for each CU, but no further than each wave has a tile (one
  // row of 32 heads over 2048 keys: 9.1 us, divided twice as far 10.7), or two for each CU where each wave still has eight and no other row tile
  // reads the same keys at its own pace (eight rows of 8 K/V heads over 10923 to 32768 keys: 66 us, with one 72; 32 rows
  // of 32 heads over 16416, two tiles a head: 46 us, with one 34).
  const long long most = (c->seq_len + 64LL * kWaves - 1) / (64 * kWaves);
  p.nsplit = p.many ? 1 : (int)max(1LL, min(most, min((long long)kMaxSplit, kAttnUnits / p.units)));
  if (p.nsplit > 1 && p.tiles == 1 && most >= 16 * p.nsplit) p.nsplit = min(2 * p.nsplit, kMaxSplit);
  return p;
}

// A call's rows count in an int, its row tiles in one launch.
static bool attn_fits(const Q8KVCache* c, int n_batches, int n_tokens, int n_heads) {
  const long long rows = (long long)n_tokens * (n_heads / c->n_kv_heads);
  const unsigned __int128 pairs = (unsigned __int128)n_batches * c->n_kv_heads;
  if (rows > 0x7fffffffLL - 64 || !q8kv_grid_ok(pairs * ((rows + 63) / 64), 64 * kWaves)) return false;
  const AttnPlan p = attn_plan(c, n_batches, n_tokens, n_heads);
  return q8kv_grid_ok((unsigned __int128)p.units * p.nsplit, 64 * kWaves);
}

template <int KS>
static hipError_t attn_launch(const Q8AttnArgs& a, const AttnPlan& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.units * p.nsplit)), block(64 * kWaves);
  if (p.many) {
    hipLaunchKernelGGL((k_q8_attn_many<KS, KS == 1 ? 4 : 2>), grid, block, 0, s, a);
    return hipGetLastError();
  }
  auto kernel = p.tiles == 1 ? k_q8_attn_few<KS, true> : k_q8_attn_few<KS, false>;
  const size_t lds = (size_t)kWaves * a.lrows * (64 * KS + 4 + 4) * sizeof(float);
  if (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(kernel, grid, block, lds, s, a);
  return hipGetLastError();
}

}  // namespace tl

static bool attn_sizes_ok(const Q8KVCache* c, int n_heads) {
  return n_heads > 0 && n_heads % c->n_kv_heads == 0;
}

extern "C" size_t thaDNN_q8_attention_workspace(const Q8KVCache* c, int n_batches, int n_tokens, int n_heads) {
  if (!c || n_batches <= 0 || n_batches > c->n_batches || n_tokens <= 0 || !tl::q8kv_sizes_ok(c->n_batches, c->n_layers, c->n_kv_heads, c->head_size, c->seq_len) ||
      !tl::q8kv_supported(c->head_size, c->block) || !attn_sizes_ok(c, n_heads) ||
      !tl::attn_fits(c, n_batches, n_tokens, n_heads))
    return 0;
  // a call of fewer rows may divide its keys among more workgroups, but never has more than this many parts
  return tl::kAttnUnits * tl::kCountStep * sizeof(unsigned) + (size_t)2 * tl::kAttnUnits * 16 * tl::attn_part(c->head_size);
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
  if (!tl::attn_fits(c, n_batches, n_tokens, n_heads)) return THABLAS_STATUS_NOT_SUPPORTED;
  const tl::AttnPlan p = tl::attn_plan(c, n_batches, n_tokens, n_heads);
  const int lrows = (int)min((long long)n_tokens * mul, 16LL);
  const size_t need = p.nsplit > 1 ? tl::kAttnUnits * tl::kCountStep * sizeof(unsigned) + (size_t)p.units * p.nsplit * lrows * tl::attn_part(c->head_size) : 0;
  if (need && (!work || ((uintptr_t)work & 15) || work_bytes < need)) return THABLAS_STATUS_INVALID_VALUE;
  a.call = {pos_d, n_d, n_batches, n_tokens};
  a.q = q;
  a.out = out;
  a.arrived = static_cast<unsigned*>(work);
  a.part = reinterpret_cast<float*>(a.arrived + tl::kAttnUnits * tl::kCountStep);
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.mul = mul;
  a.tiles = (int)p.tiles;
  a.nsplit = p.nsplit;
  a.lrows = lrows;
  a.vec = tl::q8kv_vec4(c->head_size, q_stride, q, out) && out_stride % 4 == 0;
  a.c0 = (float)__builtin_ldexp(1.4426950408889634 / __builtin_sqrt((double)c->head_size) / tl::kDigits, tl::kUnit);
  tl::Q8KVDevice dev(handle->current_gpu_id);
  if (!dev.ok) return THABLAS_STATUS_INVALID_VALUE;
  const int ks = (a.l.lanes + 63) / 64;
  hipStream_t s = handle->calc_stream;
  hipError_t e;
  if (ks == 1) e = tl::attn_launch<1>(a, p, s);
  else if (ks == 2) e = tl::attn_launch<2>(a, p, s);
  else if (ks == 3) e = tl::attn_launch<3>(a, p, s);
  else e = tl::attn_launch<4>(a, p, s);
  if (e != hipSuccess) return THABLAS_STATUS_EXECUTION_FAILED;
  return THABLAS_STATUS_SUCCESS;
}
