// Attention over the cache in 8 bits (layout: kv8.hpp): row r at position p of sequence i sees the sequence's tokens 0 .. p,
//   z_t = scale q . k_t,  w_t = exp(z_t) / sum exp(z),  y = sigmoid(gate) sum_t w_t v_t.
//
// The g = hq / hkv queries of a cached head and a sequence's rows make the columns (pairs) of both products, which run on
// v_mfma_f32_16x16x32_f16 with the cache as the row operand: S^T = K Q^T, O^T = V^T P^T.  A lane then holds 16 scores of one
// column and every block of 64 tokens, the maximum of a column is 15 fmaxf and two cross-lane steps, and the weights are the second
// product's operand as they stand.  Stored bytes become fp16 exactly: byte u beside 0x64 is 1024 + u, less 1152 is q.  A query
// (bf16) is fp16 times a power of two of its own that brings its largest element into [2^12, 2^13): exact down to 2^-29 of that
// element, below it rounded by 2^-37 of it.  Weights are rounded to fp16 (2^-11 of each; the bf16 output is rounded
// by 2^-8) as 2^15 exp(z - max), so that those down to 2^-29 of the largest keep all their bits.  Running maximum, sums and both products
// are fp32; a block's k scale multiplies its scores, its v scale joins the exponent, relative to a
// power of two that no scale so far exceeds (a row's bits then do not turn on the scale of a block that it does not see).
//
// A wave walks over cached blocks by itself: no barrier, k of the next block requested as soon as this one's is used, v likewise.  Few columns:
// the four waves of a block of threads take every fourth cached block, their sums meet in LDS.  Where that leaves CUs idle the
// cached blocks are split over `splits` blocks of threads, whose sums (fp32) a second launch joins.
#include "kv8.hpp"

using namespace drm;

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int W = 4, NT = W * WAVE;
constexpr float kInf = __builtin_inff();

struct Attn {
  Kv8 c;
  const uint16_t* q;
  const float* gate;
  uint16_t* y;
  float *part, *ml;  // [splits, rows, hq, d] and [splits, rows, hq, 2]
  size_t ldq, ldg, hsg, ldy;
  float scale;
  int hq, g, splits, scan;
};

DEV half8 to_half8(uint32_t a, uint32_t b) {
  const half2v off = {(_Float16)1152.f, (_Float16)1152.f};
  union {
    half2v h[4];
    half8 v;
  } o;
  o.h[0] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)) - off;
  o.h[1] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u)) - off;
  o.h[2] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) - off;
  o.h[3] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) - off;
  return o.v;
}

DEV float quad_max(float v) { return xmax_step<32>(xmax_step<16>(v)); }
DEV float quad_sum(float v) { return xsum_step<32>(xsum_step<16>(v)); }
DEV float lane_f(float v, int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); }

// Four elements e .. of column p (row `row` of the call, query `head`): the finished output, or a part of it to be joined.
// o: sum of exp(z - m) v, l: sum of exp(z - m), up to a common factor; no token seen: o = l = 0.
DEV void emit(const Attn& a, int split, size_t row, int head, int e, const f32x4& o, float l, float m) {
  const int d = a.c.d;
  if (a.splits > 1) {
    const size_t at = ((size_t)split * a.c.rows + row) * a.hq + head;
    *reinterpret_cast<f32x4*>(a.part + at * d + e) = o;
    if (e == 0) a.ml[2 * at] = m, a.ml[2 * at + 1] = l;
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = o[i] * inv;
  if (a.gate) {
    const float4 g = ldf4(a.gate + row * a.ldg + head * a.hsg + e);
    v[0] /= 1.f + expf(-g.x), v[1] /= 1.f + expf(-g.y), v[2] /= 1.f + expf(-g.z), v[3] /= 1.f + expf(-g.w);
  }
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = to_bf16(v[i]);
  *reinterpret_cast<uint2*>(a.y + row * a.ldy + (size_t)head * d + e) = make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
}

// DC: 64-element chunks of a head (the last may be part of one: what lies past d is loaded from inside the head, times zero queries, and
// not stored).  MT: tiles of 16 columns a wave.  WQ: waves along the columns, the other W / WQ along the cached blocks.
template <int DC, int MT, int WQ, int OCC>
__global__ void __launch_bounds__(NT, OCC) k_attn_kv8(Attn a) {
  constexpr int WK = W / WQ, TP = 16 * MT * WQ, LD = 64 * DC + 4;
  __shared__ __align__(16) float sm[WK > 1 ? W * 16 * LD : 4];
  __shared__ float sml[WK > 1 ? W * 32 : 2];
  const int l = lane_id(), j = l >> 4, wv = wave_id(), wq = WQ > 1 ? wv : 0, wk = WQ > 1 ? 0 : wv;
  const int h = blockIdx.y, sp = blockIdx.z, d = a.c.d, d16 = d >> 4, g = a.g;
  int at = blockIdx.x, i = at;
  if (a.scan) i = find_item(a.c, at, [g](const Seq& s) { return (s.n * g + TP - 1) / TP; });
  else at = 0;
  if (i < 0) return;
  const Seq s = seq_of(a.c, i);
  const int np = s.n * g, c0 = at * TP + wq * 16 * MT;
  if (c0 >= np) return;  // no rows; with waves along the columns there is no barrier behind this
  const int c1 = c0 + 16 * MT < np ? c0 + 16 * MT : np;
  const long long cap = (long long)a.c.maxp * KB - 1;
  const int p_lo = s.first + c0 / g, p_end = s.first + (c1 - 1) / g, p_hi = p_end < cap ? p_end : (int)cap;
  // cached blocks of this wave: b0 + wk, b0 + wk + WK .. below b1
  const int nb = p_hi < 0 ? 0 : (p_hi >> 6) + 1, each = (nb + a.splits - 1) / a.splits, chunk = each < WK ? WK : each;
  const int b0 = sp * chunk < nb ? sp * chunk : nb, b1 = b0 + chunk < nb ? b0 + chunk : nb;
  if (a.splits > 1 && b0 == b1 && sp > 0) {
    for (int p = c0 + (WQ > 1 ? l : (int)threadIdx.x); p < c1; p += WQ > 1 ? WAVE : NT) {
      const size_t r = ((size_t)sp * a.c.rows + s.r0 + p / g) * a.hq + h * g + p % g;
      a.ml[2 * r] = -kInf, a.ml[2 * r + 1] = 0.f;
    }
    return;
  }

  // the columns' queries in fp16 (see above), their positions, the running maximum and sum
  half8 q[MT][DC][2];
  f32x4 o[MT][4 * DC];
  float m[MT], sum[MT], qm[MT];
  int pos[MT], unit = -200;  // o holds the sums over 2^unit, a power of two not below any v scale so far
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int p = c0 + 16 * t + (l & 15), row = p / g;
    const bool on = p < np;
    const uint16_t* src = a.q + (size_t)(s.r0 + row) * a.ldq + (size_t)(h * g + p - row * g) * d;
    uint4 w[DC][2];
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int e = 64 * c + 16 * j + 8 * x;
        w[c][x] = make_uint4(0, 0, 0, 0);
        if (on && e < d) w[c][x] = ld16(src + e);
      }
    float top = 0.f;
    bool num = true;
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint32_t v[4] = {w[c][x].x, w[c][x].y, w[c][x].z, w[c][x].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float lo = fabsf(bf16_lo(v[k])), hi = fabsf(bf16_hi(v[k]));
          top = fmaxf(top, fmaxf(lo, hi));
          num = num && lo < kInf && hi < kInf;
        }
      }
    top = quad_max(num ? top : kInf);
    // an infinity or NaN in a query leaves no score that is a number (infinities of both signs, or times zero)
    const bool bad = !(top < kInf);
    const int e = bad || top == 0.f ? 0 : 13 - __builtin_amdgcn_frexp_expf(top);
    const float sign = bad ? __builtin_nanf("") : a.scale < 0.f ? -1.f : 1.f;
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint32_t v[4] = {w[c][x].x, w[c][x].y, w[c][x].z, w[c][x].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          q[t][c][x][2 * k] = (_Float16)(sign * __builtin_ldexpf(bf16_lo(v[k]), e));
          q[t][c][x][2 * k + 1] = (_Float16)(sign * __builtin_ldexpf(bf16_hi(v[k]), e));
        }
      }
    qm[t] = __builtin_ldexpf(fabsf(a.scale) * 1.44269504088896341f, -e);
    const int ps = s.first + row;
    pos[t] = on ? (ps < cap ? ps : (int)cap) : -1;
    m[t] = -kInf, sum[t] = 0.f;
#pragma unroll
    for (int u = 0; u < 4 * DC; ++u) o[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  int koff[DC];
#pragma unroll
  for (int c = 0; c < DC; ++c) koff[c] = ((4 * c + j < d16 ? 4 * c + j : d16 - 1) * KB + (l & 15)) * 16;
  const int voff = (l & 15) * KB + 16 * j;
  uint4 kr[DC][4], vr[4 * DC];
  auto load_k = [&](int page) {
    const uint8_t* p = a.c.kq + ((size_t)page * a.c.hkv + h) * KB * d;
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int t = 0; t < 4; ++t) kr[c][t] = ld16(p + koff[c] + 256 * t);
  };
  auto load_v = [&](int page) {
    const uint8_t* p = a.c.vq + ((size_t)page * a.c.hkv + h) * KB * d;
#pragma unroll
    for (int u = 0; u < 4 * DC; ++u) vr[u] = ld16(p + voff + 16 * KB * (u < d16 ? u : d16 - 1));
  };

  const int cnt = (b1 - b0 - wk + WK - 1) / WK;  // 0 where b0 + wk >= b1
  for (int k0 = 0; k0 < cnt; k0 += WAVE) {
    // pages and scales of the next 64 of the wave's blocks, a lane each
    const int n = cnt - k0 < WAVE ? cnt - k0 : WAVE;
    int pg = 0;
    float sk = 0.f, sv = 0.f;
    bool there = false;
    if (l < n) {
      const int t = page_of(a.c, i, b0 + wk + WK * (k0 + l));
      there = t >= 0;
      pg = there ? t : 0;
      sk = a.c.ks[(size_t)pg * a.c.hkv + h], sv = a.c.vs[(size_t)pg * a.c.hkv + h];
    }
    const unsigned long long have = __ballot(there);
    load_k(__builtin_amdgcn_readlane(pg, 0));
    load_v(__builtin_amdgcn_readlane(pg, 0));
    for (int k = 0; k < n; ++k) {
      const int b = b0 + wk + WK * (k0 + k), nx = __builtin_amdgcn_readlane(pg, k + 1 < n ? k + 1 : k);
      const float ks = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(sk), k));
      const float vs = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(sv), k));
      const bool exists = (have >> k) & 1;
      f32x4 sc[MT][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int x = 0; x < MT; ++x) sc[x][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < DC; ++c) {
          const half8 k8a = to_half8(kr[c][t].x, kr[c][t].y), k8b = to_half8(kr[c][t].z, kr[c][t].w);
#pragma unroll
          for (int x = 0; x < MT; ++x) sc[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8a, q[x][c][0], sc[x][t], 0, 0, 0);
#pragma unroll
          for (int x = 0; x < MT; ++x) sc[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8b, q[x][c][1], sc[x][t], 0, 0, 0);
        }
      }
      if (k + 1 < n) load_k(nx);

      // v's scale enters relative to `unit`; a block whose scale is no number leaves none to the rows that see it
      const bool vnum = vs >= 0.f && vs < kInf;
      const int ve = vnum && vs > 0.f ? __builtin_amdgcn_frexp_expf(vs) : -200, unew = unit > ve ? unit : ve;
      const float ratio = vnum ? fmaxf(__builtin_ldexpf(vs, -unew), 0x1p-40f) : 0x1p-40f, ushrink = __builtin_ldexpf(1.f, unit - unew);
      const float lw = 15.f + __builtin_amdgcn_logf(ratio), iw = 1.f / ratio;
      const bool edge = !exists || b * KB + KB - 1 > p_lo;
      half8 pf[MT][2];
#pragma unroll
      for (int x = 0; x < MT; ++x) {
        // places t <= lim of the block are seen by the lane's column
        const int lim = exists ? pos[x] - b * KB : -1;
        const float f = qm[x] * ks;
        float mx = -kInf;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float z = edge && 16 * t + 4 * j + e > lim ? -kInf : sc[x][t][e];
            mx = fmaxf(mx, z);
          }
        mx = quad_max(mx);
        const float mnew = fmaxf(m[x], mx * f), ms = mnew == -kInf ? 0.f : mnew;
        if (__any(mnew > m[x]) || unew > unit) {
          const float al = __builtin_amdgcn_exp2f(m[x] - ms), ao = al * ushrink;
          sum[x] *= al;
#pragma unroll
          for (int u = 0; u < 4 * DC; ++u) o[x][u] *= ao;
          m[x] = mnew;
        }
        if (!vnum && lim >= 0) sum[x] = __builtin_nanf("");
        float add = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float w = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[x][t][e], f, lw - ms));
            if (edge && 16 * t + 4 * j + e > lim) w = 0.f;
            add += w;
            pf[x][t >> 1][4 * (t & 1) + e] = (_Float16)w;
          }
        sum[x] += add * iw;
      }
      unit = unew;
#pragma unroll
      for (int u = 0; u < 4 * DC; ++u) {
        const half8 v8a = to_half8(vr[u].x, vr[u].y), v8b = to_half8(vr[u].z, vr[u].w);
#pragma unroll
        for (int x = 0; x < MT; ++x) o[x][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8a, pf[x][0], o[x][u], 0, 0, 0);
#pragma unroll
        for (int x = 0; x < MT; ++x) o[x][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8b, pf[x][1], o[x][u], 0, 0, 0);
      }
      if (k + 1 < n) load_v(nx);
    }
  }

#pragma unroll
  for (int x = 0; x < MT; ++x) {
    // both sums less 2^16, so that a v scale next to fp32's largest does not leave it
    const float us = __builtin_ldexpf(1.f, unit - 16);
    sum[x] = quad_sum(sum[x]) * 0x1p-16f;
    if constexpr (WK == 1) {
      const int p = c0 + 16 * x + (l & 15), row = p / g;
      if (p < np)
#pragma unroll
        for (int u = 0; u < 4 * DC; ++u)
          if (u < d16) emit(a, sp, (size_t)s.r0 + row, h * g + p - row * g, 16 * u + 4 * j, o[x][u] * us, sum[x], m[x]);
    } else {
      if (x) __syncthreads();
      if (j == 0) sml[wv * 32 + 2 * l] = m[x], sml[wv * 32 + 2 * l + 1] = sum[x];
#pragma unroll
      for (int u = 0; u < 4 * DC; ++u) *reinterpret_cast<f32x4*>(sm + (wv * 16 + (l & 15)) * LD + 16 * u + 4 * j) = o[x][u] * us;
      __syncthreads();
      const int col = threadIdx.x >> 4, p = c0 + 16 * x + col, row = p / g;
      float wt[W], mm = -kInf, ll = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) mm = fmaxf(mm, sml[w * 32 + 2 * col]);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        wt[w] = mm == -kInf ? 1.f : __builtin_amdgcn_exp2f(sml[w * 32 + 2 * col] - mm);
        ll += wt[w] * sml[w * 32 + 2 * col + 1];
      }
      if (p < np)
        for (int e = 4 * (threadIdx.x & 15); e < d; e += 64) {
          f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int w = 0; w < W; ++w) v += wt[w] * *reinterpret_cast<const f32x4*>(sm + (w * 16 + col) * LD + e);
          emit(a, sp, (size_t)s.r0 + row, h * g + p - row * g, e, v, ll, mm);
        }
    }
  }
}

// Joins the parts of a row's query: a block of threads each, groups of LE lanes (LE 4 >= d) take every NT / LE'th part.
__global__ void __launch_bounds__(NT) k_attn_join(Attn a, int LE) {
  __shared__ __align__(16) float sm[NT * 4];
  __shared__ float red[2 * W];
  const int head = blockIdx.x % a.hq, row = blockIdx.x / a.hq, s0 = a.c.start[0], s1 = a.c.start[a.c.seqs];
  if (row < s0 || row >= s1) return;
  const int l = threadIdx.x & (LE - 1), grp = threadIdx.x / LE, n = NT / LE, d = a.c.d;
  const size_t at = (size_t)row * a.hq + head, step = (size_t)a.c.rows * a.hq;
  float m = -kInf;
  if ((int)threadIdx.x < a.splits) m = a.ml[2 * (at + threadIdx.x * step)];
  float mm = wave_max(m);
  if (lane_id() == 0) red[wave_id()] = mm;
  __syncthreads();
  mm = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float ms = mm == -kInf ? 0.f : mm;
  float ls = 0.f;
  if ((int)threadIdx.x < a.splits) ls = a.ml[2 * (at + threadIdx.x * step) + 1] * __builtin_amdgcn_exp2f(m == -kInf && mm == -kInf ? 0.f : m - ms);
  ls = wave_sum(ls);
  if (lane_id() == 0) red[W + wave_id()] = ls;
  f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int sp = grp; sp < a.splits; sp += n) {
    const size_t r = at + sp * step;
    const float pm = a.ml[2 * r], pl = a.ml[2 * r + 1];
    if (pl == 0.f || 4 * l >= d) continue;  // a part that saw no token has no sums
    v += __builtin_amdgcn_exp2f(pm - ms) * *reinterpret_cast<const f32x4*>(a.part + r * d + 4 * l);
  }
  *reinterpret_cast<f32x4*>(sm + 4 * threadIdx.x) = v;
  __syncthreads();
  if (grp == 0 && 4 * l < d) {
    for (int t = 1; t < n; ++t) v += *reinterpret_cast<const f32x4*>(sm + 4 * (t * LE + l));
    Attn o = a;
    o.splits = 1;
    emit(o, 0, row, head, 4 * l, v, red[W] + red[W + 1] + red[W + 2] + red[W + 3], 0.f);
  }
}

// How a call is cut: from sizes alone, so that the workspace is known before.
struct Plan {
  int mt, wq, splits, scan;
  long long tiles;
};
Plan plan(int rows, int seqs, int max_rows, int max_len, int hq, int hkv, int d) {
  Plan p;
  const long long pairs = (long long)(max_rows < rows ? max_rows : rows) * (hq / hkv);
  p.mt = pairs <= 16 || d > 128 ? 1 : 2;
  p.wq = pairs <= 16 * p.mt ? 1 : W;
  const long long tp = 16ll * p.mt * p.wq, per = (pairs + tp - 1) / tp;
  p.scan = per > 1;
  p.tiles = per > 1 ? (long long)rows * (hq / hkv) / tp + seqs : seqs;
  if (per > 1 && p.tiles > per * seqs) p.tiles = per * seqs;
  const long long blocks = ((long long)max_len + KB - 1) / KB, units = p.tiles * hkv;
  long long s = (1024 + units - 1) / units;
  const long long most = (blocks + W - 1) / W;
  if (s > most) s = most;
  if (s > 128) s = 128;
  p.splits = s < 1 || blocks <= 16 ? 1 : (int)s;
  return p;
}

bool attn_shape_ok(int rows, int seqs, int max_rows, int max_len, int hq, int hkv, int d) {
  return rows >= 0 && rows <= (1 << 20) && seqs >= 0 && seqs <= (1 << 20) && max_rows >= 0 && max_len >= 0 && hkv >= 1 && hkv <= 1024 && hq >= hkv &&
         hq <= 1024 && hq % hkv == 0 && d >= 16 && d <= 256 && d % 16 == 0;
}

}  // namespace

API size_t dr_attn_kv8_ws(int rows, int seqs, int max_rows, int max_len, int hq, int hkv, int d) {
  if (!attn_shape_ok(rows, seqs, max_rows, max_len, hq, hkv, d)) return 0;
  if (rows == 0 || seqs == 0) return 256;
  const Plan p = plan(rows, seqs, max_rows, max_len, hq, hkv, d);
  return p.splits > 1 ? ((size_t)p.splits * rows * hq * (d + 2) * sizeof(float) + 255) & ~(size_t)255 : 256;
}

API int dr_attn_kv8(const uint16_t* q, int ldq, const int* start, const int* len, const int* table, int maxp, const uint8_t* kq, const float* ks,
                    const uint8_t* vq, const float* vs, int pages, float scale, const float* gate, int ldg, int hsg, void* ws, uint16_t* y, int ldy,
                    int rows, int seqs, int max_rows, int max_len, int hq, int hkv, int d, hipStream_t st) {
  const Kv8 c{start, len, table, maxp, const_cast<uint8_t*>(kq), const_cast<float*>(ks), const_cast<uint8_t*>(vq), const_cast<float*>(vs),
              pages, rows, seqs, hkv, d};
  if (!attn_shape_ok(rows, seqs, max_rows, max_len, hq, hkv, d) || !kv8_ok(c) || ldq < hq * d || ldq % 8 || ldy < hq * d || ldy % 4) return -1;
  if (gate && (hsg < d || hsg % 4 || ldg % 4 || ldg < (long long)(hq - 1) * hsg + d || ((uintptr_t)gate & 15))) return -1;
  if (rows == 0 || seqs == 0 || max_rows == 0) return 0;
  if (!kv8_buffers_ok(c) || !q || !y || !ws || ((uintptr_t)q & 15) || ((uintptr_t)y & 7) || ((uintptr_t)ws & 15)) return -1;
  const Plan p = plan(rows, seqs, max_rows, max_len, hq, hkv, d);
  const size_t n = (size_t)p.splits * rows * hq;
  float* part = reinterpret_cast<float*>(ws);
  const Attn a{c, q, gate, y, part, part + n * d, (size_t)ldq, (size_t)(gate ? ldg : 0), (size_t)(gate ? hsg : 0), (size_t)ldy, scale, hq, hq / hkv,
               p.splits, p.scan};
  const dim3 grid((unsigned)p.tiles, hkv, p.splits);
  auto go = [&](auto dc, auto mt, auto wq, auto occ) {
    hipLaunchKernelGGL((k_attn_kv8<decltype(dc)::value, decltype(mt)::value, decltype(wq)::value, decltype(occ)::value>), grid, dim3(NT), 0, st, a);
  };
  constexpr std::integral_constant<int, 1> i1{};
  constexpr std::integral_constant<int, 2> i2{};
  constexpr std::integral_constant<int, 3> i3{};
  constexpr std::integral_constant<int, 4> i4{};
  auto one = [&](auto dc) { p.wq == 1 ? go(dc, i1, i1, i1) : go(dc, i1, i4, i1); };
  auto two = [&](auto dc) {
    if (p.mt == 1) go(dc, i1, i1, i1);
    else p.wq == 1 ? go(dc, i2, i1, i1) : go(dc, i2, i4, i1);
  };
  if (d <= 64) two(i1);
  else if (d <= 128) two(i2);
  else if (d <= 192) one(i3);
  else one(i4);
  if (p.splits > 1) {
    int le = 4;
    while (4 * le < d) le <<= 1;
    hipLaunchKernelGGL(k_attn_join, dim3((unsigned)(rows * hq)), dim3(NT), 0, st, a, le);
  }
  return 0;
}
