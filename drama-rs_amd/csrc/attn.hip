// Attention over the cache in 8 bits (layout: kv8.hpp): row r at position p of sequence i sees the sequence's tokens 0 .. p,
//   z_t = scale q . k_t,  w_t = exp(z_t) / sum exp(z),  y = sigmoid(gate) sum_t w_t v_t.
//
// The g = hq / hkv queries of a cached head and a sequence's rows make the columns (pairs) of both products, which run on the fp16 matrix
// instructions with the cache as the row operand: S^T = K Q^T, O^T = V^T P^T.  A lane then holds scores of one column only, a column's maximum
// and sum are a lane's own and one or two cross-lane steps, and the weights are the second product's operand as they stand.
// Stored bytes become fp16 exactly: byte u beside 0x64 is 1024 + u, less 1152 is q.  A query
// (bf16) is fp16 times a power of two of its own that brings its largest element into [2^12, 2^13): exact down to 2^-29 of that
// element, below it rounded by 2^-37 of it.  Weights are rounded to fp16 (2^-11 of each; the bf16 output is rounded by 2^-8) as
// 2^15 exp(z - max) with few columns, 2^4 exp(z - reference) with many, so that at least those down to 2^-29 and 2^-18 of the largest keep all their
// bits and smaller ones are rounded by 2^-40 and 2^-29 of it; in units of a power of two up to twice the largest v scale so far.  Running maximum, sums and both products
// are fp32; a block's k scale multiplies its scores, its v scale joins the exponent, relative to a
// power of two that no scale so far exceeds (a row's bits then do not turn on the scale of a block that it does not see).
//
// Two kernels.  Few columns (a decode step): a wave walks over cached blocks by itself with no barrier, the next block's bytes requested as soon
// as this one's are used.  Many (prompts): a block's bytes are converted once for all waves, in LDS.  Where the columns alone leave CUs
// idle the cached blocks are split over blocks of threads, whose sums (fp32) a second launch joins.  plan() chooses.
#include "attn_plan.hpp"
#include "kv8.hpp"

using namespace drm;

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int W = kPlanWaves, NT = W * WAVE;
static_assert(KB == kPlanBlock, "the plan's blocks are the cache's");
constexpr float kInf = __builtin_inff();
constexpr float kLow = -__FLT_MAX__;  // the maximum of scores that all lie below fp32's range (none seen: -infinity)
constexpr int kUnit = -200;  // an exponent below that of any scale
constexpr float kFar = 0x1p20f;  // log2 scores from here on: see is_far()

struct Attn {
  Kv8 c;
  const uint16_t* q;
  const float* gate;
  uint16_t* y;
  float *part, *ml;  // [splits, prows, hq, d] and [splits, prows, hq, 2]: see part_rows()
  size_t ldq, ldg, hsg, ldy;
  float scale;
  int hq, g, splits, chunk, scan, fold, most, prows, by_seq;  // most: rows of a sequence that the cut has room for
};

// The rows of a sequence that the call computes.  More than the host said are left out here: their tiles and columns would be others'.
DEV int rows_of(const Attn& a, const Seq& s) { return s.n < a.most ? s.n : a.most; }

// The part of sequence i's first row: parts are a row each, or, where rows of no sequence outnumber what the sequences can have, `most` a
// sequence, so that neither the workspace nor the launch that joins is sized by the rows of none.
DEV size_t part_of(const Attn& a, const Seq& s, int i) { return a.by_seq ? (size_t)i * a.most : (size_t)s.r0; }

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

// What becomes of a row's query `head`: elements e .. e + 3, o: sum of exp(z - m) v, l: sum of exp(z - m), up to a common factor (no token seen:
// both 0).  The finished output, or, not alone, a part of it to be joined; alone, an l of kAlone tells the launch that joins.
// Scores past fp32's range count as infinities of their sign, whichever way a call is cut: one of +infinity leaves NaN sums by itself; all of
// -infinity (m kLow) weigh nothing in a part, which stays a part that saw tokens, and are no number where they are all that there is.
constexpr float kAlone = -1.f;
struct Out {
  uint16_t* y;
  float *part, inv;
  bool alone, gated;
  DEV Out(const Attn& a, bool alone, int split, size_t row, size_t prow, int head, float l, float m, bool first) : alone(alone), gated(a.gate != nullptr) {
    const size_t at = ((size_t)split * a.prows + prow) * a.hq + head;
    y = a.y + row * a.ldy + (size_t)head * a.c.d, part = a.part + at * a.c.d;
    if (m == kLow) l = alone ? __builtin_nanf("") : l == 0.f ? 1.f : l;
    inv = l == 0.f ? 0.f : 1.f / l;
    if (first && !alone) a.ml[2 * at] = m;
    if (first && (!alone || a.splits > 1)) a.ml[2 * at + 1] = alone ? kAlone : l;
  }
  // sigmoid by the hardware's exp2 and reciprocal (1 ulp each): far below the output's rounding to bf16
  DEV static float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896341f * g)); }
  DEV void put(int e, const f32x4& o, const float4& g) const {
    if (!alone) {
      *reinterpret_cast<f32x4*>(part + e) = o;
      return;
    }
    store(e, gated ? gate(o * inv, g) : o * inv);
  }
  DEV static f32x4 gate(const f32x4& v, const float4& g) { return v * f32x4{sigmoid(g.x), sigmoid(g.y), sigmoid(g.z), sigmoid(g.w)}; }
  DEV void store(int e, const f32x4& v) const { *reinterpret_cast<uint2*>(y + e) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])); }
};
// The gate's logits of those elements (an output waits for memory once where all of a lane's are asked for together).
DEV float4 gate_of(const Attn& a, bool on, size_t row, int head, int e) {
  float4 g = make_float4(0.f, 0.f, 0.f, 0.f);
  if (a.gate && on) g = ldf4(a.gate + row * a.ldg + head * a.hsg + e);
  return g;
}

// A wave's columns: MT tiles of 16, lane l holds column l & 15 of each.  DC: 64-element chunks of a head.
template <int DC, int MT>
struct Cols {
  half8 q[MT][DC][2];      // elements 64 c + 16 (l >> 4) + 8 x + (0 .. 7), times a power of two
  f32x4 o[MT][4 * DC];     // O^T, elements 16 u + 4 (l >> 4) + (0 .. 3), over 2^(unit - below - 15)
  float m[MT], sum[MT], qm[MT];  // maximum of the log2 scores, the lane's share of the sum, log2 score of a unit of S and of k's scale
  int pos[MT];             // the columns' positions, -1 where there is none
  int unit;                // 2^unit: a power of two not below any v scale so far
  int below[MT];           // by how much it rose for blocks that a column does not see: all that it sees lie before them
};

// A lane's share of the queries of columns c0 .. of the np pairs (row, query) of sequence s and cached head h; begin makes columns of them.
template <int DC, int MT>
DEV void load_q(const Attn& a, const Seq& s, int h, int c0, int np, uint4 (&q)[MT][DC][2]) {
  const int l = lane_id(), j = l >> 4, d = a.c.d, g = a.g;
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int p = c0 + 16 * t + (l & 15), row = p / g;
    const uint16_t* src = a.q + (size_t)(s.r0 + row) * a.ldq + (size_t)(h * g + p - row * g) * d;
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int e = 64 * c + 16 * j + 8 * x;
        q[t][c][x] = make_uint4(0, 0, 0, 0);
        if (p < np && e < d) q[t][c][x] = ld16(src + e);
      }
  }
}
template <int DC, int MT>
DEV void begin(Cols<DC, MT>& w, const Attn& a, const Seq& s, int c0, int np, const uint4 (&q)[MT][DC][2]) {
  const int l = lane_id();
  const long long cap = (long long)a.c.maxp * KB - 1;
  w.unit = kUnit;
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int p = c0 + 16 * t + (l & 15), row = p / a.g;
    const bool on = p < np;
    const uint4(&r)[DC][2] = q[t];
    float top = 0.f;
    bool num = true;
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint32_t v[4] = {r[c][x].x, r[c][x].y, r[c][x].z, r[c][x].w};
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
        const uint32_t v[4] = {r[c][x].x, r[c][x].y, r[c][x].z, r[c][x].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          w.q[t][c][x][2 * k] = (_Float16)(sign * __builtin_ldexpf(bf16_lo(v[k]), e));
          w.q[t][c][x][2 * k + 1] = (_Float16)(sign * __builtin_ldexpf(bf16_hi(v[k]), e));
        }
      }
    w.qm[t] = __builtin_ldexpf(fabsf(a.scale) * 1.44269504088896341f, -e);
    const int ps = s.first + row;
    w.pos[t] = on ? (ps < cap ? ps : (int)cap) : -1;
    w.m[t] = -kInf, w.sum[t] = 0.f, w.below[t] = 0;
#pragma unroll
    for (int u = 0; u < 4 * DC; ++u) w.o[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

// Pages and scales of up to 64 blocks of a sequence, a lane each.
struct Pages {
  int page, ve;          // v's scale is a fraction in [1/2, 1) times 2^ve,
  float ks, lv, rv;      // the fraction's log2 and reciprocal
  unsigned long long have, num;  // blocks in the cache; those whose scales are numbers
  // ask() asks for the scales, behind which blocks can be asked for; take() waits for them
  DEV void ask(const Attn& a, int seq, int h, int block, bool on) { ask(a, h, on ? page_of(a.c, seq, block) : -1, on); }
  DEV void ask(const Attn& a, int h, int p, bool on) {
    have = __ballot(p >= 0);
    page = p >= 0 ? p : 0;
    ks = lv = 0.f;
    if (on) ks = a.c.ks[(size_t)page * a.c.hkv + h], lv = a.c.vs[(size_t)page * a.c.hkv + h];
  }
  DEV void take() {
    const float vs = lv;
    const bool ok = vs >= 0.f && vs < kInf && ks >= 0.f && ks < kInf;
    num = __ballot(ok);
    if (!ok) ks = 0.f;
    // a scale of 0 weighs nothing, by an exponent far below any; nor does a block that is not there
    const bool pos = ok && (have >> lane_id() & 1) && vs > 0.f;
    ve = pos ? __builtin_amdgcn_frexp_expf(vs) : kUnit;
    const float fr = pos ? __builtin_amdgcn_frexp_mantf(vs) : 0.5f;
    lv = __builtin_amdgcn_logf(fr), rv = 1.f / fr;
  }
  DEV static float lane(float v, int k) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), k)); }
  DEV int at(int k) const { return __builtin_amdgcn_readlane(page, k); }
};

// The common weight, 2^fma(score, f, base) with base = lw - m (m: the maximum, lw: a weight at it), keeps the exact product beside a rounded m and
// rounds lw - m once more: 2 2^-24 |m| in all, an eighth up to kFar, but octaves from 2^24 on, which lift weights past fp16 or sink the
// largest to zero.  From kFar on a column's scores become their distances to m first, the product rounded as m was (0 at the maximum).  What that
// costs the calls that never get there: nothing with few columns, up to 1% in tiles, 2% with
// heads of 192 and 4% with heads of 256 (more registers in memory).
DEV bool is_far(float m) { return fabsf(m) >= kFar && m > -kInf; }
// A score's factor: above 0, so that what is hidden (-infinity) stays it with a k scale of 0, and below infinity, so that a product of nothing
// stays 0.  The words of positive floats are in their order.
DEV float factor_of(float f) { return __uint_as_float(min(__float_as_uint(fmaxf(f, 0x1p-126f)), 0x7f7fffffu)); }
// The maximum of scores from that of their products (-infinity: none is seen).
DEV float top_of(float mx, float f) { return mx > -kInf ? fmaxf(mx * f, kLow) : -kInf; }
DEV float distance(float sc, float f, float m) {
#pragma clang fp contract(off)
  const float z = sc * f;
  return z - m;
}

// One step of the softmax: the scores sc of block k of pg, its first place at position b0, become fp16 weights.
// lo: every column sees the places up to lo.
template <int DC, int MT>
DEV void soften(Cols<DC, MT>& w, f32x4 (&sc)[MT][4], half8 (&pf)[MT][2], const Pages& pg, int k, int b0, int lo) {
  const int j = lane_id() >> 4;
  const bool there = pg.have >> k & 1;
  if (!there || b0 + KB - 1 > lo) {
#pragma unroll
    for (int x = 0; x < MT; ++x) {
      const int lim = there ? w.pos[x] - b0 - 4 * j : -1000;  // of the lane's places 16 t + 4 j + e those with 16 t + e <= lim are seen
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[x][t][e] = 16 * t + e > lim ? -kInf : sc[x][t][e];
    }
  }
  // v's scale enters relative to 2^unit
  const float ks = Pages::lane(pg.ks, k);
  const int ve = __builtin_amdgcn_readlane(pg.ve, k), unew = w.unit > ve ? w.unit : ve, dv = ve - unew > -40 ? ve - unew : -40;
  const float lw = 15.f + Pages::lane(pg.lv, k) + (float)dv;
  float f[MT], mnew[MT];
  bool up = unew > w.unit;
#pragma unroll
  for (int x = 0; x < MT; ++x) {
    f[x] = factor_of(w.qm[x] * ks);
    float mx = -kInf;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = fmaxf(mx, sc[x][t][e]);
    mnew[x] = fmaxf(w.m[x], top_of(quad_max(mx), f[x]));
    up = up || mnew[x] > w.m[x];
  }
  if (__any(up)) {
#pragma unroll
    for (int x = 0; x < MT; ++x) {
      const bool seen = w.pos[x] >= b0;
      if (!seen) w.below[x] += unew - w.unit;
      const float al = mnew[x] == -kInf ? 0.f : __builtin_amdgcn_exp2f(w.m[x] - mnew[x]), ao = __builtin_ldexpf(al, seen ? w.unit - unew : 0);
      w.sum[x] *= al;
#pragma unroll
      for (int u = 0; u < 4 * DC; ++u) w.o[x][u] *= ao;
      w.m[x] = mnew[x];
    }
    w.unit = unew;
  }
  if (!(pg.num >> k & 1)) {
    // a block whose scales are no numbers leaves none to the columns that see it
#pragma unroll
    for (int x = 0; x < MT; ++x)
      if (there && w.pos[x] >= b0) w.sum[x] = __builtin_nanf("");
  }
  bool any_far = false;
#pragma unroll
  for (int x = 0; x < MT; ++x) any_far = any_far || is_far(w.m[x]);
  if (__any(any_far)) {
    // by columns, so that no other has a part in a column's bits
#pragma unroll
    for (int x = 0; x < MT; ++x) {
      if (!is_far(w.m[x])) continue;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[x][t][e] = distance(sc[x][t][e], f[x], w.m[x]);
      f[x] = 1.f;
    }
  }
  const float iw = __builtin_ldexpf(Pages::lane(pg.rv, k), -dv);
#pragma unroll
  for (int x = 0; x < MT; ++x) {
    const float base = lw - (fabsf(w.m[x]) >= kFar ? 0.f : w.m[x]);
    float add = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[x][t][e], f[x], base));
        add += v;
        pf[x][t >> 1][4 * (t & 1) + e] = (_Float16)v;
      }
    w.sum[x] += add * iw;
  }
}

// The blocks [b0, b1) of a sequence that split sp takes of the nb blocks that its columns see; true where the first takes all.
DEV bool share(const Attn& a, int nb, int sp, int& b0, int& b1) {
  const int each = (nb + a.splits - 1) / a.splits, n = each > a.chunk ? each : a.chunk;
  b0 = (long long)sp * n < nb ? sp * n : nb, b1 = nb - b0 > n ? b0 + n : nb;
  return nb <= n;
}

// A split without blocks leaves word of that for its columns [c0, c1).
DEV void emit_none(const Attn& a, size_t part, int h, int sp, int c0, int c1, int t, int nt) {
  for (int p = c0 + t; p < c1; p += nt) {
    const size_t r = ((size_t)sp * a.prows + part + p / a.g) * a.hq + h * a.g + p % a.g;
    a.ml[2 * r] = -kInf, a.ml[2 * r + 1] = 0.f;
  }
}

// Few columns: the four waves of a block of threads hold the same MT tiles of them and take every fourth cached block.  The last chunk of a
// head may be part of one: what lies past d is loaded from inside the head, times zero queries, and not stored.  More pairs than a block of threads
// holds are several blocks (z), which find the cache in L2.
// Memory bounds it where sequences are long: 48 ragged sequences of 115191 tokens in all, 8 cached heads of 128, 216 MB in 53 us (4.1 TB/s), 32 of 8000
// in 104 with the join (5.07 TB/s of 5.12 that a copy reaches); one of 60001 tokens with 2 heads of 256 is two blocks a wave,
// 61 MB in 18.  7 prompts of 33 to 373 rows, 12 heads of 64: 11.4.  Short ones are a chain of loads (length and table, scales and bytes, LDS): 300 tokens 7.4 us, of which 3 to 4 are the launch.
template <int DC, int MT>
__global__ void __launch_bounds__(NT, DC <= 2 ? 2 : 1) k_attn_few(Attn a) {
  constexpr int TP = 16 * MT, LD = 64 * DC + 4;
  __shared__ __align__(16) float sm[W * 16 * LD];
  __shared__ float sml[W * 32];
  const int l = lane_id(), j = l >> 4, wv = __builtin_amdgcn_readfirstlane(wave_id());
  // Consecutive blocks go to the eight dies in turn: heads first, and each split one sequence further, so that no die gets the long
  // sequences (48 ragged ones: 81 us with the sequences in turn, 53).
  const int h = blockIdx.x % a.c.hkv, sp = blockIdx.y, i = (int)((blockIdx.x / a.c.hkv + sp) % a.c.seqs), d = a.c.d, d16 = d >> 4, g = a.g;
  // the table's entries as the host's word for the lengths has it, beside the sequence's length itself
  const int ahead = page_of(a.c, i, (int)((long long)sp * a.chunk + wv + W * l < a.c.maxp ? sp * a.chunk + wv + W * l : -1));
  const Seq s = seq_of(a.c, i);
  const int c0 = blockIdx.z * TP, all = rows_of(a, s) * g;
  if (all <= c0) return;
  const int np = all - c0 < TP ? all : c0 + TP;
  const long long cap = (long long)a.c.maxp * KB - 1;
  const int p_lo = s.first + c0 / g, p_end = s.first + (np - 1) / g, p_hi = p_end < cap ? p_end : (int)cap;
  const int nb = p_hi < 0 ? 0 : (p_hi >> 6) + 1;
  int b0, b1;
  const bool alone = share(a, nb, sp, b0, b1);
  if (b0 == b1 && sp > 0) {
    if (!alone) emit_none(a, part_of(a, s, i), h, sp, c0, np, threadIdx.x, NT);
    return;
  }
  const int cnt = (b1 - b0 - wv + W - 1) / W;  // the wave's blocks b0 + wv, b0 + wv + W ..

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

  Pages pg;
  Cols<DC, MT> w;
  // loads come back in order: the queries are converted while the first block's bytes are on their way
  uint4 qr[MT][DC][2];
  load_q<DC, MT>(a, s, h, c0, np, qr);
  if (b0 == sp * a.chunk) pg.ask(a, h, l < cnt ? ahead : -1, l < cnt);
  else pg.ask(a, i, h, b0 + wv + W * l, l < cnt);
  if (cnt > 0) load_k(pg.at(0)), load_v(pg.at(0));
  begin(w, a, s, c0, np, qr);
  pg.take();
  for (int k0 = 0; k0 < cnt; k0 += WAVE) {
    const int n = cnt - k0 < WAVE ? cnt - k0 : WAVE;
    if (k0) {
      pg.ask(a, i, h, b0 + wv + W * (k0 + l), l < n);
      load_k(pg.at(0)), load_v(pg.at(0));
      pg.take();
    }
    for (int k = 0; k < n; ++k) {
      const int b = b0 + wv + W * (k0 + k), nx = pg.at(k + 1 < n ? k + 1 : k);
      f32x4 sc[MT][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int x = 0; x < MT; ++x) sc[x][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < DC; ++c) {
          const half8 ka = to_half8(kr[c][t].x, kr[c][t].y), kb = to_half8(kr[c][t].z, kr[c][t].w);
#pragma unroll
          for (int x = 0; x < MT; ++x) sc[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, w.q[x][c][0], sc[x][t], 0, 0, 0);
#pragma unroll
          for (int x = 0; x < MT; ++x) sc[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, w.q[x][c][1], sc[x][t], 0, 0, 0);
        }
      }
      if (k + 1 < n) load_k(nx);
      half8 pf[MT][2];
      soften(w, sc, pf, pg, k, b * KB, p_lo);
#pragma unroll
      for (int u = 0; u < 4 * DC; ++u) {
        const half8 va = to_half8(vr[u].x, vr[u].y), vb = to_half8(vr[u].z, vr[u].w);
#pragma unroll
        for (int x = 0; x < MT; ++x) w.o[x][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pf[x][0], w.o[x][u], 0, 0, 0);
#pragma unroll
        for (int x = 0; x < MT; ++x) w.o[x][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vb, pf[x][1], w.o[x][u], 0, 0, 0);
      }
      if (k + 1 < n) load_v(nx);
    }
  }

  // the waves' sums joined in LDS, both less 2^16 so that a v scale next to fp32's largest does not leave it
#pragma unroll
  for (int x = 0; x < MT; ++x) {
    const float us = __builtin_ldexpf(1.f, w.unit - w.below[x] - 16);
    w.sum[x] = quad_sum(w.sum[x]) * 0x1p-16f;
    const int col = threadIdx.x >> 4, p = c0 + 16 * x + col, row = p / g, e0 = 4 * (threadIdx.x & 15);
    float4 gate[DC];
#pragma unroll
    for (int c = 0; c < DC; ++c) gate[c] = gate_of(a, alone && p < np && e0 + 64 * c < d, (size_t)s.r0 + row, h * g + p - row * g, e0 + 64 * c);
    if (x) __syncthreads();
    if (j == 0) sml[wv * 32 + 2 * l] = w.m[x], sml[wv * 32 + 2 * l + 1] = w.sum[x];
#pragma unroll
    for (int u = 0; u < 4 * DC; ++u) *reinterpret_cast<f32x4*>(sm + (wv * 16 + (l & 15)) * LD + 16 * u + 4 * j) = w.o[x][u] * us;
    __syncthreads();
    float wt[W], mm = -kInf, ll = 0.f;
#pragma unroll
    for (int v = 0; v < W; ++v) mm = fmaxf(mm, sml[v * 32 + 2 * col]);
#pragma unroll
    for (int v = 0; v < W; ++v) {
      wt[v] = mm == -kInf ? 1.f : __builtin_amdgcn_exp2f(sml[v * 32 + 2 * col] - mm);
      ll += wt[v] * sml[v * 32 + 2 * col + 1];
    }
    if (p < np) {
      const Out out(a, alone, sp, (size_t)s.r0 + row, part_of(a, s, i) + row, h * g + p - row * g, ll, mm, e0 == 0);
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        const int e = e0 + 64 * c;
        if (e >= d) break;
        f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int z = 0; z < W; ++z) v += wt[z] * *reinterpret_cast<const f32x4*>(sm + (z * 16 + col) * LD + e);
        out.put(e, v, gate[c]);
      }
    }
  }
}

// Many columns: each of the NW waves holds 32 of its own, and all go through the cached blocks together.  A block is loaded once for
// all of them (a 1 / NW of it a wave), becomes fp16 once, and lies in LDS as the operands are read: 1 KB a fragment, lane by lane, so neither
// the writes nor the reads of 16 bytes meet in a bank.  A step has two halves, each ended by a barrier: products (O += V P of the
// block before, S = K Q of this one) and softmax.  With eight waves the second four are half a step behind, so that on every SIMD one wave
// multiplies while the other's softmax has the vector unit.  k of block n + 1 and v of block n are written beside the products of S of block
// n, into buffers whose last readers ended before them.
// What bounds it is the vector unit, which a product keeps for 10 to 12 cycles whatever its size: hence 32 x 32 x 16 products, and a
// softmax without a maximum where it can be: a column's reference is the maximum of an earlier block, and only where a lane's sum says that a
// weight may have passed fp16 (or the column has no reference yet) is the block's maximum taken, O rescaled and the weights formed again.
// 4096 rows of 16 heads of 128 behind 8192 tokens (2 cached heads): 335 to 346 us, 0.99 to 1.03 PFLOP/s (a large library product in fp16: 1.33); the matrix
// unit is busy 40% of the time, the vector unit's own instructions and what products keep it for take the rest.  8192 rows of 32 heads 533 us (1.03),
// heads of 64 108 us (0.64: the softmax is as long for half the products), of 256 267 us for 2048 rows on 6144 (0.64: four waves a CU,
// no other wave's products beside a softmax, and 147 of a lane's registers in memory, which are read where a turn or the epilogue starts).
// Short prompts are steps of 1 to 1.2 us (2.8 with heads of 256) behind a start of 5 (15), most of it the fetch of code that runs once: 1000 rows
// of 32 heads of 128 29.8 us.
template <int DC>
struct Cols32 {
  half8 q[2 * DC];   // 32-element chunk i, half y: elements 32 i + 16 (l >> 5) + 8 y + (0 .. 7), times a power of two
  f32x16 o[DC];      // O^T: elements 32 u + 8 (r >> 2) + 4 (l >> 5) + (r & 3), over 2^(unit - below - kBase)
  float m, sum, qm;  // reference of the log2 scores, the lane's share of the sum, log2 score of a unit of S and of k's scale
  int pos, unit, below;  // as in Cols
};
constexpr float kBase = 4.f;      // a weight is 2^kBase times its ratio to the reference's: 2^11 above it before fp16 ends,
constexpr float kMost = 40000.f;  // which a lane's sum of weights up to kMost rules out

// A lane's share of the queries of columns c0 .. of the np pairs of sequence s and cached head h; begin32 makes columns of them.
template <int DC>
DEV void load_q32(const Attn& a, const Seq& s, int h, int c0, int np, uint4 (&r)[2 * DC]) {
  const int l = lane_id(), hh = l >> 5, d = a.c.d, g = a.g, p = c0 + (l & 31), row = p / g;
  const uint16_t* src = a.q + (size_t)(s.r0 + row) * a.ldq + (size_t)(h * g + p - row * g) * d;
#pragma unroll
  for (int i = 0; i < 2 * DC; ++i) {
    const int e = 32 * (i >> 1) + 16 * hh + 8 * (i & 1);
    r[i] = make_uint4(0, 0, 0, 0);
    if (p < np && e < d) r[i] = ld16(src + e);
  }
}
template <int DC>
DEV void begin32(Cols32<DC>& w, const Attn& a, const Seq& s, int c0, int np, const uint4 (&r)[2 * DC]) {
  const long long cap = (long long)a.c.maxp * KB - 1;
  const int p = c0 + (lane_id() & 31), row = p / a.g;
  const bool on = p < np;
  float top = 0.f;
  bool num = true;
#pragma unroll
  for (int i = 0; i < 2 * DC; ++i) {
    const uint32_t v[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float lo = fabsf(bf16_lo(v[k])), hi = fabsf(bf16_hi(v[k]));
      top = fmaxf(top, fmaxf(lo, hi));
      num = num && lo < kInf && hi < kInf;
    }
  }
  top = xmax_step<32>(num ? top : kInf);
  const bool bad = !(top < kInf);  // as in begin()
  const int e = bad || top == 0.f ? 0 : 13 - __builtin_amdgcn_frexp_expf(top);
  const float sign = bad ? __builtin_nanf("") : a.scale < 0.f ? -1.f : 1.f;
#pragma unroll
  for (int i = 0; i < 2 * DC; ++i) {
    const uint32_t v[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      w.q[i][2 * k] = (_Float16)(sign * __builtin_ldexpf(bf16_lo(v[k]), e));
      w.q[i][2 * k + 1] = (_Float16)(sign * __builtin_ldexpf(bf16_hi(v[k]), e));
    }
  }
  w.qm = __builtin_ldexpf(fabsf(a.scale) * 1.44269504088896341f, -e);
  const int ps = s.first + row;
  w.pos = on ? (ps < cap ? ps : (int)cap) : -1;
  w.m = -kInf, w.sum = 0.f, w.unit = kUnit, w.below = 0;
#pragma unroll
  for (int u = 0; u < DC; ++u)
#pragma unroll
    for (int k = 0; k < 16; ++k) w.o[u][k] = 0.f;
}

// The scores sc of block k of pg (first place at position b0, every column sees the places up to lo) become fp16 weights.
template <int DC>
DEV void soften32(Cols32<DC>& w, f32x16 (&sc)[2], half8 (&pf)[2][2], const Pages& pg, int k, int b0, int lo) {
  const int hh = lane_id() >> 5;
  const bool there = pg.have >> k & 1;
  const int lim = there ? w.pos - b0 : -1000;
  if (!there || b0 + KB - 1 > lo) {
    const int mine = lim - 4 * hh;  // of the lane's places 32 t + 8 (r >> 2) + 4 hh + (r & 3)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[t][r] = 32 * t + 8 * (r >> 2) + (r & 3) > mine ? -kInf : sc[t][r];
  }
  const int ve = __builtin_amdgcn_readlane(pg.ve, k), unew = w.unit > ve ? w.unit : ve, dv = ve - unew > -40 ? ve - unew : -40;
  float f = factor_of(w.qm * Pages::lane(pg.ks, k));  // as in soften()
  if (unew > w.unit) {
    const int sh = lim >= 0 ? w.unit - unew : 0;
    if (lim < 0) w.below += unew - w.unit;
    if (w.unit > kUnit) {  // before there are no sums
#pragma unroll
      for (int u = 0; u < DC; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) w.o[u][r] = __builtin_ldexpf(w.o[u][r], sh);
    }
    w.unit = unew;
  }
  if (!(pg.num >> k & 1) && lim >= 0) w.sum = __builtin_nanf("");  // scales that are no numbers
  float add = 0.f, at = kBase + Pages::lane(pg.lv, k) + (float)dv - (fabsf(w.m) >= kFar ? -kInf : w.m);
  auto form = [&]() {
    add = 0.f;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][r], f, at));
        add += v;
        pf[t][r >> 2 & 1][4 * (r >> 3) + (r & 3)] = (_Float16)v;
      }
  };
  form();
  // without a reference yet, or with one far from zero, the weights above are infinite and the block's maximum is taken in any case
  if (__any(!(add <= kMost))) {
    float mx = -kInf;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[t][r]);
    // a column's own lanes alone decide, so that what is in the other columns has no part in its bits (2% of a long chunk's time)
    const float most = xmax_step<32>(add), high = top_of(xmax_step<32>(mx), f), top = !(most <= kMost) || fabsf(w.m) >= kFar ? high : w.m;
    if (top > w.m) {
      // less than the reference stays as it is; without one (m -infinity) there are no sums to scale
      const float al = w.m == -kInf ? 1.f : __builtin_amdgcn_exp2f(w.m - top);
      w.m = top;
      w.sum *= al;
#pragma unroll
      for (int u = 0; u < DC; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) w.o[u][r] *= al;
    }
    int k2 = k, d2 = dv;  // worked out again: a value kept from above costs a register where there is none (heads of 256: 267 us, 274)
    asm volatile("" : "+s"(k2), "+s"(d2));
    at = kBase + Pages::lane(pg.lv, k2) + (float)d2 - (fabsf(w.m) >= kFar ? 0.f : w.m);
    if (is_far(w.m)) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[t][r] = distance(sc[t][r], f, w.m);
      f = 1.f;
    }
    form();
  }
  w.sum += add * __builtin_ldexpf(Pages::lane(pg.rv, k), -dv);
}

template <int DC, int NW, int OCC>
__global__ void __launch_bounds__(64 * NW, OCC) k_attn_tiles(Attn a) {
  constexpr int TP = 32 * NW, F = 2 * DC, PER = (F + NW - 1) / NW;  // F: 16-byte loads a lane of k, and of v, for one block
  __shared__ __align__(16) half8 kb[2 * 2 * F * WAVE], vb[2 * 2 * F * WAVE];  // [2][F][2][64]
  const int l = lane_id(), hh = l >> 5, wv = __builtin_amdgcn_readfirstlane(wave_id());
  const bool late = NW == 8 && wv >= 4;
  // the last rows of all heads, which see most, first; heads beside each other, so that a die's share of the blocks is of few heads
  const int h = blockIdx.x % a.c.hkv, sp = blockIdx.y, d = a.c.d, d16 = d >> 4, g = a.g;
  int at = (gridDim.x - 1 - blockIdx.x) / a.c.hkv, i = at;
  Seq s;
  const int most = a.most;
  if (a.scan) i = find_item(a.c, at, s, [g, most](const Seq& q) { return ((q.n < most ? q.n : most) * g + TP - 1) / TP; });
  else at = 0, s = seq_of(a.c, i);
  if (i < 0) return;
  s.n = rows_of(a, s);
  const int np = a.scan || s.n * g < TP ? s.n * g : TP;
  // folded: the first four waves have a half tile, the others (none in the middle one) its mirror image in the sequence, which ends later
  const bool fold = NW == 8 && a.fold;
  const int half = fold ? TP / 2 : TP, c0 = at * half, m0 = fold ? ((np - 1) / half - at) * half : c0;
  if (c0 >= np || m0 < c0) return;
  const int c1 = m0 + half < np ? m0 + half : np;
  const long long cap = (long long)a.c.maxp * KB - 1;
  const int p_end = s.first + (c1 - 1) / g, p_hi = p_end < cap ? p_end : (int)cap;
  int b0, b1;
  const bool alone = share(a, p_hi < 0 ? 0 : (p_hi >> 6) + 1, sp, b0, b1);
  if (b0 == b1 && sp > 0) {
    if (!alone) emit_none(a, part_of(a, s, i), h, sp, c0, c1, threadIdx.x, 64 * NW);  // not folded: that is without splits
    return;
  }
  const int cnt = b1 - b0;
  // the wave's columns and how many of the blocks they see
  const int w0 = !fold || wv < 4 ? c0 + 32 * wv : m0 > c0 ? m0 + 32 * (wv - 4) : np, w1 = w0 + 32 < c1 ? w0 + 32 : c1;
  const int w_lo = s.first + w0 / g, w_end = s.first + (w1 - 1) / g, w_cnt = w0 < c1 && w_end >= 0 ? (w_end >> 6) + 1 - b0 : 0;

  // load f of the wave: k of 32 tokens (tile t) and of 32 elements (chunk c), 16 of them a lane; v of 32 elements (tile) and of the tokens
  // 16 .. + 8 jj + 4 hh + .. (see kv8.hpp)
  int koff[PER], voff[PER];
#pragma unroll
  for (int f = 0; f < PER; ++f) {
    const int u = wv * PER + f, c = u >> 1, b = u & 1, e = 32 * c + (l & 31);
    koff[f] = ((2 * c + hh < d16 ? 2 * c + hh : d16 - 1) * KB + 32 * b + (l & 31)) * 16;
    voff[f] = (e < d ? e : d - 1) * KB + 16 * (2 * b + hh);
  }
  uint4 kr[PER], vr[PER];
  auto mine = [&](int f) { return F % NW == 0 || wv * PER + f < F; };
  auto load_k = [&](int page) {
    const uint8_t* p = a.c.kq + ((size_t)page * a.c.hkv + h) * KB * d;
#pragma unroll
    for (int f = 0; f < PER; ++f)
      if (mine(f)) kr[f] = ld16(p + koff[f]);
  };
  auto load_v = [&](int page) {
    const uint8_t* p = a.c.vq + ((size_t)page * a.c.hkv + h) * KB * d;
#pragma unroll
    for (int f = 0; f < PER; ++f)
      if (mine(f)) vr[f] = ld16(p + voff[f]);
  };

  Pages pg, px;  // of 64 blocks, and of the 64 behind them
  uint4 qr[2 * DC];
  load_q32<DC>(a, s, h, w0, c1, qr);
  pg.ask(a, i, h, b0 + l, l < cnt);
  if (cnt > 0) load_k(pg.at(0)), load_v(pg.at(0));
  px.ask(a, i, h, b0 + WAVE + l, WAVE + l < cnt);
  pg.take();
  int base = 0;
  auto page = [&](int n) {
    const int p = pg.at((n - base) & (WAVE - 1)), x = px.at((n - base) & (WAVE - 1));  // no branch
    return n - base < WAVE ? p : x;
  };
  // k of block n + 1 and v of block n into LDS, the wave's share in 4 PER parts; the loads of the blocks behind them (past the last one again
  // that one, into a buffer that nobody reads any more): no branch, so that it goes between the products.
  auto put_part = [&](int n, int f) {
    const bool isk = f >= 2 * PER;
    const int i = (f % (2 * PER)) >> 1, y = f & 1, u = wv * PER + i;
    const uint4 r = isk ? kr[i] : vr[i];
    half8* b = (isk ? kb : vb) + ((n + isk) & 1) * 2 * F * WAVE + l;
    if (mine(i)) b[(2 * u + y) * WAVE] = y ? to_half8(r.z, r.w) : to_half8(r.x, r.y);
  };
  auto put_loads = [&](int n) {
    load_v(page(n + 1 < cnt ? n + 1 : cnt - 1));
    load_k(page(n + 2 < cnt ? n + 2 : cnt - 1));
  };
  auto put = [&](int n) {
#pragma unroll
    for (int f = 0; f < 4 * PER; ++f) put_part(n, f);
    put_loads(n);
  };
  Cols32<DC> w;
  begin32(w, a, s, w0, c1, qr);
  if (w.pos < b0 * KB) w.m = 0.f;  // a column that sees none of the blocks asks for no reference
  if (cnt > 0) {
#pragma unroll
    for (int f = 2 * PER; f < 4 * PER; ++f) put_part(-1, f);
    load_k(page(cnt > 1 ? 1 : 0));
  }
  lds_barrier();
  if (late) lds_barrier();
  f32x16 sc[2], zero;
#pragma unroll
  for (int r = 0; r < 16; ++r) zero[r] = 0.f;
  half8 pf[2][2];
  // Products in turns of four, with the next turn's operands on their way from LDS and a share of put(n) between: left to itself the compiler
  // waits for every read before it issues the next, and a product that waits for the one before it on the same sum takes twice its time, so
  // those of O += V P of block k and of S = K Q of block k + 1 alternate.
  enum { WEIGH = 1, SCORE = 2 };
  auto products = [&](auto what, int k, int n) {
    constexpr int M = decltype(what)::value, N = M == 3 ? 8 * DC : 4 * DC, T = N / 4;
    const half8* vf = vb + (k & 1) * 2 * F * WAVE + l;
    const half8* kf = kb + ((k + 1) & 1) * 2 * F * WAVE + l;
    auto is_score = [](int x) { return M == SCORE || (M == 3 && (x & 1)); };
    auto operand = [&](int x) {
      const int y = M == 3 ? x >> 1 : x;
      if (is_score(x)) return kf[(2 * (2 * (y >> 2) + (y & 1)) + (y >> 1 & 1)) * WAVE];
      return vf[(2 * (2 * (y % DC) + (y / DC >> 1)) + (y / DC & 1)) * WAVE];
    };
    half8 fr[2][4];
#pragma unroll
    for (int x = 0; x < 4; ++x) fr[0][x] = operand(x);
#pragma unroll
    for (int c = 0; c < T; ++c) {
      if (c + 1 < T)
#pragma unroll
        for (int x = 0; x < 4; ++x) fr[(c + 1) & 1][x] = operand(4 * c + 4 + x);
      if (n >= 0 && M == 3) {
#pragma unroll
        for (int f = 0; f < 4 * PER; ++f)
          if (T - 1 - (4 * PER - f) * (T - 2) / (4 * PER + 2) == c) put_part(n, f);
        if (c == T - 1) put_loads(n);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int z = 4 * c + x, y = M == 3 ? z >> 1 : z;
        if (is_score(z))
          sc[y & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fr[c & 1][x], w.q[y >> 1], y < 2 ? zero : sc[y & 1], 0, 0, 0);
        else
          w.o[y % DC] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fr[c & 1][x], pf[y / DC & 1][y / DC >> 1], w.o[y % DC], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  constexpr std::integral_constant<int, WEIGH> weigh{};
  constexpr std::integral_constant<int, SCORE> score{};
  constexpr std::integral_constant<int, WEIGH + SCORE> both{};
  // blocks later than all of the wave's columns are left out
  const int mine_cnt = cnt < w_cnt ? cnt : w_cnt;
  if (mine_cnt > 0) products(score, -1, -1);
  if (cnt > 0) put(0);
  auto soft = [&](int k) {
    lds_barrier();
    if (k - base == WAVE) {
      pg = px, base = k;
      pg.take();
      px.ask(a, i, h, b0 + k + WAVE + l, k + WAVE + l < cnt);
    }
    if (k < mine_cnt) soften32(w, sc, pf, pg, k - base, (b0 + k) * KB, w_lo);
    if (NW == 8) lds_barrier();  // four waves are not out of step: what their products read was written before the barrier above
  };
  int k = 0;
  for (; k + 1 < mine_cnt; ++k) {
    soft(k);
    __builtin_amdgcn_s_setprio(3);  // the products' few issues before the other wave's vector work: 342 us for 366
    products(both, k, k + 1);
    __builtin_amdgcn_s_setprio(0);
  }
  for (; k < cnt; ++k) {
    soft(k);
    if (k < mine_cnt) products(weigh, k, -1);
    if (k + 1 < cnt) put(k + 1);
  }
  if (NW == 8 && !late) lds_barrier();
  const float us = __builtin_ldexpf(1.f, w.unit - w.below - 16), sum = xsum_step<32>(w.sum) * 0x1p-16f;
  int z = threadIdx.x & 63;  // worked out again: values kept from begin32() would cost registers through the loop
  asm volatile("" : "+v"(z));
  const int p = w0 + (z & 31), row = p / g, head = h * g + p - row * g;
  if (p >= c1) return;
  const size_t rw = (size_t)s.r0 + row;
  const Out out(a, alone, sp, rw, part_of(a, s, i) + row, head, sum, w.m, z < 32);
  const float fin = __builtin_ldexpf(out.inv, w.unit - w.below - 16);
  // A block runs through this once, and what it costs is the fetch of its code: few branches (d ends on a multiple of 16), gates of as many
  // elements at a time as registers allow.
  auto each = [&](int u0, int n, auto f) {
#pragma unroll
    for (int u = 0; u < n; ++u)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (32 * (u0 + u) + 16 * x >= d) break;
#pragma unroll
        for (int r = 2 * x; r < 2 * x + 2; ++r) f(u0 + u, r, 32 * (u0 + u) + 8 * r + 4 * (z >> 5));
      }
  };
  auto o4 = [&](int u, int r, float s) { return f32x4{w.o[u][4 * r] * s, w.o[u][4 * r + 1] * s, w.o[u][4 * r + 2] * s, w.o[u][4 * r + 3] * s}; };
  if (!alone) {
    each(0, DC, [&](int u, int r, int e) { *reinterpret_cast<f32x4*>(out.part + e) = o4(u, r, us); });
  } else if (!a.gate) {
    each(0, DC, [&](int u, int r, int e) { out.store(e, o4(u, r, fin)); });
  } else {
    constexpr int GU = DC > 4 ? DC / 2 : DC;
#pragma unroll
    for (int u0 = 0; u0 < DC; u0 += GU) {
      float4 gate[GU][4];
      each(u0, GU, [&](int u, int r, int e) { gate[u - u0][r] = gate_of(a, true, rw, head, e); });
      each(u0, GU, [&](int u, int r, int e) { out.store(e, Out::gate(o4(u, r, fin), gate[u - u0][r])); });
    }
  }
}

// Joins the parts of a row's query, or of 4 LE elements of it where the queries are few: G groups of LE lanes of four elements, each group every
// G'th part, eight at a time in flight, with a maximum of its own; the groups meet in LDS.  As many queries a block as that
// leaves room for.  A launch and two rounds of loads: 4 to 5 us for all of the above.
constexpr int kJoin = 8;      // parts of a group in flight
__global__ void __launch_bounds__(NT) k_attn_join(Attn a, int LE, int G) {
  __shared__ __align__(16) f32x4 so[NT];
  __shared__ float sm[NT / 16], sl[NT / 16];
  const int t = threadIdx.x, gi = t / LE, grp = gi & (G - 1), d = a.c.d, n = a.prows * a.hq;
  const int item = blockIdx.x * (NT / (LE * G)) + gi / G, at = item < n ? item : n - 1, pr = at / a.hq, head = at - pr * a.hq;
  const int e = 4 * (LE * blockIdx.y + (t & (LE - 1)));
  int row = pr;
  bool own;
  if (a.by_seq) {
    const int i = pr / a.most;
    const Seq s = seq_of(a.c, i);
    row = s.r0 + (pr - i * a.most), own = pr - i * a.most < s.n;
  } else {
    own = row >= a.c.start[0] && row < a.c.start[a.c.seqs];
  }
  const bool on = item < n && e < d && own;
  const size_t step = n;
  const float4 gate = gate_of(a, on && grp == 0, row, head, e);
  float m = -kInf, s = 0.f;
  f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
  bool whole = false;
  for (int s0 = grp; s0 < a.splits; s0 += kJoin * G) {
    uint2 w[kJoin];
    f32x4 r[kJoin];
#pragma unroll
    for (int k = 0; k < kJoin; ++k) {
      const size_t sp = at + (s0 + G * k) * step;
      w[k] = make_uint2(0, 0), r[k] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (on && s0 + G * k < a.splits) w[k] = ld8(a.ml + 2 * sp), r[k] = gld<f32x4>(a.part + sp * d + e);
    }
    float mn = m;
#pragma unroll
    for (int k = 0; k < kJoin; ++k)
      if (w[k].y != 0) mn = fmaxf(mn, __uint_as_float(w[k].x));  // a part that saw no token (l = 0) has no sums
    if (s0 == 0) whole = __uint_as_float(w[0].y) == kAlone;
    const float ms = mn == -kInf ? 0.f : mn, c0 = __builtin_amdgcn_exp2f(m - ms);
    v *= c0, s *= c0, m = mn;
#pragma unroll
    for (int k = 0; k < kJoin; ++k) {
      if (w[k].y == 0) continue;
      const float c = __builtin_amdgcn_exp2f(__uint_as_float(w[k].x) - ms);
      v += c * r[k], s += c * __uint_as_float(w[k].y);
    }
  }
  if (G > 1) {
    so[t] = v;
    if ((t & (LE - 1)) == 0) sm[gi] = m, sl[gi] = s;
    __syncthreads();
    float mn = -kInf;
#pragma unroll
    for (int k = 0; k < NT / 16; ++k)
      if (k < G) mn = fmaxf(mn, sm[gi - grp + k]);
    const float ms = mn == -kInf ? 0.f : mn;
    s = 0.f, v = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NT / 16; ++k)
      if (k < G) {
        const float c = __builtin_amdgcn_exp2f(sm[gi - grp + k] - ms);
        v += c * so[t + (k - grp) * LE], s += c * sl[gi - grp + k];
      }
    m = mn;
  }
  if (on && grp == 0 && !whole) Out(a, true, 0, row, 0, head, s, m, false).put(e, v, gate);
}

bool attn_shape_ok(int rows, int seqs, int max_rows, int max_len, int hq, int hkv, int d) {
  return rows >= 0 && rows <= (1 << 20) && seqs >= 0 && seqs <= (1 << 20) && max_rows >= 0 && max_len >= 0 && hkv >= 1 && hkv <= 1024 && hq >= hkv &&
         hq <= 1024 && hq % hkv == 0 && d >= 16 && d <= 256 && d % 16 == 0;
}

// A launch has fewer than 2^32 threads in a dimension.
bool too_many(const Plan& p, int hkv) { return p.tiles * hkv >= 1 << 23; }

}  // namespace

API size_t dr_attn_kv8_ws(int rows, int seqs, int max_rows, int max_len, int hq, int hkv, int d) {
  if (!attn_shape_ok(rows, seqs, max_rows, max_len, hq, hkv, d)) return 0;
  if (rows == 0 || seqs == 0 || max_rows == 0) return 256;
  const Plan p = plan(rows, seqs, max_rows, max_len, hq, hkv, d);
  if (too_many(p, hkv)) return 0;
  return p.splits > 1 ? ((size_t)p.splits * part_rows(rows, seqs, max_rows) * hq * (d + 2) * sizeof(float) + 255) & ~(size_t)255 : 256;
}

API int dr_attn_kv8(const uint16_t* q, int ldq, const int* start, const int* len, const int* table, int maxp, const uint8_t* kq, const float* ks,
                    const uint8_t* vq, const float* vs, int pages, float scale, const float* gate, int ldg, int hsg, void* ws, uint16_t* y, int ldy,
                    int rows, int seqs, int max_rows, int max_len, int hq, int hkv, int d, hipStream_t st) {
  const Kv8 c{start, len, table, maxp, const_cast<uint8_t*>(kq), const_cast<float*>(ks), const_cast<uint8_t*>(vq), const_cast<float*>(vs),
              pages, rows, seqs, hkv, d};
  if (!attn_shape_ok(rows, seqs, max_rows, max_len, hq, hkv, d) || !kv8_ok(c) || ldq < hq * d || ldq % 8 || ldy < hq * d || ldy % 4) return -1;
  if (gate && (hsg < d || hsg % 4 || ldg % 4 || ldg < (long long)(hq - 1) * hsg + d || ((uintptr_t)gate & 15))) return -1;
  if (!(fabsf(scale) < kInf)) return -1;
  if (rows == 0 || seqs == 0 || max_rows == 0) return 0;
  if (!kv8_buffers_ok(c) || !q || !y || !ws || ((uintptr_t)q & 15) || ((uintptr_t)y & 7) || ((uintptr_t)ws & 15)) return -1;
  const Plan p = plan(rows, seqs, max_rows, max_len, hq, hkv, d);
  const int prows = part_rows(rows, seqs, max_rows);
  float* part = reinterpret_cast<float*>(ws);
  const Attn a{c, q, gate, y, part, part + (size_t)p.splits * prows * hq * d, (size_t)ldq, (size_t)(gate ? ldg : 0), (size_t)(gate ? hsg : 0),
               (size_t)ldy, scale, hq, hq / hkv, p.splits, p.chunk, p.scan, p.fold, max_rows, prows, prows < rows};
  if (too_many(p, hkv)) return -1;
  const dim3 grid((unsigned)(p.tiles * hkv), p.splits, p.cols);
  auto few = [&](auto dc, auto mt) {
    hipLaunchKernelGGL((k_attn_few<decltype(dc)::value, decltype(mt)::value>), grid, dim3(NT), 0, st, a);
  };
  auto tiles = [&](auto dc) {
    constexpr int DC = decltype(dc)::value;
    if constexpr (DC <= 4) {
      if (p.nw == 8) hipLaunchKernelGGL((k_attn_tiles<DC, 8, 2>), grid, dim3(512), 0, st, a);
      else hipLaunchKernelGGL((k_attn_tiles<DC, 4, 2>), grid, dim3(256), 0, st, a);
    } else {
      hipLaunchKernelGGL((k_attn_tiles<DC, 4, 1>), grid, dim3(256), 0, st, a);
    }
  };
  constexpr std::integral_constant<int, 1> i1{};
  constexpr std::integral_constant<int, 2> i2{};
  constexpr std::integral_constant<int, 3> i3{};
  constexpr std::integral_constant<int, 4> i4{};
  constexpr std::integral_constant<int, 6> i6{};
  constexpr std::integral_constant<int, 8> i8{};
  if (p.few) {
    if (d <= 64) p.mt == 1 ? few(i1, i1) : few(i1, i2);
    else if (d <= 128) p.mt == 1 ? few(i2, i1) : few(i2, i2);
    else d <= 192 ? few(i3, i1) : few(i4, i1);
  } else {
    if (d <= 64) tiles(i2);
    else if (d <= 128) tiles(i4);
    else d <= 192 ? tiles(i6) : tiles(i8);
  }
  if (p.splits > 1) {
    int le = 16, grps = 1;
    const long long items = (long long)prows * hq;
    if (items >= 512)
      while (4 * le < d) le <<= 1;
    while (grps * kJoin < p.splits && 2 * grps * le <= NT) grps <<= 1;
    const int per = NT / (le * grps);
    hipLaunchKernelGGL(k_attn_join, dim3((unsigned)((items + per - 1) / per), (d + 4 * le - 1) / (4 * le)), dim3(NT), 0, st, a, le, grps);
  }
  return 0;
}
