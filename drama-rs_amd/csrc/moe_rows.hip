// A whole MoE layer for a few rows (1 .. 64) of any size: per row x (bf16)
//   l = R x, picks by (l desc, index asc), w = softmax(l) renormalised over the picks,
//   y = res + sigmoid(l_E) D_s (silu(G_s x) * (U_s x)) + sum_k w_k D_k (silu(G_k x) * (U_k x)).
//
// An expert is fetched once for all the rows that picked it.  Matrix products run on
// v_mfma_f32_16x16x32_bf16 with A = 16 rows of x and B = 16 weight rows, converted exactly to bf16
// in registers (int4: 16 + q, with the rest of q scale + min in one fp32 MFMA of the group sums of x), so x
// enters exactly.  The activations are fp32; they travel as three bf16 planes of 8 mantissa
// bits each (their sum is the fp32 value), three MFMAs per weight fragment, so nothing is rounded but the fp32 sums.
#include "canon.hpp"

using namespace drm;

namespace {

constexpr int MR_NW = 8, MR_NT = MR_NW * 64, MR_ROWS = 64, MR_TOPK = 32, MR_PAIRS = MR_ROWS * MR_TOPK;
constexpr int MR_GRID = 512;  // two blocks per CU
constexpr int MR_SETS = 8;    // row sets of the router

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

DEV f32x4 mfma(const uint4& a, const uint4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

struct MoeRows {
  const uint16_t* router;
  const uint8_t *gu_q, *d_q;
  const void *gu_s, *d_s;
  const int8_t *sgu_q, *sd_q;
  const uint16_t *sgu_s, *sd_s;
  const uint16_t* x;
  const float* res;
  int* idx;
  float *wts, *sgate, *y;
  uint32_t* counter;  // [MR_SETS] words 128 bytes apart, 0 between calls
  float* logits;      // [rows, e + shared]
  uint16_t* act;      // 3 planes of [(topk + 1) rows, i]
  float* yp;          // [(topk + 1) rows, h]: each pick's expert output, then the shared expert's
  int rows, e, h, i, topk, shared;
};

// ---- weight formats --------------------------------------------------------------------------
// One wave's part of a 16-row tile: 256 inputs of each row, lane l holding 16-byte pieces of row l % 16
// (g = l / 16).  Fragment f of x (two for each group of 64 inputs) covers inputs 64 (f / 2) + xoff(g) + 8 (f % 2) .. + 8.
// half: only the chunk's first 128 inputs exist.

template <class SC>
struct RowsQ4 {
  static constexpr bool perm = true;  // fragment order 0 4 1 5 2 6 3 7
  uint4 w[2];
  uint2 s[2];
  static DEV int xoff(int g) { return 32 * (g & 1) + 16 * (g >> 1); }
  DEV void load(const uint8_t* Q, const void* S, size_t expert, int n, int N, int K, int c, bool half) {
    const size_t row = expert * N + n;
    const uint8_t* p = Q + row * (K / 2) + c * 128 + 16 * (lane_id() >> 4);
    const uint32_t* q = reinterpret_cast<const uint32_t*>(S) + row * (K / 64) + c * 4;
    w[0] = ld16(p), s[0] = ld8(q);
    w[1] = make_uint4(0, 0, 0, 0), s[1] = make_uint2(0, 0);
    if (!half) w[1] = ld16(p + 64), s[1] = ld8(q + 2);
  }
  // nibbles of a word as 16 + q in bf16: the nibble is the top four mantissa bits of a number in [16, 32)
  static DEV uint4 frag(uint32_t v) {
    constexpr uint32_t m = 0x00780078u, b = 0x41804180u;
    return make_uint4(((v << 3) & m) | b, ((v >> 1) & m) | b, ((v >> 5) & m) | b, ((v >> 9) & m) | b);
  }
  // xsum: lane's sum of x over group l / 16 of row l % 16
  template <int NP>
  DEV void mac(const uint4 (&x)[NP][8], float xsum, f32x4& out) const {
    const int g = lane_id() >> 4;
    const uint32_t own = (g & 2) ? ((g & 1) ? s[1].y : s[1].x) : ((g & 1) ? s[0].y : s[0].x);
    const float2 o = SC::pair(own);
    out = __builtin_amdgcn_mfma_f32_16x16x4f32(xsum, o.y - 16.f * o.x, out, 0, 0, 0);
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      // lanes g = 0, 1 hold group 2 p, g = 2, 3 group 2 p + 1: two words of each change places
      const auto s02 = __builtin_amdgcn_permlane32_swap(w[p].x, w[p].z, false, false);
      const auto s13 = __builtin_amdgcn_permlane32_swap(w[p].y, w[p].w, false, false);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 b0 = frag(s02[h]), b1 = frag(s13[h]);
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < NP; ++q) a = mfma(x[q][4 * p + 2 * h], b0, a), a = mfma(x[q][4 * p + 2 * h + 1], b1, a);
        const float sc = SC::pair(h ? s[p].y : s[p].x).x;
#pragma unroll
        for (int r = 0; r < 4; ++r) out[r] = __builtin_fmaf(sc, a[r], out[r]);
      }
    }
  }
};

struct Rows8 {  // one byte per weight: 64 inputs of a row per 16-byte load of four lanes
  static constexpr bool perm = false;
  uint4 w[4];
  float s[2];
  static DEV int xoff(int g) { return 16 * g; }
  DEV void load_bytes(const uint8_t* row, int c, bool half) {
    const uint8_t* p = row + c * 256 + 16 * (lane_id() >> 4);
    w[0] = ld16(p), w[1] = ld16(p + 64);
    w[2] = w[3] = make_uint4(0, 0, 0, 0);
    if (!half) w[2] = ld16(p + 128), w[3] = ld16(p + 192);
  }
};

template <int SF>
struct RowsFP8 : Rows8 {
  DEV void load(const uint8_t* Q, const void* S, size_t expert, int n, int N, int K, int c, bool half) {
    load_bytes(Q + (expert * N + n) * (size_t)K, c, half);
    const size_t b = (expert * (N / 128) + (n >> 7)) * (size_t)(K / 128) + 2 * c;
    s[0] = blk_scale<SF>(S, b);
    s[1] = half ? 0.f : blk_scale<SF>(S, b + 1);
  }
  static DEV uint4 frag(uint32_t a, uint32_t b) {
    auto cv = [](uint32_t v, auto hi) {
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, 1.0f, decltype(hi)::value));
    };
    constexpr std::integral_constant<bool, false> lo{};
    constexpr std::integral_constant<bool, true> hi{};
    return make_uint4(cv(a, lo), cv(a, hi), cv(b, lo), cv(b, hi));
  }
  template <int NP>
  DEV void mac(const uint4 (&x)[NP][8], float, f32x4& out) const {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4& v = w[2 * p + h];
        const uint4 b0 = frag(v.x, v.y), b1 = frag(v.z, v.w);
#pragma unroll
        for (int q = 0; q < NP; ++q) a = mfma(x[q][4 * p + 2 * h], b0, a), a = mfma(x[q][4 * p + 2 * h + 1], b1, a);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) out[r] = __builtin_fmaf(s[p], a[r], out[r]);
    }
  }
};

template <class SH>
struct RowsQ8 : Rows8 {
  DEV void load(const uint8_t* Q, const void* S, size_t, int n, int, int K, int c, bool half) {
    load_bytes(Q + (size_t)n * K, c, half);
    const uint16_t* sp = reinterpret_cast<const uint16_t*>(S);
    s[0] = SH::scale(sp, n, c * 256, K);
    s[1] = half ? 0.f : SH::scale(sp, n, c * 256 + 128, K);
  }
  static DEV uint32_t pk(uint32_t v, int i) {  // bytes i, i + 1 as bf16 (exact)
    const float a = (float)(int8_t)(v >> (8 * i)), b = (float)(int8_t)(v >> (8 * i + 8));
    return (__float_as_uint(b) & 0xffff0000u) | (__float_as_uint(a) >> 16);
  }
  static DEV uint4 frag(uint32_t a, uint32_t b) { return make_uint4(pk(a, 0), pk(a, 2), pk(b, 0), pk(b, 2)); }
  template <int NP>
  DEV void mac(const uint4 (&x)[NP][8], float, f32x4& out) const {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4& v = w[2 * p + h];
        const uint4 b0 = frag(v.x, v.y), b1 = frag(v.z, v.w);
#pragma unroll
        for (int q = 0; q < NP; ++q) a = mfma(x[q][4 * p + 2 * h], b0, a), a = mfma(x[q][4 * p + 2 * h + 1], b1, a);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) out[r] = __builtin_fmaf(s[p], a[r], out[r]);
    }
  }
};

// A lane's fragments of 256 inputs of its row (planes `plane` elements apart); inputs past the chunk are zero
template <class F, int NP>
DEV void load_x(const uint16_t* row, size_t plane, int c, bool half, uint4 (&x)[NP][8]) {
#pragma unroll
  for (int q = 0; q < NP; ++q) {
    const uint16_t* p = row + q * plane + c * 256 + F::xoff(lane_id() >> 4);
#pragma unroll
    for (int f = 0; f < 8; ++f) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (f < 4 || !half) v = ld16(p + 64 * (f >> 1) + 8 * (f & 1));
      if constexpr (F::perm)
        v = make_uint4(__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
                       __builtin_amdgcn_perm(v.w, v.y, 0x05040100u), __builtin_amdgcn_perm(v.w, v.y, 0x07060302u));
      x[q][f] = v;
    }
  }
}
template <class F, int NP>
DEV float group_sum(const uint4 (&x)[NP][8]) {
  if constexpr (!F::perm) return 0.f;
  float own = 0.f;
#pragma unroll
  for (int G = 0; G < 4; ++G) {
    float t = 0.f;
#pragma unroll
    for (int q = NP - 1; q >= 0; --q)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint4& v = x[q][2 * G + j];
        t += ((bf16_lo(v.x) + bf16_hi(v.x)) + (bf16_lo(v.y) + bf16_hi(v.y))) +
             ((bf16_lo(v.z) + bf16_hi(v.z)) + (bf16_lo(v.w) + bf16_hi(v.w)));
      }
    t = xsum_step<32>(xsum_step<16>(t));
    own = (lane_id() >> 4) == G ? t : own;
  }
  return own;
}

// ---- router -----------------------------------------------------------------------------------
// Logits of TS rows (set blockIdx.y) in the canonical order of canon.hpp, wave w of block b taking router row
// 8 b + w; the set's last block selects each row's picks, a wave per row.  The logits travel to it
// as agent-scope stores that have completed (s_waitcnt, barrier) before the block counts itself in, and are
// read back with agent-scope loads.
template <int TS>
__global__ void __launch_bounds__(MR_NT) k_moe_rows_router(MoeRows a) {
#pragma clang fp contract(off)
  __shared__ float lg[TS][257];
  __shared__ int s_last;
  const int lane = lane_id(), wave = wave_id(), r0 = blockIdx.y * TS, E1 = a.e + a.shared;
  const int n = blockIdx.x * MR_NW + wave;
  if (n < E1) {
    float acc[TS];
#pragma unroll
    for (int t = 0; t < TS; ++t) acc[t] = 0.f;
    const uint16_t* wr = a.router + (size_t)n * a.h;
    const uint16_t* xr[TS];
#pragma unroll
    for (int t = 0; t < TS; ++t) xr[t] = a.x + (size_t)(r0 + t < a.rows ? r0 + t : a.rows - 1) * a.h;
#pragma unroll 4
    for (int c = lane * 8; c < a.h; c += WAVE * 8) {
      const uint4 w = ld16(wr + c);
#pragma unroll
      for (int t = 0; t < TS; ++t) {
        const uint4 v = ld16(xr[t] + c);
        acc[t] = __builtin_fmaf(bf16_lo(w.x), bf16_lo(v.x), acc[t]);
        acc[t] = __builtin_fmaf(bf16_hi(w.x), bf16_hi(v.x), acc[t]);
        acc[t] = __builtin_fmaf(bf16_lo(w.y), bf16_lo(v.y), acc[t]);
        acc[t] = __builtin_fmaf(bf16_hi(w.y), bf16_hi(v.y), acc[t]);
        acc[t] = __builtin_fmaf(bf16_lo(w.z), bf16_lo(v.z), acc[t]);
        acc[t] = __builtin_fmaf(bf16_hi(w.z), bf16_hi(v.z), acc[t]);
        acc[t] = __builtin_fmaf(bf16_lo(w.w), bf16_lo(v.w), acc[t]);
        acc[t] = __builtin_fmaf(bf16_hi(w.w), bf16_hi(v.w), acc[t]);
      }
    }
#pragma unroll
    for (int t = 0; t < TS; ++t) {
      const float v = wave_sum(acc[t]);
      if (lane == 0 && r0 + t < a.rows)
        __hip_atomic_store(a.logits + (size_t)(r0 + t) * E1 + n, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  uint32_t* counter = a.counter + blockIdx.y * 32;
  if (threadIdx.x == 0)
    s_last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
  __syncthreads();
  if (!s_last) return;
  if (threadIdx.x == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const int nr = a.rows - r0 < TS ? a.rows - r0 : TS;
  for (int q = threadIdx.x; q < nr * E1; q += MR_NT)
    lg[q / E1][q % E1] = __hip_atomic_load(a.logits + (size_t)r0 * E1 + q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (wave < nr) {
    int id;
    float w;
    canon_softmax_topk(lg[wave], a.e, a.topk, &id, &w);
    const size_t r = r0 + wave;
    if (lane < a.topk) a.idx[r * a.topk + lane] = id, a.wts[r * a.topk + lane] = w;
    if (lane == 0 && a.shared) a.sgate[r] = lg[wave][a.e];
  }
}

// ---- experts ----------------------------------------------------------------------------------
// MODE 0: gate_up (unit: gate rows 16 t and up rows i + 16 t, K = h), MODE 1: down (unit: rows 32 t, K = i).
// The units of all experts that were picked, ascending, then of the shared expert, are dealt to the blocks in
// even, contiguous runs.  KS waves share a tile's inputs (256 each, a wave taking more than one chunk where
// K is larger), the others take further tiles.
template <int MODE, class F, class FS>
__global__ void __launch_bounds__(MR_NT) k_moe_rows_experts(MoeRows a, int KS) {
  constexpr int NP = MODE == 0 ? 1 : 3;
  __shared__ uint16_t s_pick[MR_PAIRS];
  __shared__ uint32_t s_mask[8];
  __shared__ int s_list[MR_ROWS], s_n;
  __shared__ f32x4 red[2][MR_NW][2][64];
  const int lane = lane_id(), wave = wave_id();
  const int pairs = a.rows * a.topk;
  const int K = MODE == 0 ? a.h : a.i, tiles = MODE == 0 ? a.i / 16 : a.h / 32;
  const int N = MODE == 0 ? 2 * a.i : a.h, second = MODE == 0 ? a.i : 16;
  const int nch = (K + 255) / 256, RG = MR_NW / KS, wk = wave % KS, rg = wave / KS;
  if (threadIdx.x < 8) s_mask[threadIdx.x] = 0;
  __syncthreads();
  for (int p = threadIdx.x; p < pairs; p += MR_NT) {
    const int e = a.idx[p];
    s_pick[p] = (uint16_t)e;
    atomicOr(&s_mask[e >> 5 & 7], 1u << (e & 31));
  }
  __syncthreads();
  int D = 0;
#pragma unroll
  for (int q = 0; q < 8; ++q) D += __builtin_popcount(s_mask[q]);
  const long long U = (long long)(D + a.shared) * tiles;
  int u = (int)(U * blockIdx.x / gridDim.x);
  const int u1 = (int)(U * (blockIdx.x + 1) / gridDim.x);
  int par = 0;
  while (u < u1) {
    const int d = u / tiles, t0 = u - d * tiles, t1 = t0 + (u1 - u) < tiles ? t0 + (u1 - u) : tiles;
    u += t1 - t0;
    const bool sh = d == D;
    int e = 0;
    if (!sh) {  // the d-th set bit
      int left = d;
      for (int q = 0; q < 8; ++q) {
        uint32_t m = s_mask[q];
        const int c = __builtin_popcount(m);
        if (left >= c) {
          left -= c;
          continue;
        }
        for (; left > 0; --left) m &= m - 1;
        e = 32 * q + __builtin_ctz(m);
        break;
      }
    }
    __syncthreads();  // the previous segment's list has been read
    if (wave == 0) {
      int n = 0;
      if (sh) {
        n = a.rows;
        if (lane < n) s_list[lane] = pairs + lane;
      } else {
        for (int b = 0; b < pairs; b += 64) {
          const bool hit = b + lane < pairs && s_pick[b + lane] == e;
          const unsigned long long m = __ballot(hit);
          if (hit) s_list[n + __builtin_popcountll(m & ((1ull << lane) - 1))] = b + lane;
          n += __builtin_popcountll(m);
        }
      }
      if (lane == 0) s_n = n;
    }
    __syncthreads();
    const int cnt = s_n;
    auto segment = [&](auto fmt, const uint8_t* Q, const void* S) __attribute__((always_inline)) {
      using Fm = decltype(fmt);
      for (int t = t0; t < t1; t += RG) {
        const int tile = t + rg;
        const int n0 = (MODE == 0 ? 16 : 32) * tile + (lane & 15);
        for (int p0 = 0; p0 < cnt; p0 += 16) {
          f32x4 o0 = {0.f, 0.f, 0.f, 0.f}, o1 = o0;
          if (tile < t1) {
            const int pr = s_list[p0 + (lane & 15) < cnt ? p0 + (lane & 15) : cnt - 1];
            const uint16_t* xr;
            if constexpr (MODE == 0) xr = a.x + (size_t)(sh ? pr - pairs : pr / a.topk) * K;
            else xr = a.act + (size_t)pr * K;
            const size_t plane = (size_t)(pairs + a.rows) * a.i;
            for (int c = wk; c < nch; c += KS) {
              const bool half = c * 256 + 128 >= K;
              Fm w0, w1;
              w0.load(Q, S, e, n0, N, K, c, half), w1.load(Q, S, e, n0 + second, N, K, c, half);
              uint4 x[NP][8];
              load_x<Fm, NP>(xr, plane, c, half, x);
              const float xs = group_sum<Fm, NP>(x);
              w0.mac(x, xs, o0), w1.mac(x, xs, o1);
            }
          }
          red[par][wave][0][lane] = o0, red[par][wave][1][lane] = o1;
          __syncthreads();
          // thread q of a row group's 64 KS: D register r of lane l is row 4 (l / 16) + r of x, column l % 16
          const int np = cnt - p0 < 16 ? cnt - p0 : 16;
          for (int q = threadIdx.x % (64 * KS); q < (MODE == 0 ? 256 : 512); q += 64 * KS) {
            const int l = q & 63, r = q >> 6 & 3, row = 4 * (l >> 4) + r;
            if (row >= np || tile >= t1) continue;
            const int pr = s_list[p0 + row];
            if constexpr (MODE == 0) {
              float g = 0.f, v = 0.f;
              for (int k = 0; k < KS; ++k) g += red[par][rg * KS + k][0][l][r], v += red[par][rg * KS + k][1][l][r];
              const float act = g / (1.f + expf(-g)) * v;
              uint16_t* o = a.act + (size_t)pr * a.i + 16 * tile + (l & 15);
              const size_t plane = (size_t)(pairs + a.rows) * a.i;
              const float hi = __uint_as_float(__float_as_uint(act) & 0xffff0000u), r1 = act - hi;
              const float mi = __uint_as_float(__float_as_uint(r1) & 0xffff0000u), r2 = r1 - mi;
              o[0] = (uint16_t)(__float_as_uint(hi) >> 16);
              o[plane] = (uint16_t)(__float_as_uint(mi) >> 16);
              o[2 * plane] = (uint16_t)(__float_as_uint(r2) >> 16);
            } else {
              const int half = q >> 8;
              float v = 0.f;
              for (int k = 0; k < KS; ++k) v += red[par][rg * KS + k][half][l][r];
              a.yp[(size_t)pr * a.h + 32 * tile + 16 * half + (l & 15)] = v;
            }
          }
          par ^= 1;
        }
      }
    };
    if (sh) segment(FS{}, reinterpret_cast<const uint8_t*>(MODE == 0 ? a.sgu_q : a.sd_q), MODE == 0 ? a.sgu_s : a.sd_s);
    else segment(F{}, MODE == 0 ? a.gu_q : a.d_q, MODE == 0 ? a.gu_s : a.d_s);
  }
}

__global__ void __launch_bounds__(256) k_moe_rows_combine(MoeRows a) {
  const int r = blockIdx.x, c = (blockIdx.y * 256 + threadIdx.x) * 4;
  if (c >= a.h) return;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (a.shared) {
    const float g = 1.f / (1.f + expf(-a.sgate[r]));
    const float4 v = ldf4(a.yp + (size_t)(a.rows * a.topk + r) * a.h + c);
    acc = make_float4(g * v.x, g * v.y, g * v.z, g * v.w);
  }
#pragma unroll 8
  for (int k = 0; k < a.topk; ++k) {
    const float w = a.wts[r * a.topk + k];
    const float4 v = ldf4(a.yp + (size_t)(r * a.topk + k) * a.h + c);
    acc.x += w * v.x, acc.y += w * v.y, acc.z += w * v.z, acc.w += w * v.w;
  }
  const size_t o = (size_t)r * a.h + c;
  if (a.res) {
    const float4 v = ldf4(a.res + o);
    acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
  }
  *reinterpret_cast<float4*>(a.y + o) = acc;
}

// ---- host -------------------------------------------------------------------------------------
bool rows_shape_ok(int rows, int e, int h, int i, int topk) {
  return rows >= 1 && rows <= MR_ROWS && e >= 1 && e <= 256 && topk >= 1 && topk <= MR_TOPK && topk <= e && h >= 128 && h <= 8192 &&
         h % 128 == 0 && i >= 128 && i <= 8192 && i % 128 == 0;
}
constexpr size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
struct WsLayout {
  size_t logits, act, yp, bytes;
  WsLayout(int rows, int e, int h, int i, int topk) {
    const size_t pr = (size_t)rows * (topk + 1);
    logits = 128 * MR_SETS;
    act = logits + up256((size_t)rows * (e + 1) * 4);
    yp = act + up256(pr * i * 6);
    bytes = yp + up256(pr * h * 4);
  }
};

int waves_on_k(int K) {
  const int nch = (K + 255) / 256;
  return nch >= 8 ? 8 : nch >= 4 ? 4 : nch >= 2 ? 2 : 1;
}

template <class F, class FS>
int moe_rows(MoeRows a, void* ws, hipStream_t st) {
  if (!rows_shape_ok(a.rows, a.e, a.h, a.i, a.topk)) return -1;
  const int given = (a.sgu_q != nullptr) + (a.sgu_s != nullptr) + (a.sd_q != nullptr) + (a.sd_s != nullptr);
  if (given != 0 && given != 4) return -1;
  a.shared = given == 4;
  if (!a.router || !a.gu_q || !a.gu_s || !a.d_q || !a.d_s || !a.x || !a.idx || !a.wts || !a.y || !ws || (a.shared && !a.sgate)) return -1;
  for (const void* p : {(const void*)a.router, (const void*)a.gu_q, a.gu_s, (const void*)a.d_q, a.d_s, (const void*)a.sgu_q,
                        (const void*)a.sd_q, (const void*)a.x, (const void*)a.res, (const void*)a.y, (const void*)ws})
    if ((uintptr_t)p & 15) return -1;
  const WsLayout l(a.rows, a.e, a.h, a.i, a.topk);
  char* w = static_cast<char*>(ws);
  a.counter = reinterpret_cast<uint32_t*>(w);
  a.logits = reinterpret_cast<float*>(w + l.logits);
  a.act = reinterpret_cast<uint16_t*>(w + l.act);
  a.yp = reinterpret_cast<float*>(w + l.yp);
  const int nb = (a.e + a.shared + MR_NW - 1) / MR_NW;
  if (a.rows <= 2) hipLaunchKernelGGL(k_moe_rows_router<1>, dim3(nb, a.rows), dim3(MR_NT), 0, st, a);
  else if (a.rows <= 8) hipLaunchKernelGGL(k_moe_rows_router<2>, dim3(nb, (a.rows + 1) / 2), dim3(MR_NT), 0, st, a);
  else if (a.rows <= 32) hipLaunchKernelGGL(k_moe_rows_router<4>, dim3(nb, (a.rows + 3) / 4), dim3(MR_NT), 0, st, a);
  else hipLaunchKernelGGL(k_moe_rows_router<8>, dim3(nb, (a.rows + 7) / 8), dim3(MR_NT), 0, st, a);
  hipLaunchKernelGGL((k_moe_rows_experts<0, F, FS>), dim3(MR_GRID), dim3(MR_NT), 0, st, a, waves_on_k(a.h));
  hipLaunchKernelGGL((k_moe_rows_experts<1, F, FS>), dim3(MR_GRID), dim3(MR_NT), 0, st, a, waves_on_k(a.i));
  hipLaunchKernelGGL(k_moe_rows_combine, dim3(a.rows, (a.h + 1023) / 1024), dim3(256), 0, st, a);
  return 0;
}

}  // namespace

API size_t dr_moe_layer_rows_ws(int rows, int e, int h, int i, int topk) {
  return rows_shape_ok(rows, e, h, i, topk) ? WsLayout(rows, e, h, i, topk).bytes : 0;
}

#define MOE_ROWS_ENTRY(NAME, S, F, FS)                                                                              \
  API int NAME(const uint16_t* router, const uint8_t* gu_q, const S* gu_s, const uint8_t* d_q, const S* d_s,              \
               const int8_t* sgu_q, const uint16_t* sgu_s, const int8_t* sd_q, const uint16_t* sd_s, const uint16_t* x,   \
               const float* res, int* idx, float* wts, float* sgate, void* ws, float* y, int rows, int e, int h, int i,   \
               int topk, hipStream_t st) {                                                                                \
    const MoeRows a{router, gu_q, d_q, gu_s, d_s, sgu_q, sd_q, sgu_s, sd_s, x, res, idx, wts, sgate, y, nullptr, nullptr, \
                    nullptr, nullptr, rows, e, h, i, topk, 0};                                                            \
    return moe_rows<F, FS>(a, ws, st);                                                                                    \
  }
MOE_ROWS_ENTRY(dr_moe_layer_rows, uint16_t, RowsQ4<ScaleF16>, RowsQ8<Q8G128F16>)
MOE_ROWS_ENTRY(dr_moe_layer_rows_bf16s, uint16_t, RowsQ4<ScaleBF16>, RowsQ8<Q8RowBF16>)
MOE_ROWS_ENTRY(dr_moe_layer_rows_fp8, float, RowsFP8<0>, RowsQ8<Q8G128F16>)
MOE_ROWS_ENTRY(dr_moe_layer_rows_fp8_bf16s, uint16_t, RowsFP8<1>, RowsQ8<Q8RowBF16>)
