// A whole MoE layer for a few rows (1 .. 64) of any size: per row x (bf16)
//   l = R x, picks by (l desc, index asc), w = softmax(l) renormalised over the picks,
//   y = res + sigmoid(l_E) D_s (silu(G_s x) * (U_s x)) + sum_k w_k D_k (silu(G_k x) * (U_k x)).
//
// An expert is fetched once for each pass of rows that picked it (gate_up: 16 rows, down: 8, fewer of large sizes).  Matrix products run on
// v_mfma_f32_16x16x32_bf16 with A = up to 16 rows of x and B = 16 weight rows, converted exactly to bf16
// in registers (int4: 16 + q, with the rest of q scale + min in one fp32 MFMA of the group sums of x), so x
// enters exactly.  The activations are fp32; they travel as three bf16 planes of 8 mantissa
// bits each (their sum is the fp32 value), so nothing is rounded but the fp32 sums.
// Four launches: router, gate_up, down, combine; for one row three, the last of which completes y.
#include "canon.hpp"

using namespace drm;

namespace {

constexpr int MR_NW = 8, MR_NT = MR_NW * 64, MR_ROWS = 64, MR_TOPK = 32, MR_PAIRS = MR_ROWS * MR_TOPK;
constexpr int MR_GRID = 256;             // a block per CU
constexpr int MR_X = 120 * 1024;         // LDS bytes for rows of x
constexpr int MR_ITEMS = MR_PAIRS + MR_ROWS;  // passes, the experts' and the shared expert's, of one row each at worst
constexpr int MR_SETS = 8;               // row sets of the router

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

DEV f32x4 mfma(const uint4& a, const uint4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

DEV uint32_t pick(bool c, uint32_t a, uint32_t b) { return c ? a : b; }

// f(0), .., f(N - 1) with the index a constant, so that arrays it selects from live in registers
template <int N, int I = 0, class Fn>
DEV void static_for(Fn f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    static_for<N, I + 1>(f);
  }
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
// One wave's part of a 16-row tile: chunk c of 256 inputs of each row.  For the product lane l has row l % 16 and
// (g = l / 16) fragment f (two for each group of 64 inputs) the inputs 64 (f / 2) + xoff(g) + 8 (f % 2) .. + 8.
// A load takes 128 bytes of 8 rows, a whole line each (16 rows of 64 bytes would ask for every line twice: 5 to 10% of
// the kernels' time); rows of a pair of loads change places in pair_up.
// The loads go through buffer resources of one expert's matrix, so a piece past the row's inputs (half: only the
// chunk's first 128 exist) and a tile that does not exist (off: nothing left to prefetch) read zeros without a
// fetch, and the code in flight stays free of branches, which keeps the load counter exact.
typedef __amdgpu_buffer_rsrc_t Rsrc;
DEV Rsrc rsrc(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
}
constexpr uint32_t NOWHERE = 0x80000000u;  // past every matrix
DEV gu32x4 buf16(const Rsrc& r, uint32_t off) { return __builtin_bit_cast(gu32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0)); }
DEV uint4 words(const gu32x4& v) { return make_uint4(v.x, v.y, v.z, v.w); }

// Where lane l's piece of a row pair's loads lies: row l % 8 (+ 8 in the second load), bytes 16 (4 (l / 8 % 2) + l / 16) of the 128
DEV int pair_row() { return lane_id() & 7; }
DEV int pair_byte() { return ((lane_id() >> 1) & 4) * 16 + (lane_id() >> 4) * 16; }
// a: rows 0 .. 7, b: rows 8 .. 15 -> a: bytes 16 g of the first 64 of row l % 16, b: of the second 64.  Lanes 8 .. 15 of each 16 of a
// take lanes 0 .. 7 of b, and the other way round.
DEV void pair_up(uint4& a, uint4& b) {
  auto sw = [](uint32_t& p, uint32_t& q) __attribute__((always_inline)) {
    const int o = (int)p, n = (int)q;
    p = (uint32_t)__builtin_amdgcn_update_dpp(o, n, 0x128, 0xF, 0xC, false);  // row_ror:8 into lanes 8 .. 15
    q = (uint32_t)__builtin_amdgcn_update_dpp(n, o, 0x128, 0xF, 0x3, false);  // into lanes 0 .. 7
  };
  sw(a.x, b.x), sw(a.y, b.y), sw(a.z, b.z), sw(a.w, b.w);
}

template <class SC>
struct RowsQ4 {
  static constexpr bool perm = true;  // fragment order 0 4 1 5 2 6 3 7
  static constexpr bool sums = true;  // needs the sums of x's groups
  // as loaded, each a register quadruple that stays one (split into words, the ring's loop would copy them, and wait for them)
  struct Raw {
    gu32x4 w[2], s;
  };
  uint4 w[2], s;
  static DEV size_t q_bytes(int N, int K) { return (size_t)N * K / 2; }
  static DEV size_t s_bytes(int N, int K) { return (size_t)N * K / 16; }
  static DEV int xoff(int g) { return 32 * (g & 1) + 16 * (g >> 1); }
  // n: the tile's first row.  WIN: the chunks of a tile come in order, so the scales of four (16 bytes a row each, of as many
  // lines) come with the first, chunk c + l / 16 in lane l; `scales` hands them out (gate_up of 64 rows, 256 experts, h 2048, i
  // 512: 64 -> 57 us; down, of two chunks there, 36.4 -> 36.8, asks for each chunk's).
  template <bool WIN>
  static DEV void load(Raw& f, const Rsrc& Q, const Rsrc& S, int n, int K, int c, bool half, bool off) {
    const bool none = off || (half && (lane_id() & 8));
    const uint32_t p = (n + pair_row()) * (K / 2) + c * 128 + pair_byte();
    f.w[0] = buf16(Q, none ? NOWHERE : p);
    f.w[1] = buf16(Q, none ? NOWHERE : p + 4 * K);
    f.s = buf16(S, off || (WIN && (c & 3)) ? NOWHERE : ((n + (lane_id() & 15)) * (K / 64) + (WIN ? c + (lane_id() >> 4) : c) * 4) * 4);
  }
  struct Win {
    gu32x4 s;
  };
  template <bool WIN>
  static DEV uint4 scales(Win& win, const Raw& f, int c) {
    if constexpr (!WIN) return words(f.s);
    if ((c & 3) == 0) win.s = f.s;
    const int from = ((c & 3) * 16 + (lane_id() & 15)) * 4;
    auto of = [&](uint32_t v) __attribute__((always_inline)) { return (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)v); };
    return make_uint4(of(win.s.x), of(win.s.y), of(win.s.z), of(win.s.w));
  }
  // nibbles of a word as 16 + q in bf16: the nibble is the top four mantissa bits of a number in [16, 32)
  // (the two constants in registers, so that each pair of nibbles is a shift and one v_and_or_b32)
  static DEV uint4 frag(uint32_t v) {
    uint32_t m = 0x00780078u, b = 0x41804180u;
    asm("" : "+s"(m));
    asm("" : "+v"(b));
    return make_uint4(((v << 3) & m) | b, ((v >> 1) & m) | b, ((v >> 5) & m) | b, ((v >> 9) & m) | b);
  }
  // The tile's words in the order of the products: w[p].x, .y the fragments of group 2 p, .z, .w of group 2 p + 1
  DEV void prep(const Raw& f, bool half, const uint4& sc) {
    w[0] = words(f.w[0]), w[1] = words(f.w[1]);
    pair_up(w[0], w[1]);
    s = make_uint4(sc.x, sc.y, pick(half, 0, sc.z), pick(half, 0, sc.w));
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      // lanes g = 0, 1 hold group 2 p, g = 2, 3 group 2 p + 1: two words of each change places
      const auto s02 = __builtin_amdgcn_permlane32_swap(w[p].x, w[p].z, false, false);
      const auto s13 = __builtin_amdgcn_permlane32_swap(w[p].y, w[p].w, false, false);
      w[p] = make_uint4(s02[0], s13[0], s02[1], s13[1]);
    }
  }
  // Weight row n of the matrix at q, s times x(k), k < K, by the formula itself: sum of (q scale + min) x.  A wave; every lane
  // gets the sum.
  template <class X>
  static DEV float dot(const uint8_t* q, const void* s, int n, int K, X x) {
    const uint8_t* qr = q + (size_t)n * (K / 2);
    const uint32_t* sr = reinterpret_cast<const uint32_t*>(s) + (size_t)n * (K / 64);
    float sum = 0.f;
    for (int k = 8 * lane_id(); k < K; k += 8 * WAVE) {
      const uint32_t w = gld<uint32_t>(qr + k / 2);
      const float2 o = SC::pair(gld<uint32_t>(sr + k / 64));
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = __builtin_fmaf(__builtin_fmaf((float)(w >> (4 * j) & 15u), o.x, o.y), x(k + j), sum);
    }
    return wave_sum(sum);
  }
  // what 16 + q leaves of q scale + min; xsum: the lane's sum of x over group l / 16 of row l % 16
  DEV void rest(float xsum, f32x4& out) const {
    const int g = lane_id() >> 4;
    // (by value: a choice between members would keep them in memory)
    const uint32_t lo = pick(g & 1, s.y, s.x), hi = pick(g & 1, s.w, s.z);
    const float2 o = SC::pair(pick(g & 2, hi, lo));
    out = __builtin_amdgcn_mfma_f32_16x16x4f32(xsum, o.y - 16.f * o.x, out, 0, 0, 0);
  }
  // group 2 p + h of the chunk, the x fragments x[q] into out[q][i]
  template <int NQ, int MQ, int TL>
  DEV void group(int p, int h, const uint4 (&x)[NQ][2], f32x4 (&)[NQ][TL], f32x4 (&out)[MQ][TL], int i) const {
    const uint4 b0 = frag(pick(h, w[p].z, w[p].x)), b1 = frag(pick(h, w[p].w, w[p].y));
    const float sc = SC::pair(p ? pick(h, s.w, s.z) : pick(h, s.y, s.x)).x;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const f32x4 a = mfma(x[q][1], b1, mfma(x[q][0], b0, f32x4{0.f, 0.f, 0.f, 0.f}));
#pragma unroll
      for (int r = 0; r < 4; ++r) out[q][i][r] = __builtin_fmaf(sc, a[r], out[q][i][r]);
    }
  }
};

// One byte per weight: 64 inputs of a row per 16-byte load of four lanes, scales per 128 inputs.  D: the
// format's conversions
template <class D, bool PERM>
struct Rows8 {
  static constexpr bool perm = PERM, sums = false;
  struct Raw {
    gu32x4 w[4];
    uint32_t s[2];
  };
  uint4 w[4];
  uint32_t s[2];
  static DEV size_t q_bytes(int N, int K) { return (size_t)N * K; }
  static DEV int xoff(int g) { return 16 * g; }
  template <bool>
  static DEV void load(Raw& f, const Rsrc& Q, const Rsrc& S, int n, int K, int c, bool half, bool off) {
    const uint32_t p = (n + pair_row()) * K + c * 256 + pair_byte();
    f.w[0] = buf16(Q, off ? NOWHERE : p), f.w[1] = buf16(Q, off ? NOWHERE : p + 8 * K);
    f.w[2] = buf16(Q, half ? NOWHERE : p + 128), f.w[3] = buf16(Q, half ? NOWHERE : p + 128 + 8 * K);
    f.s[0] = D::scale_raw(S, n + (lane_id() & 15), 2 * c, K, off);
    f.s[1] = D::scale_raw(S, n + (lane_id() & 15), 2 * c + 1, K, half);
  }
  struct Win {};
  template <bool>
  static DEV uint4 scales(Win&, const Raw&, int) { return make_uint4(0, 0, 0, 0); }
  DEV void prep(const Raw& f, bool, const uint4&) {
#pragma unroll
    for (int q = 0; q < 4; ++q) w[q] = words(f.w[q]);
    pair_up(w[0], w[1]), pair_up(w[2], w[3]);
    s[0] = f.s[0], s[1] = f.s[1];
  }
  DEV void rest(float, f32x4&) const {}
  template <int NQ, int MQ, int TL>
  DEV void group(int p, int h, const uint4 (&x)[NQ][2], f32x4 (&acc)[NQ][TL], f32x4 (&out)[MQ][TL], int i) const {
    const uint4& v = w[2 * p + h];
    const uint4 b0 = D::frag(v.x, v.y), b1 = D::frag(v.z, v.w);
    const float sc = D::scale_cvt(s[p]);
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      f32x4& a = acc[q][i];
      if (h == 0) a = f32x4{0.f, 0.f, 0.f, 0.f};
      a = mfma(x[q][1], b1, mfma(x[q][0], b0, a));
      if (h == 0) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) out[q][i][r] = __builtin_fmaf(sc, a[r], out[q][i][r]);
    }
  }
};
DEV uint32_t buf_half(const Rsrc& S, uint32_t off) { return (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(S, off, 0, 0); }

template <int SF>
struct RowsFP8 : Rows8<RowsFP8<SF>, false> {
  static DEV size_t s_bytes(int N, int K) { return (size_t)(N / 128) * (K / 128) * (SF ? 2 : 4); }
  static DEV uint32_t scale_raw(const Rsrc& S, int n, int b, int K, bool off) {
    const uint32_t i = (n >> 7) * (K / 128) + b;
    if constexpr (SF) return buf_half(S, off ? NOWHERE : 2 * i);
    else return __builtin_amdgcn_raw_buffer_load_b32(S, off ? NOWHERE : 4 * i, 0, 0);
  }
  static DEV float scale_cvt(uint32_t r) { return blk_cvt<SF>(r); }
  static DEV uint4 frag(uint32_t a, uint32_t b) {
    return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true)));
  }
};

// PERM: the fragment order of int4, beside whose experts it stands
template <class SH, bool PERM>
struct RowsQ8 : Rows8<RowsQ8<SH, PERM>, PERM> {
  static DEV size_t s_bytes(int N, int K) { return (size_t)N * (SH::per_row ? 1 : K / 128) * 2; }
  static DEV uint32_t scale_raw(const Rsrc& S, int n, int b, int K, bool off) {
    return buf_half(S, off ? NOWHERE : 2 * (SH::per_row ? n : n * (K / 128) + b));
  }
  static DEV float scale_cvt(uint32_t r) { return SH::cvt(r); }
  // as RowsQ4::dot
  template <class X>
  static DEV float dot(const int8_t* q, const uint16_t* s, int n, int K, X x) {
    float sum = 0.f;
    for (int k = lane_id(); k < K; k += WAVE) sum = __builtin_fmaf(SH::scale(s, n, k, K) * (float)q[(size_t)n * K + k], x(k), sum);
    return wave_sum(sum);
  }
  static DEV uint32_t pk(uint32_t u, int i, uint32_t v, int j) {  // byte i of u and byte j of v as bf16 (exact)
    const float a = (float)(int8_t)(u >> (8 * i)), b = (float)(int8_t)(v >> (8 * j));
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
  }
  static DEV uint4 frag(uint32_t a, uint32_t b) {
    if constexpr (PERM) return make_uint4(pk(a, 0, b, 0), pk(a, 1, b, 1), pk(a, 2, b, 2), pk(a, 3, b, 3));
    else return make_uint4(pk(a, 0, a, 1), pk(a, 2, a, 3), pk(b, 0, b, 1), pk(b, 2, b, 3));
  }
};

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
    // 2048 inputs at a time: the row of the router, then the rows of x one after the other with the next one in flight;
    // chunks past h are neither loaded nor added
    for (int c0 = lane * 8; c0 - lane * 8 < a.h; c0 += 2048) {
      uint4 w[4], v[2][4];
      auto load = [&](const uint16_t* p, uint4 (&d)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) d[j] = ld16(p + (c0 + 512 * j < a.h ? c0 + 512 * j : 0));
      };
      auto row = [&](int t) { return a.x + (size_t)(r0 + t < a.rows ? r0 + t : a.rows - 1) * a.h; };
      load(wr, w);
      load(row(0), v[0]);
      static_for<TS>([&](auto tt) __attribute__((always_inline)) {
        constexpr int t = decltype(tt)::value;
        if constexpr (t + 1 < TS) load(row(t + 1), v[(t + 1) & 1]);
        issue_fence();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint4 q = w[j], u = v[t & 1][j];
          float s = acc[t];
          s = __builtin_fmaf(bf16_lo(q.x), bf16_lo(u.x), s);
          s = __builtin_fmaf(bf16_hi(q.x), bf16_hi(u.x), s);
          s = __builtin_fmaf(bf16_lo(q.y), bf16_lo(u.y), s);
          s = __builtin_fmaf(bf16_hi(q.y), bf16_hi(u.y), s);
          s = __builtin_fmaf(bf16_lo(q.z), bf16_lo(u.z), s);
          s = __builtin_fmaf(bf16_hi(q.z), bf16_hi(u.z), s);
          s = __builtin_fmaf(bf16_lo(q.w), bf16_lo(u.w), s);
          s = __builtin_fmaf(bf16_hi(q.w), bf16_hi(u.w), s);
          acc[t] = c0 + 512 * j < a.h ? s : acc[t];
        }
      });
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
  {
    // every row's logits requested at once
    constexpr int NL = (TS * 257 + MR_NT - 1) / MR_NT;
    float v[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int q = threadIdx.x + MR_NT * i;
      v[i] = q < nr * E1 ? __hip_atomic_load(a.logits + (size_t)r0 * E1 + q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int q = threadIdx.x + MR_NT * i;
      if (q < nr * E1) lg[q / E1][q % E1] = v[i];
    }
  }
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
// inclusive sum over the lanes
DEV int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

// MODE 0: gate_up (tile t: gate rows 16 t and up rows i + 16 t, K = h), MODE 1: down (tile t: rows 32 t, K = i).
//
// Items are passes of up to P rows (16; down: 8, two fragments of four rows and their planes) of an expert, ascending, then of
// the shared expert (whose rows are all); their tiles are dealt to the blocks in contiguous runs of even length.  The
// shared expert has blocks of its own (a block with tiles of both formats would stage and wait twice: gate_up of 4 rows, 256
// experts, h 2048, i 512, 25 us instead of 19), three times as many for its tiles as the others: its passes are the fullest and
// its format the widest (2 / 3 / 4 times: 64 rows 66.5 / 63.6 / 64.8 us, 8 rows of fp8 experts 26.8 / 25.4 / 25.4, 24 rows of 16
// experts of 4096 x 2048 71 / 71 / 76).  A block stages the rows of its items in LDS (as many items at a time as R rows
// hold, most often all), then each of its waves takes one tile after the other from a counter and multiplies all of its
// inputs, in chunks of 256: no sum crosses waves and no barrier stands between tiles.  A wave's weights come in a ring of
// DEPTH chunks that runs on across tiles and items.
//
// 64 rows, 256 experts, h 2048, i 512, 8 picks and the shared expert: gate_up 64 us, down 40, for 266 and 133 MB; without the
// products the loads alone take 52 (no shared expert; 58 with them) and 32, 4 of each the launch.  The down planes as rows of one
// fragment: 41 -> 38 us, 16 rows 25 -> 20.  Rings of 2 / 3 / 4 chunks: down 39.2 / 40.4 / 43.6, gate_up (19 rows, h 1280, i 896, 48
// experts) 18.6 / 21.4 / 22.4.  16 waves a block: gate_up level, down twice as long (spills); two blocks a CU with half the rows
// each: level to slower.
//
// LDS: row slot s at s * RB, its planes Kp * 2 bytes apart (Kp: K rounded up to a chunk, zeros past K), pieces of 8 inputs
// reordered for int4; RB is 16 bytes more than the planes, so that the rows of a fragment meet different banks.  In down a
// row's three planes share a fragment and meet the same ones, as Kp * 2 is a multiple of 512: 2.3 M conflict cycles for 0.41 M LDS
// instructions (gate_up 0.16 M for 1.07 M) in the case above.
// Then, for int4, the fp32 sums of each 64 inputs.
template <int MODE>
struct XLayout {
  static constexpr int NP = MODE == 0 ? 1 : 3;
  int Kp, RB, GS, R;  // padded inputs, row bytes, floats of sums a row, rows
  __host__ __device__ XLayout(int K) {
    Kp = (K + 255) & ~255;
    RB = NP * Kp * 2 + 16;
    GS = Kp / 64 + 4;
    R = MR_X / (RB + 4 * GS);
  }
};

// nrows rows (row_of(slot): of x, or of act) into the slots from 0; all threads
template <int MODE, bool PERM, bool SUMS, class RowOf>
DEV void stage_rows(const MoeRows& a, const XLayout<MODE>& L, int K, int nrows, char* xb, float* sums, size_t plane, RowOf row_of) {
  constexpr int NP = XLayout<MODE>::NP;
  const int k8 = L.Kp / 8;
  for (int q = threadIdx.x; q < nrows * k8; q += MR_NT) {
    const int slot = q / k8, k = (q - slot * k8) * 8;
    const uint16_t* src = (MODE == 0 ? a.x : a.act) + (size_t)row_of(slot) * K + k;
    float sum = 0.f;
#pragma unroll
    for (int p = NP - 1; p >= 0; --p) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (k < K) v = ld16(src + p * plane);
      if constexpr (SUMS)
        sum += ((bf16_lo(v.x) + bf16_hi(v.x)) + (bf16_lo(v.y) + bf16_hi(v.y))) + ((bf16_lo(v.z) + bf16_hi(v.z)) + (bf16_lo(v.w) + bf16_hi(v.w)));
      if constexpr (PERM)
        v = make_uint4(__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
                       __builtin_amdgcn_perm(v.w, v.y, 0x05040100u), __builtin_amdgcn_perm(v.w, v.y, 0x07060302u));
      *reinterpret_cast<uint4*>(xb + slot * L.RB + (p * L.Kp + k) * 2) = v;
    }
    if constexpr (SUMS) {
      // the 8 pieces of a group are 8 consecutive threads (k8 is a multiple of 8), all in or all past the rows
      sum = xsum_step<4>(xsum_step<2>(xsum_step<1>(sum)));
      if ((q & 7) == 0) sums[slot * L.GS + k / 64] = sum;
    }
  }
}

// o[q] += the products of chunk c of x fragments 0 .. NQ - 1 (a lane's row of each at xr[q], its group sums at sr[q], counted if
// lead) with TL tiles of weights, converted once for all of them
template <int NQ, class Fm, int TL, int MQ>
DEV void chunk_mac(const typename Fm::Raw (&raw)[TL], const uint4 (&sc)[TL], const char* const (&xr)[MQ], const float* const (&sr)[MQ], bool lead, int c, bool half,
                   f32x4 (&o)[MQ][TL]) {
  Fm f[TL];
#pragma unroll
  for (int i = 0; i < TL; ++i) f[i].prep(raw[i], half, sc[i]);
  if constexpr (Fm::sums)
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const float xs = lead ? sr[q][4 * c] : 0.f;
#pragma unroll
      for (int i = 0; i < TL; ++i) f[i].rest(xs, o[q][i]);
    }
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    f32x4 acc[NQ][TL];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 x[NQ][2];
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        const uint4* src = reinterpret_cast<const uint4*>(xr[q] + (c * 256 + 128 * p + 64 * h) * 2);
        x[q][0] = src[0], x[q][1] = src[1];
      }
#pragma unroll
      for (int i = 0; i < TL; ++i) f[i].template group<NQ>(p, h, x, acc, o, i);
    }
  }
}

// down: the planes of four rows share a fragment, plane p of row s in its row 4 s + p (the last of each four unused): lane l has the
// outputs of row l / 16, its planes' in registers 0 .. 2
DEV int quad_row() { return (lane_id() & 15) >> 2; }
DEV int quad_plane() { return min(lane_id() & 3, 2); }
DEV bool quad_lead() { return (lane_id() & 3) == 0; }
DEV float quad_sum(const f32x4& o) { return o[0] + o[1] + o[2]; }

// silu(g) u as three bf16 planes: 8 mantissa bits each, the last exact; returns it
// (no contraction: act - hi of the product before its rounding would leave planes that are not act, nor their group sums for int4)
DEV float store_act(const MoeRows& a, size_t plane, int pair, int col, float g, float u) {
#pragma clang fp contract(off)
  const float act = g / (1.f + expf(-g)) * u;
  uint16_t* dst = a.act + (size_t)pair * a.i + col;
  const float hi = __uint_as_float(__float_as_uint(act) & 0xffff0000u), r1 = act == hi ? 0.f : act - hi;  // (an infinity stays one)
  const float mi = __uint_as_float(__float_as_uint(r1) & 0xffff0000u), r2 = r1 - mi;
  dst[0] = (uint16_t)(__float_as_uint(hi) >> 16);
  dst[plane] = (uint16_t)(__float_as_uint(mi) >> 16);
  dst[2 * plane] = (uint16_t)(__float_as_uint(r2) >> 16);
  return act;
}

// The two parts of an int4 product, 16 + q and min - 16 scale, are up to 31 times (q scale + min) x and of opposite signs: they
// leave fp32 before it does, and an infinite activation gives them infinities of both signs.  So what comes out of them as no finite
// number is summed again from the formula (RowsQ4::dot), where it is an infinity, NaN or a number after all; which outputs
// are, depends on themselves alone, so a row keeps its bits in any company.  Rows with a NaN among their inputs are NaN
// either way and are left.  One wave each, all lanes.  Where nothing overflows this costs the check of the outputs: one row 23.5 -> 23.9 us,
// 19 rows of 48 experts 43.6 -> 43.7, 64 rows of 256 118.2 -> 118.5.
DEV bool no_number(uint32_t bits) { return !__builtin_isfinite(__uint_as_float(bits)); }
DEV float act_at(const MoeRows& a, size_t plane, int pair, int k) {
  const uint16_t* p = a.act + (size_t)pair * a.i + k;
  return bf16f(p[0]) + bf16f(p[plane]) + bf16f(p[2 * plane]);
}
template <class X>
DEV bool has_nan(int K, X x) {
  bool nan = false;
  for (int k = lane_id(); k < K; k += WAVE) nan = nan || x(k) != x(k);
  return __any(nan);
}
// activations 16 tile + c of the pair whose row of x is xr, for each bit c of odd
template <class F>
DEV void acts_again(const MoeRows& a, size_t plane, int e, const uint16_t* xr, int pair, int tile, uint32_t odd) {
  auto x = [&](int k) { return bf16f(xr[k]); };
  if (has_nan(a.h, x)) return;
  const uint8_t* q = a.gu_q + (size_t)e * F::q_bytes(2 * a.i, a.h);
  const char* s = reinterpret_cast<const char*>(a.gu_s) + (size_t)e * F::s_bytes(2 * a.i, a.h);
  for (; odd; odd &= odd - 1) {
    const int n = 16 * tile + __builtin_ctz(odd);
    const float g = F::dot(q, s, n, a.h, x), u = F::dot(q, s, a.i + n, a.h, x);
    if (lane_id() == 0) store_act(a, plane, pair, n, g, u);
  }
}
// output n of the pair by expert e
template <class F>
DEV float down_again(const MoeRows& a, size_t plane, int e, int pair, int n) {
  return F::dot(a.d_q + (size_t)e * F::q_bytes(a.h, a.i), reinterpret_cast<const char*>(a.d_s) + (size_t)e * F::s_bytes(a.h, a.i), n, a.i,
                [&](int k) { return act_at(a, plane, pair, k); });
}

template <int MODE, class F, class FS>
__global__ void __launch_bounds__(MR_NT, 2) k_moe_rows_experts(MoeRows a) {
  constexpr int TL = 2, MQ = MODE == 0 ? 1 : 2;  // tiles of 16 weight rows, x fragments
  constexpr bool WIN = MODE == 0;
  extern __shared__ uint4 xlds[];
  __shared__ uint16_t s_list[MR_PAIRS + MR_ROWS];  // pairs by expert, then the shared expert's rows
  __shared__ uint16_t s_e[MR_ITEMS], s_off[MR_ITEMS], s_num[MR_ITEMS];  // items: expert, first place in s_list, rows
  __shared__ uint2 s_rows[256];
  __shared__ int s_start[256], s_d0, s_ticket, s_odd;  // s_odd: an output of this block so far is no finite number
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), tid = threadIdx.x, c16 = lane & 15, g = lane >> 4;
  const int pairs = a.rows * a.topk;
  const int K = MODE == 0 ? a.h : a.i, tiles = MODE == 0 ? a.i / 16 : a.h / 32, N = MODE == 0 ? 2 * a.i : a.h;
  const int nch = (K + 255) / 256;
  const XLayout<MODE> L(K);
  constexpr int PM = MODE == 0 ? 16 : 4 * MQ;
  const int P = L.R < PM ? L.R : PM;
  // rows of each expert as a 64-bit mask (a row picks an expert once), so that every block has the same passes
  constexpr int PPT = MR_PAIRS / MR_NT;
  int pe[PPT];
#pragma unroll
  for (int q = 0; q < PPT; ++q) pe[q] = tid + MR_NT * q < pairs ? a.idx[tid + MR_NT * q] & 255 : -1;
  if (tid < 256) s_rows[tid] = make_uint2(0, 0);
  lds_barrier();
#pragma unroll
  for (int q = 0; q < PPT; ++q)
    if (pe[q] >= 0) {
      const int r = (tid + MR_NT * q) / a.topk;
      atomicOr(r < 32 ? &s_rows[pe[q]].x : &s_rows[pe[q]].y, 1u << (r & 31));
    }
  lds_barrier();
  if (wave == 0) {
    // lane l: experts 4 l .. 4 l + 3; rows and passes summed over the experts before, in the halves of a word
    int n[4], v = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint2 m = s_rows[4 * lane + j];
      n[j] = __builtin_popcount(m.x) + __builtin_popcount(m.y);
      v += n[j] | (n[j] + P - 1) / P << 16;
    }
    int at = wave_scan(v) - v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int off = at & 0xffff, d = at >> 16;
      s_start[4 * lane + j] = off;
      at += n[j] | (n[j] + P - 1) / P << 16;
      for (int left = n[j]; left > 0; left -= P, off += P, ++d) s_e[d] = 4 * lane + j, s_off[d] = off, s_num[d] = left < P ? left : P;
    }
    if (lane == 63) {
      int d = at >> 16;
      s_d0 = d, s_ticket = 0, s_odd = 0;
      if (a.shared)
        for (int r = 0; r < a.rows; r += P, ++d) s_e[d] = 256, s_off[d] = pairs + r, s_num[d] = a.rows - r < P ? a.rows - r : P;
    }
  }
  lds_barrier();
#pragma unroll
  for (int q = 0; q < PPT; ++q)
    if (pe[q] >= 0) {
      const int r = (tid + MR_NT * q) / a.topk;
      const uint2 m = s_rows[pe[q]];
      const uint32_t below = (1u << (r & 31)) - 1;
      s_list[s_start[pe[q]] + (r < 32 ? __builtin_popcount(m.x & below) : __builtin_popcount(m.x) + __builtin_popcount(m.y & below))] =
          tid + MR_NT * q;
    }
  if (a.shared && tid < a.rows) s_list[pairs + tid] = pairs + tid;
  lds_barrier();
  // the shared expert's blocks, in the measure of its cost, and this block's tiles lo .. hi - 1 of the items from dbase on
  const int D0 = __builtin_amdgcn_readfirstlane(s_d0), DS = a.shared ? (a.rows + P - 1) / P : 0;
  const int grid = gridDim.x, cost = 3 * DS, nS = DS == 0 ? 0 : max(1, min(grid - 1, (2 * grid * cost + D0 + cost) / (2 * (D0 + cost))));
  const bool sh = (int)blockIdx.x < nS;
  const int b = sh ? blockIdx.x : blockIdx.x - nS, nb = sh ? nS : grid - nS, all = (sh ? DS : D0) * tiles, dbase = sh ? D0 : 0;
  const int lo = (int)((long long)all * b / nb), hi = (int)((long long)all * (b + 1) / nb);
  if (lo >= hi) return;
  const int dfirst = dbase + lo / tiles, dend = dbase + (hi - 1) / tiles + 1;
  const size_t plane = (size_t)(pairs + a.rows) * a.i;
  char* xb = reinterpret_cast<char*>(xlds);
  float* sums = reinterpret_cast<float*>(xb + (size_t)L.R * L.RB);
  // the block's tiles [t0, t1) of item d
  auto range = [&](int d, int& t0, int& t1) __attribute__((always_inline)) {
    const int cum = (d - dbase) * tiles;
    t0 = lo > cum ? lo - cum : 0, t1 = hi - cum < tiles ? hi - cum : tiles;
  };
  // items dA .. dB - 1, their rows in the slots from 0
  auto run = [&](auto fmt, const int dA, const int dB, const bool sh, const uint8_t* Wq, const void* Ws) __attribute__((always_inline)) {
    using Fm = decltype(fmt);
    constexpr int DEPTH = 2;
    const int pos = s_off[dA], nrows = s_off[dB - 1] + s_num[dB - 1] - pos;
    // the position to load next: chunk lc of tile lt of item ld, whose tiles here are the counter's lbase .. lbase + ln - 1
    int ld = dA, lbase = 0, lt = 0, lt0, lt1, lc = nch;
    bool over = false;
    range(ld, lt0, lt1);
    Rsrc Q, S;
    auto open = [&]() __attribute__((always_inline)) {
      const size_t m = sh ? 0 : __builtin_amdgcn_readfirstlane(s_e[ld]);
      Q = rsrc(Wq + m * Fm::q_bytes(N, K), (uint32_t)Fm::q_bytes(N, K));
      S = rsrc(reinterpret_cast<const char*>(Ws) + m * Fm::s_bytes(N, K), (uint32_t)Fm::s_bytes(N, K));
    };
    open();
    int td[DEPTH], tt[DEPTH], tc[DEPTH];  // item (-1: none), tile and chunk of the ring's places
    typename Fm::Raw w[DEPTH][TL];
    auto advance = [&](typename Fm::Raw (&f)[TL], int& d, int& t, int& c) __attribute__((always_inline)) {
      if (++lc >= nch && !over) {
        int k = 0;
        if (lane == 0) k = atomicAdd(&s_ticket, 1);
        k = __builtin_amdgcn_readfirstlane(k);
        if (k >= lbase + lt1 - lt0) {
          do {
            lbase += lt1 - lt0;
            if (++ld >= dB) {
              over = true;
              break;
            }
            range(ld, lt0, lt1);
          } while (k >= lbase + lt1 - lt0);
          if (!over) open();
        }
        lt = lt0 + k - lbase, lc = 0;
      }
      d = over ? -1 : ld, t = lt, c = lc;
      const bool none = over | (lc * 256 + 128 >= K);
#pragma unroll
      for (int i = 0; i < TL; ++i) Fm::template load<WIN>(f[i], Q, S, MODE == 0 ? 16 * lt + i * a.i : 32 * lt + 16 * i, K, lc, none, over);
      __builtin_amdgcn_sched_barrier(0);
    };
    static_for<DEPTH>([&](auto k) __attribute__((always_inline)) { advance(w[k.value], td[k.value], tt[k.value], tc[k.value]); });
    // the rows, requested behind the first weights: the two waits are one
    stage_rows<MODE, Fm::perm, Fm::sums>(a, L, K, nrows, xb, sums, plane, [&](int slot) {
      const int pr = s_list[pos + slot];
      return MODE == 0 ? (sh ? pr - pairs : pr / a.topk) : pr;
    });
    lds_barrier();
    f32x4 o[MQ][TL];
    const char* xr[MQ];
    const float* sr[MQ];
    int cnt = 0;
    float odd = 0.f;  // NaN once an output of this lane is no finite number
    typename Fm::Win win[TL] = {};
#pragma unroll
    for (int q = 0; q < MQ; ++q) xr[q] = xb, sr[q] = sums;
    auto body = [&](typename Fm::Raw (&raw)[TL], int& d, int& t, int& c) __attribute__((always_inline)) {  // one chunk
      if (c == 0 && d >= 0) {
        cnt = s_num[d];
#pragma unroll
        for (int q = 0; q < MQ; ++q) {
          const int row = MODE == 0 ? c16 : 4 * q + quad_row(), slot = s_off[d] - pos + (row < cnt ? row : cnt - 1);
          xr[q] = xb + slot * L.RB + 2 * Fm::xoff(g) + (MODE == 0 ? 0 : quad_plane() * L.Kp * 2);
          sr[q] = sums + slot * L.GS + g;
#pragma unroll
          for (int i = 0; i < TL; ++i) o[q][i] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
      }
      const bool half = c * 256 + 128 >= K, lead = MODE == 0 || quad_lead();
      uint4 sc[TL];
#pragma unroll
      for (int i = 0; i < TL; ++i) sc[i] = Fm::template scales<WIN>(win[i], raw[i], c);
      if (MODE == 0 || cnt <= 4) chunk_mac<1, Fm>(raw, sc, xr, sr, lead, c, half, o);
      else chunk_mac<MQ, Fm>(raw, sc, xr, sr, lead, c, half, o);
      if (c == nch - 1 && d >= 0) {
        const int off = s_off[d];
        if constexpr (MODE == 0) {
          // register r of lane l: row 4 (l / 16) + r of x, column l % 16
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (r >= cnt) break;
            const int row = 4 * g + r;
            if (row >= cnt) continue;
            const float act = store_act(a, plane, s_list[off + row], 16 * t + c16, o[0][0][r], o[0][1][r]);
            if constexpr (Fm::sums) odd = __builtin_fmaf(0.f, act, odd);
          }
        } else {
#pragma unroll
          for (int q = 0; q < MQ; ++q) {
            if (4 * q >= cnt) break;
            const int row = 4 * q + g;
            if (row >= cnt) continue;
            float* dst = a.yp + (size_t)s_list[off + row] * a.h + 32 * t + c16;
#pragma unroll
            for (int i = 0; i < TL; ++i) {
              const float v = quad_sum(o[q][i]);
              dst[16 * i] = v;
              if constexpr (Fm::sums) odd = __builtin_fmaf(0.f, v, odd);
            }
          }
        }
      }
      advance(raw, d, t, c);
    };
    // One exit, at the head: places of the ring without a tile are computed too (zeros, not stored), since paths that
    // skip loads and join the loop again would make every wait in it a wait for all loads.
    while (td[0] >= 0) static_for<DEPTH>([&](auto k) __attribute__((always_inline)) { body(w[k.value], td[k.value], tt[k.value], tc[k.value]); });
    if (odd != 0.f) s_odd = 1;
    lds_barrier();  // the rows may be replaced, the counter starts again
    if (tid == 0) s_ticket = 0;
    lds_barrier();
  };
  for (int d = dfirst; d < dend;) {
    int e = d + 1;
    while (e < dend && s_off[e] + s_num[e] - s_off[d] <= L.R) ++e;
    if (sh) run(FS{}, d, e, true, reinterpret_cast<const uint8_t*>(MODE == 0 ? a.sgu_q : a.sd_q), MODE == 0 ? a.sgu_s : a.sd_s);
    else run(F{}, d, e, false, MODE == 0 ? a.gu_q : a.d_q, MODE == 0 ? a.gu_s : a.d_s);
    d = e;
  }
  if constexpr (F::sums) {
    if (!s_odd) return;  // (behind the last barrier of run, so the same for all waves)
    __syncthreads();     // the waves' stores
    for (int d = dfirst; d < dend; ++d) {
      const int cnt = s_num[d], e = s_e[d];
      int t0, t1;
      range(d, t0, t1);
      for (int q = wave; q < (t1 - t0) * cnt; q += MR_NW) {
        const int t = t0 + q / cnt, pr = s_list[s_off[d] + q % cnt];
        if constexpr (MODE == 0) {
          const uint32_t odd = (uint32_t)__ballot(lane < 16 && no_number((uint32_t)a.act[(size_t)pr * a.i + 16 * t + c16] << 16));
          if (odd) acts_again<F>(a, plane, e, a.x + (size_t)(pr / a.topk) * a.h, pr, t, odd);
        } else {
          float* y = a.yp + (size_t)pr * a.h + 32 * t;
          uint32_t odd = (uint32_t)__ballot(lane < 32 && no_number(__float_as_uint(y[lane & 31])));
          if (!odd || has_nan(a.i, [&](int k) { return act_at(a, plane, pr, k); })) continue;
          for (; odd; odd &= odd - 1) {
            const int n = __builtin_ctz(odd);
            const float v = down_again<F>(a, plane, e, pr, 32 * t + n);
            if (lane == 0) y[n] = v;
          }
        }
      }
    }
  }
}

// ---- experts of one row -----------------------------------------------------------------------
// With so few tiles the kernels above wait for one wave's walk through all inputs of a tile, and their last launch (the
// combine) costs little but its start.  gate_up: the eight waves of a block share the inputs of a tile (16 gate and 16 up rows),
// their sums meet in LDS.  down: a block owns 16 outputs; its waves share out (pick, chunk), weight and add the
// products, and the block joins those with res: y is complete.  The row stands in all rows of the fragments.
// 256 experts, h 2048, i 512, 8 picks and the shared expert: 9.6 + 8.4 us, the kernels above 12.8 + 8.2 + 4.1 and one launch
// more (two rows, in kernels like these: 12.6 + 14.3 against 13.8 + 9.2 + 4.0).
// Two chunks under way per wave in down; four cost 4 us more (places without work are multiplied too).
template <int MODE, class F, class FS>
__global__ void __launch_bounds__(MR_NT, MODE == 0 ? 4 : 2) k_moe_rows_one(MoeRows a) {
  constexpr int TL = MODE == 0 ? 2 : 1, RING = 2;
  extern __shared__ uint4 xlds[];
  __shared__ float red[2][MR_NW][TL][16];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), c16 = lane & 15, g = lane >> 4;
  const int K = MODE == 0 ? a.h : a.i, tiles = MODE == 0 ? a.i / 16 : a.h / 16, N = MODE == 0 ? 2 * a.i : a.h;
  const int nch = (K + 255) / 256, S = a.shared ? 1 : 0, grid = gridDim.x, blk = blockIdx.x;
  const XLayout<MODE> L(K);
  const int slots = MODE == 0 ? 1 : a.topk + S;
  const size_t plane = (size_t)(a.topk + 1) * a.i;
  char* xb = reinterpret_cast<char*>(xlds);
  float* sums = reinterpret_cast<float*>(xb + (size_t)slots * L.RB);
  // pick p in lane p, with its weight in y (the shared expert's the last)
  const int mine = lane < a.topk ? a.idx[lane] & 255 : 0;
  float wt = 0.f;
  if constexpr (MODE == 1) {
    wt = lane < a.topk ? a.wts[lane] : 0.f;
    if (S && lane == a.topk) wt = 1.f / (1.f + expf(-a.sgate[0]));
  }
  // chunk c of tile `tile` of pick d (none: nothing is fetched)
  auto load = [&](auto fmt, auto& raw, const bool sh, const uint8_t* Wq, const void* Ws, int d, int tile, int c, bool none) __attribute__((always_inline)) {
    using Fm = decltype(fmt);
    const size_t m = sh || none ? 0 : __builtin_amdgcn_readlane(mine, d);
    const Rsrc Q = rsrc(Wq + m * Fm::q_bytes(N, K), (uint32_t)Fm::q_bytes(N, K));
    const Rsrc Z = rsrc(reinterpret_cast<const char*>(Ws) + m * Fm::s_bytes(N, K), (uint32_t)Fm::s_bytes(N, K));
#pragma unroll
    for (int i = 0; i < TL; ++i) Fm::template load<false>(raw[i], Q, Z, 16 * tile + i * a.i, K, c, none || c * 256 + 128 >= K, none);
    __builtin_amdgcn_sched_barrier(0);
  };
  bool staged = false;
  auto stage = [&]() __attribute__((always_inline)) {  // behind the first weights
    if (staged) return;
    stage_rows<MODE, F::perm, F::sums>(a, L, K, slots, xb, sums, plane, [](int slot) { return slot; });
    lds_barrier();
    staged = true;
  };
  if constexpr (MODE == 0) {
    const float* const sr[1] = {sums + g};
    int par = 0;
    // tiles u0, u0 + grid, .. of the picks or of the shared expert
    auto run = [&](auto fmt, int u0, int units, const bool sh, const uint8_t* Wq, const void* Ws) __attribute__((always_inline)) {
      using Fm = decltype(fmt);
      if (u0 >= units) return;
      const char* const xr[1] = {xb + 2 * Fm::xoff(g)};
      typename Fm::Raw raw[TL];
      load(fmt, raw, sh, Wq, Ws, u0 / tiles, u0 % tiles, wave, wave >= nch);
      stage();
      for (int u = u0; u < units; u += grid) {
        const int d = u / tiles, tile = u - d * tiles, v = u + grid;
        f32x4 o[1][TL];
#pragma unroll
        for (int i = 0; i < TL; ++i) o[0][i] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int c = wave; c < nch; c += MR_NW) {
          if (c != wave) load(fmt, raw, sh, Wq, Ws, d, tile, c, false);
          typename Fm::Win win;
          uint4 sc[TL];
#pragma unroll
          for (int i = 0; i < TL; ++i) sc[i] = Fm::template scales<false>(win, raw[i], c);
          chunk_mac<1, Fm>(raw, sc, xr, sr, true, c, c * 256 + 128 >= K, o);
        }
        load(fmt, raw, sh, Wq, Ws, v / tiles, v % tiles, wave, v >= units || wave >= nch);
        if (g == 0)
#pragma unroll
          for (int i = 0; i < TL; ++i) red[par][wave][i][c16] = o[0][i][0];
        lds_barrier();
        if (wave == 4 * par) {
          float s[TL] = {0.f, 0.f};
#pragma unroll
          for (int k = 0; k < MR_NW; ++k)
#pragma unroll
            for (int i = 0; i < TL; ++i) s[i] += red[par][k][i][c16];
          float act = 0.f;
          if (g == 0) act = store_act(a, plane, sh ? a.topk : d, 16 * tile + c16, s[0], s[1]);
          if constexpr (Fm::sums) {
            const uint32_t odd = (uint32_t)__ballot(no_number(__float_as_uint(act)));
            if (odd) acts_again<Fm>(a, plane, __builtin_amdgcn_readlane(mine, d), a.x, d, tile, odd);
          }
        }
        par ^= 1;
      }
    };
    const int us = S * tiles;
    if (S) run(FS{}, blk, us, true, reinterpret_cast<const uint8_t*>(a.sgu_q), a.sgu_s);
    run(F{}, (blk + grid - us % grid) % grid, a.topk * tiles, false, a.gu_q, a.gu_s);
  } else {
    int par = 0;
    for (int tile = blk; tile < tiles; tile += grid) {
      float sum = 0.f;
      // (pick, chunk) q0, q0 + 8, .. of one format
      auto run = [&](auto fmt, int q0, int units, const bool sh, const uint8_t* Wq, const void* Ws) __attribute__((always_inline)) {
        using Fm = decltype(fmt);
        typename Fm::Raw raw[RING][TL];
        auto ask = [&](typename Fm::Raw (&f)[TL], int q) __attribute__((always_inline)) {
          load(fmt, f, sh, Wq, Ws, q / nch, tile, q % nch, q >= units);
        };
        auto body = [&](typename Fm::Raw (&f)[TL], int q) __attribute__((always_inline)) {
          const int d = q < units ? q / nch : 0, c = q % nch, slot = sh ? a.topk : d;
          const char* const xr[1] = {xb + slot * L.RB + 2 * Fm::xoff(g) + quad_plane() * L.Kp * 2};
          const float* const sr[1] = {sums + slot * L.GS + g};
          f32x4 o[1][TL] = {{f32x4{0.f, 0.f, 0.f, 0.f}}};
          typename Fm::Win win;
          const uint4 sc[TL] = {Fm::template scales<false>(win, f[0], c)};
          chunk_mac<1, Fm>(f, sc, xr, sr, quad_lead(), c, c * 256 + 128 >= K, o);
          ask(f, q + RING * MR_NW);
          const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(wt), slot));
          if (q < units) sum += w * quad_sum(o[0][0]);
        };
        static_for<RING>([&](auto j) __attribute__((always_inline)) { ask(raw[j], q0 + j * MR_NW); });
        stage();
        for (int q = q0; q < units; q += RING * MR_NW)
          static_for<RING>([&](auto j) __attribute__((always_inline)) { body(raw[j], q + j * MR_NW); });
      };
      const int ur = a.topk * nch;
      run(F{}, wave, ur, false, a.d_q, a.d_s);
      if (S) run(FS{}, (wave + MR_NW - ur % MR_NW) % MR_NW, nch, true, reinterpret_cast<const uint8_t*>(a.sd_q), a.sd_s);
      if (g == 0) red[par][wave][0][c16] = sum;
      lds_barrier();
      if (wave == 0) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < MR_NW; ++k) v += red[par][k][0][c16];
        if constexpr (F::sums) {
          uint32_t odd = (uint32_t)__ballot(no_number(__float_as_uint(v))) & 0xffffu;
          if (odd && !__any(wt != wt) && !has_nan(slots * a.i, [&](int k) { return act_at(a, plane, 0, k); }))
            for (; odd; odd &= odd - 1) {
              const int n = __builtin_ctz(odd);
              float y = 0.f;
              for (int d = 0; d < a.topk; ++d)
                y += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(wt), d)) *
                     down_again<F>(a, plane, __builtin_amdgcn_readlane(mine, d), d, 16 * tile + n);
              if (S)
                y += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(wt), a.topk)) *
                     FS::dot(a.sd_q, a.sd_s, 16 * tile + n, K, [&](int k) { return act_at(a, plane, a.topk, k); });
              v = c16 == n ? y : v;
            }
        }
        const int o = 16 * tile + c16;
        if (lane < 16) a.y[o] = a.res ? a.res[o] + v : v;
      }
      par ^= 1;
    }
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

template <class F, class SH>
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
  // the smallest sets that MR_SETS counters allow: shorter chains for the last block (1 / 2 / 4 / 8 rows a set in us: 1 row 6.0 / 6.5 /
  // 7.0 / 8.2, 8 rows 6.7 / 6.6 / 7.3 / 8.9, 16 rows - / 7.8 / 7.9 / 9.3, 32 rows - / - / 9.7 / 10.0; 64 rows 12.9)
  if (a.rows <= 4) hipLaunchKernelGGL(k_moe_rows_router<1>, dim3(nb, a.rows), dim3(MR_NT), 0, st, a);
  else if (a.rows <= 16) hipLaunchKernelGGL(k_moe_rows_router<2>, dim3(nb, (a.rows + 1) / 2), dim3(MR_NT), 0, st, a);
  else if (a.rows <= 32) hipLaunchKernelGGL(k_moe_rows_router<4>, dim3(nb, (a.rows + 3) / 4), dim3(MR_NT), 0, st, a);
  else hipLaunchKernelGGL(k_moe_rows_router<8>, dim3(nb, (a.rows + 7) / 8), dim3(MR_NT), 0, st, a);
  const XLayout<0> gl(a.h);
  const XLayout<1> dl(a.i);
  const int slots = a.topk + a.shared;
  if (a.rows == 1 && slots <= dl.R) {
    const int ug = a.i / 16 * slots, ud = a.h / 16;
    hipLaunchKernelGGL((k_moe_rows_one<0, F, RowsQ8<SH, F::perm>>), dim3(ug < 512 ? ug : 512), dim3(MR_NT), gl.RB + 4 * gl.GS, st, a);
    hipLaunchKernelGGL((k_moe_rows_one<1, F, RowsQ8<SH, F::perm>>), dim3(ud < 256 ? ud : 256), dim3(MR_NT), slots * (dl.RB + 4 * dl.GS), st, a);
    return 0;
  }
  hipLaunchKernelGGL((k_moe_rows_experts<0, F, RowsQ8<SH, F::perm>>), dim3(MR_GRID), dim3(MR_NT), MR_X, st, a);
  hipLaunchKernelGGL((k_moe_rows_experts<1, F, RowsQ8<SH, F::perm>>), dim3(MR_GRID), dim3(MR_NT), MR_X, st, a);
  hipLaunchKernelGGL(k_moe_rows_combine, dim3(a.rows, (a.h + 1023) / 1024), dim3(256), 0, st, a);
  return 0;
}

}  // namespace

API size_t dr_moe_layer_rows_ws(int rows, int e, int h, int i, int topk) {
  return rows_shape_ok(rows, e, h, i, topk) ? WsLayout(rows, e, h, i, topk).bytes : 0;
}

#define MOE_ROWS_ENTRY(NAME, S, F, SH)                                                                             \
  API int NAME(const uint16_t* router, const uint8_t* gu_q, const S* gu_s, const uint8_t* d_q, const S* d_s,              \
               const int8_t* sgu_q, const uint16_t* sgu_s, const int8_t* sd_q, const uint16_t* sd_s, const uint16_t* x,   \
               const float* res, int* idx, float* wts, float* sgate, void* ws, float* y, int rows, int e, int h, int i,   \
               int topk, hipStream_t st) {                                                                                \
    const MoeRows a{router, gu_q, d_q, gu_s, d_s, sgu_q, sd_q, sgu_s, sd_s, x, res, idx, wts, sgate, y, nullptr, nullptr, \
                    nullptr, nullptr, rows, e, h, i, topk, 0};                                                            \
    return moe_rows<F, SH>(a, ws, st);                                                                             \
  }
MOE_ROWS_ENTRY(dr_moe_layer_rows, uint16_t, RowsQ4<ScaleF16>, Q8G128F16)
MOE_ROWS_ENTRY(dr_moe_layer_rows_bf16s, uint16_t, RowsQ4<ScaleBF16>, Q8RowBF16)
MOE_ROWS_ENTRY(dr_moe_layer_rows_fp8, float, RowsFP8<0>, Q8G128F16)
MOE_ROWS_ENTRY(dr_moe_layer_rows_fp8_bf16s, uint16_t, RowsFP8<1>, Q8RowBF16)
