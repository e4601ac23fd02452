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
constexpr int MR_GRID = 256;  // a block per CU
constexpr int MR_ITEMS = 256 + MR_PAIRS / 16 + MR_ROWS / 16;  // passes of 16 rows, the experts' and the shared expert's
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
DEV uint4 buf16(const Rsrc& r, uint32_t off) { return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0)); }

// Where lane l's piece of a row pair's loads lies: row l % 8 (+ 8 in the second load), bytes 16 (4 (l / 8 % 2) + l / 16) of the 128
DEV int pair_row() { return lane_id() & 7; }
DEV int pair_byte() { return ((lane_id() >> 1) & 4) * 16 + (lane_id() >> 4) * 16; }
// a: rows 0 .. 7, b: rows 8 .. 15 -> a: bytes 16 g of the first 64 of row l % 16, b: of the second 64.  Lanes 8 .. 15 of each 16 of a
// take lanes 0 .. 7 of b, and the other way round.
DEV void pair_up(uint4& a, uint4& b) {
  auto sw = [](uint32_t& p, uint32_t& q) {
    const int o = (int)p, n = (int)q;
    p = (uint32_t)__builtin_amdgcn_update_dpp(o, n, 0x128, 0xF, 0xC, false);  // row_ror:8 into lanes 8 .. 15
    q = (uint32_t)__builtin_amdgcn_update_dpp(n, o, 0x128, 0xF, 0x3, false);  // into lanes 0 .. 7
  };
  sw(a.x, b.x), sw(a.y, b.y), sw(a.z, b.z), sw(a.w, b.w);
}

template <class SC>
struct RowsQ4 {
  static constexpr bool perm = true;  // fragment order 0 4 1 5 2 6 3 7
  uint4 w[2], s;
  static DEV size_t q_bytes(int N, int K) { return (size_t)N * K / 2; }
  static DEV size_t s_bytes(int N, int K) { return (size_t)N * K / 16; }
  static DEV int xoff(int g) { return 32 * (g & 1) + 16 * (g >> 1); }
  // n: the tile's first row
  DEV void load(const Rsrc& Q, const Rsrc& S, int n, int K, int c, bool half, bool off) {
    const bool none = off || (half && (lane_id() & 8));
    const uint32_t p = (n + pair_row()) * (K / 2) + c * 128 + pair_byte();
    w[0] = buf16(Q, none ? NOWHERE : p);
    w[1] = buf16(Q, none ? NOWHERE : p + 4 * K);
    s = buf16(S, off ? NOWHERE : ((n + (lane_id() & 15)) * (K / 64) + c * 4) * 4);
  }
  // nibbles of a word as 16 + q in bf16: the nibble is the top four mantissa bits of a number in [16, 32)
  // (the two constants in registers, so that each pair of nibbles is a shift and one v_and_or_b32)
  static DEV uint4 frag(uint32_t v) {
    uint32_t m = 0x00780078u, b = 0x41804180u;
    asm("" : "+s"(m));
    asm("" : "+v"(b));
    return make_uint4(((v << 3) & m) | b, ((v >> 1) & m) | b, ((v >> 5) & m) | b, ((v >> 9) & m) | b);
  }
  // xsum: lane's sum of x over group l / 16 of row l % 16 (0 past the chunk's groups)
  template <int NP>
  DEV void mac(const uint4 (&x)[NP][8], float xsum, bool half, f32x4& out) {
    const int g = lane_id() >> 4;
    const uint32_t sw[4] = {s.x, s.y, half ? 0u : s.z, half ? 0u : s.w};
    const uint32_t lo = g & 1 ? sw[1] : sw[0], hi = g & 1 ? sw[3] : sw[2];
    const float2 o = SC::pair(g & 2 ? hi : lo);
    out = __builtin_amdgcn_mfma_f32_16x16x4f32(xsum, o.y - 16.f * o.x, out, 0, 0, 0);
    pair_up(w[0], w[1]);
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
        const float sc = SC::pair(sw[2 * p + h]).x;
#pragma unroll
        for (int r = 0; r < 4; ++r) out[r] = __builtin_fmaf(sc, a[r], out[r]);
      }
    }
  }
};

// One byte per weight: 64 inputs of a row per 16-byte load of four lanes, scales per 128 inputs.  D: the
// format's conversions
template <class D>
struct Rows8 {
  static constexpr bool perm = false;
  uint4 w[4];
  uint32_t s[2];
  static DEV size_t q_bytes(int N, int K) { return (size_t)N * K; }
  static DEV int xoff(int g) { return 16 * g; }
  DEV void load(const Rsrc& Q, const Rsrc& S, int n, int K, int c, bool half, bool off) {
    const uint32_t p = (n + pair_row()) * K + c * 256 + pair_byte();
    w[0] = buf16(Q, off ? NOWHERE : p), w[1] = buf16(Q, off ? NOWHERE : p + 8 * K);
    w[2] = buf16(Q, half ? NOWHERE : p + 128), w[3] = buf16(Q, half ? NOWHERE : p + 128 + 8 * K);
    s[0] = D::scale_raw(S, n + (lane_id() & 15), 2 * c, K, off);
    s[1] = D::scale_raw(S, n + (lane_id() & 15), 2 * c + 1, K, half);
  }
  template <int NP>
  DEV void mac(const uint4 (&x)[NP][8], float, bool, f32x4& out) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      pair_up(w[2 * p], w[2 * p + 1]);
      f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4& v = w[2 * p + h];
        const uint4 b0 = D::frag(v.x, v.y), b1 = D::frag(v.z, v.w);
#pragma unroll
        for (int q = 0; q < NP; ++q) a = mfma(x[q][4 * p + 2 * h], b0, a), a = mfma(x[q][4 * p + 2 * h + 1], b1, a);
      }
      const float sc = D::scale_cvt(s[p]);
#pragma unroll
      for (int r = 0; r < 4; ++r) out[r] = __builtin_fmaf(sc, a[r], out[r]);
    }
  }
};
DEV uint32_t buf_half(const Rsrc& S, uint32_t off) { return (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(S, off, 0, 0); }

template <int SF>
struct RowsFP8 : Rows8<RowsFP8<SF>> {
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

template <class SH>
struct RowsQ8 : Rows8<RowsQ8<SH>> {
  static DEV size_t s_bytes(int N, int K) { return (size_t)N * (SH::per_row ? 1 : K / 128) * 2; }
  static DEV uint32_t scale_raw(const Rsrc& S, int n, int b, int K, bool off) {
    return buf_half(S, off ? NOWHERE : 2 * (SH::per_row ? n : n * (K / 128) + b));
  }
  static DEV float scale_cvt(uint32_t r) { return SH::cvt(r); }
  static DEV uint32_t pk(uint32_t v, int i) {  // bytes i, i + 1 as bf16 (exact)
    const float a = (float)(int8_t)(v >> (8 * i)), b = (float)(int8_t)(v >> (8 * i + 8));
    return (__float_as_uint(b) & 0xffff0000u) | (__float_as_uint(a) >> 16);
  }
  static DEV uint4 frag(uint32_t a, uint32_t b) { return make_uint4(pk(a, 0), pk(a, 2), pk(b, 0), pk(b, 2)); }
};

// A lane's fragments of chunk c of the row at byte `row` (planes `plane` bytes apart); inputs past the row are zero
template <class F, int NP>
DEV void load_x(const Rsrc& X, uint32_t row, uint32_t plane, int c, bool half, uint4 (&x)[NP][8]) {
  const uint32_t p = row + (c * 256 + F::xoff(lane_id() >> 4)) * 2;
#pragma unroll
  for (int q = 0; q < NP; ++q)
#pragma unroll
    for (int f = 0; f < 8; ++f)
      x[q][f] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(X, f >= 4 && half ? NOWHERE : p + 2 * (64 * (f >> 1) + 8 * (f & 1)),
                                                                                 q * plane, 0));
}
// the fragments in the weights' order, and the lane's group sum (RowsQ4)
template <class F, int NP>
DEV float order_x(uint4 (&x)[NP][8]) {
  if constexpr (!F::perm) return 0.f;
  float own = 0.f;
#pragma unroll
  for (int G = 0; G < 4; ++G) {
    float t = 0.f;
#pragma unroll
    for (int q = NP - 1; q >= 0; --q)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint4& v = x[q][2 * G + j];
        t += ((bf16_lo(v.x) + bf16_hi(v.x)) + (bf16_lo(v.y) + bf16_hi(v.y))) +
             ((bf16_lo(v.z) + bf16_hi(v.z)) + (bf16_lo(v.w) + bf16_hi(v.w)));
        v = make_uint4(__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
                       __builtin_amdgcn_perm(v.w, v.y, 0x05040100u), __builtin_amdgcn_perm(v.w, v.y, 0x07060302u));
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
// MODE 0: gate_up (tile t: gate rows 16 t and up rows i + 16 t, K = h), MODE 1: down (tile t: rows 32 t, K = i).
// KS waves share a tile's inputs, a chunk each (cpw > 1: further chunks in turn); the other groups of waves (RG)
// take further tiles, a step of the block being RG tiles.  Items are passes of up to 16 rows of an expert, ascending,
// then of the shared expert (whose rows are all); their steps are dealt to the blocks in contiguous runs of even
// cost, the shared expert's counting twice where its bytes are twice the others'.  (All passes of an expert as one
// item fetch its weights once but x again for every tile and pass: 64 rows 202 us against 152.)
// A wave's x fragments stay in registers for all tiles of an item (where it has one chunk).  Two steps of weights
// are in flight: a tile's registers take the tile two steps on as soon as it is used.  The KS sums meet in LDS, behind a
// barrier that leaves the loads in flight.
template <int MODE, class F, class FS>
__global__ void __launch_bounds__(MR_NT, 2) k_moe_rows_experts(MoeRows a, int KS, int cpw, int fs_cost) {
  constexpr int NP = MODE == 0 ? 1 : 3, TL = 2;
  __shared__ uint16_t s_list[MR_PAIRS + MR_ROWS];  // pairs by expert
  __shared__ uint32_t s_rows[256][2];
  __shared__ int s_start[256], s_e[MR_ITEMS], s_off[MR_ITEMS], s_num[MR_ITEMS], s_cum[MR_ITEMS + 1], s_tot[8][3], s_first;
  __shared__ float red[2][MR_NW][TL][4][64];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), tid = threadIdx.x;
  const int pairs = a.rows * a.topk;
  const int K = MODE == 0 ? a.h : a.i, RG = MR_NW / KS, tiles = MODE == 0 ? a.i / 16 : a.h / 32;
  const int steps = (tiles + RG - 1) / RG;
  const int N = MODE == 0 ? 2 * a.i : a.h;
  const int nch = (K + 255) / 256, wk = wave % KS, rg = wave / KS;
  // rows of each expert as a 64-bit mask (a row picks an expert once), so that every block has the same passes
  constexpr int PPT = MR_PAIRS / MR_NT;
  int pe[PPT];
#pragma unroll
  for (int q = 0; q < PPT; ++q) pe[q] = tid + MR_NT * q < pairs ? a.idx[tid + MR_NT * q] & 255 : -1;
  if (tid < 256) s_rows[tid][0] = s_rows[tid][1] = 0;
  lds_barrier();
#pragma unroll
  for (int q = 0; q < PPT; ++q)
    if (pe[q] >= 0) {
      const int r = (tid + MR_NT * q) / a.topk;
      atomicOr(&s_rows[pe[q]][r >> 5], 1u << (r & 31));
    }
  lds_barrier();
  // sums over the experts (thread e) of their rows, their passes and their cost
  {
    int v[3] = {0, 0, 0}, own[3];
    if (tid <= 256) {
      const bool sh = tid == 256;
      v[0] = sh ? (a.shared ? a.rows : 0) : __builtin_popcount(s_rows[tid][0]) + __builtin_popcount(s_rows[tid][1]);
      v[1] = (v[0] + 15) / 16;
      v[2] = v[1] * steps * (sh ? fs_cost : 1);
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      own[q] = v[q];
      for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(v[q], o);
        if (lane >= o) v[q] += up;
      }
      if (lane == 63) s_tot[wave][q] = v[q];
    }
    lds_barrier();
    int base[3] = {0, 0, 0};
    for (int w = 0; w < wave; ++w)
#pragma unroll
      for (int q = 0; q < 3; ++q) base[q] += s_tot[w][q];
    lds_barrier();
    if (tid <= 256) {
      const int off = base[0] + v[0] - own[0], cum = base[2] + v[2] - own[2];
      for (int p = 0; p < own[1]; ++p) {
        const int d = base[1] + v[1] - own[1] + p;
        s_e[d] = tid, s_off[d] = off + 16 * p, s_num[d] = own[0] - 16 * p < 16 ? own[0] - 16 * p : 16, s_cum[d] = cum + own[2] / own[1] * p;
      }
      if (tid < 256) s_start[tid] = off;
    }
    if (tid == 256) s_cum[base[1] + v[1]] = base[2] + v[2], s_tot[0][0] = base[1] + v[1];
    lds_barrier();
  }
  const int D = s_tot[0][0];
  const int lo = (int)((long long)s_cum[D] * blockIdx.x / gridDim.x), hi = (int)((long long)s_cum[D] * (blockIdx.x + 1) / gridDim.x);
  if (tid < D && s_cum[tid] <= lo && lo < s_cum[tid + 1]) s_first = tid;
#pragma unroll
  for (int q = 0; q < PPT; ++q)
    if (pe[q] >= 0) {
      const int r = (tid + MR_NT * q) / a.topk;
      const uint32_t lo32 = s_rows[pe[q]][0], hi32 = s_rows[pe[q]][1], below = (1u << (r & 31)) - 1;
      s_list[s_start[pe[q]] + (r < 32 ? __builtin_popcount(lo32 & below) : __builtin_popcount(lo32) + __builtin_popcount(hi32 & below))] =
          tid + MR_NT * q;
    }
  if (a.shared && tid < a.rows) s_list[pairs + tid] = pairs + tid;
  lds_barrier();
  if (lo >= hi) return;
  int par = 0;
  const size_t plane = (size_t)(pairs + a.rows) * a.i;
  for (int d = s_first; d < D && s_cum[d] < hi; ++d) {
    const int e = __builtin_amdgcn_readfirstlane(s_e[d]), off = s_off[d], cnt = s_num[d];
    const int cum = s_cum[d], tc = (s_cum[d + 1] - cum) / steps;
    const int t0 = lo > cum ? (lo - cum + tc - 1) / tc : 0, t1 = (hi - cum + tc - 1) / tc < steps ? (hi - cum + tc - 1) / tc : steps;
    if (t0 >= t1) continue;
    const bool sh = e == 256;
    auto segment = [&](auto fmt, const void* Qp, const void* Sp) __attribute__((always_inline)) {
      using Fm = decltype(fmt);
      const Rsrc Q = rsrc(Qp, (uint32_t)Fm::q_bytes(N, K)), S = rsrc(Sp, (uint32_t)Fm::s_bytes(N, K));
      const Rsrc X = MODE == 0 ? rsrc(a.x, (uint32_t)a.rows * K * 2) : rsrc(a.act, (uint32_t)(6 * plane));
      Fm w[2][TL];
      uint4 x[NP][8];
      auto half_of = [&](int c) { return c * 256 + 128 >= K; };
      auto load_w = [&](Fm& f, int i, int t, int ci) __attribute__((always_inline)) {
        const int c = wk + KS * ci, tile = t * RG + rg;
        const bool none = (t >= t1) | (tile >= tiles) | (rg >= RG) | (c >= nch);
        f.load(Q, S, MODE == 0 ? 16 * tile + i * a.i : 32 * tile + 16 * i, K, c, none | half_of(c), none);
        __builtin_amdgcn_sched_barrier(0);
      };
      auto fetch_x = [&](int ci) __attribute__((always_inline)) {
        const int m = lane & 15, pr = s_list[off + (m < cnt ? m : cnt - 1)], c = wk + KS * ci;
        const int row = MODE == 1 ? pr : sh ? pr - pairs : pr / a.topk;
        load_x<Fm, NP>(X, c < nch ? (uint32_t)(row * K * 2) : NOWHERE, (uint32_t)(2 * plane), c, half_of(c), x);
        __builtin_amdgcn_sched_barrier(0);
      };
      // the KS sums of step t's tiles, and what becomes of them
      auto finish = [&](const f32x4 (&o)[TL], int t) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < TL; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) red[par][wave][i][r][lane] = o[i][r];
        lds_barrier();
        const int tile = t * RG + rg, nr = tile < tiles && rg < RG ? cnt : 0;
        // register r of lane l: row 4 (l / 16) + r of x, column l % 16; the KS waves share the registers
        auto part = [&](auto ks) __attribute__((always_inline)) {
          constexpr int KK = decltype(ks)::value;
          const int base = rg * KS;
          auto total = [&](int i, int r) {
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < KK; ++k) {
              const float q = red[par][base + (k < KS ? k : 0)][i][r][lane];
              v += k < KS ? q : 0.f;
            }
            return v;
          };
          for (int q = MODE == 0 && KS == 8 ? wk ^ (4 * par) : wk; q < (MODE == 0 ? 4 : 4 * TL); q += KS) {
            const int r = q & 3, row = 4 * (lane >> 4) + r;
            if (r >= nr) continue;
            const bool live = row < nr;
            const int pr = s_list[off + (live ? row : 0)];
            if constexpr (MODE == 0) {
              const float g = total(0, r), v = total(1, r);
              if (live) {
                const float act = g / (1.f + expf(-g)) * v;
                uint16_t* dst = a.act + (size_t)pr * a.i + 16 * tile + (lane & 15);
                const float hi8 = __uint_as_float(__float_as_uint(act) & 0xffff0000u), r1 = act - hi8;
                const float mi8 = __uint_as_float(__float_as_uint(r1) & 0xffff0000u), r2 = r1 - mi8;
                dst[0] = (uint16_t)(__float_as_uint(hi8) >> 16);
                dst[plane] = (uint16_t)(__float_as_uint(mi8) >> 16);
                dst[2 * plane] = (uint16_t)(__float_as_uint(r2) >> 16);
              }
            } else {
              const float v = total(q >> 2, r);
              if (live) a.yp[(size_t)pr * a.h + 32 * tile + 16 * (q >> 2) + (lane & 15)] = v;
            }
          }
        };
        if (KS > 4) part(std::integral_constant<int, 8>{});
        else if (KS > 2) part(std::integral_constant<int, 4>{});
        else if (KS == 2) part(std::integral_constant<int, 2>{});
        else part(std::integral_constant<int, 1>{});
        par ^= 1;
      };
      const f32x4 z = {0.f, 0.f, 0.f, 0.f};
      f32x4 o[TL];
      if (cpw == 1) {  // x stays
#pragma unroll
        for (int i = 0; i < TL; ++i) load_w(w[0][i], i, t0, 0);
        fetch_x(0);
#pragma unroll
        for (int i = 0; i < TL; ++i) load_w(w[1][i], i, t0 + 1, 0);
        const float xs = order_x<Fm, NP>(x);
        auto body = [&](Fm (&f)[TL], int t) __attribute__((always_inline)) {
#pragma unroll
          for (int i = 0; i < TL; ++i) o[i] = z, f[i].template mac<NP>(x, xs, half_of(wk), o[i]), load_w(f[i], i, t + 2, 0);
          finish(o, t);
        };
        for (int t = t0;;) {
          body(w[0], t);
          if (++t >= t1) break;
          body(w[1], t);
          if (++t >= t1) break;
        }
      } else {
        // step and chunk, and those of the one ahead (x) and the two ahead (weights)
        int t = t0, ci = 0, tx = t0, cx = 0, tw = t0, cw = 0;
        auto next = [&](int& t, int& ci) {
          if (++ci == cpw) ci = 0, ++t;
        };
#pragma unroll
        for (int i = 0; i < TL; ++i) load_w(w[0][i], i, t0, 0);
        fetch_x(0);
        next(tw, cw), next(tx, cx);
#pragma unroll
        for (int i = 0; i < TL; ++i) load_w(w[1][i], i, tw, cw);
        auto body = [&](Fm (&f)[TL]) __attribute__((always_inline)) {
          const float xs = order_x<Fm, NP>(x);
          if (ci == 0)
#pragma unroll
            for (int i = 0; i < TL; ++i) o[i] = z;
#pragma unroll
          for (int i = 0; i < TL; ++i) f[i].template mac<NP>(x, xs, half_of(wk + KS * ci), o[i]);
          fetch_x(cx);
          next(tx, cx), next(tw, cw);
#pragma unroll
          for (int i = 0; i < TL; ++i) load_w(f[i], i, tw, cw);
          if (ci == cpw - 1) finish(o, t);
          next(t, ci);
        };
        for (;;) {
          body(w[0]);
          if (t >= t1) break;
          body(w[1]);
          if (t >= t1) break;
        }
      }
    };
    if (sh) segment(FS{}, MODE == 0 ? a.sgu_q : a.sd_q, MODE == 0 ? a.sgu_s : a.sd_s);
    else
      segment(F{}, (MODE == 0 ? a.gu_q : a.d_q) + e * F::q_bytes(N, K),
              reinterpret_cast<const char*>(MODE == 0 ? a.gu_s : a.d_s) + e * F::s_bytes(N, K));
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

// The waves that share a tile's K inputs and the chunks each takes: a wave per chunk up to all eight.
struct Split {
  int ks, cpw;
  Split(int K) {
    const int nch = (K + 255) / 256;
    cpw = (nch + MR_NW - 1) / MR_NW;
    ks = (nch + cpw - 1) / cpw;
  }
};

template <class F, class SH, bool BYTES>
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
  const Split g(a.h), d(a.i);
  hipLaunchKernelGGL((k_moe_rows_experts<0, F, RowsQ8<SH>>), dim3(MR_GRID), dim3(MR_NT), 0, st, a, g.ks, g.cpw, BYTES ? 1 : 2);
  hipLaunchKernelGGL((k_moe_rows_experts<1, F, RowsQ8<SH>>), dim3(MR_GRID), dim3(MR_NT), 0, st, a, d.ks, d.cpw, BYTES ? 1 : 2);
  hipLaunchKernelGGL(k_moe_rows_combine, dim3(a.rows, (a.h + 1023) / 1024), dim3(256), 0, st, a);
  return 0;
}

}  // namespace

API size_t dr_moe_layer_rows_ws(int rows, int e, int h, int i, int topk) {
  return rows_shape_ok(rows, e, h, i, topk) ? WsLayout(rows, e, h, i, topk).bytes : 0;
}

#define MOE_ROWS_ENTRY(NAME, S, F, SH, BYTES)                                                                             \
  API int NAME(const uint16_t* router, const uint8_t* gu_q, const S* gu_s, const uint8_t* d_q, const S* d_s,              \
               const int8_t* sgu_q, const uint16_t* sgu_s, const int8_t* sd_q, const uint16_t* sd_s, const uint16_t* x,   \
               const float* res, int* idx, float* wts, float* sgate, void* ws, float* y, int rows, int e, int h, int i,   \
               int topk, hipStream_t st) {                                                                                \
    const MoeRows a{router, gu_q, d_q, gu_s, d_s, sgu_q, sd_q, sgu_s, sd_s, x, res, idx, wts, sgate, y, nullptr, nullptr, \
                    nullptr, nullptr, rows, e, h, i, topk, 0};                                                            \
    return moe_rows<F, SH, BYTES>(a, ws, st);                                                                             \
  }
MOE_ROWS_ENTRY(dr_moe_layer_rows, uint16_t, RowsQ4<ScaleF16>, Q8G128F16, false)
MOE_ROWS_ENTRY(dr_moe_layer_rows_bf16s, uint16_t, RowsQ4<ScaleBF16>, Q8RowBF16, false)
MOE_ROWS_ENTRY(dr_moe_layer_rows_fp8, float, RowsFP8<0>, Q8G128F16, true)
MOE_ROWS_ENTRY(dr_moe_layer_rows_fp8_bf16s, uint16_t, RowsFP8<1>, Q8RowBF16, true)
