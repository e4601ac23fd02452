// A whole MoE layer for a few rows (1 .. 64) of any size: per row x (bf16)
//   l = R x, picks by (l desc, index asc), w = softmax(l) renormalised over the picks,
//   y = res + sigmoid(l_E) D_s (silu(G_s x) * (U_s x)) + sum_k w_k D_k (silu(G_k x) * (U_k x)).
//
// An expert is fetched once for all the rows that picked it.  Matrix products run on
// v_mfma_f32_16x16x32_bf16 with A = up to 16 rows of x and B = 16 weight rows, converted exactly to bf16
// in registers (int4: 16 + q, with the rest of q scale + min in one fp32 MFMA of the group sums of x), so x
// enters exactly.  The activations are fp32; they travel as three bf16 planes of 8 mantissa
// bits each (their sum is the fp32 value), three MFMAs per weight fragment, so nothing is rounded but the fp32 sums.
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
  // as loaded, each a register quadruple that stays one (split into words, the ring's loop would copy them, and wait for them)
  struct Raw {
    gu32x4 w[2], s;
  };
  uint4 w[2], s;
  static DEV size_t q_bytes(int N, int K) { return (size_t)N * K / 2; }
  static DEV size_t s_bytes(int N, int K) { return (size_t)N * K / 16; }
  static DEV int xoff(int g) { return 32 * (g & 1) + 16 * (g >> 1); }
  // n: the tile's first row
  static DEV void load(Raw& f, const Rsrc& Q, const Rsrc& S, int n, int K, int c, bool half, bool off) {
    const bool none = off || (half && (lane_id() & 8));
    const uint32_t p = (n + pair_row()) * (K / 2) + c * 128 + pair_byte();
    f.w[0] = buf16(Q, none ? NOWHERE : p);
    f.w[1] = buf16(Q, none ? NOWHERE : p + 4 * K);
    f.s = buf16(S, off ? NOWHERE : ((n + (lane_id() & 15)) * (K / 64) + c * 4) * 4);
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
  DEV void prep(const Raw& f, bool half) {
    w[0] = words(f.w[0]), w[1] = words(f.w[1]);
    pair_up(w[0], w[1]);
    s = make_uint4(f.s.x, f.s.y, pick(half, 0, f.s.z), pick(half, 0, f.s.w));
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      // lanes g = 0, 1 hold group 2 p, g = 2, 3 group 2 p + 1: two words of each change places
      const auto s02 = __builtin_amdgcn_permlane32_swap(w[p].x, w[p].z, false, false);
      const auto s13 = __builtin_amdgcn_permlane32_swap(w[p].y, w[p].w, false, false);
      w[p] = make_uint4(s02[0], s13[0], s02[1], s13[1]);
    }
  }
  // what 16 + q leaves of q scale + min; xsum: the lane's sum of x over group l / 16 of row l % 16
  DEV void rest(float xsum, f32x4& out) const {
    const int g = lane_id() >> 4;
    // (by value: a choice between members would keep them in memory)
    const uint32_t lo = pick(g & 1, s.y, s.x), hi = pick(g & 1, s.w, s.z);
    const float2 o = SC::pair(pick(g & 2, hi, lo));
    out = __builtin_amdgcn_mfma_f32_16x16x4f32(xsum, o.y - 16.f * o.x, out, 0, 0, 0);
  }
  // group 2 p + h of the chunk
  template <int NP>
  DEV void group(int p, int h, const uint4 (&x)[NP][2], f32x4&, f32x4& out) const {
    const uint4 b0 = frag(pick(h, w[p].z, w[p].x)), b1 = frag(pick(h, w[p].w, w[p].y));
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < NP; ++q) a = mfma(x[q][0], b0, a), a = mfma(x[q][1], b1, a);
    const float sc = SC::pair(p ? pick(h, s.w, s.z) : pick(h, s.y, s.x)).x;
#pragma unroll
    for (int r = 0; r < 4; ++r) out[r] = __builtin_fmaf(sc, a[r], out[r]);
  }
};

// One byte per weight: 64 inputs of a row per 16-byte load of four lanes, scales per 128 inputs.  D: the
// format's conversions
template <class D>
struct Rows8 {
  static constexpr bool perm = false;
  struct Raw {
    gu32x4 w[4];
    uint32_t s[2];
  };
  uint4 w[4];
  uint32_t s[2];
  static DEV size_t q_bytes(int N, int K) { return (size_t)N * K; }
  static DEV int xoff(int g) { return 16 * g; }
  static DEV void load(Raw& f, const Rsrc& Q, const Rsrc& S, int n, int K, int c, bool half, bool off) {
    const uint32_t p = (n + pair_row()) * K + c * 256 + pair_byte();
    f.w[0] = buf16(Q, off ? NOWHERE : p), f.w[1] = buf16(Q, off ? NOWHERE : p + 8 * K);
    f.w[2] = buf16(Q, half ? NOWHERE : p + 128), f.w[3] = buf16(Q, half ? NOWHERE : p + 128 + 8 * K);
    f.s[0] = D::scale_raw(S, n + (lane_id() & 15), 2 * c, K, off);
    f.s[1] = D::scale_raw(S, n + (lane_id() & 15), 2 * c + 1, K, half);
  }
  DEV void prep(const Raw& f, bool) {
#pragma unroll
    for (int q = 0; q < 4; ++q) w[q] = words(f.w[q]);
    pair_up(w[0], w[1]), pair_up(w[2], w[3]);
    s[0] = f.s[0], s[1] = f.s[1];
  }
  DEV void rest(float, f32x4&) const {}
  template <int NP>
  DEV void group(int p, int h, const uint4 (&x)[NP][2], f32x4& a, f32x4& out) const {
    const uint4& v = w[2 * p + h];
    const uint4 b0 = D::frag(v.x, v.y), b1 = D::frag(v.z, v.w);
    if (h == 0) a = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < NP; ++q) a = mfma(x[q][0], b0, a), a = mfma(x[q][1], b1, a);
    if (h == 0) return;
    const float sc = D::scale_cvt(s[p]);
#pragma unroll
    for (int r = 0; r < 4; ++r) out[r] = __builtin_fmaf(sc, a[r], out[r]);
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
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
  }
  static DEV uint4 frag(uint32_t a, uint32_t b) { return make_uint4(pk(a, 0), pk(a, 2), pk(b, 0), pk(b, 2)); }
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

// MODE 0: gate_up (tile t: gate rows 16 t and up rows i + 16 t, K = h), MODE 1: down (tile t: rows 64 t, K = i).
//
// Items are passes of up to P rows of an expert, ascending, then of the shared expert (whose rows are all); their
// tiles are dealt to the blocks in contiguous runs of even cost, the shared expert's counting twice where its bytes are
// twice the others'.  A block stages the rows of its items in LDS (as many items at a time as R rows hold, most
// often all), then each of its waves takes one tile after the other from a counter and multiplies all of its inputs, in chunks
// of 256: no sum crosses waves and no barrier stands between tiles.  A wave's weights come in a ring of DEPTH chunks that
// runs on across tiles and items.
//
// LDS: row slot s at s * RB, its planes Kp * 2 bytes apart (Kp: K rounded up to a chunk, zeros past K), pieces of 8 inputs
// reordered for int4; RB is 16 bytes more than the planes, so that the 16 rows of a fragment meet different banks.
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

template <int MODE, class F, class FS>
__global__ void __launch_bounds__(MR_NT, 2) k_moe_rows_experts(MoeRows a, int fs_cost) {
  constexpr int NP = MODE == 0 ? 1 : 3, TL = MODE == 0 ? 2 : 4;
  extern __shared__ uint4 xlds[];
  __shared__ uint16_t s_list[MR_PAIRS + MR_ROWS];  // pairs by expert, then the shared expert's rows
  __shared__ uint16_t s_e[MR_ITEMS], s_off[MR_ITEMS], s_num[MR_ITEMS];  // items: expert, first place in s_list, rows
  __shared__ uint2 s_rows[256];
  __shared__ int s_start[256], s_d0, s_ticket;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), tid = threadIdx.x, c16 = lane & 15, g = lane >> 4;
  const int pairs = a.rows * a.topk;
  const int K = MODE == 0 ? a.h : a.i, tiles = MODE == 0 ? a.i / 16 : a.h / 64, N = MODE == 0 ? 2 * a.i : a.h;
  const int nch = (K + 255) / 256;
  const XLayout<MODE> L(K);
  const int P = L.R < 16 ? L.R : 16;
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
      s_d0 = d, s_ticket = 0;
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
  // items of the routed experts, of all; cost of the items before d: 1 a tile, fs_cost a tile of the shared expert
  const int D0 = __builtin_amdgcn_readfirstlane(s_d0), D = D0 + (a.shared ? (a.rows + P - 1) / P : 0);
  auto cost_before = [&](int d) { return d <= D0 ? d * tiles : D0 * tiles + (d - D0) * tiles * fs_cost; };
  const long long all = cost_before(D);
  const int lo = (int)(all * blockIdx.x / gridDim.x), hi = (int)(all * (blockIdx.x + 1) / gridDim.x);
  if (lo >= hi) return;
  auto item_at = [&](int c) { return c < D0 * tiles ? c / tiles : D0 + (c - D0 * tiles) / (tiles * fs_cost); };
  const int dfirst = item_at(lo), dend = item_at(hi - 1) + 1;  // this block's items
  const size_t plane = (size_t)(pairs + a.rows) * a.i;
  char* xb = reinterpret_cast<char*>(xlds);
  float* sums = reinterpret_cast<float*>(xb + (size_t)L.R * L.RB);
  // the block's tiles [t0, t1) of item d
  auto range = [&](int d, int& t0, int& t1) __attribute__((always_inline)) {
    const int cum = cost_before(d), tc = d < D0 ? 1 : fs_cost;
    t0 = lo > cum ? (lo - cum + tc - 1) / tc : 0;
    t1 = (hi - cum + tc - 1) / tc;
    t0 = t0 < tiles ? t0 : tiles, t1 = t1 < tiles ? t1 : tiles;
  };
  // items dA .. dB - 1, of one weight format, their rows in the slots from 0
  auto run = [&](auto fmt, const int dA, const int dB, const bool sh, const uint8_t* Wq, const void* Ws) __attribute__((always_inline)) {
    using Fm = decltype(fmt);
    constexpr int DEPTH = Fm::perm ? 8 / TL : MODE == 0 ? 3 : 2;
    const int pos = s_off[dA], nrows = s_off[dB - 1] + s_num[dB - 1] - pos, k8 = L.Kp / 8;
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
      for (int i = 0; i < TL; ++i) Fm::load(f[i], Q, S, MODE == 0 ? 16 * lt + i * a.i : 64 * lt + 16 * i, K, lc, none, over);
      __builtin_amdgcn_sched_barrier(0);
    };
    static_for<DEPTH>([&](auto k) __attribute__((always_inline)) { advance(w[k.value], td[k.value], tt[k.value], tc[k.value]); });
    // the rows, requested behind the first weights: the two waits are one
    for (int q = tid; q < nrows * k8; q += MR_NT) {
      const int slot = q / k8, k = (q - slot * k8) * 8, pr = s_list[pos + slot];
      float sum = 0.f;
#pragma unroll
      for (int p = NP - 1; p >= 0; --p) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (k < K) v = ld16(MODE == 0 ? a.x + (size_t)(sh ? pr - pairs : pr / a.topk) * K + k : a.act + p * plane + (size_t)pr * K + k);
        if constexpr (Fm::perm) {
          sum += ((bf16_lo(v.x) + bf16_hi(v.x)) + (bf16_lo(v.y) + bf16_hi(v.y))) + ((bf16_lo(v.z) + bf16_hi(v.z)) + (bf16_lo(v.w) + bf16_hi(v.w)));
          v = make_uint4(__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
                         __builtin_amdgcn_perm(v.w, v.y, 0x05040100u), __builtin_amdgcn_perm(v.w, v.y, 0x07060302u));
        }
        *reinterpret_cast<uint4*>(xb + slot * L.RB + (p * L.Kp + k) * 2) = v;
      }
      if constexpr (Fm::perm) {
        // the 8 pieces of a group are 8 consecutive threads (k8 is a multiple of 8), all in or all past the rows
        sum = xsum_step<4>(xsum_step<2>(xsum_step<1>(sum)));
        if ((q & 7) == 0) sums[slot * L.GS + k / 64] = sum;
      }
    }
    lds_barrier();
    f32x4 o[TL];
    const char* xr = xb;
    const float* sr = sums;
    auto body = [&](typename Fm::Raw (&raw)[TL], int& d, int& t, int& c) __attribute__((always_inline)) {  // one chunk
      if (c == 0 && d >= 0) {
        const int cnt = s_num[d], slot = s_off[d] - pos + (c16 < cnt ? c16 : cnt - 1);
        xr = xb + slot * L.RB + 2 * Fm::xoff(g);
        sr = sums + slot * L.GS + g;
#pragma unroll
        for (int i = 0; i < TL; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      const bool half = c * 256 + 128 >= K;
      Fm f[TL];
      const float xs = Fm::perm ? sr[4 * c] : 0.f;
#pragma unroll
      for (int i = 0; i < TL; ++i) f[i].prep(raw[i], half), f[i].rest(xs, o[i]);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        f32x4 acc[TL];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint4 x[NP][2];
#pragma unroll
          for (int q = 0; q < NP; ++q) {
            const uint4* src = reinterpret_cast<const uint4*>(xr + q * L.Kp * 2 + (c * 256 + 128 * p + 64 * h) * 2);
            x[q][0] = src[0], x[q][1] = src[1];
          }
#pragma unroll
          for (int i = 0; i < TL; ++i) f[i].template group<NP>(p, h, x, acc[i], o[i]);
        }
      }
      if (c == nch - 1 && d >= 0) {
        // register r of lane l: row 4 (l / 16) + r of x, column l % 16
        const int off = s_off[d], cnt = s_num[d];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (r >= cnt) break;
          const int row = 4 * g + r;
          if (row >= cnt) continue;
          const int pr = s_list[off + row];
          if constexpr (MODE == 0) {
            const float act = o[0][r] / (1.f + expf(-o[0][r])) * o[1][r];
            uint16_t* dst = a.act + (size_t)pr * a.i + 16 * t + c16;
            const float hi8 = __uint_as_float(__float_as_uint(act) & 0xffff0000u), r1 = act - hi8;
            const float mi8 = __uint_as_float(__float_as_uint(r1) & 0xffff0000u), r2 = r1 - mi8;
            dst[0] = (uint16_t)(__float_as_uint(hi8) >> 16);
            dst[plane] = (uint16_t)(__float_as_uint(mi8) >> 16);
            dst[2 * plane] = (uint16_t)(__float_as_uint(r2) >> 16);
          } else {
#pragma unroll
            for (int i = 0; i < TL; ++i) a.yp[(size_t)pr * a.h + 64 * t + 16 * i + c16] = o[i][r];
          }
        }
      }
      advance(raw, d, t, c);
    };
    // One exit, at the head: places of the ring without a tile are computed too (zeros, not stored), since paths that
    // skip loads and join the loop again would make every wait in it a wait for all loads.
    while (td[0] >= 0) static_for<DEPTH>([&](auto k) __attribute__((always_inline)) { body(w[k.value], td[k.value], tt[k.value], tc[k.value]); });
    lds_barrier();  // the rows may be replaced, the counter starts again
    if (tid == 0) s_ticket = 0;
    lds_barrier();
  };
  for (int d = dfirst; d < dend;) {
    int e = d + 1;
    const bool sh = d >= D0;
    while (e < dend && (e >= D0) == sh && s_off[e] + s_num[e] - s_off[d] <= L.R) ++e;
    if (sh) run(FS{}, d, e, true, reinterpret_cast<const uint8_t*>(MODE == 0 ? a.sgu_q : a.sd_q), MODE == 0 ? a.sgu_s : a.sd_s);
    else run(F{}, d, e, false, MODE == 0 ? a.gu_q : a.d_q, MODE == 0 ? a.gu_s : a.d_s);
    d = e;
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
  hipLaunchKernelGGL((k_moe_rows_experts<0, F, RowsQ8<SH>>), dim3(MR_GRID), dim3(MR_NT), MR_X, st, a, BYTES ? 1 : 2);
  hipLaunchKernelGGL((k_moe_rows_experts<1, F, RowsQ8<SH>>), dim3(MR_GRID), dim3(MR_NT), MR_X, st, a, BYTES ? 1 : 2);
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
