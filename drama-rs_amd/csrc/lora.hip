// An int8 projection shared by all rows with each row's own low-rank adapter:
//   y[r] = res[r] + W x[r] + s_a B_a (A_a x[r]),   a = adapter[r].
//
// Two launches.  k_lora_down: t[r] = s_a A_a x[r] (fp32), a block per 16 rows and distinct adapter among them, so
// rows that share an adapter share its fetch whatever their order.  k_lora_gemm_rows (few rows) and k_lora_gemm_tiles:
// W x on v_mfma_f32_16x16x32_bf16 (int8 is exact in bf16, the scales enter the fp32 sums), with B_a t and the residual
// added to each output before its one store.
#include "common.hpp"

using namespace drm;

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

DEV f32x4 mfma(const uint4& a, const uint4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

struct Lora {
  const int8_t* w;
  const uint16_t* s;
  const uint16_t* x;
  const int* adapter;
  const uint16_t *la, *lb;
  const int* rank;
  const float* lscale;
  const float* res;
  float *t, *y;
  size_t ldx, ldy;
  int adapters, rmax, rows, n, k;
  uint16_t* planes;  // t as three bf16 planes [rows, rp] whose sum it is, zero past the rank (k_lora_gemm_tiles), or null
  int rp;            // rmax rounded up to the 32 of an MFMA
};

typedef __amdgpu_buffer_rsrc_t Rsrc;

constexpr int LR_NW = 8, LR_NT = LR_NW * 64;

// adapter of row r, -1 for none (an id outside 0 .. adapters - 1, an adapter without rank)
DEV int adapter_of(const Lora& a, int r) {
  if (!a.adapter || r >= a.rows) return -1;
  const int v = a.adapter[r];
  return v >= 0 && v < a.adapters && a.rank[v] > 0 ? v : -1;
}
DEV int rank_of(const Lora& a, int v) { return a.rank[v] < a.rmax ? a.rank[v] : a.rmax; }

// ---- t = s_a A_a x --------------------------------------------------------------------------
// Block: 16 rows (blockIdx.x), 16 RT ranks (blockIdx.z), the distinct adapters blockIdx.y, + gridDim.y, ... of
// those rows.  The eight waves take 128 inputs each in turn.  Bound by the latency of a short chain of loads (ids, ranks,
// inputs) and, with many rows, by the requests of 16 rows a fetch (two turns in flight: 20 -> 31 us at 4096 rows).
template <int RT>
__global__ void __launch_bounds__(LR_NT) k_lora_down(Lora a) {
  __shared__ float red[LR_NW][RT][4][64];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), c16 = lane & 15, g = lane >> 4;
  const int r0 = blockIdx.x * 16, j0 = blockIdx.z * 16 * RT;
  const uint16_t* xr = a.x + (size_t)(r0 + c16 < a.rows ? r0 + c16 : a.rows - 1) * a.ldx + 8 * g;
  // the first turn's x is requested ahead of the ids (12 adapters in any order over 4096 rows: 104 -> 89 us)
  uint4 x0[4];
#pragma unroll
  for (int f = 0; f < 4; ++f) x0[f] = ld16(xr + (wave * 128 < a.k ? wave * 128 : 0) + 32 * f);
  __builtin_amdgcn_sched_barrier(0);
  const int mine = adapter_of(a, r0 + c16);
  // row c16 is the first of its adapter: no earlier row of the 16 has it
  bool first = mine >= 0;
#pragma unroll
  for (int q = 0; q < 15; ++q) first = first && !(q < c16 && __builtin_amdgcn_readlane(mine, q) == mine);
  uint32_t firsts = (uint32_t)__ballot(first) & 0xffffu;
  for (int q = 0; q < (int)blockIdx.y && firsts; ++q) firsts &= firsts - 1;
  while (firsts) {
    const int ad = __builtin_amdgcn_readlane(mine, __builtin_ctz(firsts));
    for (int q = 0; q < (int)gridDim.y && firsts; ++q) firsts &= firsts - 1;
    const uint32_t rows = (uint32_t)__ballot(mine == ad) & 0xffffu;
    const int rk = rank_of(a, ad);
    const float scale = a.lscale[ad];
    f32x4 acc[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (j0 < rk) {
      const uint16_t* ar[RT];
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int j = j0 + 16 * t + c16;
        ar[t] = a.la + ((size_t)ad * a.rmax + (j < rk ? j : rk - 1)) * a.k + 8 * g;
      }
      for (int c = wave * 128; c < a.k; c += LR_NW * 128) {
        uint4 xv[4], av[RT][4];
#pragma unroll
        for (int f = 0; f < 4; ++f) xv[f] = c == wave * 128 ? x0[f] : ld16(xr + c + 32 * f);
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int f = 0; f < 4; ++f) av[t][f] = ld16(ar[t] + c + 32 * f);
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
          for (int t = 0; t < RT; ++t) acc[t] = mfma(xv[f], av[t][f], acc[t]);
      }
    }
    lds_barrier();
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int q = 0; q < 4; ++q) red[wave][t][q][lane] = acc[t][q];
    lds_barrier();
    for (int o = wave; o < 4 * RT; o += LR_NW) {
      const int q = o & 3, t = o >> 2, i = 4 * g + q, row = r0 + i, j = j0 + 16 * t + c16;
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < LR_NW; ++w) v += red[w][t][q][lane];
      if (!(rows >> i & 1)) continue;
      v = j < rk ? scale * v : 0.f;
      if (!a.planes) {
        if (j < a.rmax) a.t[(size_t)row * a.rmax + j] = v;
      } else if (j < a.rp) {
        // 8 mantissa bits each, the last exact: hi + mid + lo = v
        const float hi = __uint_as_float(__float_as_uint(v) & 0xffff0000u), r1 = v == hi ? 0.f : v - hi;  // (an infinity stays one)
        const float mi = __uint_as_float(__float_as_uint(r1) & 0xffff0000u), r2 = r1 - mi;
        uint16_t* p = a.planes + (size_t)row * a.rp + j;
        const size_t plane = (size_t)a.rows * a.rp;
        p[0] = (uint16_t)(__float_as_uint(hi) >> 16);
        p[plane] = (uint16_t)(__float_as_uint(mi) >> 16);
        p[2 * plane] = (uint16_t)(__float_as_uint(r2) >> 16);
      }
    }
  }
}

// ---- y = res + W x + B t -----------------------------------------------------------------------
DEV uint32_t pk8(uint32_t v, int i) {  // bytes i, i + 1 as bf16 (exact)
  const float a = (float)(int8_t)(v >> (8 * i)), b = (float)(int8_t)(v >> (8 * i + 8));
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);  // the upper halves
}
DEV uint4 frag8(uint32_t a, uint32_t b) { return make_uint4(pk8(a, 0), pk8(a, 2), pk8(b, 0), pk8(b, 2)); }

// Few rows: a block owns 16 columns and all rows, MT tiles of 16; its eight waves take 128 inputs each in turn and
// add their sums through LDS.  48 rows, n 4096, k 2048, 40 adapters of 32 ranks: 12.6 us behind 8 to 9 of k_lora_down, 18 MB
// in all (3.8 at the copy rate); an empty launch takes 4 of each, the rest are the chains of dependent loads.  Column l % 16 of the weights in lane l, 16 inputs (16 (l / 16)) of each 64.
template <class SH, int MT>
__global__ void __launch_bounds__(LR_NT) k_lora_gemm_rows(Lora a) {
  __shared__ float red[LR_NW][MT][4][64];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), c16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const size_t n = n0 + c16 < a.n ? n0 + c16 : a.n - 1;
  // the rows and columns of this thread's outputs: output o = tid + 512 i is row 16 (o / 256) + 4 (o / 16 % 4) + o / 64 % 4 of
  // the block; what the epilogue needs of them is requested ahead of the product
  constexpr int OPT = (256 * MT + LR_NT - 1) / LR_NT;
  int row[OPT], ad[OPT], rk[OPT];
  float base[OPT];
  const int col = n0 + c16;
#pragma unroll
  for (int i = 0; i < OPT; ++i) {
    const int o = threadIdx.x + LR_NT * i;
    row[i] = 16 * (o >> 8) + 4 * (o >> 4 & 3) + (o >> 6 & 3);
    const bool live = o < 256 * MT && row[i] < a.rows && col < a.n;
    if (!live) row[i] = -1;
    base[i] = live && a.res ? a.res[row[i] * a.ldy + col] : 0.f;
    ad[i] = live ? adapter_of(a, row[i]) : -1;
    rk[i] = ad[i] >= 0 ? rank_of(a, ad[i]) : 0;
  }
  f32x4 acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
  const uint8_t* wr = reinterpret_cast<const uint8_t*>(a.w) + n * a.k + 16 * g;
  const uint16_t* xr[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = 16 * m + c16;
    xr[m] = a.x + (size_t)(r < a.rows ? r : a.rows - 1) * a.ldx + 16 * g;
  }
  for (int c = wave * 128; c < a.k; c += LR_NW * 128) {
    const uint4 w0 = ld16(wr + c), w1 = ld16(wr + c + 64);
    const float sc = SH::scale(a.s, n, c, a.k);
    uint4 x[MT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int f = 0; f < 4; ++f) x[m][f] = ld16(xr[m] + c + 64 * (f >> 1) + 8 * (f & 1));
    const uint4 b0 = frag8(w0.x, w0.y), b1 = frag8(w0.z, w0.w), b2 = frag8(w1.x, w1.y), b3 = frag8(w1.z, w1.w);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      f32x4 p = {0.f, 0.f, 0.f, 0.f};
      p = mfma(x[m][0], b0, p), p = mfma(x[m][1], b1, p), p = mfma(x[m][2], b2, p), p = mfma(x[m][3], b3, p);
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[m][q] = __builtin_fmaf(sc, p[q], acc[m][q]);
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int q = 0; q < 4; ++q) red[wave][m][q][lane] = acc[m][q];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < OPT; ++i) {
    if (row[i] < 0) continue;
    const int o = threadIdx.x + LR_NT * i;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < LR_NW; ++w) v += red[w][o >> 8][o >> 6 & 3][lane];
    // eight ranks at a time; t is 0 past the rank, where B's padding must not count
    const uint16_t* b = a.lb + ((size_t)(ad[i] < 0 ? 0 : ad[i]) * a.n + col) * a.rmax;
    const float* t = a.t + (size_t)row[i] * a.rmax;
    float d = 0.f;
#pragma unroll 4
    for (int j = 0; j < rk[i]; j += 8) {
      const uint4 q = ld16(b + j);
      const float4 t0 = ldf4(t + j), t1 = ldf4(t + j + 4);
      const int on = rk[i] - j;
      d = __builtin_fmaf(bf16_lo(q.x), t0.x, d);
      d = on > 1 ? __builtin_fmaf(bf16_hi(q.x), t0.y, d) : d;
      d = on > 2 ? __builtin_fmaf(bf16_lo(q.y), t0.z, d) : d;
      d = on > 3 ? __builtin_fmaf(bf16_hi(q.y), t0.w, d) : d;
      d = on > 4 ? __builtin_fmaf(bf16_lo(q.z), t1.x, d) : d;
      d = on > 5 ? __builtin_fmaf(bf16_hi(q.z), t1.y, d) : d;
      d = on > 6 ? __builtin_fmaf(bf16_lo(q.w), t1.z, d) : d;
      d = on > 7 ? __builtin_fmaf(bf16_hi(q.w), t1.w, d) : d;
    }
    a.y[row[i] * a.ldy + col] = base[i] + (v + d);
  }
}

// One row whose adapters have at most 16 ranks: every block computes t itself, beside its columns and from the same x, so no
// launch goes before it (n = k = 2048: 6.4 us; A x and the product apart 5.0 + 3.8 and the second launch.  Each further 16
// ranks or row cost 3 to 4 us here, as all blocks ask for the same lines: 2 rows 9.3 against 5.2 + 3.9).
template <class SH>
__global__ void __launch_bounds__(LR_NT) k_lora_gemm_one(Lora a) {
  __shared__ float red[LR_NW][2][16];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), c16 = lane & 15, g = lane >> 4;
  const int col = blockIdx.x * 16 + c16;
  const size_t n = col < a.n ? col : a.n - 1;
  const uint16_t* xr = a.x + 16 * g;
  const uint8_t* wr = reinterpret_cast<const uint8_t*>(a.w) + n * a.k + 16 * g;
  const bool mine = threadIdx.x < 16 && col < a.n;
  const float base = mine && a.res ? a.res[col] : 0.f;
  const int ad = __builtin_amdgcn_readfirstlane(adapter_of(a, 0)), rk = ad < 0 ? 0 : __builtin_amdgcn_readfirstlane(rank_of(a, ad));
  const uint16_t* ar = a.la + ((size_t)(ad < 0 ? 0 : ad) * a.rmax + (c16 < rk ? c16 : rk > 0 ? rk - 1 : 0)) * a.k + 16 * g;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f}, at = acc;
  for (int c = wave * 128; c < a.k; c += LR_NW * 128) {
    const uint4 w0 = ld16(wr + c), w1 = ld16(wr + c + 64);
    const float sc = SH::scale(a.s, n, c, a.k);
    uint4 x[4], av[4];
#pragma unroll
    for (int f = 0; f < 4; ++f) x[f] = ld16(xr + c + 64 * (f >> 1) + 8 * (f & 1));
#pragma unroll
    for (int f = 0; f < 4; ++f) av[f] = ld16(ar + c + 64 * (f >> 1) + 8 * (f & 1));
    f32x4 p = {0.f, 0.f, 0.f, 0.f};
    p = mfma(x[0], frag8(w0.x, w0.y), p), p = mfma(x[1], frag8(w0.z, w0.w), p), p = mfma(x[2], frag8(w1.x, w1.y), p), p = mfma(x[3], frag8(w1.z, w1.w), p);
    acc[0] = __builtin_fmaf(sc, p[0], acc[0]);
#pragma unroll
    for (int f = 0; f < 4; ++f) at = mfma(x[f], av[f], at);
  }
  // all 16 rows of the products are the one row
  if (g == 0) red[wave][0][c16] = acc[0], red[wave][1][c16] = at[0];
  uint4 b[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (mine)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (8 * i < rk) b[i] = ld16(a.lb + ((size_t)ad * a.n + col) * a.rmax + 8 * i);
  __syncthreads();
  if (wave != 0) return;
  float v = 0.f, t = 0.f, d = 0.f;
#pragma unroll
  for (int w = 0; w < LR_NW; ++w) v += red[w][0][c16], t += red[w][1][c16];
  t *= ad < 0 ? 0.f : a.lscale[ad];
  // ranks in order; those past the rank, where A's and B's padding must not count, are left out
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t q[4] = {b[i].x, b[i].y, b[i].z, b[i].w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float tj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(t), 8 * i + j));
      if (8 * i + j < rk) d = __builtin_fmaf(j & 1 ? bf16_hi(q[j >> 1]) : bf16_lo(q[j >> 1]), tj, d);
    }
  }
  if (mine) a.y[col] = base + (v + d);
}

// Many rows: a block of 2 x 2 waves owns 32 MT rows x 32 NT columns, a wave 16 MT x 16 NT of them.  Slices of 64 inputs
// go through two LDS buffers, a slice's global loads in flight for the whole of the slice before; the barrier between slices
// leaves them in flight.  W stays int8 in LDS and is converted in the registers of the wave that multiplies it (in bf16 a wave tile
// of 64 x 64 would read 64 KB a slice, at ~64 bytes a clock twice the time of its products), and the tile is as wide as the
// registers allow; the widest keeps 22 of them in memory.
// x: row r's 16-byte piece j lies at j ^ (r % 8), so its fragment reads meet no bank twice; W: four pieces a row in order, a
// fragment pair being 1 KB in a row, but 64 bytes from lane to lane: its reads do meet (4.2 M conflict cycles for 1.6 M LDS
// instructions in the case below).  Lane (l % 16, g = l / 16) has the inputs 16 g .. 16 g + 15 of a slice, 8 a product.
// 8 XCDs take the tiles in 8 contiguous runs, down columns of 8 row tiles, so that an XCD's blocks share x and W in its L2.
// KS = 2 (the small tile): two groups of 2 x 2 waves take half of the inputs each and join their sums through LDS, since
// small products wait for a tile's slices in turn (700 rows, n 1031, k 1024: 14.9 -> 11.2 us; 300 x 2048 x 2048: 19.3 -> 15.2).
// 4096 rows, n 4096, k 2048, runs of 12 adapters of up to 64 ranks, one scale a row: 113 us, of which the product 79 (870
// TFLOP/s; no one pipe fills them, they wait for each other: LDS reads 27, its writes 14, matrix unit 29, the conversions of W, done by two waves
// each, and the rest of the VALU 35), the residual and the store 24 (128 MB, the card's copy rate; nothing is left to overlap them with when
// every CU has its two tiles at once) and the adapters the rest.
constexpr int LG_K = 64;
// 16 bytes of each lane to dst + 16 lane
DEV void to_lds(const void* src, uint4* dst) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}
template <class SH, int MT, int NT, int KS>
__global__ void __launch_bounds__(256 * KS, 2 * KS) k_lora_gemm_tiles(Lora a, int tm, int tn) {
  constexpr int BM = 32 * MT, BN = 32 * NT, PX = BM * 8 / 256, PW = BN * 4 / 256;
  constexpr int ME = MT / KS;  // row tiles of a wave once the parts of K are joined
  static_assert(PX * 256 == BM * 8 && PW * 256 == BN * 4 && PX % KS == 0, "pieces per thread");
  __shared__ uint4 lds_x[KS][2][BM * 8], lds_w[KS][2][BN * 4];
  const int part = KS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  auto& lx = lds_x[part];
  auto& lw = lds_w[part];
  const int tid = threadIdx.x & 255, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()) & 3, c16 = lane & 15, g = lane >> 4;
  // tile of this block
  const int total = tm * tn, per = (total + 7) / 8, q = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || q >= total) return;
  const int band = q / (8 * tn), bh = tm - 8 * band < 8 ? tm - 8 * band : 8, in = q - band * 8 * tn;
  const int m0 = (8 * band + in % bh) * BM, n0 = in / bh * BN;
  const int wm = (wave >> 1) * 16 * MT, wn = (wave & 1) * 16 * NT, we = wm + 16 * ME * part;
  // adapters of the wave's rows and their ranks, known before the product ends
  int mine[ME], ranks[ME];
#pragma unroll
  for (int m = 0; m < ME; ++m) mine[m] = adapter_of(a, m0 + we + 16 * m + c16), ranks[m] = mine[m] < 0 ? 0 : rank_of(a, mine[m]);
  // this part's inputs, whole pairs of slices
  const int pairs = a.k / 128, k0 = part * ((pairs + KS - 1) / KS) * 128, k1 = KS == 1 || part ? a.k : (pairs + KS - 1) / KS * 128;
  const uint16_t* xp[PX];
  const uint8_t* wp[PW];
#pragma unroll
  for (int i = 0; i < PX; ++i) {
    const int r = m0 + (tid + 256 * i) / 8;
    xp[i] = a.x + (size_t)(r < a.rows ? r : a.rows - 1) * a.ldx + 8 * (tid & 7) + (k0 < a.k ? k0 : 0);
  }
#pragma unroll
  for (int i = 0; i < PW; ++i) {
    const int n = n0 + (tid + 256 * i) / 4;
    wp[i] = reinterpret_cast<const uint8_t*>(a.w) + (size_t)(n < a.n ? n : a.n - 1) * a.k + 16 * (tid & 3) + (k0 < a.k ? k0 : 0);
  }
  uint4 xv[PX], wv[PW];
  auto load = [&](int k) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PX; ++i) xv[i] = ld16(xp[i] + k);
#pragma unroll
    for (int i = 0; i < PW; ++i) wv[i] = ld16(wp[i] + k);
  };
  auto store = [&](int b) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PX; ++i) {
      const int r = (tid + 256 * i) / 8, j = tid & 7;
      lx[b][r * 8 + (j ^ (r & 7))] = xv[i];
    }
#pragma unroll
    for (int i = 0; i < PW; ++i) lw[b][tid + 256 * i] = wv[i];
  };
  // SH::per_row: the scale is applied once at the end; else the sums of a group (two slices) are scaled into `sum`
  f32x4 acc[MT][NT], sum[SH::per_row ? 1 : MT][SH::per_row ? 1 : NT];
  const f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      acc[m][n] = z;
      if constexpr (!SH::per_row) sum[m][n] = z;
    }
  int col[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int c = n0 + wn + 16 * n + c16;
    col[n] = c < a.n ? c : a.n - 1;
  }
  const int steps = (k1 - k0) / LG_K, most = KS == 1 ? steps : (pairs + KS - 1) / KS * 2;  // even
  load(0);
  store(0);
  load(steps > 0 ? LG_K : 0);
  lds_barrier();
  auto step = [&](auto odd, int s) __attribute__((always_inline)) {
    constexpr int B = decltype(odd)::value;
    if (KS > 1 && s >= steps) {  // the longer part's barriers
      lds_barrier();
      return;
    }
    if (s + 1 < steps) {
      store(B ^ 1);
      load(s + 2 < steps ? (s + 2) * LG_K : (s + 1) * LG_K);
    }
    float sc[NT];
    if constexpr (B == 1 && !SH::per_row) {
#pragma unroll
      for (int n = 0; n < NT; ++n) sc[n] = SH::scale(a.s, col[n], k0 + s * LG_K, a.k);
    }
    uint4 xf[2][MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = wm + 16 * m + c16;
      xf[0][m] = lx[B][r * 8 + ((2 * g) ^ (r & 7))], xf[1][m] = lx[B][r * 8 + ((2 * g + 1) ^ (r & 7))];
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint4 v = lw[B][(wn + 16 * n + c16) * 4 + g];
      const uint4 w0 = frag8(v.x, v.y), w1 = frag8(v.z, v.w);
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[m][n] = mfma(xf[0][m], w0, acc[m][n]);
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[m][n] = mfma(xf[1][m], w1, acc[m][n]);
      if constexpr (B == 1 && !SH::per_row) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
          for (int r = 0; r < 4; ++r) sum[m][n][r] = __builtin_fmaf(sc[n], acc[m][n][r], sum[m][n][r]);
          acc[m][n] = z;
        }
      }
    }
    lds_barrier();
  };
  for (int s = 0; s < most; s += 2) {
    step(std::integral_constant<int, 0>{}, s);
    step(std::integral_constant<int, 1>{}, s + 1);
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float sc = SH::per_row ? SH::scale(a.s, col[n], 0, a.k) : 1.f;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if constexpr (SH::per_row) {
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[m][n][r] *= sc;
      } else {
        acc[m][n] = sum[m][n];
      }
    }
  }
  f32x4 out[ME][NT];
  if constexpr (KS == 1) {
#pragma unroll
    for (int m = 0; m < ME; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) out[m][n] = acc[m][n];
  } else {
    // each wave joins its share of the row tiles with the other part's sums
    static_assert(KS == 1 || (KS == 2 && sizeof(lds_x) >= 8 * ME * NT * 64 * 16), "sums on their way");
    f32x4* ex = reinterpret_cast<f32x4*>(&lds_x[0][0][0]);
#pragma unroll
    for (int m = 0; m < ME; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) ex[(((part ^ 1) * 4 + wave) * ME * NT + m * NT + n) * 64 + lane] = part ? acc[m][n] : acc[ME + m][n];
    lds_barrier();
#pragma unroll
    for (int m = 0; m < ME; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) out[m][n] = (part ? acc[ME + m][n] : acc[m][n]) + ex[((part * 4 + wave) * ME * NT + m * NT + n) * 64 + lane];
    lds_barrier();
  }
  // B t, 64 ranks at a time: t of the block's rows goes to LDS (plane p in place of the x and W slices, laid out as a slice of x), then each wave
  // multiplies the distinct adapters of its rows and adds what belongs to each row; B's fragments serve all row tiles.
  // (B of two or four adapters asked for at once: level, 700 rows of 40 adapters 59 -> 64 and 71 us.)
  if (a.adapter) {
    static_assert(sizeof(lds_w[0]) >= sizeof(lds_x[0][0]), "plane 2 of t");
    uint4 *l0 = lds_x[0][0], *l1 = lds_x[0][1], *l2 = lds_w[0][0];
    const size_t plane = (size_t)a.rows * a.rp;
    uint32_t rows_of[ME];
#pragma unroll
    for (int m = 0; m < ME; ++m) rows_of[m] = (uint32_t)__ballot(mine[m] >= 0) & 0xffffu;
    uint4 b[2][NT];
    auto load_b = [&](int h, int ad, int rk, int j0) __attribute__((always_inline)) {  // ranks j0 + 32 h ..
      const int last = n0 + BN < a.n ? BN : a.n - n0, j = j0 + 32 * h + 8 * g;
      const Rsrc B = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(a.lb + ((size_t)ad * a.n + n0) * a.rmax), 0, (uint32_t)(last * a.rmax * 2), 0x00020000);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint32_t off = ((wn + 16 * n + c16) * a.rmax + j) * 2;
        b[h][n] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(B, j < rk ? off : 0x80000000u, 0, 0));
      }
    };
    for (int j0 = 0; j0 < a.rp; j0 += 64) {
      uint32_t left[ME];
#pragma unroll
      for (int m = 0; m < ME; ++m) left[m] = rows_of[m];
      // the next adapter and its rank, -1 for none: its rows leave `left` and are those of `has`
      uint32_t has[ME];
      int rk = 0;
      auto next = [&]() __attribute__((always_inline)) {
        int ad = -1;
#pragma unroll
        for (int m = ME - 1; m >= 0; --m)
          if (left[m]) {
            const int at = __builtin_ctz(left[m]);
            ad = __builtin_amdgcn_readlane(mine[m], at), rk = __builtin_amdgcn_readlane(ranks[m], at);
          }
#pragma unroll
        for (int m = 0; m < ME; ++m) {
          has[m] = ad < 0 ? 0u : (uint32_t)__ballot(mine[m] == ad) & 0xffffu;
          left[m] &= ~has[m];
        }
        return ad;
      };
      int ad = next();
      if (ad >= 0) load_b(0, ad, rk, j0), load_b(1, ad, rk, j0);
      if (j0) lds_barrier();
      // straight to LDS, 64 pieces a wave in order: no registers beside the sums and B's fragments
#pragma unroll
      for (int i = part; i < PX; i += KS) {
        const int at = 256 * i + 64 * wave, rl = (at + lane) >> 3, r = m0 + rl, j = j0 + 8 * ((lane & 7) ^ (rl & 7));
        const uint16_t* src = a.planes + (size_t)(r < a.rows ? r : a.rows - 1) * a.rp + (j < a.rp ? j : 0);
        to_lds(src, l0 + at), to_lds(src + plane, l1 + at), to_lds(src + 2 * plane, l2 + at);
      }
      __builtin_amdgcn_s_waitcnt(0);
      lds_barrier();
      while (ad >= 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int on = rk - j0 - 32 * h - 8 * g;  // of this lane's 8 ranks, those below rk
          const uint32_t k0 = on >= 2 ? 0xffffffffu : on == 1 ? 0xffffu : 0u, k1 = on >= 4 ? 0xffffffffu : on == 3 ? 0xffffu : 0u;
          const uint32_t k2 = on >= 6 ? 0xffffffffu : on == 5 ? 0xffffu : 0u, k3 = on >= 8 ? 0xffffffffu : on == 7 ? 0xffffu : 0u;
#pragma unroll
          for (int n = 0; n < NT; ++n) b[h][n] = make_uint4(b[h][n].x & k0, b[h][n].y & k1, b[h][n].z & k2, b[h][n].w & k3);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (rk <= j0 + 32 * h) continue;
#pragma unroll
          for (int m = 0; m < ME; ++m) {
            if (!has[m]) continue;
            const int r = we + 16 * m + c16, at = r * 8 + ((4 * h + g) ^ (r & 7));
            const uint4 tf[3] = {l0[at], l1[at], l2[at]};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              f32x4 s = z;
#pragma unroll
              for (int q3 = 0; q3 < 3; ++q3) s = mfma(tf[q3], b[h][n], s);
              // (chosen, not multiplied by zero: another row's adapter may hold infinities)
#pragma unroll
              for (int i = 0; i < 4; ++i) out[m][n][i] += has[m] >> (4 * g + i) & 1 ? s[i] : 0.f;
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        ad = next();
        if (ad >= 0) load_b(0, ad, rk, j0), load_b(1, ad, rk, j0);
      }
    }
  }
  // the residual of 16 rows in flight at a time (y may be res: its loads could not pass the stores)
#pragma unroll
  for (int m = 0; m < ME; ++m) {
    float rv[4][NT];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = m0 + we + 16 * m + 4 * g + r;
#pragma unroll
      for (int n = 0; n < NT; ++n) rv[r][n] = a.res ? gld<float>(a.res + (size_t)(row < a.rows ? row : a.rows - 1) * a.ldy + col[n]) : 0.f;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = m0 + we + 16 * m + 4 * g + r;
#pragma unroll
      for (int n = 0; n < NT; ++n)
        if (row < a.rows && n0 + wn + 16 * n + c16 < a.n) a.y[row * a.ldy + col[n]] = rv[r][n] + out[m][n][r];
    }
  }
}

bool lora_shape_ok(int rows, int n, int k, int rmax) {
  return rows >= 0 && rows <= (1 << 20) && n >= 1 && k >= 128 && k <= 16384 && k % 128 == 0 && rmax >= 8 && rmax <= 128 && rmax % 8 == 0;
}

template <class SH>
int gemm_lora(Lora a, int ldx, int ldy, hipStream_t st) {
  if (!lora_shape_ok(a.rows, a.n, a.k, a.rmax) || ldx < a.k || ldx % 8 || ldy < a.n || a.adapters < 0) return -1;
  if (a.rows == 0) return 0;
  if (!a.w || !a.s || !a.x || !a.y || ((uintptr_t)a.w & 15) || ((uintptr_t)a.x & 15)) return -1;
  if (a.adapters == 0) a.adapter = nullptr;
  if (a.adapter && (!a.la || !a.lb || !a.rank || !a.lscale || !a.t || ((uintptr_t)a.la & 15) || ((uintptr_t)a.lb & 15) || ((uintptr_t)a.t & 15)))
    return -1;
  a.ldx = ldx, a.ldy = ldy;
  const int tiles = (a.rows + 15) / 16;
  const bool few = a.rows <= 64;
  a.rp = (a.rmax + 31) & ~31;
  a.planes = few || !a.adapter ? nullptr : reinterpret_cast<uint16_t*>(a.t);
  if (a.adapter && a.rows == 1 && a.rmax <= 16) {
    hipLaunchKernelGGL((k_lora_gemm_one<SH>), dim3((a.n + 15) / 16), dim3(LR_NT), 0, st, a);
    return 0;
  }
  // Blocks along the distinct adapters: 16 rows may have 16, but runs of rows have one or two, and blocks without one cost
  // their start (4096 rows in runs: 21 us with 2, 54 with 16; in any order 300 rows of 40 adapters: 38 and 14, 48 rows: 26 and 7.5).
  // 32 ranks a block take x half as often as 16 and have fewer blocks: from 65 rows on (4096 rows: 21 and 25 us; 48: 8.9 and 7.5).
  const unsigned ny = 256 / tiles < 2 ? 2 : 256 / tiles > 16 ? 16 : 256 / tiles;
  if (a.adapter && few) hipLaunchKernelGGL(k_lora_down<1>, dim3(tiles, ny, (a.rmax + 15) / 16), dim3(LR_NT), 0, st, a);
  else if (a.adapter) hipLaunchKernelGGL(k_lora_down<2>, dim3(tiles, ny, a.rp / 32), dim3(LR_NT), 0, st, a);
  if (few) {
    const dim3 g((a.n + 15) / 16), b(LR_NT);
    if (tiles == 1) hipLaunchKernelGGL((k_lora_gemm_rows<SH, 1>), g, b, 0, st, a);
    else if (tiles == 2) hipLaunchKernelGGL((k_lora_gemm_rows<SH, 2>), g, b, 0, st, a);
    else if (tiles == 3) hipLaunchKernelGGL((k_lora_gemm_rows<SH, 3>), g, b, 0, st, a);
    else hipLaunchKernelGGL((k_lora_gemm_rows<SH, 4>), g, b, 0, st, a);
    return 0;
  }
  auto go = [&](auto mt, auto nt, auto ks) {
    constexpr int M = decltype(mt)::value, N = decltype(nt)::value, KS = decltype(ks)::value;
    const long long tm = (a.rows + 32ll * M - 1) / (32 * M), tn = (a.n + 32ll * N - 1) / (32 * N), per = (tm * tn + 7) / 8;
    hipLaunchKernelGGL((k_lora_gemm_tiles<SH, M, N, KS>), dim3((unsigned)(8 * per)), dim3(256 * KS), 0, st, a, (int)tm, (int)tn);
  };
  constexpr std::integral_constant<int, 1> i1{};
  constexpr std::integral_constant<int, 2> i2{};
  constexpr std::integral_constant<int, 4> i4{};
  constexpr std::integral_constant<int, SH::per_row ? 8 : 4> wide{};
  // the wide tile once there are two for each CU, the middle one once there is one (4096 x 4096 x 2048, ranks to 64, W with one
  // scale a row: wide 113 us, middle 128; 2048 rows: 74 and 67), else the small one with two parts of K a block
  const long long m128 = (a.rows + 127) / 128;
  if (m128 * ((a.n + 32 * wide.value - 1) / (32 * wide.value)) >= 512) go(i4, wide, i1);
  else if (m128 * ((a.n + 127) / 128) >= 256) go(i4, i4, i1);
  else go(i2, i2, i2);
  return 0;
}

}  // namespace

API size_t dr_gemm_q8_lora_ws(int rows, int n, int k, int rmax) {
  // t: fp32 of rmax ranks or three bf16 planes of rmax rounded up to 32
  return lora_shape_ok(rows, n, k, rmax) ? ((size_t)(rows ? rows : 1) * ((rmax + 31) & ~31) * 6 + 255) & ~(size_t)255 : 0;
}

API int dr_gemm_q8_lora(const int8_t* w, const uint16_t* s, const uint16_t* x, int ldx, const int* adapter, const uint16_t* la,
                        const uint16_t* lb, const int* rank, const float* lscale, int adapters, int rmax, void* ws,
                        const float* res, float* y, int ldy, int rows, int n, int k, hipStream_t st) {
  return gemm_lora<Q8G128F16>(Lora{w, s, x, adapter, la, lb, rank, lscale, res, static_cast<float*>(ws), y, 0, 0, adapters, rmax, rows, n, k, nullptr, 0},
                              ldx, ldy, st);
}

API int dr_gemm_q8_lora_bf16s(const int8_t* w, const uint16_t* s, const uint16_t* x, int ldx, const int* adapter,
                              const uint16_t* la, const uint16_t* lb, const int* rank, const float* lscale, int adapters, int rmax,
                              void* ws, const float* res, float* y, int ldy, int rows, int n, int k, hipStream_t st) {
  return gemm_lora<Q8RowBF16>(Lora{w, s, x, adapter, la, lb, rank, lscale, res, static_cast<float*>(ws), y, 0, 0, adapters, rmax, rows, n, k, nullptr, 0},
                              ldx, ldy, st);
}
