// The norms between two blocks of a layer with the gate and the residual scale, one pass over a row:
//   n  = b rsqrt(mean(b^2) + eps) pw            norm behind the block (pw null: n = b)
//   xo = xscale x + bscale cs[c] sigmoid(gate) n
//   hn = bf16(xo rsqrt(mean(xo^2) + eps) nw)    norm before the next block
// b is the block's output (f32 or bf16), or the weighted sum of a prefill's expert rows,
//   b = sigmoid(sgate) shared + sum_k wts[k] y[slot_of[k]]  (k ascending, as dr_moe_combine).
//
// Every element of a row is read once and stays in the registers of the L lanes that share the row
// (8 elements a lane, 16 beyond 4096 columns), so b's sum of squares, xo and xo's sum of squares
// need no second read and xo may be x or b.  Bound by HBM: 4096 rows of 4096, 235 MB, 53 us = 4.4 TB/s where a large copy
// reaches 4.7 (single elements where something is not aligned: 58); with few rows by the chain load, two row sums, store: 3.2 us for one
// row of 2048.  The combine form reads topk rows of y besides: 300 rows of 2048, top 8, 28 MB in 9.8 us.
#include "common.hpp"

using namespace drm;

namespace {

struct BlockNorm {
  const void* b;  // block output, or y of the combine form
  const float* x;
  const float *pw, *gate, *cs, *nw;
  float* xo;
  uint16_t* hn;
  size_t ldb, ldx, ldg, ldo, ldh;
  float bscale, xscale, eps;
  int gate_mode, rows, h;
  // combine form
  const int* slot_of;
  const float *wts, *sgate, *shared;  // sgate null without shared: the kernel reads what it is given
  int topk;
};

enum { B_NONE, B_F32, B_BF16, B_COMBINE };

template <int V>
DEV void ld_f32(const float* p, float (&o)[V]) {
  if constexpr (V == 4) {
    const float4 v = ldf4(p);
    o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w;
  } else {
    o[0] = gld<float>(p);
  }
}

// sum over the L lanes of a row; red: one word per wave of the block (L > 64)
template <int L>
DEV float row_sum(float v, float* red) {
  v = wave_sum(v);
  if constexpr (L > WAVE) {
    if (lane_id() == 0) red[wave_id()] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < L / WAVE; ++w) v += red[w];
    __syncthreads();
  }
  return v;
}

// V elements per load (4, or 1 where sizes, strides or addresses are no multiple of 16 bytes), PER
// loads per lane; blocks of max(L, 256) threads, grid-stride over the rows.  The vectors pw, cs and nw
// are requested with the row (a single row then waits for memory once) up to 8 elements a lane, after the
// sums beyond that (all at once they would not fit the registers of 1024 threads).
template <int BK, int V, int L, int PER>
__global__ void __launch_bounds__(L > 256 ? L : 256) k_block_norm(BlockNorm a) {
  constexpr int NT = L > 256 ? L : 256, RPB = NT / L;
  constexpr bool EARLY = PER * V <= 8;
  constexpr int KG = 32 / (PER * V);  // picks in flight: at most 32 elements a lane
  __shared__ float red[NT / WAVE];
  const int t = threadIdx.x % L;
  for (long long r0 = (long long)blockIdx.x * RPB; r0 < a.rows; r0 += (long long)gridDim.x * RPB) {
    const long long r = r0 + threadIdx.x / L;
    // a wave without a row (L = 64) has nothing to wait for; with L > 64 a block is one row
    if (r >= a.rows) break;
    float b[PER][V], x[PER][V], g[PER][V], pw[PER][V], nw[PER][V], cs[PER][V];
    if constexpr (BK == B_COMBINE) {
      const float sg = a.sgate ? 1.f / (1.f + expf(-a.sgate[r])) : 0.f;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int c = (t + L * j) * V;
#pragma unroll
        for (int v = 0; v < V; ++v) b[j][v] = 0.f;
        if (c < a.h && a.shared) {
          float s[V];
          ld_f32<V>(a.shared + (size_t)r * a.h + c, s);
#pragma unroll
          for (int v = 0; v < V; ++v) b[j][v] = sg * s[v];
        }
      }
      const float* y = reinterpret_cast<const float*>(a.b);
      for (int k0 = 0; k0 < a.topk; k0 += KG) {
        float w[KG], q[KG][PER][V];
#pragma unroll
        for (int k = 0; k < KG; ++k) {
          const bool on = k0 + k < a.topk;
          w[k] = on ? a.wts[(size_t)r * a.topk + k0 + k] : 0.f;
          const float* yr = y + (on ? (size_t)a.slot_of[(size_t)r * a.topk + k0 + k] : 0) * a.h;
#pragma unroll
          for (int j = 0; j < PER; ++j) {
            const int c = (t + L * j) * V;
#pragma unroll
            for (int v = 0; v < V; ++v) q[k][j][v] = 0.f;
            if (on && c < a.h) ld_f32<V>(yr + c, q[k][j]);
          }
        }
#pragma unroll
        for (int k = 0; k < KG; ++k)
          if (k0 + k < a.topk)
#pragma unroll
            for (int j = 0; j < PER; ++j)
#pragma unroll
              for (int v = 0; v < V; ++v) b[j][v] += w[k] * q[k][j][v];
      }
    }
    const float grow = a.gate_mode == 1 ? a.gate[r] : 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int c = (t + L * j) * V;
      const bool in = c < a.h;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if constexpr (BK != B_COMBINE) b[j][v] = 0.f;
        x[j][v] = 0.f, g[j][v] = grow, pw[j][v] = 1.f, nw[j][v] = 0.f, cs[j][v] = 1.f;
      }
      if (!in) continue;
      if constexpr (BK == B_F32) ld_f32<V>(reinterpret_cast<const float*>(a.b) + r * a.ldb + c, b[j]);
      if constexpr (BK == B_BF16) {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(a.b) + r * a.ldb + c;
        if constexpr (V == 4) {
          const uint2 w = ld8(p);
          b[j][0] = bf16_lo(w.x), b[j][1] = bf16_hi(w.x), b[j][2] = bf16_lo(w.y), b[j][3] = bf16_hi(w.y);
        } else {
          b[j][0] = bf16f(ld2(p));
        }
      }
      if (a.x) ld_f32<V>(a.x + r * a.ldx + c, x[j]);
      if (a.gate_mode == 2) ld_f32<V>(a.gate + r * a.ldg + c, g[j]);
      if (EARLY && a.pw) ld_f32<V>(a.pw + c, pw[j]);
      if (EARLY && a.cs) ld_f32<V>(a.cs + c, cs[j]);
      if (EARLY && a.hn) ld_f32<V>(a.nw + c, nw[j]);
    }
    float inv = 1.f;
    if (BK != B_NONE && a.pw) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < PER; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) ss += b[j][v] * b[j][v];
      inv = rsqrtf(row_sum<L>(ss, red) / (float)a.h + a.eps);
    }
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (!EARLY && (t + L * j) * V < a.h) {
        if (a.pw) ld_f32<V>(a.pw + (t + L * j) * V, pw[j]);
        if (a.cs) ld_f32<V>(a.cs + (t + L * j) * V, cs[j]);
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float o = a.xscale * x[j][v];
        if constexpr (BK != B_NONE) {
          float n = b[j][v] * inv * pw[j][v] * (a.bscale * cs[j][v]);
          if (a.gate_mode) n = n / (1.f + expf(-g[j][v]));
          // a lane past the row holds zeros, but 0 inv is no number where the row has none
          if (a.x) o += n;
          else o = n;
        }
        o = (t + L * j) * V < a.h ? o : 0.f;
        x[j][v] = o;
        ss += o * o;
      }
    }
    if (a.xo)
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int c = (t + L * j) * V;
        if (c >= a.h) continue;
        float* p = a.xo + r * a.ldo + c;
        if constexpr (V == 4) *reinterpret_cast<float4*>(p) = make_float4(x[j][0], x[j][1], x[j][2], x[j][3]);
        else *p = x[j][0];
      }
    if (a.hn) {
      const float i2 = rsqrtf(row_sum<L>(ss, red) / (float)a.h + a.eps);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int c = (t + L * j) * V;
        if (c >= a.h) continue;
        uint16_t* p = a.hn + r * a.ldh + c;
        if (!EARLY) ld_f32<V>(a.nw + c, nw[j]);
        uint32_t q[V];
#pragma unroll
        for (int v = 0; v < V; ++v) q[v] = to_bf16(x[j][v] * i2 * nw[j][v]);
        if constexpr (V == 4) *reinterpret_cast<uint2*>(p) = make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
        else *p = (uint16_t)q[0];
      }
    }
  }
}

template <int BK, int V, int L, int PER>
void launch(const BlockNorm& a, hipStream_t st) {
  constexpr int NT = L > 256 ? L : 256, RPB = NT / L;
  const long long blocks = ((long long)a.rows + RPB - 1) / RPB;
  hipLaunchKernelGGL((k_block_norm<BK, V, L, PER>), dim3((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20)), dim3(NT), 0, st, a);
}

// The fewest lanes that hold the row in 8 elements each, 16 beyond 4096 columns: more in a lane hide less of the next load (4096 rows:
// h 2048 20.6 us, 29.0 with 16; h 4096 54.0 and 55.3), but blocks of 1024 threads leave a CU idle while a row ends (2000
// rows of 8192: 56.5 us with 512 lanes of 16, 67.9 with 1024 of 8; above 8192 512 lanes of 32 spill: 66 and 73).  Of the
// kernels here those for unaligned rows past 8192 columns keep 44 to 56 registers in memory.
template <int BK, int V>
void launch_l(const BlockNorm& a, hipStream_t st) {
  constexpr int P = 8 / V;
  if (a.h <= 512) launch<BK, V, 64, P>(a, st);
  else if (a.h <= 1024) launch<BK, V, 256, P / 2>(a, st);
  else if (a.h <= 2048) launch<BK, V, 256, P>(a, st);
  else if (a.h <= 4096) launch<BK, V, 512, P>(a, st);
  else if (a.h <= 8192) launch<BK, V, 512, 2 * P>(a, st);
  else launch<BK, V, 1024, 2 * P>(a, st);
}

template <int BK>
int block_norm(BlockNorm a, hipStream_t st) {
  if (a.rows < 0 || a.h < 1 || a.h > 16384 || a.gate_mode < 0 || a.gate_mode > 2 || (a.gate_mode && !a.gate)) return -1;
  if ((!a.xo && !a.hn) || (a.hn && !a.nw) || (BK == B_NONE && !a.x)) return -1;
  const size_t h = a.h;
  if ((a.b && BK != B_COMBINE && a.ldb < h) || (a.x && a.ldx < h) || (a.gate_mode == 2 && a.ldg < h) || (a.xo && a.ldo < h) ||
      (a.hn && a.ldh < h))
    return -1;
  if (a.rows == 0) return 0;
  auto a16 = [](const void* p) { return ((uintptr_t)p & 15) == 0; };
  auto a8 = [](const void* p) { return ((uintptr_t)p & 7) == 0; };
  const bool bok = BK == B_NONE || (BK == B_BF16 ? a8(a.b) : a16(a.b));
  const bool vec = h % 4 == 0 && bok && (BK == B_NONE || a.ldb % 4 == 0) && a16(a.pw) && a16(a.cs) && a16(a.nw) && a16(a.shared) &&
                   (!a.x || (a16(a.x) && a.ldx % 4 == 0)) && (a.gate_mode != 2 || (a16(a.gate) && a.ldg % 4 == 0)) &&
                   (!a.xo || (a16(a.xo) && a.ldo % 4 == 0)) && (!a.hn || (a8(a.hn) && a.ldh % 4 == 0));
  if (vec) launch_l<BK, 4>(a, st);
  else launch_l<BK, 1>(a, st);
  return 0;
}

BlockNorm norm_args(const void* b, int ldb, const float* x, int ldx, const float* pw, const float* gate, int gate_mode, int ldg,
                    const float* cs, float bscale, float xscale, const float* nw, float eps, float* xo, int ldo, uint16_t* hn,
                    int ldh, int rows, int h) {
  // a negative stride is below every row size
  auto ld = [](int v) { return v < 0 ? (size_t)0 : (size_t)v; };
  return BlockNorm{b, x, pw, gate, cs, nw, xo, hn, ld(ldb), ld(ldx), ld(ldg), ld(ldo), ld(ldh), bscale, xscale, eps, gate_mode,
                   rows, h, nullptr, nullptr, nullptr, nullptr, 0};
}

}  // namespace

API int dr_block_norm(const float* b, int ldb, const float* x, int ldx, const float* pw, const float* gate, int gate_mode,
                      int ldg, const float* cs, float bscale, float xscale, const float* nw, float eps, float* xo, int ldo,
                      uint16_t* hn, int ldh, int rows, int h, hipStream_t st) {
  const BlockNorm a = norm_args(b, ldb, x, ldx, pw, gate, gate_mode, ldg, cs, bscale, xscale, nw, eps, xo, ldo, hn, ldh, rows, h);
  return b ? block_norm<B_F32>(a, st) : block_norm<B_NONE>(a, st);
}

API int dr_block_norm_bf16(const uint16_t* b, int ldb, const float* x, int ldx, const float* pw, const float* gate,
                           int gate_mode, int ldg, const float* cs, float bscale, float xscale, const float* nw, float eps,
                           float* xo, int ldo, uint16_t* hn, int ldh, int rows, int h, hipStream_t st) {
  const BlockNorm a = norm_args(b, ldb, x, ldx, pw, gate, gate_mode, ldg, cs, bscale, xscale, nw, eps, xo, ldo, hn, ldh, rows, h);
  return b ? block_norm<B_BF16>(a, st) : block_norm<B_NONE>(a, st);
}

API int dr_moe_combine_norm(const float* y, const int* slot_of, const float* wts, const float* sgate, const float* shared,
                            int topk, const float* x, int ldx, const float* pw, const float* gate, int gate_mode, int ldg,
                            const float* cs, float bscale, float xscale, const float* nw, float eps, float* xo, int ldo,
                            uint16_t* hn, int ldh, int rows, int h, hipStream_t st) {
  if (topk < 1 || topk > 32 || (rows > 0 && (!y || !slot_of || !wts || (shared && !sgate)))) return -1;
  BlockNorm a = norm_args(y, h, x, ldx, pw, gate, gate_mode, ldg, cs, bscale, xscale, nw, eps, xo, ldo, hn, ldh, rows, h);
  a.slot_of = slot_of, a.wts = wts, a.sgate = shared ? sgate : nullptr, a.shared = shared, a.topk = topk;
  return block_norm<B_COMBINE>(a, st);
}
