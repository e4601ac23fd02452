// The norm of each head and its rotary positions:
//   n = x rsqrt(mean(x^2) + eps) nw          over a head's d elements (nw null: n = x)
//   th = pos freq[j], c = mscale cos th, s = mscale sin th,  j < rot / 2
//   (a, b) = (n[j], n[j + rot/2]) or, in pairs, (n[2 j], n[2 j + 1]) -> (a c - b s, b c + a s); elements from rot on stay n.
//
// A block takes a row (or a share of its heads, or as many rows as give its lanes work): it requests its elements, works out the rows' cosines and
// sines once for all heads (LDS), and turns.  The lanes of a head (a power of two within a wave) hold both partners of
// each pair, so the norm is a butterfly and nothing else crosses lanes, and y may be x.  Angles: the product of a position
// and a frequency in 64 bits, its whole turns taken off there (at position 10^6 fp32 would be 0.06 rad off), the
// sine and cosine of the rest in fp32.
//
// Every element is loaded once and stored once, so memory bounds large calls: 8192 rows of 16 heads of 256 (64 turned, gates between the heads, fp32
// in, bf16 out) 38.4 us, 5.24 TB/s.  Small ones are a launch and one chain of loads, sums and stores: one row of 20 heads of 128 3.5 us; 777 rows of
// 15 heads of 80 in bf16, 36 turned in pairs, 3.9 us (5.4 with a load an element).
#include "common.hpp"

using namespace drm;

namespace {

constexpr int NT = 256;

struct Rope {
  const void* x;
  const float* nw;
  const int* pos;
  const float* freq;
  float* y;
  uint16_t* yb;
  size_t ldx, hsx, ldn, ldy, ldb;
  float eps, mscale;
  int rows, heads, d, rot, pairs;
};

// V elements of a row from `at` on
template <bool B16, int V>
DEV void ld_x(const void* x, size_t at, float (&o)[V]) {
  if constexpr (B16) {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(x) + at;
    if constexpr (V == 4) {
      const uint2 w = ld8(p);
      o[0] = bf16_lo(w.x), o[1] = bf16_hi(w.x), o[2] = bf16_lo(w.y), o[3] = bf16_hi(w.y);
    } else {
      o[0] = bf16f(ld2(p));
    }
  } else {
    const float* p = reinterpret_cast<const float*>(x) + at;
    if constexpr (V == 4) {
      const float4 v = ldf4(p);
      o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w;
    } else {
      o[0] = gld<float>(p);
    }
  }
}

template <int V>
DEV void st_y(const Rope& a, size_t row, int at, const float (&o)[V]) {
  if (a.y) {
    float* p = a.y + row * a.ldy + at;
    if constexpr (V == 4) *reinterpret_cast<float4*>(p) = make_float4(o[0], o[1], o[2], o[3]);
    else *p = o[0];
  }
  if (a.yb) {
    uint16_t* p = a.yb + row * a.ldb + at;
    if constexpr (V == 4) *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]));
    else *p = to_bf16(o[0]);
  }
}

// Sum over the L lanes of a head; all lanes of the wave take part.
DEV float head_sum(float v, int L) {
  if (L > 1) v = xsum_step<1>(v);
  if (L > 2) v = xsum_step<2>(v);
  if (L > 4) v = xsum_step<4>(v);
  if (L > 8) v = xsum_step<8>(v);
  if (L > 16) v = xsum_step<16>(v);
  if (L > 32) v = xsum_step<32>(v);
  return v;
}

// V elements a load (4, or 1 where sizes, strides or addresses allow no more).  A unit is a vector of the first half of the turned elements and
// its counterpart in the second (the partners), or two vectors of the elements behind rot likewise; in pairs a vector of the first half
// of the head and one of the second, as each holds both partners: lanes beside each other load and store beside each other.  2^LS lanes a head, up to PER units a lane; RB rows a block; U heads a lane at a time.
template <bool B16, int V, int PER, int U>
__global__ void __launch_bounds__(NT) k_rope(Rope a, int LS, int RB) {
  extern __shared__ float2 cs[];  // [RB][rot / 2]
  const bool whole = V > 1 && a.pairs;
  const int half = a.rot >> 1, turned = whole ? 0 : half / V, tail = (a.d - (whole ? 0 : a.rot) + 2 * V - 1) / (2 * V), units = turned + tail;
  const long long r0 = (long long)blockIdx.x * RB;
  const int hb = (a.heads + gridDim.y - 1) / gridDim.y, h0 = blockIdx.y * hb, nh = a.heads - h0 < hb ? a.heads - h0 : hb;
  const int nr = a.rows - r0 < RB ? (int)(a.rows - r0) : RB, items = (nr * nh) << LS, l = threadIdx.x & ((1 << LS) - 1);
  int e0[PER], e1[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int k = l + (u << LS);
    e0[u] = k < turned ? V * k : (whole ? 0 : a.rot) + V * (k - turned);
    e1[u] = k < turned ? e0[u] + half : e0[u] + V * tail;
    if (V == 1 && a.pairs && k < turned) e0[u] = 2 * k, e1[u] = 2 * k + 1;  // a unit is one pair
    if (k >= units) e0[u] = e1[u] = a.d;
  }
  bool ready = false;
  for (int w0 = threadIdx.x; w0 - (int)threadIdx.x < items; w0 += U * NT) {
    float p[U][PER][2][V], nw[U][PER][2][V];
    int h[U], rl[U];
#pragma unroll
    for (int x = 0; x < U; ++x) {
      const int w = w0 + NT * x, hr = w >> LS;
      rl[x] = RB == 1 ? 0 : hr / nh, h[x] = h0 + hr - rl[x] * nh;
      const size_t xb = (size_t)(r0 + rl[x]) * a.ldx + (size_t)h[x] * a.hsx;
#pragma unroll
      for (int u = 0; u < PER; ++u)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int e = b ? e1[u] : e0[u];
#pragma unroll
          for (int v = 0; v < V; ++v) p[x][u][b][v] = 0.f, nw[x][u][b][v] = 1.f;
          if (w < items && e < a.d) {
            ld_x<B16, V>(a.x, xb + e, p[x][u][b]);
            if (a.nw) ld_x<false, V>(a.nw, h[x] * a.ldn + e, nw[x][u][b]);
          }
        }
    }
    if (!ready) {
      // behind the first loads, which are on their way meanwhile
      for (int t = threadIdx.x; t < nr * half; t += NT) {
        const int tr = RB == 1 ? 0 : t / half;
        double turns = (double)a.pos[r0 + tr] * (double)a.freq[t - tr * half] * 0.15915494309189533577;
        turns -= rint(turns);
        float sn, cn;
        sincospif(2.f * (float)turns, &sn, &cn);
        cs[t] = make_float2(a.mscale * cn, a.mscale * sn);
      }
      __syncthreads();
      ready = true;
    }
#pragma unroll
    for (int x = 0; x < U; ++x) {
      if (a.nw) {
        float ss = 0.f;
#pragma unroll
        for (int u = 0; u < PER; ++u)
#pragma unroll
          for (int v = 0; v < V; ++v) ss += p[x][u][0][v] * p[x][u][0][v] + p[x][u][1][v] * p[x][u][1][v];
        const float inv = rsqrtf(head_sum(ss, 1 << LS) / (float)a.d + a.eps);
#pragma unroll
        for (int u = 0; u < PER; ++u)
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int v = 0; v < V; ++v) p[x][u][b][v] *= inv * nw[x][u][b][v];
      }
      if (w0 + NT * x >= items) continue;
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        if (e0[u] >= a.d) continue;
        const float2* c = cs + rl[x] * half;
        auto turn = [](float& m, float& n, const float2& t) {
          const float y = m * t.x - n * t.y;
          n = n * t.x + m * t.y, m = y;
        };
        if (whole) {
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int e = b ? e1[u] : e0[u];
            if (e >= a.rot) continue;
#pragma unroll
            for (int v = 0; v < V; v += 2) turn(p[x][u][b][v], p[x][u][b][(v + 1) % V], c[(e + v) >> 1]);
          }
        } else if (e0[u] < a.rot) {
#pragma unroll
          for (int v = 0; v < V; ++v) turn(p[x][u][0][v], p[x][u][1][v], c[V == 1 && a.pairs ? e0[u] >> 1 : e0[u] + v]);
        }
        st_y<V>(a, (size_t)(r0 + rl[x]), h[x] * a.d + e0[u], p[x][u][0]);
        if (e1[u] < a.d) st_y<V>(a, (size_t)(r0 + rl[x]), h[x] * a.d + e1[u], p[x][u][1]);
      }
    }
  }
}

template <bool B16>
int rope(const Rope& a, int ldx, int hsx, int ldn, int ldy, int ldb, hipStream_t st) {
  const long long n = (long long)a.heads * a.d;
  if (a.rows < 0 || a.rows > 1 << 23 || a.heads < 1 || a.heads > 4096 || a.d < 1 || a.d > 512 || a.rot < 0 || a.rot > a.d || a.rot % 2 || a.pairs < 0 || a.pairs > 1) return -1;
  if (hsx < a.d || ldx < (long long)(a.heads - 1) * hsx + a.d || (a.nw && ldn != 0 && ldn < a.d) || (a.y && ldy < n) || (a.yb && ldb < n)) return -1;
  if (a.rows == 0) return 0;  // before the buffers: an empty one may have no address
  if ((!a.y && !a.yb) || (a.rot && (!a.pos || !a.freq)) || !a.x) return -1;
  auto al = [](const void* p, uintptr_t m) { return ((uintptr_t)p & (m - 1)) == 0; };
  const bool vec = a.d % 4 == 0 && a.rot % (a.pairs ? 4 : 8) == 0 && al(a.x, B16 ? 8 : 16) && ldx % 4 == 0 && hsx % 4 == 0 && al(a.nw, 16) && ldn % 4 == 0 &&
                   (!a.y || (al(a.y, 16) && ldy % 4 == 0)) && (!a.yb || (al(a.yb, 8) && ldb % 4 == 0));
  const int V = vec ? 4 : 1, units = vec && a.pairs ? (a.d + 7) / 8 : (a.rot >> 1) / V + (a.d - a.rot + 2 * V - 1) / (2 * V);
  int LS = 0;
  while ((1 << LS) < units && LS < 6) ++LS;
  const int per_row = a.heads << LS, RB = per_row >= NT ? 1 : NT / per_row;
  // rows that do not fill the card share their heads out to several blocks: 67 rows of 39 heads of 219 4.3 us (15.4 with a block a row), one of 40
  // heads of 256 3.8 (6.2)
  const int loops = (per_row + NT - 1) / NT, U = vec && loops > 1 ? 2 : 1, room = a.rows < 2048 ? 2048 / a.rows : 1, most = (loops + U - 1) / U;
  const dim3 g((unsigned)(((long long)a.rows + RB - 1) / RB), most < room ? most : room), b(NT);
  const size_t lds = (size_t)RB * (a.rot >> 1) * sizeof(float2);
  if (U == 2) hipLaunchKernelGGL((k_rope<B16, 4, 1, 2>), g, b, lds, st, a, LS, RB);
  else if (vec) hipLaunchKernelGGL((k_rope<B16, 4, 1, 1>), g, b, lds, st, a, LS, RB);
  else if (units <= 1 << LS) hipLaunchKernelGGL((k_rope<B16, 1, 1, 1>), g, b, lds, st, a, LS, RB);
  else hipLaunchKernelGGL((k_rope<B16, 1, 4, 1>), g, b, lds, st, a, LS, RB);
  return 0;
}

Rope rope_args(const void* x, int ldx, int hsx, const float* nw, int ldn, float eps, const int* pos, const float* freq, float mscale, int pairs,
               float* y, int ldy, uint16_t* yb, int ldb, int rows, int heads, int d, int rot) {
  auto ld = [](int v) { return v < 0 ? (size_t)0 : (size_t)v; };
  return Rope{x, nw, pos, freq, y, yb, ld(ldx), ld(hsx), ld(ldn), ld(ldy), ld(ldb), eps, mscale, rows, heads, d, rot, pairs};
}

}  // namespace

API int dr_rope(const float* x, int ldx, int hsx, const float* nw, int ldn, float eps, const int* pos, const float* freq, float mscale, int layout,
                float* y, int ldy, uint16_t* yb, int ldb, int rows, int heads, int d, int rot, hipStream_t st) {
  return rope<false>(rope_args(x, ldx, hsx, nw, ldn, eps, pos, freq, mscale, layout, y, ldy, yb, ldb, rows, heads, d, rot), ldx, hsx, ldn, ldy, ldb, st);
}

API int dr_rope_bf16(const uint16_t* x, int ldx, int hsx, const float* nw, int ldn, float eps, const int* pos, const float* freq, float mscale, int layout,
                     float* y, int ldy, uint16_t* yb, int ldb, int rows, int heads, int d, int rot, hipStream_t st) {
  return rope<true>(rope_args(x, ldx, hsx, nw, ldn, eps, pos, freq, mscale, layout, y, ldy, yb, ldb, rows, heads, d, rot), ldx, hsx, ldn, ldy, ldb, st);
}
