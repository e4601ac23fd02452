// Tokens into and out of the cache in 8 bits (layout: kv8.hpp).
//
// A block of threads owns one head's k or v of one cached block: it takes the call's tokens of that block into registers, reduces their largest
// magnitude A, and stores round(x / s).  With the block's first token in the call s = fl(A / 127); otherwise s is the
// block's scale, doubled until A <= 127 s, and where it grew by 2^j the block's earlier integers become round(q / 2^j).  Growth by
// powers of two bounds what repeated rounding adds: every earlier rounding is worth at most half of the next one's step, so an element is
// never off by a whole step of the block's present scale, however often single tokens made it grow.  Integers are exact roundings of
// the quotient (half to even): x - q s needs at most 24 bits where q is next to x / s, so one fma tells on which side x lies.
#include "kv8.hpp"

using namespace drm;

namespace {

constexpr int NT = 256;
constexpr int VROW = KB + 16;  // LDS row of v's 64 bytes: 16-byte pieces, four banks further each row

struct Append {
  Kv8 c;
  const void *k, *v;
  size_t ldk, ldv;
};

template <bool B16>
DEV void ld_elems(const void* p, size_t at, float (&o)[16]) {
  if constexpr (B16) {
    const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + at);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint4 w = ld16(q + i);
      const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) o[8 * i + 2 * e] = bf16_lo(ww[e]), o[8 * i + 2 * e + 1] = bf16_hi(ww[e]);
    }
  } else {
    const float* q = reinterpret_cast<const float*>(p) + at;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 w = ldf4(q + 4 * i);
      o[4 * i] = w.x, o[4 * i + 1] = w.y, o[4 * i + 2] = w.z, o[4 * i + 3] = w.w;
    }
  }
}

// round(x / s), half to even; inv is 1 / s within a few ulp, |x| <= 127 s (1 + 2^-23)
DEV int quant(float x, float s, float inv) {
  float q = rintf(x * inv);
  const float r = __builtin_fmaf(-q, s, x), h = 0.5f * s;
  const bool odd = (int)q & 1;
  if (r > h || (r == h && odd)) q += 1.f;
  if (r < -h || (r == -h && odd)) q -= 1.f;
  return (int)fminf(fmaxf(q, -127.f), 127.f);
}

// round(q / 2^j), half to even
DEV int shrink(int q, int j) {
  return (int)rintf(__builtin_ldexpf((float)q, -j));
}

// the four stored bytes of w shrunk
DEV uint32_t shrink4(uint32_t w, int j) {
  uint32_t o = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) o |= (uint32_t)(shrink((int)((w >> (8 * e)) & 255) - 128, j) + 128) << (8 * e);
  return o;
}

DEV int v_at(int t) { return 16 * ((t >> 2) & 3) + 4 * (t >> 4) + (t & 3); }

template <bool B16>
__global__ void __launch_bounds__(NT) k_kv8_append(Append a) {
  __shared__ float red[NT / WAVE + 1];
  __shared__ __align__(16) uint8_t vt[256 * VROW];
  int at = blockIdx.x;
  const int i = find_item(a.c, at, seq_blocks);
  if (i < 0) return;
  const Seq s = seq_of(a.c, i);
  const int b = (s.first >> 6) + at, page = page_of(a.c, i, b);
  if (page < 0) return;
  const int h = blockIdx.y >> 1, d = a.c.d, d16 = d >> 4;
  const bool isv = blockIdx.y & 1;
  // the block's places [t0, t1) get rows r .. of the call
  const int t0 = s.first > b * KB ? s.first - b * KB : 0, t1 = s.len - b * KB < KB ? s.len - b * KB : KB;
  const size_t r = (size_t)s.r0 + (b * KB + t0 - s.first), ld = isv ? a.ldv : a.ldk;
  const void* src = isv ? a.v : a.k;
  const size_t ph = (size_t)page * a.c.hkv + h;
  uint8_t* blk = (isv ? a.c.vq : a.c.kq) + ph * KB * d;
  float* scale = (isv ? a.c.vs : a.c.ks) + ph;
  if (threadIdx.x == 0) red[NT / WAVE] = *scale;  // read by the thread that writes it
  const int units = (t1 - t0) * d16;
  float x[4][16];
  float top = 0.f;
  bool fine = true;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int w = threadIdx.x + NT * u;
    if (w >= units) break;
    const int t = w / d16, c = w - t * d16;
    ld_elems<B16>(src, (r + t) * ld + (size_t)h * d + 16 * c, x[u]);
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    if ((int)threadIdx.x + NT * u >= units) break;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      top = fmaxf(top, fabsf(x[u][e]));
      fine = fine && fabsf(x[u][e]) < __builtin_inff();
    }
  }
  top = wave_max(fine ? top : __builtin_inff());  // an infinity or NaN among them: infinity
  if (lane_id() == 0) red[wave_id()] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float s_old = red[NT / WAVE];

  const bool fresh = t0 == 0 || s_old == 0.f;
  float sc;
  int grow = 0;
  if (!(top < __builtin_inff()) || (t0 > 0 && !(s_old < __builtin_inff()))) {
    sc = __builtin_nanf("");  // the block stands for no numbers
  } else if (fresh) {
    sc = (float)((double)top / 127.0);
  } else {
    const double ratio = (double)top / (127.0 * (double)s_old);
    if (ratio > 1.0) {
      int e;
      const double m = frexp(ratio, &e);
      grow = m == 0.5 ? e - 1 : e;
    }
    sc = __builtin_ldexpf(s_old, grow);
  }
  // tiny scales are lifted by a power of two, so that their reciprocal is a normal number
  const bool none = !(sc > 0.f);
  const float lift = sc < 0x1p-90f ? 0x1p90f : 1.f, sl = sc * lift, inv = none ? 0.f : 1.f / sl;
  // places that keep what they held are rewritten only where the scale grew
  const bool keep = t0 > 0 && grow > 0;
  if (!isv) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int w = threadIdx.x + NT * u;
      if (w >= units) break;
      const int t = w / d16, c = w - t * d16;
      uint32_t o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[e] = 0;
#pragma unroll
        for (int f = 0; f < 4; ++f) o[e] |= (uint32_t)((none ? 0 : quant(x[u][4 * e + f] * lift, sl, inv)) + 128) << (8 * f);
      }
      *reinterpret_cast<uint4*>(blk + ((size_t)c * KB + t0 + t) * 16) = make_uint4(o[0], o[1], o[2], o[3]);
    }
    if (keep)
      for (int w = threadIdx.x; w < t0 * d16; w += NT) {
        uint4* p = reinterpret_cast<uint4*>(blk + ((size_t)(w / t0) * KB + w % t0) * 16);
        uint4 o = *p;
        o.x = shrink4(o.x, grow), o.y = shrink4(o.y, grow), o.z = shrink4(o.z, grow), o.w = shrink4(o.w, grow);
        *p = o;
      }
  } else {
    // whole rows where every place is written or the call began the block, the new bytes alone otherwise
    const bool rows = keep || t0 == 0;
    if (rows && (keep || t1 < KB)) {
      for (int w = threadIdx.x; w < d * 4; w += NT) {
        uint4 o = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
        if (keep) {
          o = *reinterpret_cast<const uint4*>(blk + (size_t)w * 16);
          o.x = shrink4(o.x, grow), o.y = shrink4(o.y, grow), o.z = shrink4(o.z, grow), o.w = shrink4(o.w, grow);
        }
        *reinterpret_cast<uint4*>(vt + (w >> 2) * VROW + (w & 3) * 16) = o;
      }
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int w = threadIdx.x + NT * u;
      if (w >= units) break;
      const int t = w / d16, c = w - t * d16, p = v_at(t0 + t);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint8_t q = (uint8_t)((none ? 0 : quant(x[u][e] * lift, sl, inv)) + 128);
        if (rows) vt[(16 * c + e) * VROW + p] = q;
        else blk[(size_t)(16 * c + e) * KB + p] = q;
      }
    }
    if (rows) {
      __syncthreads();
      for (int w = threadIdx.x; w < d * 4; w += NT)
        *reinterpret_cast<uint4*>(blk + (size_t)w * 16) = *reinterpret_cast<const uint4*>(vt + (w >> 2) * VROW + (w & 3) * 16);
    }
  }
  if (threadIdx.x == 0) *scale = sc;
}

struct Read {
  Kv8 c;
  float *k, *v;
  size_t ldk, ldv;
};

__global__ void __launch_bounds__(NT) k_kv8_read(Read a) {
  __shared__ __align__(16) uint8_t vt[256 * VROW];
  int at = blockIdx.x;
  const int i = find_item(a.c, at, seq_blocks);
  if (i < 0) return;
  const Seq s = seq_of(a.c, i);
  const int b = (s.first >> 6) + at, page = page_of(a.c, i, b);
  const int h = blockIdx.y >> 1, d = a.c.d;
  const bool isv = blockIdx.y & 1;
  const int t0 = s.first > b * KB ? s.first - b * KB : 0, t1 = s.len - b * KB < KB ? s.len - b * KB : KB;
  const size_t r = (size_t)s.r0 + (b * KB + t0 - s.first), ld = isv ? a.ldv : a.ldk;
  float* dst = (isv ? a.v : a.k) + r * ld + (size_t)h * d;
  const size_t ph = (size_t)(page < 0 ? 0 : page) * a.c.hkv + h;
  const uint8_t* blk = (isv ? a.c.vq : a.c.kq) + ph * KB * d;
  const float sc = page < 0 ? 0.f : (isv ? a.c.vs : a.c.ks)[ph];
  if (isv && page >= 0) {
    for (int w = threadIdx.x; w < d * 4; w += NT) *reinterpret_cast<uint4*>(vt + (w >> 2) * VROW + (w & 3) * 16) = ld16(blk + (size_t)w * 16);
    __syncthreads();
  }
  // four elements a thread, a token's elements beside each other
  const int d4 = d >> 2;
  for (int w = threadIdx.x; w < (t1 - t0) * d4; w += NT) {
    const int t = w / d4, e = 4 * (w - t * d4);
    uint32_t q = 0x80808080u;
    if (page >= 0) {
      if (isv) {
        const uint8_t* p = vt + e * VROW + v_at(t0 + t);
        q = p[0] | p[VROW] << 8 | p[2 * VROW] << 16 | (uint32_t)p[3 * VROW] << 24;
      } else {
        q = ld4(blk + ((size_t)(e >> 4) * KB + t0 + t) * 16 + (e & 15));
      }
    }
    float4 o;
    o.x = sc * (float)((int)(q & 255) - 128), o.y = sc * (float)((int)((q >> 8) & 255) - 128);
    o.z = sc * (float)((int)((q >> 16) & 255) - 128), o.w = sc * (float)((int)(q >> 24) - 128);
    *reinterpret_cast<float4*>(dst + t * ld + e) = o;
  }
}

template <bool B16>
int append(const Append& a, int ldk, int ldv, hipStream_t st) {
  const int n = a.c.hkv * a.c.d, per = B16 ? 8 : 4;
  if (!kv8_ok(a.c) || ldk < n || ldv < n || ldk % per || ldv % per) return -1;
  if (a.c.rows == 0 || a.c.seqs == 0) return 0;
  if (!kv8_buffers_ok(a.c) || !a.k || !a.v || ((uintptr_t)a.k & 15) || ((uintptr_t)a.v & 15)) return -1;
  hipLaunchKernelGGL((k_kv8_append<B16>), dim3((unsigned)max_blocks(a.c.rows, a.c.seqs), 2 * a.c.hkv), dim3(NT), 0, st, a);
  return 0;
}

Append append_args(const void* k, int ldk, const void* v, int ldv, const int* start, const int* len, const int* table, int maxp, uint8_t* kq, float* ks,
                   uint8_t* vq, float* vs, int pages, int rows, int seqs, int hkv, int d) {
  return Append{Kv8{start, len, table, maxp, kq, ks, vq, vs, pages, rows, seqs, hkv, d}, k, v, ldk < 0 ? 0 : (size_t)ldk, ldv < 0 ? 0 : (size_t)ldv};
}

}  // namespace

API int dr_kv8_append(const float* k, int ldk, const float* v, int ldv, const int* start, const int* len, const int* table, int maxp, uint8_t* kq,
                      float* ks, uint8_t* vq, float* vs, int pages, int rows, int seqs, int hkv, int d, hipStream_t st) {
  return append<false>(append_args(k, ldk, v, ldv, start, len, table, maxp, kq, ks, vq, vs, pages, rows, seqs, hkv, d), ldk, ldv, st);
}

API int dr_kv8_append_bf16(const uint16_t* k, int ldk, const uint16_t* v, int ldv, const int* start, const int* len, const int* table, int maxp,
                           uint8_t* kq, float* ks, uint8_t* vq, float* vs, int pages, int rows, int seqs, int hkv, int d, hipStream_t st) {
  return append<true>(append_args(k, ldk, v, ldv, start, len, table, maxp, kq, ks, vq, vs, pages, rows, seqs, hkv, d), ldk, ldv, st);
}

API int dr_kv8_read(const int* start, const int* len, const int* table, int maxp, const uint8_t* kq, const float* ks, const uint8_t* vq,
                    const float* vs, int pages, float* k, int ldk, float* v, int ldv, int rows, int seqs, int hkv, int d, hipStream_t st) {
  const Kv8 c{start, len, table, maxp, const_cast<uint8_t*>(kq), const_cast<float*>(ks), const_cast<uint8_t*>(vq), const_cast<float*>(vs),
              pages, rows, seqs, hkv, d};
  if (!kv8_ok(c) || ldk < hkv * d || ldv < hkv * d || ldk % 4 || ldv % 4) return -1;
  if (rows == 0 || seqs == 0) return 0;
  if (!kv8_buffers_ok(c) || !k || !v || ((uintptr_t)k & 15) || ((uintptr_t)v & 15)) return -1;
  const Read a{c, k, v, (size_t)ldk, (size_t)ldv};
  hipLaunchKernelGGL(k_kv8_read, dim3((unsigned)max_blocks(rows, seqs), 2 * hkv), dim3(NT), 0, st, a);
  return 0;
}
