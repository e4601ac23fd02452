// Tokens into and out of the cache in 8 bits (layout: kv8.hpp).
//
// One owner (a block of threads, or a wave where few tokens come) takes one head's k or v of one cached block: the call's tokens of that block go
// into registers, their largest magnitude A is reduced, and round(x / s) is stored.  With the block's first token in the call s = fl(A / 127);
// otherwise s is the block's scale, doubled until A <= 127 s, and where it grew by 2^j the block's earlier integers become round(q / 2^j).
// Growth by powers of two bounds what repeated rounding adds: every earlier rounding is worth at most half of the next one's step, so an element
// is never off by a whole step of the block's present scale, however often single tokens made it grow.  Integers are exact roundings of the
// quotient (half to even): |x - q s| below half a step says that q = round(x / s), and one fma compares it without an error that counts.
//
// Nothing is read or written twice, so memory bounds the large calls and a chain of loads (where a sequence's rows are, the table, the scale)
// the small ones.  Kernels alone: 4844 rows of 4 heads of 128 in fp32, 9 sequences: 9.9 us into the cache (2.5 TB/s of rows and bytes; 2.7 us
// more with every integer by quant()) and 7.8 us out of it (3.2 TB/s); 63 sequences with one token of 8 heads of 128 in bf16 5.9 us,
// their last blocks out 8.5 us; one token 3.7 us.
#include "kv8.hpp"

using namespace drm;

namespace {

constexpr int NT = 512;
constexpr int UNITS = 1024 / NT;  // of 4 tokens x 4 elements a thread: 64 tokens of up to 256 elements

struct Append {
  Kv8 c;
  const void *k, *v;
  size_t ldk, ldv;
};

// Unit n of a block (16 d / 4 of them) is four dwords of it.  k: elements e .. e + 3 of tokens t + 16 i, a dword a token; v: tokens t .. t + 3 of
// elements e + i, a dword an element.  Either way a wave's dwords lie beside each other in runs of 64 bytes or more, and the 16-byte pieces
// of the rows outside in runs of 64.
struct Unit {
  int t, e;
  size_t at[4];  // of the dwords in the block
};
DEV Unit unit_of(bool isv, int n) {
  Unit u;
  if (isv) {
    const int m = n & 15;  // dword of a row: tokens 16 (m & 3) + 4 (m >> 2) ..
    u.t = 16 * (m & 3) + 4 * (m >> 2), u.e = n >> 4 << 2;
#pragma unroll
    for (int i = 0; i < 4; ++i) u.at[i] = (size_t)(u.e + i) * KB + 4 * m;
  } else {
    u.t = n >> 2 & 15, u.e = (n >> 6) * 16 + 4 * (n & 3);
#pragma unroll
    for (int i = 0; i < 4; ++i) u.at[i] = ((size_t)(n >> 6) * KB + u.t + 16 * i) * 16 + 4 * (n & 3);
  }
  return u;
}
DEV int token_of(bool isv, const Unit& u, int i) { return isv ? u.t + i : u.t + 16 * i; }

template <bool B16>
DEV float4 ld4_elems(const void* p, size_t at) {
  if constexpr (B16) {
    const uint2 w = ld8(reinterpret_cast<const uint16_t*>(p) + at);
    return make_float4(bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y));
  } else {
    return ldf4(reinterpret_cast<const float*>(p) + at);
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

// A block's scale s with tokens of largest magnitude `top` (infinity: some are no numbers) in it, 2^grow times s_old; first: its first token is
// among them.
struct Scale {
  float s, lift, sl, inv;
  int grow;
  bool none;
  DEV uint32_t byte(float v) const { return (uint32_t)((none ? 0 : quant(v * lift, sl, inv)) + 128); }
  // Four bytes by the reciprocal alone, and in `off` the largest distance of an element to its integer's value: right where that is
  // below half a step (and never past 127, but for scales that are subnormal or no numbers).
  DEV uint32_t guess(float a, float b, float c, float e, float& off) const {
    uint32_t w = 0;
    const float v[4] = {a, b, c, e};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float q = rintf(v[k] * inv);
      off = fmaxf(off, fabsf(__builtin_fmaf(-q, s, v[k])));
      w = __builtin_amdgcn_cvt_pk_u8_f32(q + 128.f, k, w);
    }
    return w;
  }
  DEV bool sure(float off) const { return lift == 1.f && !none && off < 0.5f * s; }
  DEV uint32_t exact(float a, float b, float c, float e) const { return byte(a) | byte(b) << 8 | byte(c) << 16 | byte(e) << 24; }
};
DEV Scale scale_of(float top, float s_old, bool first) {
  Scale q;
  q.grow = 0;
  if (!(top < __builtin_inff()) || (!first && !(s_old < __builtin_inff()))) {
    q.s = __builtin_nanf("");  // the block stands for no numbers
  } else if (first || s_old == 0.f) {
    q.s = top / 127.f;  // rounded correctly
  } else {
    // 127 s_old and the comparisons are exact in 64 bits
    const double most = 127.0 * (double)s_old;
    if ((double)top > most) {
      int e;
      const double m = frexp((double)top / most, &e);
      q.grow = m == 0.5 ? e - 1 : e;
    }
    q.s = __builtin_ldexpf(s_old, q.grow);
  }
  // tiny scales are lifted by a power of two, so that their reciprocal is a normal number
  q.none = !(q.s > 0.f);
  q.lift = q.s < 0x1p-90f ? 0x1p90f : 1.f, q.sl = q.s * q.lift, q.inv = q.none ? 0.f : 1.f / q.sl;
  return q;
}
DEV bool finite4(const float4& v) {
  return fabsf(v.x) < __builtin_inff() && fabsf(v.y) < __builtin_inff() && fabsf(v.z) < __builtin_inff() && fabsf(v.w) < __builtin_inff();
}
DEV float top4(const float4& v) { return fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))); }

// A few tokens a sequence (decode steps): a wave owns a head's k or v of a block, a lane four elements of each token; tokens past the fourth
// are loaded again.  Bound by its chain of loads (sequence, rows beside the table, scale): 3.7 us for one
// token and 5.9 us for 63 sequences with one of 8 heads of 128, where k_kv8_append takes 7.4 and 13.9.
template <bool B16>
__global__ void __launch_bounds__(256) k_kv8_append_few(Append a) {
  int at = blockIdx.x;
  Seq s;
  const int i = find_item(a.c, at, s, seq_blocks);
  const int y = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(wave_id());
  if (i < 0 || y >= 2 * a.c.hkv) return;
  const int b = (s.first >> 6) + at, h = y >> 1, d = a.c.d, l = lane_id(), e = 4 * l;
  const bool isv = y & 1, on = e < d;
  const int t0 = s.first > b * KB ? s.first - b * KB : 0, t1 = s.len - b * KB < KB ? s.len - b * KB : KB;
  const size_t ld = isv ? a.ldv : a.ldk, r = ((size_t)s.r0 + (b * KB + t0 - s.first)) * ld + (size_t)h * d + e;
  const void* src = isv ? a.v : a.k;
  float4 x[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (on && t0 + k < t1) x[k] = ld4_elems<B16>(src, r + k * ld);
  }
  const int page = page_of(a.c, i, b);
  if (page < 0) return;
  const size_t ph = (size_t)page * a.c.hkv + h;
  uint8_t* blk = (isv ? a.c.vq : a.c.kq) + ph * KB * d;
  float* scale = (isv ? a.c.vs : a.c.ks) + ph;
  const float s_old = *scale;
  float top = 0.f;
  bool fine = true;
#pragma unroll
  for (int k = 0; k < 4; ++k) top = fmaxf(top, top4(x[k])), fine = fine && finite4(x[k]);
  for (int t = t0 + 4; t < t1; ++t) {
    if (!on) continue;
    const float4 v = ld4_elems<B16>(src, r + (t - t0) * ld);
    top = fmaxf(top, top4(v)), fine = fine && finite4(v);
  }
  top = wave_max(fine ? top : __builtin_inff());
  const Scale q = scale_of(top, s_old, t0 == 0);
  if (q.grow && t0 > 0) {
    // 16 bytes are 16 elements of a token (k: the lane's token), or of an element 16 tokens, new ones among them that are written below
    for (int n = l; n < 4 * d; n += WAVE) {
      if (!isv && (n & (KB - 1)) >= t0) continue;
      uint4* p = reinterpret_cast<uint4*>(blk) + n;
      uint4 o = *p;
      o.x = shrink4(o.x, q.grow), o.y = shrink4(o.y, q.grow), o.z = shrink4(o.z, q.grow), o.w = shrink4(o.w, q.grow);
      *p = o;
    }
    // the new tokens' bytes come from other lanes than these
    __builtin_amdgcn_s_waitcnt(0);
  }
  auto put = [&](int t, const float4& v) {
    const uint32_t w = q.exact(v.x, v.y, v.z, v.w);
    if (isv) {
      uint8_t* p = blk + (size_t)e * KB + 16 * (t >> 2 & 3) + 4 * (t >> 4) + (t & 3);
      p[0] = (uint8_t)w, p[KB] = (uint8_t)(w >> 8), p[2 * KB] = (uint8_t)(w >> 16), p[3 * KB] = (uint8_t)(w >> 24);
    } else {
      *reinterpret_cast<uint32_t*>(blk + ((size_t)(e >> 4) * KB + t) * 16 + (e & 15)) = w;
    }
  };
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (on && t0 + k < t1) put(t0 + k, x[k]);
  for (int t = t0 + 4; t < t1; ++t)
    if (on) put(t, ld4_elems<B16>(src, r + (t - t0) * ld));
  if (l == 0) *scale = q.s;
}

// Many tokens a sequence: a block of threads owns a head's k or v of a block, and a thread loads all of its rows' pieces before it needs the
// first.  512 threads hold 64 tokens of 256 elements in 32 registers each; 256 took 12.4 us where these take 10.9.
template <bool B16>
__global__ void __launch_bounds__(NT) k_kv8_append(Append a) {
  constexpr int NW = NT / WAVE;
  __shared__ float red[NW + 1];
  int at = blockIdx.x;
  Seq s;
  const int i = find_item(a.c, at, s, seq_blocks);
  if (i < 0) return;
  const int b = (s.first >> 6) + at, h = blockIdx.y >> 1, d = a.c.d;
  const bool isv = blockIdx.y & 1;
  // the block's places [t0, t1) get rows r .. of the call
  const int t0 = s.first > b * KB ? s.first - b * KB : 0, t1 = s.len - b * KB < KB ? s.len - b * KB : KB;
  const size_t ld = isv ? a.ldv : a.ldk, r = ((size_t)s.r0 + (b * KB + t0 - s.first)) * ld + (size_t)h * d;
  const void* src = isv ? a.v : a.k;
  // the rows are on their way while the table says where they go
  float4 x[UNITS][4];
  Unit u[UNITS];
#pragma unroll
  for (int n = 0; n < UNITS; ++n) {
    u[n] = unit_of(isv, threadIdx.x + NT * n);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int t = token_of(isv, u[n], k);
      x[n][k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (u[n].e < d && t >= t0 && t < t1) x[n][k] = ld4_elems<B16>(src, r + (size_t)(t - t0) * ld + u[n].e);
    }
  }
  const int page = page_of(a.c, i, b);
  if (page < 0) return;
  const size_t ph = (size_t)page * a.c.hkv + h;
  uint8_t* blk = (isv ? a.c.vq : a.c.kq) + ph * KB * d;
  float* scale = (isv ? a.c.vs : a.c.ks) + ph;
  if (threadIdx.x == 0) red[NW] = *scale;  // read by the thread that writes it
  float top = 0.f;
  bool fine = true;
#pragma unroll
  for (int n = 0; n < UNITS; ++n)
#pragma unroll
    for (int k = 0; k < 4; ++k) top = fmaxf(top, top4(x[n][k])), fine = fine && finite4(x[n][k]);
  top = wave_max(fine ? top : __builtin_inff());  // an infinity or NaN among them: infinity
  if (lane_id() == 0) red[wave_id()] = top;
  __syncthreads();
  top = red[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) top = fmaxf(top, red[w]);
  const float s_old = red[NW];

  const Scale q = scale_of(top, s_old, t0 == 0);
  const int grow = q.grow;
  // dword o of the block: those of its bytes that `now` says are new
  auto put = [&](size_t o, uint32_t w, int now, bool old) {
    if (now == 15) {
      *reinterpret_cast<uint32_t*>(blk + o) = w;
    } else if (grow && old) {
      // places that keep what they held are rewritten only where the scale grew
      uint32_t p = shrink4(*reinterpret_cast<const uint32_t*>(blk + o), grow);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (now >> k & 1) p = (p & ~(255u << 8 * k)) | (w & (255u << 8 * k));
      *reinterpret_cast<uint32_t*>(blk + o) = p;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (now >> k & 1) blk[o + k] = (uint8_t)(w >> 8 * k);
    }
  };
#pragma unroll
  for (int n = 0; n < UNITS; ++n) {
    if (u[n].e >= d) break;
    const float* f = reinterpret_cast<const float*>(x[n]);
    // dword k is elements of token k, or tokens of element k
    uint32_t w[4];
    float off = 0.f;
    auto all = [&](auto how) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        w[k] = isv ? how(f[k], f[4 + k], f[8 + k], f[12 + k]) : how(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3]);
    };
    all([&](float a, float b, float c, float e) { return q.guess(a, b, c, e, off); });
    if (!q.sure(off)) all([&](float a, float b, float c, float e) { return q.exact(a, b, c, e); });
    if (isv) {
      int now = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) now |= (int)(u[n].t + k >= t0 && u[n].t + k < t1) << k;
      if (!now && !(grow && u[n].t < t0)) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) put(u[n].at[e], w[e], now, u[n].t < t0);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int t = u[n].t + 16 * k;
        if (t < t1 && (t >= t0 || grow)) put(u[n].at[k], w[k], t >= t0 ? 15 : 0, t < t0);
      }
    }
  }
  if (threadIdx.x == 0) *scale = q.s;
}

struct Read {
  Kv8 c;
  float *k, *v;
  size_t ldk, ldv;
};

// Out of the cache: the reverse, each thread's dwords loaded together.  512 threads are as fast (within 0.5 us either way).
constexpr int RT = 256;
__global__ void __launch_bounds__(RT) k_kv8_read(Read a) {
  int at = blockIdx.x;
  Seq s;
  const int i = find_item(a.c, at, s, seq_blocks);
  if (i < 0) return;
  const int b = (s.first >> 6) + at, page = page_of(a.c, i, b), h = blockIdx.y >> 1, d = a.c.d;
  const bool isv = blockIdx.y & 1;
  const int t0 = s.first > b * KB ? s.first - b * KB : 0, t1 = s.len - b * KB < KB ? s.len - b * KB : KB;
  const size_t ld = isv ? a.ldv : a.ldk;
  float* dst = (isv ? a.v : a.k) + ((size_t)s.r0 + (b * KB + t0 - s.first)) * ld + (size_t)h * d;
  const size_t ph = (size_t)(page < 0 ? 0 : page) * a.c.hkv + h;
  const uint8_t* blk = (isv ? a.c.vq : a.c.kq) + ph * KB * d;
  const float sc = (isv ? a.c.vs : a.c.ks)[ph];
#pragma unroll
  for (int n = 0; n < 1024 / RT; ++n) {
    const Unit u = unit_of(isv, threadIdx.x + RT * n);
    if (u.e >= d) break;
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = ld4(blk + u.at[k]);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int t = token_of(isv, u, k);
      if (t < t0 || t >= t1) continue;
      float o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int q = (int)(isv ? w[e] >> 8 * k : w[k] >> 8 * e) & 255;
        o[e] = page < 0 ? 0.f : sc * (float)(q - 128);
      }
      *reinterpret_cast<float4*>(dst + (size_t)(t - t0) * ld + u.e) = make_float4(o[0], o[1], o[2], o[3]);
    }
  }
}

template <bool B16>
int append(const Append& a, int ldk, int ldv, hipStream_t st) {
  const int n = a.c.hkv * a.c.d, per = B16 ? 8 : 4;
  if (!kv8_ok(a.c) || ldk < n || ldv < n || ldk % per || ldv % per) return -1;
  if (a.c.rows == 0 || a.c.seqs == 0) return 0;
  if (!kv8_buffers_ok(a.c) || !a.k || !a.v || ((uintptr_t)a.k & 15) || ((uintptr_t)a.v & 15)) return -1;
  const unsigned nb = (unsigned)max_blocks(a.c.rows, a.c.seqs);
  // A wave walks four rows at a time: more than four a sequence are left to a block of threads.  Kernels alone, us, a wave and (a block of threads), 8 heads of
  // 128 in bf16: 64 tokens of as many sequences 4.5 (12.8), 32 x 4 5.7 (11.5), 32 x 6 7.2 (11.6), 1 x 5 5.8 (7.8), 1 x 20 14.6 (7.3); 2 heads of 256 in fp32: 32 x 4 5.1
  // (6.4), 32 x 6 7.0 (6.6), 16 x 8 8.7 (6.5).  The rule knows the average alone: a prompt of 512 rows beside 63 single tokens takes a block of threads, 15.4
  // (53), beside 200 a wave, 56 (44; 2 heads of 256 60, 16), where a choice by each block of the cache would take both.
  if (a.c.rows <= 4ll * a.c.seqs) hipLaunchKernelGGL((k_kv8_append_few<B16>), dim3(nb, (2 * a.c.hkv + 3) / 4), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_kv8_append<B16>), dim3(nb, 2 * a.c.hkv), dim3(NT), 0, st, a);
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
  hipLaunchKernelGGL(k_kv8_read, dim3((unsigned)max_blocks(rows, seqs), 2 * hkv), dim3(RT), 0, st, a);
  return 0;
}
