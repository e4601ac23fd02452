// The cache of dr_kv8_append, dr_kv8_read and dr_attn_kv8, and the rows and sequences of a call over it.
//
// A cache holds blocks of 64 tokens of one sequence, each with its k and v of every cached head as integers q in -127 .. 127
// (stored as q + 128) and one f32 scale a block and head; which page of the cache holds block b of sequence i is table[i maxp + b].
//   kq [pages, hkv, d / 16, 64, 16]: 16 elements of a token are one 16-byte load, the same 16 of neighbouring tokens lie beside each
//     other, so a wave's load of 16 tokens (rows of an MFMA operand) x 64 elements is four runs of 256 bytes;
//   vq [pages, hkv, d, 64]: token 16 a + 4 b + c of an element at byte 16 b + 4 a + c.  The MFMA that sums over tokens takes
//     from lane quad b the tokens 16 a + 4 b + (0 .. 3), those whose scores the same lane holds, so a lane's 16 bytes are its
//     tokens of the whole block and the weights go from one product to the other without leaving their registers.
#pragma once
#include "common.hpp"

namespace drm {

constexpr int KB = 64;  // tokens of a block: the header's DR_KV8_BLOCK

struct Kv8 {
  const int *start, *len, *table;
  int maxp;
  uint8_t* kq;
  float* ks;
  uint8_t* vq;
  float* vs;
  int pages, rows, seqs, hkv, d;
};

// What every call over a cache refuses.
inline bool kv8_ok(const Kv8& a) {
  return a.rows >= 0 && a.rows <= (1 << 20) && a.seqs >= 0 && a.seqs <= (1 << 20) && a.hkv >= 1 && a.hkv <= 1024 && a.d >= 16 && a.d <= 256 &&
         a.d % 16 == 0 && a.maxp >= 1 && a.maxp < (1 << 25) && a.pages >= 1;
}
inline bool kv8_buffers_ok(const Kv8& a) {
  return a.start && a.len && a.table && a.kq && a.ks && a.vq && a.vs && !((uintptr_t)a.kq & 15) && !((uintptr_t)a.vq & 15);
}

// Sequence i of a call: its rows [r0, r0 + n) (inside the call's rows whatever start holds), the position of the first of them,
// and its tokens.
struct Seq {
  int r0, n, first, len;
};
DEV Seq seq_of(const Kv8& a, int i) {
  const int s0 = a.start[i], s1 = a.start[i + 1], len = a.len[i] > 0 ? a.len[i] : 0;
  const int r0 = s0 < 0 ? 0 : s0 > a.rows ? a.rows : s0, r1 = s1 < r0 ? r0 : s1 > a.rows ? a.rows : s1;
  return Seq{r0, r1 - r0, len - (r1 - r0), len};
}

// The page of block b of sequence i, -1 where the table has none.
DEV int page_of(const Kv8& a, int i, int b) {
  if (b < 0 || b >= a.maxp) return -1;
  const int p = a.table[(size_t)i * a.maxp + b];
  return p >= 0 && p < a.pages ? p : -1;
}

// Item `at` of the items of all sequences in order, count(sequence) of each: its sequence (s: what seq_of gives for it), and its number there in
// `at`; -1 where there are fewer.  64 sequences a step, all lanes of the wave together.
template <class Count>
DEV int find_item(const Kv8& a, int& at, Seq& s, Count count) {
  const int l = lane_id();
  for (int i0 = 0; i0 < a.seqs; i0 += WAVE) {
    Seq q{0, 0, 0, 0};
    if (i0 + l < a.seqs) q = seq_of(a, i0 + l);
    const int c = i0 + l < a.seqs ? count(q) : 0;
    int n = c;
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
      const int t = __shfl_up(n, o);
      n += l >= o ? t : 0;
    }
    const unsigned long long behind = __ballot(n > at);
    if (behind) {
      const int w = __builtin_ctzll(behind);
      at -= __builtin_amdgcn_readlane(n - c, w);
      s = Seq{__builtin_amdgcn_readlane(q.r0, w), __builtin_amdgcn_readlane(q.n, w), __builtin_amdgcn_readlane(q.first, w),
              __builtin_amdgcn_readlane(q.len, w)};
      return i0 + w;
    }
    at -= __builtin_amdgcn_readlane(n, WAVE - 1);
  }
  return -1;
}

// The blocks that the rows of a sequence lie in, the negative ones of rows before its first token among them.
DEV int seq_blocks(const Seq& s) { return s.n ? ((s.len - 1) >> 6) - (s.first >> 6) + 1 : 0; }
// An upper bound of their number over all sequences.
inline long long max_blocks(int rows, int seqs) {
  const long long m = rows / KB + 2ll * seqs;
  return m < rows ? m : rows;
}

}  // namespace drm
