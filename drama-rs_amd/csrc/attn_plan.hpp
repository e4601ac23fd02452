// How dr_attn_kv8 cuts a call into blocks of threads.  Host code alone, apart from the kernels, so that tests can ask which cut a call takes.
#pragma once
#include <initializer_list>

namespace drm {

constexpr int kPlanBlock = 64, kPlanWaves = 4;  // tokens of a cached block; waves of a block of threads with few columns
constexpr int kSplits = 128;                    // at most

// Rows of a part (part_of()).
inline int part_rows(int rows, int seqs, int max_rows) { return (long long)seqs * max_rows < rows ? seqs * max_rows : rows; }

// How a call is cut: by its sizes alone, so that the workspace is known before.
struct Plan {
  bool few, scan, fold;
  int mt, cols, nw, splits, chunk;
  long long tiles;
};
inline Plan plan(int rows, int seqs, int max_rows, int max_len, int hq, int hkv, int d) {
  Plan p;
  const long long g = hq / hkv, pairs = (max_rows < rows ? max_rows : rows) * g, blocks = ((long long)max_len + kPlanBlock - 1) / kPlanBlock, items = (long long)part_rows(rows, seqs, max_rows) * hq;
  // Few columns: each block of threads 16 or 32 pairs of a cached head and sequence.
  p.mt = pairs <= 16 || d > 128 ? 1 : 2;
  const long long cols = (pairs + 16 * p.mt - 1) / (16 * p.mt), room = rows * g / (16 * p.mt) + seqs, few = (cols * seqs < room ? cols * seqs : room) * hkv;
  // Many: tiles of 128 or 256 pairs; where sequences have several, of all rows together.  Eight waves only where a tile fills them and the tiles
  // most of the card (16 heads of 128, 2 cached; behind 8192 tokens 2800 rows 254 us with eight, 283 with four, 2100 215 and 203).
  auto cut = [&](int nw) {
    const long long tp = 32 * nw, per = (pairs + tp - 1) / tp, all = rows * g / tp + seqs;
    p.nw = nw, p.scan = per > 1, p.tiles = per > 1 && all < per * seqs ? all : per * seqs;
  };
  cut(8);
  if (d > 128 || pairs <= 128 || p.tiles * hkv < 176) cut(4);
  // us: rounds of the blocks that the card holds, each a start and its steps, `at` cached blocks a step; with splits a launch that joins, and the
  // parts out and back.  The constants are what single rounds took.  What the rule gives, and the other side:
  //   in few columns  3 sequences of 1000 tokens with 72 pairs of d 256 14.7 us (split tiles 26, whole ones 58), 8 of 500 with 192 pairs of d 64
  //                   9.1 (15.6), 7 of 33 to 373 with as many pairs of d 64 10.8 (13.2);
  //   in tiles        49 of 2000 with 122 pairs of d 128 25 (30), 12 of 420 to 3900 with 318 pairs of d 96 65 (94), 30 of 40 with 120 pairs of d 256
  //                   21 (32), 63 of 10 with 40 pairs of d 112 9.5 (15.7).
  struct Cut {
    long long s;
    float us;
  };
  const float part = (float)items * d * 8 / 3e6f;
  auto best = [&](long long units, int holds, int at, float start, float step) {
    Cut c{1, 3e38f};
    for (int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128}) {
      if (s > 1 && s * at > blocks) break;
      // up to d 128 a CU takes a second block beside the first, so that half rounds count
      const float rounds = d > 128 ? (float)((units * s + holds - 1) / holds) : units * s > holds ? .5f * (float)((2 * units * s + holds - 1) / holds) : 1.f;
      const float us = rounds * (start + step * (float)((blocks + s * at - 1) / (s * at))) + (s > 1 ? 3.f + s * part : 0.f);
      if (us < c.us) c = Cut{s, us};
    }
    return c;
  };
  Cut c;
  const int holds = d <= 128 ? 512 : 256;  // blocks of few columns
  if (pairs <= 32 || (pairs <= 64 && (blocks > 16 || 2 * few <= 3 * holds))) {
    // With lengths apart a long sequence needs many splits (48 ragged sequences: blocks of threads up to 2048 57.5 us, to 1024 75; 32 of 8000
    // tokens with heads of 256: to 512 62 us, to 2048 104).  Four waves walk over 16 blocks in less than a launch that joins takes.
    const long long want = p.mt == 1 && d <= 128 ? 2048 : 512, most = (blocks + kPlanWaves - 1) / kPlanWaves;
    p.few = true;
    c.s = blocks <= 16 ? 1 : (want + few - 1) / few;
    c.s = c.s > most ? most : c.s;
    c.s = c.s > kSplits ? kSplits : c.s;
  } else {
    const float step = p.nw == 8 ? 1.6f : d <= 64 ? 1.f : d <= 128 ? 1.2f : d <= 192 ? 2.f : 2.8f;
    c = best(p.tiles * hkv, 256, 1, d <= 128 ? 5.f : d <= 192 ? 8.f : 15.f, step);
    const Cut f = best(few, holds, kPlanWaves, d <= 64 ? 4.f : 5.f, d <= 64 ? .7f : d <= 128 ? 1.8f : 2.9f);
    // what either asks of L2, which the rounds leave out
    const float each = blocks * kPlanBlock * 2 * d / 8e6f;
    p.few = pairs <= 2048 && f.us + each * few < c.us + each * p.tiles * hkv;
    if (p.few) c = f;
  }
  if (p.few) p.scan = false, p.tiles = seqs;
  p.cols = p.few ? (int)cols : 1;
  p.splits = c.s < 1 || items >= 1 << 22 ? 1 : (int)c.s;  // with so many rows there are blocks enough
  p.chunk = (int)((blocks + p.splits - 1) / p.splits);
  if (p.few) {
    // as many blocks for each of the waves (16 sequences of 1000 to 5000 tokens, 8 heads of 128: 24.6 us, 29.6 with chunks of any number)
    p.chunk = p.chunk < kPlanWaves ? kPlanWaves : (p.chunk + kPlanWaves - 1) / kPlanWaves * kPlanWaves;
    p.splits = blocks > p.chunk ? (int)((blocks + p.chunk - 1) / p.chunk) : 1;
  }
  if (p.chunk < 1) p.chunk = 1;
  // Where all tiles run at once the last rows' take longest: folding puts an early half tile beside a late one, so that all blocks have as many
  // steps of a wave; the chain of steps is still the late half's (4096 rows of 16 heads behind 8192 tokens 341 us, 352 without; 98 and 109
  // behind none).  With more tiles than that the next ones fill the gaps (8192 rows of 32 heads 538 without, 634 folded).
  p.fold = !p.few && p.nw == 8 && p.splits == 1 && p.tiles * hkv <= 256;
  return p;
}

}  // namespace drm
