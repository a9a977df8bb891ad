// The paged 4-bit K/V cache: where things lie in a page, which arguments its entry points take, and
// what a kernel makes of a sequence's lengths and pages.  Nothing here needs a device, so a plain
// C++ compiler can check all of it.
//
// A page holds P rows of every kv head; a kv head's block in it is four pieces in a row:
//   key codes     [P][4][D/32] words   word (c, s) of a row: elements 32 s + 8 c .. + 7
//   key params    [P][D/g] pairs       fp16 (step, minimum)
//   value codes   [P/4][D/8][4] words  word (b, w, t): elements 8 w .. 8 w + 7 of row 4 b + t
//   value params  [P/4][D/g][2][4]     fp16 steps of rows 4 b .. 4 b + 3, then their minima
// A key word has element 2 i in nibble i and element 2 i + 1 in nibble 4 + i, a value word element i
// in nibble i.  The orders are those of a matrix instruction's operands: the 16 bytes (D = 128) that
// lane (row, c) of a 16 x 32 key operand needs for its D/32 steps lie together, and a 16-byte piece of
// value codes is four rows (the contracted index) of eight output elements.
#pragma once

#include <cmath>
#include <cstddef>
#include <cstdint>
#include <cstdio>

#if defined(__HIPCC__)
#define KRM_HD __host__ __device__
#else
#define KRM_HD
#endif

namespace krm {

// A group with a magnitude above this (or a NaN) gets a NaN step and reads as NaN: 15 * step, and
// step * 15 + minimum with both rounded outwards, then stay finite in fp16.
constexpr float kKv4Limit = 32640.0f;

// (row, head) pairs of a sequence and kv head that a call takes.
constexpr uint32_t kKv4MostPairs = 1u << 24;

struct Kv4Layout {
  uint32_t depth, group, page_rows, kv_heads;

  KRM_HD uint32_t groups() const { return depth / group; }
  KRM_HD uint32_t code_row() const { return depth / 2; }          // bytes of a row's codes
  KRM_HD uint32_t code_bytes() const { return page_rows * (depth / 2); }
  KRM_HD uint32_t param_bytes() const { return page_rows * groups() * 4; }
  KRM_HD uint32_t key_params() const { return code_bytes(); }
  KRM_HD uint32_t value_codes() const { return code_bytes() + param_bytes(); }
  KRM_HD uint32_t value_params() const { return 2 * code_bytes() + param_bytes(); }
  KRM_HD uint32_t block() const { return 2 * (code_bytes() + param_bytes()); }
  KRM_HD uint64_t page() const { return (uint64_t)block() * kv_heads; }
  // bytes from the start of a block
  KRM_HD uint32_t key_word(uint32_t row, uint32_t word) const {   // word: elements 8 word ..
    return row * code_row() + ((word & 3) * (depth / 32) + word / 4) * 4;
  }
  KRM_HD uint32_t key_param(uint32_t row, uint32_t g) const { return key_params() + (row * groups() + g) * 4; }
  KRM_HD uint32_t value_word(uint32_t row, uint32_t word) const {
    return value_codes() + ((row / 4 * (depth / 8) + word) * 4 + row % 4) * 4;
  }
  KRM_HD uint32_t value_param(uint32_t row, uint32_t g) const {   // the step; its minimum lies 8 bytes on
    return value_params() + (row / 4 * groups() + g) * 16 + row % 4 * 2;
  }
};

// What the rows of one sequence are in this step, from the device's words: rows first .. first +
// rows - 1 of the packed step, columns len - rows .. len - 1 of the sequence.  `ok` is false where the
// words break the limits that the launch was made for; nothing may be indexed by them then.
struct Kv4Sequence {
  int32_t first, rows, len;
  bool ok;
};
struct Kv4Limits {
  uint32_t total_rows, max_query, max_columns, table_stride, page_rows;
};
KRM_HD inline Kv4Sequence kv4_sequence(int32_t cu0, int32_t cu1, int32_t len, const Kv4Limits& a) {
  Kv4Sequence s{cu0, 0, len, false};
  if (cu0 < 0 || cu1 < cu0 || (uint32_t)cu1 > a.total_rows) return s;
  s.rows = cu1 - cu0;
  if (s.rows == 0) {   // an entry of a padded batch: nothing to do, whatever its length says
    s.ok = true;
    return s;
  }
  s.ok = (uint32_t)s.rows <= a.max_query && len >= s.rows && (uint32_t)len <= a.max_columns &&
         (uint64_t)(uint32_t)len <= (uint64_t)a.table_stride * a.page_rows;
  return s;
}

// Tiles of `tile` columns, about, that one kv head of a sequence has in a launch for sequences of least_pairs to
// most_pairs (row, head) pairs, all blocks of block_pairs of them together: none for an entry without rows (whatever its
// length says) or one of the other launch, or more pairs than any call takes, as descending offsets give.  (A refused
// sequence counts with what else its words say, within max_columns.)
KRM_HD inline float kv4_tiles(uint32_t rows, int32_t len, uint32_t share, uint32_t least_pairs, uint32_t most_pairs,
                              uint32_t block_pairs, uint32_t window, uint32_t max_columns, uint32_t tile) {
  const uint32_t pairs = rows * share, most = window && window < max_columns ? window : max_columns;
  const uint32_t n = len < 0 ? 0 : (uint32_t)len < most ? (uint32_t)len : most;
  const uint32_t past = most_pairs < kKv4MostPairs ? most_pairs : kKv4MostPairs;
  const uint32_t blocks = pairs < least_pairs || pairs > past ? 0 : (pairs + block_pairs - 1) / block_pairs;
  return (float)(n / tile + 1) * (float)blocks;
}

// Work of one kv head of a sequence in blocks of rows, each of which sees some more columns than the one before it:
// block b has first + b * step units.  All of them together are less than 2^31.
struct Kv4Blocks {
  uint32_t blocks, first, step;
  KRM_HD uint32_t of(uint32_t b) const { return first + b * step; }
  KRM_HD uint32_t before(uint32_t b) const { return b * first + (step ? b * (b - 1) / 2 * step : 0); }
  KRM_HD uint32_t all() const { return before(blocks); }
  // The block that unit `at` (less than all()) is in.
  KRM_HD uint32_t block_at(uint32_t at) const {
    const float x = (float)first - 0.5f * (float)step;   // the root of before(b) = at
    uint32_t b = (uint32_t)(2.0f * (float)at / (x + sqrtf(x * x + 2.0f * (float)step * (float)at)));
    if (b > blocks - 1) b = blocks - 1;
    while (before(b) > at) --b;
    while (b + 1 < blocks && before(b + 1) <= at) ++b;
    return b;
  }
};
// Units of 2^grain columns.  `pairs` (row, head) pairs, in blocks of `block_pairs`, of a sequence of `len` columns.
KRM_HD inline Kv4Blocks kv4_blocks(uint64_t pairs, uint32_t share, uint32_t block_pairs, int32_t len, uint32_t window,
                                   uint32_t grain) {
  Kv4Blocks b;
  const uint32_t rows = (uint32_t)(pairs / share);
  b.blocks = (uint32_t)((pairs + block_pairs - 1) / block_pairs);
  const uint32_t last = (uint32_t)((pairs < block_pairs ? pairs : block_pairs) - 1) / share;   // of the first block
  b.first = (((uint32_t)len - rows + last) >> grain) + 1;
  b.step = b.blocks > 1 ? block_pairs / share >> grain : 0;
  if (window) {   // blocks that all see a window are alike, and are all taken for such ones where some do
    const uint64_t most = (((uint64_t)window + block_pairs) >> grain) + 1;
    if (b.of(b.blocks - 1) > most) {
      b.first = (uint32_t)most;
      b.step = 0;
    }
  }
  return b;
}
// A workgroup's run of the row of work: units [at, end), of `per` units in all runs but the last.
struct Kv4Run {
  uint32_t per, at, end;
  uint32_t begin, snap;   // units that beginning a block counts as; distance at which a run's end moves to a block's
  uint32_t even;          // units are equal parts of blocks
  uint32_t fresh;         // the run has had no piece yet
};
// Its piece of the block that unit `at` is in, which has `width` units from `block_at` on.
struct Kv4Cut {
  uint32_t from, to;      // of the block's units
  uint32_t parts, first;  // pieces that the block is in, each in a run of its own; the first one's run
};
enum Kv4Dealt { kRunEnds, kBlockSkipped, kPieceDealt };
KRM_HD inline Kv4Dealt kv4_cut(Kv4Run& r, uint32_t block_at, uint32_t width, Kv4Cut& c) {
  const bool uncut = width < 2 * r.snap;
  const uint32_t near = uncut ? (width + 1) / 2 : r.snap, behind = block_at + width;
  c.from = r.at - block_at;
  c.to = width;
  if (r.fresh) {
    r.fresh = 0;
    if (c.from < near) {
      c.from = 0;
    } else if (uncut || width - c.from < r.snap) {
      r.at = behind;
      return r.at < r.end ? kBlockSkipped : kRunEnds;
    }
  }
  if (r.end < behind) {
    if (r.end - block_at < near) return kRunEnds;
    if (!uncut && behind - r.end >= r.snap) c.to = r.end - block_at;
  }
  r.at = block_at + c.to;
  const uint32_t first_cut = (block_at + r.snap + r.per - 1) / r.per, last_cut = (behind - r.snap) / r.per;
  c.parts = uncut || last_cut < first_cut ? 1 : last_cut - first_cut + 2;
  c.first = first_cut - 1;
  return kPieceDealt;
}
// The tile, of a block's `tiles`, at which its unit `unit` begins.  (Units are an estimate, rounded, of a window's
// widest block: what it leaves or lacks is the last part's.)
KRM_HD inline uint32_t kv4_tile(const Kv4Run& r, uint32_t unit, uint32_t width, uint32_t tiles, uint32_t grain,
                                uint32_t tile) {
  if (r.even) return tiles / width * unit + tiles % width * unit / width;
  if (unit == width) return tiles;
  const uint64_t at = ((uint64_t)(unit < r.begin ? 0 : unit - r.begin) << grain) / tile;
  return at < tiles ? (uint32_t)at : tiles;
}
// First column that a row at `position` sees.
KRM_HD inline int32_t kv4_first_column(int32_t position, uint32_t window) {
  return window == 0 || (uint32_t)position < window ? 0 : position - (int32_t)window + 1;
}

// Rows of a sequence that a launch has to make room for.
inline uint32_t kv4_rows(uint32_t max_query, uint32_t total_rows) { return max_query < total_rows ? max_query : total_rows; }

// ---- argument checks (host) -----------------------------------------------------------------
struct Kv4Shape {
  uint32_t nseq, max_query, total_rows, heads, kv_heads, depth, group, page_rows, pages, table_stride;
};
// Writes why `s` is refused and returns false.
inline bool kv4_refused(char* why, size_t size, const char* text, uint32_t a, uint32_t b) {
  snprintf(why, size, text, a, b);
  return false;
}
inline bool kv4_layout_ok(const Kv4Shape& s, char* why, size_t size) {
  if (s.kv_heads < 1 || s.kv_heads > 65535)
    return kv4_refused(why, size, "kv_heads %u (1 to 65535)", s.kv_heads, 0);
  if (s.depth != 64 && s.depth != 128 && s.depth != 256)
    return kv4_refused(why, size, "depth %u (64, 128 or 256)", s.depth, 0);
  if ((s.group != 32 && s.group != 64 && s.group != 128) || s.group > s.depth)
    return kv4_refused(why, size, "group %u (32, 64 or 128, within a depth of %u)", s.group, s.depth);
  if (s.page_rows < 16 || s.page_rows > 256 || (s.page_rows & (s.page_rows - 1)) != 0)
    return kv4_refused(why, size, "page_rows %u (a power of two from 16 to 256)", s.page_rows, 0);
  return true;
}
inline bool kv4_shape_ok(const Kv4Shape& s, char* why, size_t size) {
  if (!kv4_layout_ok(s, why, size)) return false;
  if (s.heads < s.kv_heads || s.heads > 65535 || s.heads % s.kv_heads != 0)
    return kv4_refused(why, size, "heads %u are no multiple of kv_heads %u", s.heads, s.kv_heads);
  if (s.nseq > 65535) return kv4_refused(why, size, "nseq %u (65535 at most)", s.nseq, 0);
  if (s.total_rows > 0x7fffffffu || (s.total_rows && !s.max_query))
    return kv4_refused(why, size, "max_query %u beside total_rows %u", s.max_query, s.total_rows);
  if (s.pages < 1 || s.pages > 0x7fffffffu) return kv4_refused(why, size, "pages %u", s.pages, 0);
  if (s.table_stride < 1 || s.table_stride > 0x7fffffffu)
    return kv4_refused(why, size, "table_stride %u", s.table_stride, 0);
  return true;
}
inline bool kv4_turn_ok(uint32_t depth, uint32_t rotary, int32_t layout, uint32_t table_rows, uint32_t table_width,
                        char* why, size_t size) {
  if (rotary % 2 != 0 || rotary > depth)
    return kv4_refused(why, size, "rotary_dim %u (even, within a head of %u)", rotary, depth);
  if (layout != 0 && layout != 1) return kv4_refused(why, size, "layout %u", (uint32_t)layout, 0);
  if (rotary && (table_rows < 1 || table_width < rotary / 2))
    return kv4_refused(why, size, "tables of %u rows of %u angles", table_rows, table_width);
  return true;
}

}  // namespace krm
