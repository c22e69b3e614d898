// wir_pages.h -- the index arithmetic of paged 8-bit caches: which tokens,
// pages and work a program has.  No device code: the kernels
// (kv_cache.hip, attn_cached.hip) and a host program that checks it against
// plain counting compile the same functions.
#pragma once

#if defined(__HIPCC__) || defined(__HIP__)
#define WIR_HD __host__ __device__ __forceinline__
#else
#define WIR_HD inline
#endif

namespace wir {

typedef long long i64;

WIR_HD int imin(int a, int b) { return a < b ? a : b; }
WIR_HD int imax(int a, int b) { return a > b ? a : b; }

// One sequence of the batch: its new tokens t = 0 .. count - 1 have the
// positions start + t, and the cache holds positions 0 .. held - 1.  Lengths
// and counts are data: whatever they hold, 0 <= count <= tokens and
// 0 <= held <= capacity (< 2^31).  `start` may be negative: tokens before
// position 0 have no place.
struct Span {
  int start, count, held;
};

WIR_HD Span span_of(int length, int count, int tokens, int capacity) {
  Span s;
  length = imax(length, 0);
  s.count = imin(imax(count, 0), tokens);
  s.start = length - s.count;
  s.held = imin(length, capacity);
  return s;
}

// First new position that has a place.
WIR_HD int first_new(const Span& s) { return imax(s.start, 0); }

// A page id of the table, or -1 for one that is no page of the cache or lies
// past the table's columns.
WIR_HD int checked_page(int id, int pages) { return id >= 0 && id < pages ? id : -1; }

// Smallest e with amax <= 448 * 2^e, at least -126, as the bits of 2^e.  amax
// by its fp32 bits (finite): 448 = 1.75 * 2^8, so e is the exponent - 8, and
// one more where the fraction is past 0.75.
WIR_HD unsigned scale_bits(unsigned amax) {
  const int e = (int)((amax + 0x1fffffu) >> 23) - 127 - 8;
  return (unsigned)(imax(e, -126) + 127) << 23;
}

// ---------------------------------------------------------------------------
// Attention: rows and tiles.  The query rows of one sequence and key/value
// head are r = t * group + j, token t of query head j of the group; a block
// has `rows_per_block` of them.  A tile is TILE positions.
// ---------------------------------------------------------------------------
constexpr int TILE = 64;

// Positions that some row of block rb sees: 0 .. keys - 1.
WIR_HD int block_keys(const Span& s, int rb, int rows_per_block, int rows, int group) {
  const int first = rb * rows_per_block / group;
  const int last = imin((imin(rows, (rb + 1) * rows_per_block) - 1) / group, s.count - 1);
  if (first >= s.count || s.start + last < 0) return 0;
  return imin(s.start + last + 1, s.held);
}

// Its units of work: tiles, and one where there are none (its rows are written all the same).
WIR_HD int block_units(int keys) { return imax((int)(((unsigned)keys + TILE - 1) / TILE), 1); }

// All units together, and so any unit's index, have to stay below 2^30 (64-bit
// divisions cost microseconds here).
//
// Division of the units of all (sequence, block) pairs, heads of a pair in
// turn, tiles of a head in turn, over the programs.
//
// With more heads than programs can have one each, a program takes `share`
// consecutive units, parts of one or more heads.  One that takes part of a
// head's units leaves a partial result in one of its two slots: the first
// segment of its share in slot 2 * program, another one, which is then its
// last, in 2 * program + 1.
//
// With fewer heads, a head's units go to parts_even(units) programs of its
// own in equal parts, and program w's slot is w.
WIR_HD int share_of(int total, int programs, int least) { return imax((total + programs - 1) / programs, least); }

struct Segment {
  int head, first, last;   // tiles first .. last - 1 of the head's
  bool whole;              // all of the head's
  int slot, parts;         // of its partial result; partial results of the head
};

// Slot of the partial result of a segment that starts at unit u.
WIR_HD int slot_of(int u, int share) { return 2 * (u / share) + (u % share ? 1 : 0); }

// The segment at unit u of a pair whose units start at `base`, `units` a head; the program's share ends at `end`.
WIR_HD Segment segment_at(int u, int base, int units, int end, int share) {
  Segment g;
  g.head = (u - base) / units;
  g.first = (u - base) % units;
  g.last = imin(units, g.first + end - u);
  g.whole = g.first == 0 && g.last == units;
  const int begin = u - g.first;
  g.slot = slot_of(u, share);
  g.parts = (begin + units - 1) / share - begin / share + 1;
  return g;
}

// Slot of a head's n-th partial result, from that of its first.
WIR_HD int slot_of_part(int first, int n, bool even) { return even ? first + n : n == 0 ? first : 2 * (first / 2 + n); }

// Equal parts: the share that gives all heads together at most `programs` of them (heads < programs).
WIR_HD int share_even(int total, int programs, int heads, int least) { return share_of(total, programs - heads, least); }
WIR_HD int parts_even(int units, int share) { return (units + share - 1) / share; }

// Part n of the pair's parts, which start with program `base`.
WIR_HD Segment segment_even(int program, int base, int units, int share) {
  Segment g;
  g.parts = parts_even(units, share);
  g.head = (program - base) / g.parts;
  const int n = (program - base) % g.parts;
  // the first units % parts of them have one more
  const int each = units / g.parts, more = units % g.parts;
  g.first = n * each + imin(n, more);
  g.last = g.first + each + (n < more ? 1 : 0);
  g.whole = g.parts == 1;
  g.slot = program;
  return g;
}

}  // namespace wir
