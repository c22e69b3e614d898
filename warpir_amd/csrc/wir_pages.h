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
  int first = 0, last = rows;   // tokens; one block has them all (and needs no division)
  if (rows > rows_per_block) {
    first = rb * rows_per_block / group;
    last = (imin(rows, (rb + 1) * rows_per_block) - 1) / group;
  }
  last = imin(last, s.count - 1);
  if (first >= s.count || s.start + last < 0) return 0;
  return imin(s.start + last + 1, s.held);
}

// Its units of work: tiles, and one where there are none (its rows are written all the same).
WIR_HD int block_tiles(int keys) { return (int)(((unsigned)keys + TILE - 1) / TILE); }
WIR_HD int block_units(int keys) { return imax(block_tiles(keys), 1); }

// Division of the work: a head's units go to parts_of(units) programs in
// equal parts of at most `share`, in the order of (sequence, block) pairs,
// their heads, and tiles.  `extra` bounds the programs: at most one a head and
// `extra` more.  All units together have to stay below 2^30 (64-bit divisions
// cost microseconds here).
WIR_HD int share_of(int total, int extra, int least) { return imax((total + extra - 1) / extra, least); }
WIR_HD int parts_of(int units, int share) { return (units + share - 1) / share; }

// First unit of part n; the first units % parts of them have one more.
WIR_HD int part_begin(int n, int units, int parts) {
  const int each = units / parts;
  return n * each + imin(n, units - each * parts);
}

// Where a partial result goes: the parts of divided heads have at least
// share / 2 units, so no two of them start in the same such interval of all
// units.  `begin`: the part's first unit among them.
WIR_HD int slot_width(int share) { return imax(share / 2, 1); }
WIR_HD int slots_for(int extra) { return 3 * extra + 2; }
WIR_HD int slot_of(int begin, int width, int extra) { return imin(imax(begin / width, 0), slots_for(extra) - 1); }

}  // namespace wir
