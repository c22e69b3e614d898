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

}  // namespace wir
