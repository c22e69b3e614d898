// kv_cache.hip -- new keys and values into a paged cache of e4m3 codes, and
// a cache's keys and values back as dense bf16 (warpir_amd.api.kv_cache_write,
// kv_cache_read).
//
// A page holds `page` tokens of every key/value head; each (page, head) has
// one fp32 scale for K and one for V:
//   scale = smallest 2^e with max |x| <= 448 * 2^e,  code = e4m3(x / scale).
// With a power of two x / scale is exact and the code the only rounding (half
// a step: 2^-4 of the value).  A page that already holds tokens keeps its
// scale if that is enough; where it grows, the tokens' codes are rounded
// again by a power of two, which loses nothing but what falls below 2^-9.
//
// K pages are [page, D].  V pages are [D, page]: the second product of
// attention contracts over tokens, so its operand is 16 tokens of one column,
// 16 contiguous bytes here (attn_cached.hip loads them straight into
// registers).  The transposition costs nothing on the way in: the conversion
// packs the codes of any registers, and a lane that holds 4 tokens x 8
// columns packs either way.
//
// Both kernels are bound by memory (2 bytes a value in, 1 out, and back).
// Measured (a 2 GiB copy moves 4.90 TB/s; 8 heads, D = 128, pages of 64): 8
// prompts of up to 4096 tokens written in 19.2 us, 81 MB at 4.2 TB/s; 16
// contexts of up to 8192 read back in 135 us, 654 MB at 4.84 TB/s; bytes moved
// by the counters 1.00 of that.  One token for each of 64 sequences: 4.8 - 6.7
// us, bound by its latency (table, page, store) and by V, of which a token is
// one byte in each of D lines.
#include <hip/hip_runtime.h>

#include "wir_pages.h"

namespace {

using wir::i64;

typedef __bf16 bf16;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// codes [pages, heads, page, D] (K) or [pages, heads, D, page] (V) and their scales [pages, heads]
struct kv_side {
  unsigned char* codes;
  float* scales;
  bf16* x;              // [B, heads, tokens, D] by strides
  i64 xb, xh, xt;
};

struct kv_args {
  kv_side k, v;
  const int* table;     // [B, columns]
  const int* lengths;   // [B]
  const int* counts;    // [B], or null: every token counts
  i64 tb;               // row stride of the table
  int batch, heads, tokens, page, pages, columns, slots;   // slots: pages a sequence's tokens can touch
};

__device__ __forceinline__ unsigned bits_of(bf16 x) { return (unsigned)__builtin_bit_cast(unsigned short, x); }

// Maximum over a page's threads: each `lanes` (32 or 64) of a wave, or not PACKED the workgroup's 256 (x: finite values'
// bits, ordered as unsigned).
template <bool PACKED>
__device__ __forceinline__ unsigned page_max(unsigned x, int lanes) {
#pragma unroll
  for (int m = 32; m; m >>= 1)
    if (!PACKED || m < lanes) x = max(x, (unsigned)__shfl_xor((int)x, m));
  if (PACKED) return x;
  __shared__ unsigned part[4];
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = x;
  __syncthreads();
  return max(max(part[0], part[1]), max(part[2], part[3]));
}

// A workgroup's page of one sequence and head, of K or of V.  PACKED: pages of 32 or 64 lanes, several to a workgroup,
// which has threads idle otherwise (us, one a workgroup / packed, pages of 16: 51 x 309 tokens, 12 heads of D = 64, written
// 32.8 / 16.7; 8 x up to 4096, 8 heads of D = 128 39 / 26.7; 16 x up to 8192 of D = 64 read 123 / 70.  Pages of 128 lanes
// are no faster packed: 26.4 / 27.0).
struct Unit {
  unsigned b, slot, h;
  int lane;
  bool is_v, any;
};
template <int D, bool PACKED>
__device__ __forceinline__ Unit unit_of(const kv_args& a, int lanes) {
  const unsigned first = PACKED ? threadIdx.x / (unsigned)lanes : 0;
  unsigned at = PACKED ? blockIdx.x * (256 / (unsigned)lanes) + first : blockIdx.x;
  Unit u;
  u.lane = threadIdx.x - first * lanes;
  u.is_v = at & 1;
  at >>= 1;
  u.h = at % (unsigned)a.heads;
  at /= (unsigned)a.heads;
  u.slot = at % (unsigned)a.slots, u.b = at / (unsigned)a.slots;
  u.any = !PACKED || u.b < (unsigned)a.batch;
  if (PACKED && !u.any) u.b = 0;
  return u;
}

// Two codes in the low or high half of a word.  An infinity becomes NaN, which e4m3 has and infinity not.
template <bool HIGH>
__device__ __forceinline__ unsigned pack2(float a, float b, unsigned old) {
  return __builtin_amdgcn_cvt_pk_fp8_f32(a, b, old, HIGH);
}
__device__ __forceinline__ unsigned pack4(float a, float b, float c, float d) {
  return pack2<true>(c, d, pack2<false>(a, b, 0u));
}

// The four codes of a word times `ratio`, rounded again.
__device__ __forceinline__ unsigned rescale(unsigned w, float ratio) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  return pack4(a[0] * ratio, a[1] * ratio, b[0] * ratio, b[1] * ratio);
}

__device__ __forceinline__ void rescale2(unsigned* at, float ratio) {
  const u32x2 w = *(const u32x2*)at;
  *(u32x2*)at = u32x2{rescale(w[0], ratio), rescale(w[1], ratio)};
}

// Workgroup -> one page of one sequence and head, of K or of V, or several: a
// page's scale needs all of its new values first, and so few stay in registers
// between the two.  A lane takes 4 tokens x 8 columns; PASSES of 256 lanes
// cover a page.
template <int D, int PASSES, bool PACKED>
__device__ __forceinline__ void write(const kv_args& a) {
  constexpr int COLS = D / 8;
  const int groups = a.page / 4, lanes = groups * COLS;
  const Unit u = unit_of<D, PACKED>(a, lanes);
  const unsigned h = u.h, slot = u.slot, b = u.b;
  const bool is_v = u.is_v;
  const kv_side& side = is_v ? a.v : a.k;

  const wir::Span s = wir::span_of(a.lengths[b], a.counts ? a.counts[b] : a.tokens, a.tokens, a.columns * a.page);
  const int place = min(wir::first_new(s) / a.page + (int)slot, a.columns);
  const int base = place * a.page;   // position of the page's first token
  const int lo = max(wir::first_new(s), base);
  int hi = min(s.held, base + a.page), id = -1;
  if (u.any && place < a.columns && lo < hi) id = wir::checked_page(a.table[b * a.tb + place], a.pages);
  if (!PACKED && id < 0) return;
  if (PACKED && id < 0) hi = 0;   // no tokens
  const i64 index = (i64)max(id, 0) * a.heads + h;
  unsigned* codes = (unsigned*)(side.codes + index * a.page * D);
  const bool kept = lo > base;   // (the page then holds positions base .. lo - 1)
  const float was = side.scales[index];

  // lane -> tokens 4 r .. 4 r + 3 of the page and columns 8 c .. 8 c + 7: neighbours in K's store order or, for whole
  // V pages, in V's (a few tokens then keep to few waves, and the others skip the work)
  const bool by_token = is_v && hi - lo >= 16;
  const bf16* x = side.x + b * side.xb + h * side.xh;
  bf16x8 val[PASSES][4];
  unsigned had[PASSES][8];   // V words that keep some of their codes
  unsigned top = 0;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int l = p * 256 + u.lane, r = by_token ? l % groups : l / COLS, c = by_token ? l / groups : l % COLS;
    const int pos = base + 4 * r;
    if (l >= lanes || pos >= hi || pos + 4 <= lo) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      val[p][i] = bf16x8{};
      if (pos + i >= lo && pos + i < hi) val[p][i] = *(const bf16x8*)(x + (pos + i - s.start) * side.xt + 8 * c);
    }
    if (is_v && (pos < lo || pos + 4 > hi)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) had[p][j] = codes[(8 * c + j) * groups + r];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const unsigned m = bits_of(val[p][i][j]) & 0x7fffu;
        top = max(top, m < 0x7f80u ? m : 0u);
      }
  }
  const float enough = __uint_as_float(wir::scale_bits(page_max<PACKED>(top, lanes) << 16));
  const float scale = kept && was >= enough ? was : enough;
  const bool grown = kept && !(scale == was);
  const float inv = 1.0f / scale, ratio = was / scale;
  if (u.lane == 0 && (!PACKED || id >= 0)) side.scales[index] = scale;

#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int l = p * 256 + u.lane, r = by_token ? l % groups : l / COLS, c = by_token ? l / groups : l % COLS;
    const int pos = base + 4 * r;
    if (l >= lanes || pos >= hi) continue;
    unsigned* to = codes + (8 * c * a.page + 4 * r) / 4;   // V: word j the four tokens of column 8 c + j
    if (pos + 4 <= lo) {   // tokens that were there
      if (!grown) continue;
      if (is_v) {
#pragma unroll
        for (int j = 0; j < 8; ++j) to[j * groups] = rescale(to[j * groups], ratio);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) rescale2(codes + ((4 * r + i) * D + 8 * c) / 4, ratio);
      }
      continue;
    }
    float y[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float z = (float)val[p][i][j];
        y[i][j] = __builtin_fabsf(z) < __builtin_inff() ? z * inv : __builtin_nanf("");
      }
    if (is_v) {
      unsigned fresh = 0, old = 0;   // masks of the word's bytes
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (pos + i >= lo && pos + i < hi) fresh |= 0xffu << 8 * i;
        if (pos + i < lo) old |= 0xffu << 8 * i;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        unsigned w = pack4(y[0][j], y[1][j], y[2][j], y[3][j]);
        if (fresh != ~0u) {
          const unsigned again = grown ? rescale(had[p][j], ratio) : had[p][j];
          w = (w & fresh) | (again & old) | (had[p][j] & ~(fresh | old));
        }
        to[j * groups] = w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        unsigned* row = codes + ((4 * r + i) * D + 8 * c) / 4;
        if (pos + i >= lo && pos + i < hi)
          *(u32x2*)row = u32x2{pack4(y[i][0], y[i][1], y[i][2], y[i][3]), pack4(y[i][4], y[i][5], y[i][6], y[i][7])};
        else if (pos + i < lo && grown)
          rescale2(row, ratio);
      }
    }
  }
}

// Workgroup -> one page's places of one sequence and head, of K or of V, or
// several, as dense rows; places past the sequence and those of no page
// become 0.
template <int D, int PASSES, bool PACKED>
__device__ __forceinline__ void read(const kv_args& a) {
  constexpr int COLS = D / 8;
  const int groups = a.page / 4, lanes = groups * COLS;
  const Unit u = unit_of<D, PACKED>(a, lanes);
  if (!u.any) return;
  const unsigned h = u.h, slot = u.slot, b = u.b;
  const bool is_v = u.is_v;
  const kv_side& side = is_v ? a.v : a.k;
  const int held = wir::span_of(a.lengths[b], 0, 0, a.columns * a.page).held;
  const int base = (int)slot * a.page;
  int id = -1;
  if ((int)slot < a.columns && base < held) id = wir::checked_page(a.table[b * a.tb + slot], a.pages);
  const int there = id < 0 ? 0 : held - base;   // tokens of the page that the sequence holds
  const i64 index = (i64)(id < 0 ? 0 : id) * a.heads + h;
  const unsigned* codes = (const unsigned*)(side.codes + index * a.page * D);
  const float scale = side.scales[index];
  bf16* x = side.x + b * side.xb + h * side.xh;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int l = p * 256 + u.lane, r = is_v ? l % groups : l / COLS, c = is_v ? l / groups : l % COLS;
    if (l >= lanes || base + 4 * r >= a.tokens) continue;
    // word (i, u): columns 4 u .. of token i (K), or w[j]: tokens of column j (V)
    unsigned w[8] = {};
    if (4 * r >= there) {
    } else if (is_v) {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = codes[(8 * c + j) * groups + r];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32x2 y = *(const u32x2*)(codes + ((4 * r + i) * D + 8 * c) / 4);
        w[2 * i] = y[0], w[2 * i + 1] = y[1];
      }
    }
    f32x2 y[8][2];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      y[j][0] = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], false);
      y[j][1] = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], true);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int tok = 4 * r + i;
      if (base + tok >= a.tokens) break;
      bf16x8 out;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float z = is_v ? y[j][i / 2][i % 2] : y[2 * i + j / 4][j % 4 / 2][j % 2];
        out[j] = (bf16)(tok < there ? z * scale : 0.f);
      }
      *(bf16x8*)(x + (i64)(base + tok) * side.xt + 8 * c) = out;
    }
  }
}

}  // namespace

#define KV_KERNEL(NAME, CALL) \
  extern "C" __global__ void __launch_bounds__(256) NAME(const kv_args args) { CALL(args); }

KV_KERNEL(wir_kv_write_d64, (write<64, 1, false>))
KV_KERNEL(wir_kv_write_d64_packed, (write<64, 1, true>))     // pages of 16 and 32 tokens
KV_KERNEL(wir_kv_write_d128, (write<128, 1, false>))
KV_KERNEL(wir_kv_write_d128_packed, (write<128, 1, true>))   // pages of 16
KV_KERNEL(wir_kv_write_d128_p128, (write<128, 2, false>))    // pages of 128
KV_KERNEL(wir_kv_read_d64, (read<64, 1, false>))
KV_KERNEL(wir_kv_read_d64_packed, (read<64, 1, true>))
KV_KERNEL(wir_kv_read_d128, (read<128, 1, false>))
KV_KERNEL(wir_kv_read_d128_packed, (read<128, 1, true>))
KV_KERNEL(wir_kv_read_d128_p128, (read<128, 2, false>))
