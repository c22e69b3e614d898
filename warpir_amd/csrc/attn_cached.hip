// attn_cached.hip -- attention of new queries over a paged cache of e4m3
// codes (warpir_amd.api.attention_cached; kv_cache.hip writes the cache).
//
// A token's key is k = code * ks and its value v = code * vs, ks and vs one
// scale for each page and head.  For query row r at position p:
//   s_j = q . code_j * ks / sqrt(D) for j <= p,  O = sum_j softmax(s)_j vs code_j.
//
// Both products run on bf16 matrix instructions: e4m3 codes are exact in bf16,
// also times a power of two, and one instruction converts two of them.  ks
// multiplies the fp32 score; the power of two of vs goes to the values in
// their conversion, what vs has beside it to the probabilities (which are
// rounded to bf16 once).  (The first product on fp8 matrix instructions, with
// q as the sum of two e4m3 terms, spares half the conversions, but those add
// up with about 16 bits: scores were off by 1.4e-5 of sum |q k|.)
//
// Both products are taken transposed, S^T = K Q^T and O^T = V^T P^T, with the
// query rows (the heads that share a key/value head, and the new tokens) as
// the columns.  A lane then holds scores of one query row, and those of a
// 64-token tile are turned into the second product's operand without leaving
// the lane: the rows of K go to the matrix core in an order that gives each
// lane group 16 tokens that follow one another.  V pages are [D, token], so
// that operand's other side is 16 contiguous bytes of one column.
//
// Few rows (16 or 32 of a key/value head, on 16x16x32 products): K and V come
// from memory straight into registers, every byte once, with no LDS and no
// barrier in the loop; a workgroup's waves take every WK-th tile and are joined
// at the end.  Bound by the cache's bytes: one token over 131072 (32/8 heads, D
// = 128) 45 us, 268 MB at 5.9 TB/s, and 5 for the join; 64 sequences of up to
// 8192 113 us, 598 MB at 5.3 TB/s, and 5; 16 sequences of up to 2050, 4 tokens,
// 16 heads of D = 64, pages of 16: 11 us, 41 MB at 3.7 TB/s.  (Reading 4 GiB
// alone goes at 7.1 TB/s.)  32 rows at D = 128 need 11 registers more than the 256
// that two programs a CU leave: four 8-byte loads, a 4-byte load and store of
// scratch memory in each tile.  One program without them is slower: 8 x 64
// queries over 2000 keys (32/8 heads) 46.0 us, so 42.5; 4 x 8 over 8000 32.2, so 28.9.
// Many rows: a workgroup's waves take 32 rows each, on 32x32x16 products (half
// the steps between lanes, and half the instructions to issue, of 16x16x32:
// 5% at D = 128, 3% at 64), and share the tiles: each wave converts its part
// of the next tile's codes and leaves them in LDS as operands (a fragment is 64
// lanes' 16 bytes in lane order), so that a code is converted once for 128
// rows.  (Eight waves, for launches of one block a CU: two such groups divide the
// tiles and are joined at the end; 1 x 1000 queries over 8192 keys 180 -> 156 us.)
// 2 x 1000 queries over 8192 keys (32/8 heads, D = 128): 278 us, 907
// TFLOP/s, 68% of a large matrix product's 1328, with the matrix cores busy 42%
// and the vector ALU 56% of the cycles at 2.1 GHz, to which the card's power
// holds it (on 16x16x32 products 2.3 GHz, and 16% more cycles).  No one thing
// bounds it: taken out of a copy each by itself, the next tile's loads are 10%
// of the time, its conversion and LDS stores 10%, the softmax 14%, the barrier
// 1.5%, half of the LDS reads 2.5%; two waves a SIMD cover each other only in
// part, and the registers of 32 rows leave no room for a third.  The next tile's
// scores under this one's exponentials, 64 rows a wave, 256 rows a workgroup
// with the halves of its waves in opposite phases, loads two tiles ahead, and
// higher priorities for either phase changed nothing.
#include "wir_cdna4.h"
#include "wir_pages.h"

namespace {

using wir::i64;
using wir::bf16;
using wir::bf16x8;
using wir::f32x4;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) bf16x8 lds_bf16x8;

constexpr float kLn2 = 0.6931471805599453f;

struct attn_args {
  const bf16* q;               // [B, H, T, D]
  const unsigned char* k;      // [pages, heads, page, D]
  const unsigned char* v;      // [pages, heads, D, page]
  const float* k_scale;        // [pages, heads]
  const float* v_scale;
  const int* table;            // [B, columns]
  const int* lengths;          // [B]
  const int* counts;           // [B] or null
  bf16* out;                   // [B, H, T, D]
  float* lse;                  // [B, H, T]
  float* partial;              // [slots][block rows][D], then [slots][block rows][2]
  int* info;                   // [items][4]: first unit, units, parts, width of a slot
  i64 qb, qh, qt, ob, oh, ot, lb, lh, lt, tb;
  int batch, heads, group, tokens, page_shift, pages, columns;
  int blocks;                  // row blocks of a sequence and head
  int extra;                   // programs beyond one for each (sequence, block, head) at most; 0: no division
  int least;                   // tiles of a part at least, unless the head has fewer
};

// The arguments where the launch put them.  They fill most of the scalar registers: `fresh` makes the compiler read them
// again in each phase instead of keeping them (spilled) through the tiles' loop, where reading a spilled one back costs
// a vector instruction (95 of 470 a tile).
typedef const __attribute__((address_space(4))) attn_args* args_ptr;
__device__ __forceinline__ args_ptr fresh(args_ptr a) {
  unsigned long long p = (unsigned long long)a;
  asm volatile("" : "+s"(p));
  return (args_ptr)p;
}

// The eight codes of two words, times a power of two, in bf16 (exact).
__device__ __forceinline__ bf16x8 unpack8(unsigned a, unsigned b, float scale) {
  const bf16x2 w = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, false);
  const bf16x2 x = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, true);
  const bf16x2 y = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, false);
  const bf16x2 z = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, true);
  return bf16x8{w[0], w[1], x[0], x[1], y[0], y[1], z[0], z[1]};
}

// op over lanes l, l ^ 16, l ^ 32, l ^ 48
template <class F>
__device__ __forceinline__ float over_groups(float x, F op) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Inclusive sums over the lanes of a wave.
__device__ __forceinline__ int wave_scan(int x) {
  const int lane = wir::lane_id();
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  return x;
}

// One of a sequence's row blocks of one head, over some of its tiles: W waves, of 16 * NQ rows each, WR side by side
// and the others dividing the tiles.  WIDE: a page holds whole tiles.
template <int D, int NQ, int WR, int W, bool WIDE = false>
struct Program {
  static constexpr int WK = W / WR;              // waves that divide the tiles
  static constexpr bool SHARED = WR > 1;         // tiles go through LDS
  static constexpr int ROWS = 16 * NQ;           // query rows of a wave
  static constexpr int BLOCK = ROWS * WR;        // and of the workgroup
  static constexpr int KC = D / 64, DT = D / 16, PITCH = D + 4;
  static constexpr int CHUNKS = D / 8;           // of a tile's codes, 64 lanes' 16 bytes each
  static_assert(!SHARED || (WR == 4 && NQ == 2), "");

  // What the workgroup does, worked out by its first wave.  The lengths are read here and nowhere else, and every index
  // that follows from them is bounded: a program that changes them under a running launch gets wrong rows, no more.
  struct Plan {
    int pair, head, first, last, slot;
    wir::Span span;
  };

  struct Results {
    float o[W * ROWS * PITCH];
    float ml[W * ROWS * 2];
  };
  struct Shared {
    union {
      Results r;
      char ring[SHARED ? WK * 2 * CHUNKS * 2048 : 16];   // two tiles as operands, for each that divide the tiles
    };
    int nan_from[D];   // first position with a NaN code in the column, of the tiles that not all rows see whole
    int nan_any;
    Plan plan;
  };

  args_ptr a;
  Shared& sh;
  int lane, col, grp, wave, wr, wk;
  // the pair's
  int b, rb;
  wir::Span span;

  __device__ __forceinline__ Program(args_ptr args, Shared& shared) : a(args), sh(shared) {
    lane = wir::lane_id();
    col = lane % 16;
    grp = lane / 16;
    wave = wir::wave_id();
    wr = wave % WR;
    wk = wave / WR;
  }

  __device__ __forceinline__ int rows() const { return a->tokens * a->group; }

  __device__ __forceinline__ wir::Span span_at(int seq) const {
    return wir::span_of(a->lengths[seq], a->counts ? a->counts[seq] : a->tokens, a->tokens, a->columns << a->page_shift);
  }
  // (divisions that the plain decode step does not need are branched over: a step's whole path is a few microseconds)
  __device__ __forceinline__ int sequence_of(int pair) const { return a->blocks == 1 ? pair : pair / a->blocks; }
  __device__ __forceinline__ int token_of(int r) const { return a->tokens == 1 ? 0 : r / a->group; }
  __device__ __forceinline__ int keys_of(const wir::Span& s, int pair) const {
    return wir::block_keys(s, pair - sequence_of(pair) * a->blocks, BLOCK, rows(), a->group);
  }

  // Position that new token t sees up to; -1: none.
  __device__ __forceinline__ int position_of(int t) const { return t < span.count ? max(span.start + t, -1) : -1; }

  // A wave's running softmax and output, and its queries as operands.
  struct State {
    bf16x8 q[NQ][2 * KC];   // in the order of K's 16-byte pieces
    int pos[NQ];
    int low;              // no row that sees anything sees less
    f32x4 o[DT][NQ];
    float m[NQ], l[NQ];
  };

  // The lane's 16 tokens of a tile.
  struct Tokens {
    float ks, vs;
    int have;             // how many the sequence holds
  };

  __device__ __forceinline__ void begin(State& s, int head) const {
    const int row0 = rb * BLOCK + wr * ROWS;
    s.low = max(span.start + min(token_of(row0), span.count), 0);
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int r = row0 + n * 16 + col;
      const int rr = r < rows() ? r : 0, t = token_of(rr);
      s.pos[n] = r < rows() ? position_of(t) : -1;
      const bf16* p = a->q + b * a->qb + (i64)(head * a->group + rr - t * a->group) * a->qh + t * a->qt + 16 * grp;
#pragma unroll
      for (int u = 0; u < 2 * KC; ++u) s.q[n][u] = *(const bf16x8*)(p + u / 2 * 64 + u % 2 * 8);
      s.m[n] = -__builtin_inff(), s.l[n] = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) s.o[d][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // A lane's value scale vs = 2^e g by its bits: 2^e goes to the values, g to the probabilities (and out of their sum
  // again).  Where the lane has no token it is 1.
  static __device__ __forceinline__ unsigned scale_of(const Tokens& k) { return __float_as_uint(k.have ? k.vs : 1.f); }
  static __device__ __forceinline__ float power_of(unsigned bits) {
    return __uint_as_float(max(bits & 0x7f800000u, 0x00800000u));
  }

  // One tile: key(j, u) the K operand of tokens 16 g + 4 j .. + 3, read() what to do once the keys are used, value(d) the
  // codes of column 16 d + col.
  template <class Key, class Read, class Value>
  __device__ __forceinline__ void tile(State& s, int t, const Tokens& k, Key key, Read read, Value value) const {
    f32x4 x[4][NQ];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) x[j][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < 2 * KC; ++u) {
        const bf16x8 y = key(j, u);
#pragma unroll
        for (int n = 0; n < NQ; ++n) x[j][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(y, s.q[n][u], x[j][n], 0, 0, 0);
      }
    }
    const int at = t * wir::TILE + 16 * grp;   // the lane's tokens: at .. at + have - 1
    const bool edge = __builtin_amdgcn_ballot_w64(k.have < 16 || at + 15 > s.low) != 0;
    read();
    const float g = __uint_as_float((scale_of(k) & 0x7fffffu) | 0x3f800000u);
    const float log_g = __builtin_amdgcn_logf(g), inv_g = __builtin_amdgcn_rcpf(g);
    // ks log2(e) / sqrt(D)
    const float scale = (k.have ? k.ks : 1.f) * (float)(1.4426950408889634 / (D == 64 ? 8.0 : 11.313708498984761));
    const float f = edge ? 1.f : scale;
    if (edge) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const int seen = min(k.have, s.pos[n] - at + 1);   // of the lane's tokens
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[j][n][i] = 4 * j + i < seen ? x[j][n][i] * scale : -__builtin_inff();
      }
    }
    float corr[NQ], shift[NQ];
    bool rescale = false;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float top = x[0][n][0];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, x[j][n][i]);
      top = fmaxf(over_groups(top * f, [](float y, float z) { return fmaxf(y, z); }), s.m[n]);
      const float base = top == -__builtin_inff() ? 0.f : top;
      corr[n] = __builtin_amdgcn_exp2f(s.m[n] - base);
      shift[n] = log_g - base;
      s.m[n] = top;
      s.l[n] *= corr[n];
      rescale |= corr[n] != 1.0f;
    }
    if (__builtin_amdgcn_ballot_w64(rescale) != 0) {
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int d = 0; d < DT; ++d) s.o[d][n] *= corr[n];
    }
    bf16x8 p[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(x[j][n][i], f, shift[n]));
          sum[i % 2] += y;
          p[n][j / 2][j % 2 * 4 + i] = (bf16)y;
        }
      s.l[n] += (sum[0] + sum[1]) * inv_g;
    }
    const unsigned bits = scale_of(k);
    const float power = power_of(bits);
    u32x4 v[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) v[d] = value(d);
    if (__builtin_amdgcn_ballot_w64(bits >= 0x7f800000u) != 0) {
#pragma unroll
      for (int d = 0; d < DT; ++d) v[d] = scaled_codes(v[d], bits);
    }
    if (edge) {
      const u32x4 held = held_bytes(k.have);
#pragma unroll
      for (int d = 0; d < DT; ++d) v[d] &= held;
      if (unseen(k.have, at, s.low)) take_nans<DT>(v, col, 16, at);
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bf16x8 w = unpack8(v[d][2 * u], v[d][2 * u + 1], power);
#pragma unroll
        for (int n = 0; n < NQ; ++n) s.o[d][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, p[n][u], s.o[d][n], 0, 0, 0);
      }
  }

  // Value codes past the sequence's end become 0 (0 * NaN is NaN in the product); those of a scale that is no number
  // NaN.  NaN codes of a tile that not all rows see whole are marked instead.
  static __device__ __forceinline__ u32x4 held_bytes(int n) {   // 0xff where a lane's 16 bytes hold a token
    u32x4 m;
#pragma unroll
    for (int w = 0; w < 4; ++w) m[w] = n >= 4 * w + 4 ? ~0u : n <= 4 * w ? 0u : (1u << 8 * (n - 4 * w)) - 1;
    return m;
  }
  static __device__ __forceinline__ u32x4 nan_codes(const u32x4& v) {   // 0xff where a byte is 0x7f or 0xff
    return ((((v & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu;
  }
  static __device__ __forceinline__ u32x4 scaled_codes(const u32x4& v, unsigned bits) {
    return bits >= 0x7f800000u ? u32x4{0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu} : v;
  }
  // Whether some held token of the tile may be seen by one row and not by another (never with one new token).
  static __device__ __forceinline__ bool unseen(int have, int at, int low) {
    return __builtin_amdgcn_ballot_w64(have > 0 && at + have - 1 > low) != 0;
  }
  // NaN codes out of the lane's tokens at .. of columns from, from + step, ..: a row that sees one of a column's is NaN
  // there, which is so from the first of them on, so that is all `store` has to know.
  template <int N>
  __device__ __forceinline__ void take_nans(u32x4 (&v)[N], int from, int step, int at) const {
    u32x4 some = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < N; ++i) some |= nan_codes(v[i]);
    if (__builtin_amdgcn_ballot_w64((some[0] | some[1] | some[2] | some[3]) != 0) == 0) return;
    sh.nan_any = 1;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const u32x4 n = nan_codes(v[i]);
#pragma unroll
      for (int w = 3; w >= 0; --w)
        if (n[w]) atomicMin(&sh.nan_from[from + step * i], at + 4 * w + __builtin_ctz(n[w]) / 8);
      v[i] &= ~n;
    }
  }

  // Addresses of a head's pages: a lane's place in page 0, and what a page and a place in it add.
  struct Bases {
    const float *ks, *vs;
    const unsigned char *k, *v;
    const int* table;
    int page_bytes, page_scales, shift, pages;
  };
  __device__ __forceinline__ Bases bases(int head) const {
    Bases x;
    x.ks = a->k_scale + head;
    x.vs = a->v_scale + head;
    x.page_scales = a->heads;
    x.page_bytes = (a->heads * D) << a->page_shift;
    x.shift = a->page_shift;
    x.pages = a->pages;
    x.table = a->table + b * a->tb;
    x.k = a->k + (((i64)head << a->page_shift) + col % 4) * D + 16 * grp;
    x.v = a->v + (((i64)head * D + col) << a->page_shift);
    return x;
  }
  // Page id of the tile's 16-token segment `seg`; -1 past the sequence.
  __device__ __forceinline__ int page_of(const Bases& x, int t, int seg) const {
    const int at = t * wir::TILE + 16 * seg;
    return at < span.held ? x.table[at >> x.shift] : -1;
  }
  // (a page that is none is read as page 0, and its tokens masked)
  static __device__ __forceinline__ i64 page_index(const Bases& x, int page) {
    return max(wir::checked_page(page, x.pages), 0);
  }
  static __device__ __forceinline__ int in_page(const Bases& x, int t, int seg) {
    return (t * wir::TILE + 16 * seg) & ((1 << x.shift) - 1);
  }

  // Segment `seg` of a tile, which the lane has scores of.
  __device__ __forceinline__ void scales_of(Tokens& k, const Bases& x, int t, int seg, int page) const {
    const i64 at = page_index(x, page) * x.page_scales;
    k.have = wir::checked_page(page, x.pages) < 0 ? 0 : min(max(span.held - (t * wir::TILE + 16 * seg), 0), 16);
    k.ks = x.ks[at];   // (of page 0 where there is none: `tile` sees to it, after the loads' time)
    k.vs = x.vs[at];
  }
  __device__ __forceinline__ const unsigned char* key_at(const Bases& x, int t, int page) const {
    return x.k + page_index(x, page) * x.page_bytes + in_page(x, t, col / 4) * D;
  }
  __device__ __forceinline__ const unsigned char* value_at(const Bases& x, int t, int page) const {
    return x.v + page_index(x, page) * x.page_bytes + in_page(x, t, grp);
  }

  // Tiles first .. last - 1 of `head`, every WK-th from the wave's, through registers: K of the next tile is in
  // flight during the softmax and the second product, V during the next tile's first product.
  __device__ __forceinline__ void walk_registers(State& s, int head, int first, int last) const {
    const Bases at = bases(head);
    const i64 v_step = (i64)16 << at.shift;
    u32x4 kf[4][KC], vf[DT];
    Tokens tok;
    const unsigned char* vp;
    auto load_k = [&](int t, int page_k, int page_v) {
      scales_of(tok, at, t, grp, page_v);
      const unsigned char* kp = key_at(at, t, page_k);
      vp = value_at(at, t, page_v);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int x = 0; x < KC; ++x) kf[j][x] = *(const u32x4*)(kp + 4 * j * D + 64 * x);
    };
    auto load_v = [&]() {
#pragma unroll
      for (int d = 0; d < DT; ++d) vf[d] = *(const u32x4*)(vp + d * v_step);
    };
    int t = first + wk, next_k = -1, next_v = -1;
    if (t < last) {
      load_k(t, page_of(at, t, col / 4), page_of(at, t, grp));
      if (t + WK < last) next_k = page_of(at, t + WK, col / 4), next_v = page_of(at, t + WK, grp);
      load_v();
    }
    begin(s, head);
    for (; t < last; t += WK) {
      const Tokens now = tok;
      tile(s, t, now,
           [&](int j, int u) { return unpack8(kf[j][u / 2][u % 2 * 2], kf[j][u / 2][u % 2 * 2 + 1], 1.f); },
           [&]() {
             if (t + WK >= last) return;
             const int page_k = next_k, page_v = next_v;
             if (t + 2 * WK < last) next_k = page_of(at, t + 2 * WK, col / 4), next_v = page_of(at, t + 2 * WK, grp);
             load_k(t + WK, page_k, page_v);
           },
           [&](int d) { return vf[d]; });
      if (t + WK < last) load_v();
    }
  }

  // Through LDS: 32 rows a wave on 32x32x16 products, every tile for all waves.  A lane has the scores of row lane % 32
  // and, with h = lane / 32, tokens 32 j + 16 h .. + 15 of the tile for j = 0, 1: K's rows come in the order that puts
  // those into the lane's 16 registers of product j one after another.
  struct Rows {
    bf16x8 q[D / 16];
    int pos, low;
    f32x16 o[D / 32];
    float m, l;
  };
  static __device__ __forceinline__ float max_of_halves(float x) {
    auto z = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(z[0]), __uint_as_float(z[1]));
  }

  __device__ __forceinline__ void begin(Rows& s, int head) const {
    const int row0 = rb * BLOCK + wr * ROWS, r = row0 + lane % 32, rr = r < rows() ? r : 0, t = token_of(rr);
    s.low = max(span.start + min(token_of(row0), span.count), 0);
    s.pos = r < rows() ? position_of(t) : -1;
    const bf16* p = a->q + b * a->qb + (i64)(head * a->group + rr - t * a->group) * a->qh + t * a->qt + lane / 32 * 16;
#pragma unroll
    for (int u = 0; u < D / 16; ++u) s.q[u] = *(const bf16x8*)(p + u / 2 * 32 + u % 2 * 8);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) s.o[d][i] = 0.f;
    s.m = -__builtin_inff(), s.l = 0.f;
    // (they are here before the loop, or its waits for them would count the loop's own loads)
#pragma unroll
    for (int u = 0; u < D / 16; ++u) asm volatile("" : "+v"(s.q[u]));
  }

  // Reads of N fragments, a few ahead of the products that use them.
  template <int N>
  static __device__ __forceinline__ void fragments_ahead() {
    constexpr int AHEAD = 8;
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
    for (int i = 0; i < N - AHEAD; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, AHEAD, 0);
  }

  // One tile, its operands at `from`: K's (j, u) and then V's (j, d, m).
  __device__ __forceinline__ void tile(Rows& s, int t, const Tokens (&k)[2], const lds_bf16x8* from) const {
    constexpr int U = D / 16, V = D / 32;
    f32x16 x[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) x[j][i] = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        x[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(from[(j * U + u) * 64], s.q[u], x[j], 0, 0, 0);
    fragments_ahead<2 * U>();
    const int at = t * wir::TILE + lane / 32 * 16;   // the lane's tokens: at + 32 j .. + have[j] - 1
    const bool edge = __builtin_amdgcn_ballot_w64(k[0].have < 16 || k[1].have < 16 || at + 47 > s.low) != 0;
    float f[2], log_g[2], inv_g[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float g = __uint_as_float((scale_of(k[j]) & 0x7fffffu) | 0x3f800000u);
      log_g[j] = __builtin_amdgcn_logf(g), inv_g[j] = __builtin_amdgcn_rcpf(g);
      // ks log2(e) / sqrt(D)
      f[j] = (k[j].have ? k[j].ks : 1.f) * (float)(1.4426950408889634 / (D == 64 ? 8.0 : 11.313708498984761));
    }
    if (edge) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int seen = min(k[j].have, s.pos - (at + 32 * j) + 1);   // of the lane's tokens
#pragma unroll
        for (int i = 0; i < 16; ++i) x[j][i] = i < seen ? x[j][i] * f[j] : -__builtin_inff();
        f[j] = 1.f;
      }
    }
    float top[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      top[j] = x[j][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) top[j] = fmaxf(top[j], x[j][i]);
    }
    float m = fmaxf(top[0] * f[0], top[1] * f[1]);
    m = fmaxf(max_of_halves(m), s.m);
    const float base = m == -__builtin_inff() ? 0.f : m, corr = __builtin_amdgcn_exp2f(s.m - base);
    s.m = m;
    s.l *= corr;
    if (__builtin_amdgcn_ballot_w64(corr != 1.0f) != 0) {
#pragma unroll
      for (int d = 0; d < V; ++d) s.o[d] *= corr;
    }
    bf16x8 p[2][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float sum[2] = {0.f, 0.f};
      const float shift = log_g[j] - base;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(x[j][i], f[j], shift));
        sum[i % 2] += y;
        p[j][i / 8][i % 8] = (bf16)y;
      }
      s.l += (sum[0] + sum[1]) * inv_g[j];
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int d = 0; d < V; ++d)
          s.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(from[(2 * U + 2 * (j * V + d) + m) * 64], p[j][m], s.o[d], 0, 0, 0);
    fragments_ahead<4 * V>();
  }

  // In each iteration a wave asks for its quarter of the next tile (K or V of 32 tokens), computes, and leaves what came
  // as operands in the other slot.  WIDE: a tile's page and addresses are the wave's, and a lane adds its place (pages of
  // 64 tokens, 32/8 heads, this way / by lanes' own addresses: 277 / 291 us for 2 x 1000 over 8192, 308 / 334 for 2 x 2048
  // over 8192 at D = 64).
  __device__ __forceinline__ void walk_shared(Rows& s, int head, int first, int last) const {
    constexpr int MINE = CHUNKS / WR, V = D / 32;
    const bool mine_k = wr < 2;
    const int half = wr % 2, h = lane / 32, r = lane % 32;
    // K: row r of the operand is token 16 (r / 4 % 2) + 4 (r / 8) + r % 4, bytes 32 i + 16 h; V: column 32 i + r, token 16 h
    const int mine_h = mine_k ? r / 4 % 2 : h, token = 16 * mine_h + (mine_k ? 4 * (r / 8) + r % 4 : 0);
    const Bases at = bases(head);
    const unsigned char* head_at = mine_k ? a->k + (((i64)head << at.shift) * D) : a->v + (((i64)head * D) << at.shift);
    const int token_bytes = mine_k ? D : 1, chunk_bytes = mine_k ? 32 : 32 << at.shift;
    // the lane's place: WIDE in a tile, else in a segment
    const unsigned lane_at = mine_k ? ((WIDE ? 32 * half + token : token % 16) * D + 16 * h)
                                    : (r << at.shift) + (WIDE ? 32 * half + token : 0);
    char* ring = sh.ring + wk * 2 * CHUNKS * 2048;
    u32x4 codes[MINE];
    Tokens tok[2];
    auto ask = [&](int t, const int (&page)[3]) {   // of segments h and 2 + h, and of the lane's own codes
      const unsigned char* from;
      if constexpr (WIDE) {
        const int id = __builtin_amdgcn_readfirstlane(page[0]);
        from = head_at + page_index(at, id) * at.page_bytes + in_page(at, t, 0) * token_bytes;
        scales_of(tok[0], at, t, h, id);
        tok[1] = tok[0];
        tok[1].have = wir::checked_page(id, at.pages) < 0 ? 0 : min(max(span.held - (t * wir::TILE + 16 * (2 + h)), 0), 16);
      } else {
        from = head_at + page_index(at, page[2]) * at.page_bytes + in_page(at, t, 2 * half + mine_h) * token_bytes;
        scales_of(tok[0], at, t, h, page[0]);
        scales_of(tok[1], at, t, 2 + h, page[1]);
      }
#pragma unroll
      for (int i = 0; i < MINE; ++i) codes[i] = *(const u32x4*)(from + i * chunk_bytes + lane_at);
    };
    auto pages_of = [&](int (&page)[3], int t) {
      page[0] = page_of(at, t, WIDE ? 0 : h);
      if constexpr (!WIDE) page[1] = page_of(at, t, 2 + h), page[2] = page_of(at, t, 2 * half + mine_h);
    };
    const int low = max(span.start + min(token_of(rb * BLOCK), span.count), 0);   // of all waves' rows
    auto leave = [&](int t, int slot) {
      float power = 1.f;
      if (!mine_k) {
        const Tokens mine = {0.f, half ? tok[1].vs : tok[0].vs, half ? tok[1].have : tok[0].have};   // (not by an index)
        const unsigned bits = scale_of(mine);
        power = power_of(bits);
        const int first_token = t * wir::TILE + 32 * half + 16 * h;
        if (__builtin_amdgcn_ballot_w64(bits >= 0x7f800000u || mine.have < 16 || first_token + 15 > low) != 0) {
          const u32x4 held = held_bytes(mine.have);
#pragma unroll
          for (int i = 0; i < MINE; ++i) codes[i] = scaled_codes(codes[i], bits) & held;
          if (unseen(mine.have, first_token, low)) take_nans<MINE>(codes, r, 32, first_token);
        }
      }
      lds_bf16x8* to = (lds_bf16x8*)wir::lds(ring + (slot * CHUNKS + wr * MINE) * 2048) + lane;
#pragma unroll
      for (int i = 0; i < MINE; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) to[(2 * i + u) * 64] = unpack8(codes[i][2 * u], codes[i][2 * u + 1], power);
    };
    static_assert(MINE == V, "");
    int next[3] = {-1, -1, -1}, slot = 0;
    const int start = first + wk;
    if (start < last) {
      pages_of(next, start);
      ask(start, next);
      pages_of(next, start + WK);
    }
    begin(s, head);
    if (start < last) leave(start, 0);
    for (int t = start; t < last + wk; t += WK, slot ^= 1) {   // (as often for all waves)
      __syncthreads();
      if (WK > 1 && t >= last) break;
      const Tokens now[2] = {tok[0], tok[1]};
      ask(t + WK, next);
      pages_of(next, t + 2 * WK);   // (past the end -1, or pages not used)
      tile(s, t, now, (const lds_bf16x8*)wir::lds(ring + slot * CHUNKS * 2048) + lane);
      if (t + WK < last) leave(t + WK, slot ^ 1);
    }
    __syncthreads();   // the ring is read: results go there
  }

  // Tiles first .. last - 1 of `head` -> sh.r
  __device__ __forceinline__ void walk(int head, int first, int last) {
    if constexpr (SHARED) {
      Rows s;
      walk_shared(s, head, first, last);
      const int row = wave * ROWS + lane % 32, h = lane / 32;
      auto l = __builtin_amdgcn_permlane32_swap(__float_as_uint(s.l), __float_as_uint(s.l), false, false);
      if (h == 0) sh.r.ml[2 * row] = s.m, sh.r.ml[2 * row + 1] = __uint_as_float(l[0]) + __uint_as_float(l[1]);
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *(f32x4*)(sh.r.o + row * PITCH + 32 * d + 8 * g + 4 * h) =
              f32x4{s.o[d][4 * g], s.o[d][4 * g + 1], s.o[d][4 * g + 2], s.o[d][4 * g + 3]};
    } else {
      State s;
      walk_registers(s, head, first, last);
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const float sum = over_groups(s.l[n], [](float x, float y) { return x + y; });
        const int row = wave * ROWS + n * 16 + col;
        if (grp == 0) sh.r.ml[2 * row] = s.m[n], sh.r.ml[2 * row + 1] = sum;
#pragma unroll
        for (int d = 0; d < DT; ++d) *(f32x4*)(sh.r.o + row * PITCH + 16 * d + 4 * grp) = s.o[d][n];
      }
    }
  }

  // The waves' results of a block, joined: the outputs, or the partial result of `slot`.
  __device__ __forceinline__ void store(int head, int slot) {
    constexpr int CH = D / 8;
    const int left = min(rows() - rb * BLOCK, BLOCK);
    for (int idx = threadIdx.x; idx < left * CH; idx += 64 * W) {
      const int row = idx / CH, ch = idx % CH;
      float top = -__builtin_inff();
#pragma unroll
      for (int w = 0; w < WK; ++w) top = fmaxf(top, sh.r.ml[2 * (w * BLOCK + row)]);
      const float base = top == -__builtin_inff() ? 0.f : top;
      float sum = 0.f;
      f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        const int at = w * BLOCK + row;
        const float f = __builtin_amdgcn_exp2f(sh.r.ml[2 * at] - base);
        sum += f * sh.r.ml[2 * at + 1];
        x += f * *(const f32x4*)(sh.r.o + at * PITCH + 8 * ch);
        y += f * *(const f32x4*)(sh.r.o + at * PITCH + 8 * ch + 4);
      }
      const int pos = position_of(token_of(rb * BLOCK + row));
      if (sh.nan_any) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (sh.nan_from[8 * ch + i] <= pos) x[i] = __builtin_nanf("");
          if (sh.nan_from[8 * ch + 4 + i] <= pos) y[i] = __builtin_nanf("");
        }
      }
      if (pos < 0) {   // it took part in tiles that every row with a position sees
        top = -__builtin_inff(), sum = 0.f;
        x = y = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      if (slot >= 0) {
        float* to = a->partial + ((i64)slot * BLOCK + row) * D + 8 * ch;
        *(f32x4*)to = x;
        *(f32x4*)(to + 4) = y;
        if (ch == 0)
          *(f32x2*)(a->partial + (i64)wir::slots_for(a->extra) * BLOCK * D + ((i64)slot * BLOCK + row) * 2) = f32x2{top, sum};
      } else {
        put(a, b, head, rb * BLOCK + row, ch, x, y, top, sum);
      }
    }
  }

  // 8 columns of a row's output and, with the first of them, its LSE; a row that sees nothing: 0 and -inf.
  static __device__ __forceinline__ void put(args_ptr a, int b, int head, int r, int ch, const f32x4& x,
                                             const f32x4& y, float top, float sum) {
    const int t = a->tokens == 1 ? 0 : r / a->group;
    const i64 h = head * a->group + r - t * a->group;
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    bf16x8 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (bf16)(x[i] * inv), v[4 + i] = (bf16)(y[i] * inv);
    *(bf16x8*)(a->out + b * a->ob + h * a->oh + t * a->ot + 8 * ch) = v;
    if (ch == 0)
      a->lse[b * a->lb + h * a->lh + t * a->lt] =
          sum == 0.f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(sum)) * kLn2;
  }

  // Program -> (sequence and head, block) without a division of the work; later blocks see more keys.
  // A head's blocks are next to one another on one XCD, the longest first, and a sequence's heads on all of them.  Where
  // all programs run at once, two a CU, the second ones come in the opposite order, so that a CU has a long and a short
  // one; many blocks of 128 rows go block length by block length; those of one or two heads are dealt over the XCDs, for
  // each to have long ones.  us, the blocks in turn with consecutive heads on an XCD / so, D = 128: 4096 queries over
  // 4096 keys (16/8 heads) 111 / 103, 2 x 1000 over 8192 (32/8) 285 / 281; 4 x 2048 over 2048 (32/8) 192 / 180, 4096 over
  // 4096 (24/12) 167 / 135; 8000 over 8000 (8/1) 245 / 180; 8 x 200 over up to 3000 (32/8) 104 / 77, 12 x 1024 over up to
  // 2048 (16/8) 163 / 142.  Elsewhere they cost: by length just past two a CU (3 x 700 over 3000, 32/8) 143 / 146 and where
  // a head has few blocks (64 x 100 over 2000, 32/8) 327 / 351, dealt for more heads (5 x 40 over 2000, 24/6) 30.7 / 31.9.
  __device__ __forceinline__ void in_turn(int& item, int& block) const {
    int id = blockIdx.x;
    const int total = gridDim.x;
    const int heads = a->batch * a->heads;
    if (SHARED && total >= 768 && a->blocks >= 8) {
      wir::longest_first<true, 2048>(id, a->blocks, heads, block, item);
      if (heads % 8 == 0 && total <= 2048) item = item % (heads / 8) * 8 + item / (heads / 8);   // (one range of heads)
      return;
    }
    const bool whole = heads > 2;   // a head on one XCD
    const int step = whole ? 8 : 1, per = total / step, half = min(256 / step, per);   // (the first on every CU)
    if (total <= 512 && id >= step * half && id < step * per) id = step * (per - 1 - (id / step - half)) + id % step;
    const bool spread = whole && heads % 8 == 0;
    const int xcd = id % 8;
    if (spread)
      id /= 8;
    else if (whole)
      id = wir::remap_xcd(id, total);
    item = id / a->blocks;
    block = a->blocks - 1 - (id - item * a->blocks);
    if (spread) item = 8 * item + xcd;
  }

  __device__ __forceinline__ Plan plan() const {
    Plan w;
    w.first = 0, w.slot = -1;
    if (!a->extra) {
      if (a->blocks == 1) {
        const int id = blockIdx.x;
        w.pair = id / a->heads;
        w.head = id - w.pair * a->heads;
      } else {
        int item, block;
        in_turn(item, block);
        const int seq = item / a->heads;
        w.head = item - seq * a->heads;
        w.pair = seq * a->blocks + block;
      }
      w.span = span_at(sequence_of(w.pair));
      w.last = wir::block_tiles(keys_of(w.span, w.pair));
      return w;
    }
    // a lane takes `each` pairs
    const int pairs = a->batch * a->blocks, each = (pairs + 63) / 64, from = lane * each, to = min(from + each, pairs);
    auto units_of = [&](int p) { return wir::block_units(keys_of(span_at(sequence_of(p)), p)); };
    int units = 0, parts = 0;
    for (int p = from; p < to; ++p) units += units_of(p);
    const int units_to = a->heads * (pairs == 1 ? units : wave_scan(units));
    const int share = wir::share_of(__builtin_amdgcn_readlane(units_to, pairs == 1 ? 0 : 63), a->extra, a->least);
    for (int p = from; p < to; ++p) parts += wir::parts_of(units_of(p), share);
    const int parts_to = a->heads * (pairs == 1 ? parts : wave_scan(parts));
    // the program's pair, and the units and parts before it
    const int id = blockIdx.x;
    const unsigned long long past = __builtin_amdgcn_ballot_w64(lane < pairs && id < parts_to);
    if (past == 0) {
      w.pair = -1;
      return w;
    }
    const int src = __builtin_ctzll(past);
    int p = from, units_before = units_to - a->heads * units, parts_before = parts_to - a->heads * parts;
    if (lane == src) {
      for (; p + 1 < to; ++p) {
        const int u = units_of(p), n = a->heads * wir::parts_of(u, share);
        if (id < parts_before + n) break;
        parts_before += n, units_before += a->heads * u;
      }
    }
    w.pair = __builtin_amdgcn_readlane(p, src);
    units_before = __builtin_amdgcn_readlane(units_before, src);
    parts_before = __builtin_amdgcn_readlane(parts_before, src);
    w.span = span_at(sequence_of(w.pair));
    const int keys = keys_of(w.span, w.pair);
    units = wir::block_units(keys);
    parts = wir::parts_of(units, share);
    w.head = min((id - parts_before) / parts, a->heads - 1);
    const int n = min(id - parts_before - w.head * parts, parts - 1), width = wir::slot_width(share);
    const int begin = units_before + w.head * units;
    w.first = wir::part_begin(n, units, parts);
    w.last = min(wir::part_begin(n + 1, units, parts), wir::block_tiles(keys));
    if (parts > 1) w.slot = wir::slot_of(begin + w.first, width, a->extra);
    if (lane == 0 && n == 0) {
      int* info = a->info + 4 * ((i64)w.pair * a->heads + w.head);
      info[0] = begin, info[1] = units, info[2] = parts, info[3] = width;
    }
    return w;
  }

  __device__ __forceinline__ void run() {
    if (wave == 0) {
      const Plan w = plan();
      for (int d = lane; d < D; d += 64) sh.nan_from[d] = 0x7fffffff;
      if (lane == 0) sh.plan = w, sh.nan_any = 0;
    }
    __syncthreads();
    auto read = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    const int pair = read(sh.plan.pair);
    if (pair < 0) return;
    const int head = read(sh.plan.head), slot = read(sh.plan.slot);
    b = sequence_of(pair);
    rb = pair - b * a->blocks;
    span = wir::Span{read(sh.plan.span.start), read(sh.plan.span.count), read(sh.plan.span.held)};
    walk(head, read(sh.plan.first), read(sh.plan.last));
    __syncthreads();
    a = fresh(a);
    store(head, slot);
  }
};

// Partial results of a head's rows, joined in the order of their tiles: a
// workgroup takes one row, its waves' lanes reading 1024 / D partial results
// side by side, or, for launches with many rows and so few partial results
// of each, one row a wave (ROWS = 4).
template <int D, int BLOCK, int ROWS>
__device__ __forceinline__ void join(args_ptr a) {
  constexpr int CH = D / 4, PER = 256 / ROWS / CH, EARLY = 4;   // lanes of a row; partial results read side by side
  __shared__ f32x4 sums[256];
  __shared__ float ls[ROWS * PER];
  const int per = (min(a->tokens * a->group, BLOCK) + ROWS - 1) / ROWS;   // programs of an item
  const int item = blockIdx.x / per, sub = ROWS == 1 ? 0 : wir::wave_id(), lane = threadIdx.x % (256 / ROWS);
  const int row = (blockIdx.x - item * per) * ROWS + sub;
  const int* info = a->info + 4 * (i64)item;
  const int begin = info[0], units = info[1], parts = min(info[2], wir::slots_for(a->extra)), width = max(info[3], 1);
  if (parts <= 1) return;
  const int pair = item / a->heads, head = item - pair * a->heads, b = pair / a->blocks, rb = pair - b * a->blocks;
  const int r = rb * BLOCK + row;
  const bool mine = row < BLOCK && r < a->tokens * a->group;
  const f32x2* ml = (const f32x2*)(a->partial + (i64)wir::slots_for(a->extra) * BLOCK * D);
  auto place = [&](int p) { return (i64)wir::slot_of(begin + wir::part_begin(p, units, parts), width, a->extra) * BLOCK + row; };
  const int ch = lane % CH, w = lane / CH;
  float top = -__builtin_inff(), l = 0.f;
  if (mine) {
    // the first partial results are on their way while their maxima are compared
    f32x4 early[EARLY];
    f32x2 early_ml[EARLY];
#pragma unroll
    for (int i = 0; i < EARLY; ++i) {
      const i64 at = place(min(w + i * PER, parts - 1));
      early_ml[i] = ml[at];
      early[i] = *(const f32x4*)(a->partial + at * D + 4 * ch);
    }
    for (int p = wir::lane_id(); p < parts; p += 64) top = fmaxf(top, ml[place(p)][0]);   // every wave for itself
#pragma unroll
    for (int d = 1; d < 16; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
    top = over_groups(top, [](float x, float y) { return fmaxf(x, y); });
    const float base = top == -__builtin_inff() ? 0.f : top;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](const f32x2& y, const f32x4& z) {
      const float f = __builtin_amdgcn_exp2f(y[0] - base);
      l += f * y[1];
      x += f * z;
    };
#pragma unroll
    for (int i = 0; i < EARLY; ++i)
      if (w + i * PER < parts) add(early_ml[i], early[i]);
#pragma unroll 4
    for (int p = w + EARLY * PER; p < parts; p += PER) {
      const i64 at = place(p);
      add(ml[at], *(const f32x4*)(a->partial + at * D + 4 * ch));
    }
    sums[threadIdx.x] = x;
    if (ch == 0) ls[sub * PER + w] = l;
  }
  __syncthreads();
  if (lane >= D / 8 || !mine) return;
  f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
  l = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    lo += sums[sub * (256 / ROWS) + i * CH + 2 * lane];
    hi += sums[sub * (256 / ROWS) + i * CH + 2 * lane + 1];
    l += ls[sub * PER + i];
  }
  Program<D, 1, 1, 1>::put(a, b, head, r, lane, lo, hi, top, l);
}

}  // namespace

#define ATTN_KERNEL(NAME, D, NQ, WR, W, OCC, WIDE)                                                        \
  extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(64 * W, 64 * W),                  \
                                            amdgpu_waves_per_eu(OCC, OCC))) NAME(const attn_args) {       \
    __shared__ __attribute__((aligned(1024))) Program<D, NQ, WR, W, WIDE>::Shared shared;                 \
    Program<D, NQ, WR, W, WIDE>((args_ptr)__builtin_amdgcn_kernarg_segment_ptr(), shared).run();          \
  }
#define JOIN_KERNEL(NAME, D, BLOCK, ROWS)                                             \
  extern "C" __global__ void __launch_bounds__(256) NAME(const attn_args) {           \
    join<D, BLOCK, ROWS>((args_ptr)__builtin_amdgcn_kernarg_segment_ptr());           \
  }

ATTN_KERNEL(wir_attn_cached_d64_r16, 64, 1, 1, 4, 4, false)
ATTN_KERNEL(wir_attn_cached_d64_r16_w2, 64, 1, 1, 2, 4, false)
ATTN_KERNEL(wir_attn_cached_d64_r16_w8, 64, 1, 1, 8, 4, false)
ATTN_KERNEL(wir_attn_cached_d128_r16_w2, 128, 1, 1, 2, 2, false)
ATTN_KERNEL(wir_attn_cached_d128_r16_w8, 128, 1, 1, 8, 2, false)
ATTN_KERNEL(wir_attn_cached_d64_r32_w2, 64, 2, 1, 2, 2, false)
ATTN_KERNEL(wir_attn_cached_d64_r32_w8, 64, 2, 1, 8, 2, false)
ATTN_KERNEL(wir_attn_cached_d64_r32, 64, 2, 1, 4, 2, false)
ATTN_KERNEL(wir_attn_cached_d64_r128, 64, 2, 4, 4, 3, false)
ATTN_KERNEL(wir_attn_cached_d64_r128_w8, 64, 2, 4, 8, 2, false)
ATTN_KERNEL(wir_attn_cached_d64_r128_w8_p64, 64, 2, 4, 8, 2, true)
ATTN_KERNEL(wir_attn_cached_d64_r128_p64, 64, 2, 4, 4, 3, true)   // pages of 64 tokens or more
ATTN_KERNEL(wir_attn_cached_d128_r16, 128, 1, 1, 4, 2, false)
ATTN_KERNEL(wir_attn_cached_d128_r32_w2, 128, 2, 1, 2, 2, false)
ATTN_KERNEL(wir_attn_cached_d128_r32, 128, 2, 1, 4, 2, false)
ATTN_KERNEL(wir_attn_cached_d128_r128, 128, 2, 4, 4, 2, false)
ATTN_KERNEL(wir_attn_cached_d128_r128_w8, 128, 2, 4, 8, 2, false)
ATTN_KERNEL(wir_attn_cached_d128_r128_w8_p64, 128, 2, 4, 8, 2, true)
ATTN_KERNEL(wir_attn_cached_d128_r128_p64, 128, 2, 4, 4, 2, true)   // pages of 64 tokens or more
JOIN_KERNEL(wir_attn_join_d64_r16, 64, 16, 1)
JOIN_KERNEL(wir_attn_join_d64_r32, 64, 32, 1)
JOIN_KERNEL(wir_attn_join_d64_r128, 64, 128, 1)
JOIN_KERNEL(wir_attn_join_d64_r128_w4, 64, 128, 4)
JOIN_KERNEL(wir_attn_join_d128_r16, 128, 16, 1)
JOIN_KERNEL(wir_attn_join_d128_r32, 128, 32, 1)
JOIN_KERNEL(wir_attn_join_d128_r128, 128, 128, 1)
JOIN_KERNEL(wir_attn_join_d128_r128_w4, 128, 128, 4)
