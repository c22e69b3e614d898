// attn_cached.hip -- attention of new queries over a paged cache of e4m3
// codes (warpir_amd.api.attention_cached; kv_cache.hip writes the cache).
//
// A token's key is k = code * ks and its value v = code * vs, ks and vs one
// scale for each page and head.  For query row r at position p:
//   s_j = q . code_j * ks / sqrt(D) for j <= p,  O = sum_j softmax(s)_j vs code_j.
// The scales stay out of the products: ks multiplies a score, vs a
// probability (before its rounding to bf16), and e4m3 codes are exact in bf16,
// so the products run on v_mfma_f32_16x16x32_bf16 with codes as they are.
//
// Both products are taken transposed, S^T = K Q^T and O^T = V^T P^T, with 16
// query rows (the heads that share a key/value head, and the new tokens) as
// the columns.  A lane then holds scores of one query row, and its 16 of a
// 64-token tile are turned into the second product's operand without leaving
// the lane: the rows of K go to the matrix core in an order that gives lane
// group g (16 lanes) the tokens 16 g .. 16 g + 15.  V pages are [D, token], so
// that operand's other side is 16 contiguous bytes of one column.  K and V
// come from memory straight into registers, every byte once, with no LDS and
// no barrier in the loop: K of the next tile is in flight during the softmax
// and the second product, V during the next tile's first product.
//
// What bounds it: the cache's bytes for few rows (a decode step).
#include <hip/hip_runtime.h>

#include "wir_pages.h"

namespace {

using wir::i64;

typedef __bf16 bf16;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int WAVES = 4;
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
  int* info;                   // [items][2]: slot of the first partial result, how many
  i64 qb, qh, qt, ob, oh, ot, lb, lh, lt, tb;
  int batch, heads, group, tokens, page_shift, pages, columns;
  int blocks;                  // row blocks of a sequence and head
  int programs, least;         // 0: one program for each (sequence, block, head)
};

// The eight codes of two words in bf16 (exact).
__device__ __forceinline__ bf16x8 unpack8(unsigned a, unsigned b) {
  const bf16x2 w = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false);
  const bf16x2 x = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
  const bf16x2 y = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false);
  const bf16x2 z = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
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

// One of a sequence's row blocks of one head, over some of its tiles.
template <int D, int NQ, int WR>
struct Program {
  static constexpr int WK = WAVES / WR;          // waves that divide the tiles
  static constexpr int ROWS = 16 * NQ;           // query rows of a wave
  static constexpr int BLOCK = ROWS * WR;        // and of the workgroup
  static constexpr int KC = D / 64, DT = D / 16, PITCH = D + 4;

  struct Shared {
    float o[WAVES * ROWS * PITCH];
    float ml[WAVES * ROWS * 2];
    i64 scan[256];
    i64 found_base;
    int found;
  };

  const attn_args& a;
  Shared& sh;
  int lane, col, grp, wr, wk;
  // the pair's
  int b, rb;
  wir::Span span;

  __device__ __forceinline__ Program(const attn_args& args, Shared& shared) : a(args), sh(shared) {
    lane = threadIdx.x % 64;
    col = lane % 16;
    grp = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    wr = wave % WR;
    wk = wave / WR;
  }

  __device__ __forceinline__ int rows() const { return a.tokens * a.group; }

  __device__ __forceinline__ wir::Span span_at(int seq) const {
    return wir::span_of(a.lengths[seq], a.counts ? a.counts[seq] : a.tokens, a.tokens, a.columns << a.page_shift);
  }
  __device__ __forceinline__ int keys_at(int pair) const {
    return wir::block_keys(span_at(pair / a.blocks), pair % a.blocks, BLOCK, rows(), a.group);
  }

  // Position that row r of the pair sees up to; -1: none.
  __device__ __forceinline__ int position(int r) const {
    const int t = r / a.group;
    return r < rows() && t < span.count ? max(span.start + t, -1) : -1;
  }

  struct Page {      // of a lane's 16 tokens of a tile
    int k, v;        // ids for the K operand's rows and for the scores and V, -1: none
  };

  __device__ __forceinline__ Page pages_of(int tile) const {
    const int* row = a.table + b * a.tb;
    const int tk = tile * wir::TILE + 16 * (col / 4), tv = tile * wir::TILE + 16 * grp;
    Page p;
    p.k = tk < span.held ? row[tk >> a.page_shift] : -1;
    p.v = tv < span.held ? row[tv >> a.page_shift] : -1;
    return p;
  }

  // Tiles first .. last - 1 of `head`; -> sh.o, sh.ml.
  __device__ __forceinline__ void walk(int head, int first, int last) {
    const int mask = (1 << a.page_shift) - 1;
    const float c = (float)(1.4426950408889634 / (D == 64 ? 8.0 : 11.313708498984761));   // log2(e) / sqrt(D)
    const int row0 = rb * BLOCK + wr * ROWS;
    // q: the operand's k order is that of K's 16-byte loads
    bf16x8 q[NQ][2 * KC];
    int pos[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int r = row0 + n * 16 + col;
      pos[n] = position(r);
      const int rr = r < rows() ? r : 0, t = rr / a.group;
      const bf16* p = a.q + b * a.qb + (i64)(head * a.group + rr - t * a.group) * a.qh + t * a.qt + 16 * grp;
#pragma unroll
      for (int u = 0; u < 2 * KC; ++u) q[n][u] = *(const bf16x8*)(p + u / 2 * 64 + u % 2 * 8);
    }
    const int low = max(span.start + min(row0 / a.group, span.count), 0);   // no row that sees anything sees less
    f32x4 o[DT][NQ];
    float m[NQ], l[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      m[n] = -__builtin_inff(), l[n] = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    u32x4 kf[4][KC], vf[DT];
    float ks, vs;
    int there;               // of the lane group's 16 tokens, how many the sequence holds
    const unsigned char* vp;
    auto load_k = [&](int tile, const Page& p) {
      const int tk = tile * wir::TILE + 16 * (col / 4), tv = tile * wir::TILE + 16 * grp;
      const int ik = max(wir::checked_page(p.k, a.pages), 0), iv = wir::checked_page(p.v, a.pages);
      there = iv < 0 ? 0 : min(max(span.held - tv, 0), 16);
      const i64 index_k = (i64)ik * a.heads + head, index_v = (i64)max(iv, 0) * a.heads + head;
      ks = iv < 0 ? 0.f : a.k_scale[index_v] * c;
      vs = iv < 0 ? 0.f : a.v_scale[index_v];
      const unsigned char* kp = a.k + ((index_k << a.page_shift) + (tk & mask) + col % 4) * D + 16 * grp;
      vp = a.v + (((index_v * D) + col) << a.page_shift) + (tv & mask);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int x = 0; x < KC; ++x) kf[j][x] = *(const u32x4*)(kp + 4 * j * D + 64 * x);
    };
    auto load_v = [&]() {
#pragma unroll
      for (int d = 0; d < DT; ++d) vf[d] = *(const u32x4*)(vp + ((i64)(16 * d) << a.page_shift));
    };

    int t = first + wk;
    Page next;
    if (t < last) {
      load_k(t, pages_of(t));
      if (t + WK < last) next = pages_of(t + WK);
      load_v();
    }
    for (; t < last; t += WK) {
      f32x4 s[4][NQ];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[j][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < 2 * KC; ++u) {
          const bf16x8 k = unpack8(kf[j][u / 2][u % 2 * 2], kf[j][u / 2][u % 2 * 2 + 1]);
#pragma unroll
          for (int n = 0; n < NQ; ++n) s[j][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[n][u], s[j][n], 0, 0, 0);
        }
      }
      const float f = ks, g = vs;
      const int have = there, at = t * wir::TILE + 16 * grp;   // the lane group's tokens at .. at + have - 1
      const bool edge = __builtin_amdgcn_ballot_w64(have < 16 || at + 15 > low) != 0;
      if (t + WK < last) {   // kf is read: the next tile's keys
        const Page p = next;
        if (t + 2 * WK < last) next = pages_of(t + 2 * WK);
        load_k(t + WK, p);
      }
      bf16x8 pb[NQ][2];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float top = m[n];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x = s[j][n][i] * f;
            if (edge) x = 4 * j + i < have && at + 4 * j + i <= pos[n] ? x : -__builtin_inff();
            s[j][n][i] = x;
            top = fmaxf(top, x);
          }
        top = over_groups(top, [](float x, float y) { return fmaxf(x, y); });
        const float base = top == -__builtin_inff() ? 0.f : top;
        const float corr = __builtin_amdgcn_exp2f(m[n] - base);
        m[n] = top;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p = __builtin_amdgcn_exp2f(s[j][n][i] - base);
            sum += p;
            // a key that the row does not see adds nothing, whatever its scale is
            pb[n][j / 2][j % 2 * 4 + i] = (bf16)(edge && s[j][n][i] == -__builtin_inff() ? 0.f : p * g);
          }
        l[n] = l[n] * corr + sum;
        if (__builtin_amdgcn_ballot_w64(corr != 1.0f) != 0) {
#pragma unroll
          for (int d = 0; d < DT; ++d) o[d][n] *= corr;
        }
      }
      if (edge) edge_values(vf, o, have, at, pos);
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const bf16x8 v = unpack8(vf[d][2 * u], vf[d][2 * u + 1]);
#pragma unroll
          for (int n = 0; n < NQ; ++n) o[d][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pb[n][u], o[d][n], 0, 0, 0);
        }
      if (t + WK < last) load_v();
    }

    const int wave = wk * WR + wr;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const float sum = over_groups(l[n], [](float x, float y) { return x + y; });
      const int row = wave * ROWS + n * 16 + col;
      if (grp == 0) sh.ml[2 * row] = m[n], sh.ml[2 * row + 1] = sum;
#pragma unroll
      for (int d = 0; d < DT; ++d) *(f32x4*)(sh.o + row * PITCH + 16 * d + 4 * grp) = o[d][n];
    }
  }

  // Values of a tile that not all rows see: bytes past the sequence's end
  // become 0 (0 * NaN is NaN in the product), and so do NaN codes, which
  // instead make NaN of exactly the rows that see them, by a product of
  // where they are with who sees them.
  __device__ __forceinline__ void edge_values(u32x4 (&vf)[DT], f32x4 (&o)[DT][NQ], int have, int at, const int (&pos)[NQ]) {
    unsigned keep[4], some = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int n = min(max(have - 4 * w, 0), 4);
      keep[w] = n == 4 ? ~0u : (1u << 8 * n) - 1;
    }
    u32x4 is[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const unsigned x = vf[d][w] & keep[w];
        const unsigned high = ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;   // of bytes 0x7f and 0xff
        some |= high;
        const unsigned bytes = (high >> 7) * 0xffu;
        vf[d][w] = x & ~bytes;
        is[d][w] = bytes & 0x38383838u;   // 1.0 in e4m3
      }
    if (__builtin_amdgcn_ballot_w64(some != 0) == 0) return;
    bf16x8 sees[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int e = 0; e < 16; ++e) sees[n][e / 8][e % 8] = (bf16)(e < have && at + e <= pos[n] ? 1.f : 0.f);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        f32x4 count = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < 2; ++u)
          count = __builtin_amdgcn_mfma_f32_16x16x32_bf16(unpack8(is[d][2 * u], is[d][2 * u + 1]), sees[n][u], count, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (count[i] > 0.f) o[d][n][i] = __builtin_nanf("");
      }
  }

  // The waves' results of a block, joined: the outputs, or the partial result of `slot`.
  __device__ __forceinline__ void store(int head, int slot) {
    constexpr int CH = D / 8;
    const int left = min(rows() - rb * BLOCK, BLOCK);
    for (int idx = threadIdx.x; idx < left * CH; idx += 256) {
      const int row = idx / CH, ch = idx % CH;
      float top = -__builtin_inff();
#pragma unroll
      for (int w = 0; w < WK; ++w) top = fmaxf(top, sh.ml[2 * (w * BLOCK + row)]);
      const float base = top == -__builtin_inff() ? 0.f : top;
      float sum = 0.f;
      f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        const int at = w * BLOCK + row;
        const float f = __builtin_amdgcn_exp2f(sh.ml[2 * at] - base);
        sum += f * sh.ml[2 * at + 1];
        x += f * *(const f32x4*)(sh.o + at * PITCH + 8 * ch);
        y += f * *(const f32x4*)(sh.o + at * PITCH + 8 * ch + 4);
      }
      if (position(rb * BLOCK + row) < 0) {   // it took part in tiles that every row with a position sees
        top = -__builtin_inff(), sum = 0.f;
        x = y = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      if (slot >= 0) {
        float* to = a.partial + ((i64)slot * BLOCK + row) * D + 8 * ch;
        *(f32x4*)to = x;
        *(f32x4*)(to + 4) = y;
        if (ch == 0)
          *(f32x2*)(a.partial + (i64)2 * a.programs * BLOCK * D + ((i64)slot * BLOCK + row) * 2) = f32x2{top, sum};
      } else {
        put(a, b, head, rb * BLOCK + row, ch, x, y, top, sum);
      }
    }
  }

  // 8 columns of a row's output and, with the first of them, its LSE; a row that sees nothing: 0 and -inf.
  static __device__ __forceinline__ void put(const attn_args& a, int b, int head, int r, int ch, const f32x4& x,
                                             const f32x4& y, float top, float sum) {
    const int t = r / a.group;
    const i64 h = head * a.group + r - t * a.group;
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    bf16x8 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (bf16)(x[i] * inv), v[4 + i] = (bf16)(y[i] * inv);
    *(bf16x8*)(a.out + b * a.ob + h * a.oh + t * a.ot + 8 * ch) = v;
    if (ch == 0)
      a.lse[b * a.lb + h * a.lh + t * a.lt] =
          sum == 0.f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(sum)) * kLn2;
  }

  __device__ __forceinline__ void segment(int pair, int keys, const wir::Segment& g, i64 share) {
    b = pair / a.blocks;
    rb = pair % a.blocks;
    span = span_at(b);
    walk(g.head, g.first, min(g.last, (int)(((i64)keys + wir::TILE - 1) / wir::TILE)));
    __syncthreads();
    const int slot = g.whole ? -1 : wir::slot_of(g.begin, share);
    if (threadIdx.x == 0 && a.programs && g.first == 0) {
      int* info = a.info + 2 * ((i64)pair * a.heads + g.head);
      info[0] = slot;
      info[1] = g.whole ? 1 : wir::parts_of(g.begin, wir::block_units(keys), share);
    }
    store(g.head, slot);
    __syncthreads();
  }

  __device__ __forceinline__ void run() {
    const int pairs = a.batch * a.blocks;
    if (!a.programs) {
      const int pair = blockIdx.x / a.heads, keys = keys_at(pair);
      segment(pair, keys, wir::Segment{(int)(blockIdx.x % a.heads), 0, wir::block_units(keys), 0, true}, 1);
      return;
    }
    // units before every thread's pairs
    const int each = (pairs + 255) / 256, from = threadIdx.x * each;
    i64 own = 0;
    for (int p = from; p < min(from + each, pairs); ++p) own += (i64)a.heads * wir::block_units(keys_at(p));
    sh.scan[threadIdx.x] = own;
    __syncthreads();
    for (int d = 1; d < 256; d *= 2) {
      const i64 x = threadIdx.x >= d ? sh.scan[threadIdx.x - d] : 0;
      __syncthreads();
      sh.scan[threadIdx.x] += x;
      __syncthreads();
    }
    const i64 total = sh.scan[255], share = wir::share_of(total, a.programs, a.least);
    i64 u = (i64)blockIdx.x * share;
    if (u >= total) return;
    const i64 end = u + share < total ? u + share : total;
    i64 base = sh.scan[threadIdx.x] - own;
    if (base <= u && u < base + own) {
      int p = from;
      for (;; ++p) {
        const i64 n = (i64)a.heads * wir::block_units(keys_at(p));
        if (u < base + n) break;
        base += n;
      }
      sh.found = p;
      sh.found_base = base;
    }
    __syncthreads();
    int pair = sh.found;
    base = sh.found_base;
    while (u < end) {
      const int keys = keys_at(pair), units = wir::block_units(keys);
      const wir::Segment g = wir::segment_at(u, base, units, end);
      segment(pair, keys, g, share);
      u += g.last - g.first;
      if (u == base + (i64)a.heads * units) base = u, ++pair;
    }
  }
};

// Partial results of a head's rows, joined in the order of their tiles:
// program (row of the block, item).
template <int D, int BLOCK>
__device__ __forceinline__ void join(const attn_args& a) {
  constexpr int CH = D / 4, PER = 256 / CH;   // lanes of a row; partial results read side by side
  __shared__ float tops[256];
  __shared__ f32x4 sums[256];
  __shared__ float ls[PER];
  const int per = min(a.tokens * a.group, BLOCK), item = blockIdx.x / per, row = blockIdx.x % per;
  const int pair = item / a.heads, head = item - pair * a.heads, b = pair / a.blocks, rb = pair - b * a.blocks;
  const int r = rb * BLOCK + row;
  if (r >= a.tokens * a.group) return;
  const int slot = a.info[2 * (i64)item], parts = a.info[2 * (i64)item + 1];
  if (parts <= 1) return;
  const f32x2* ml = (const f32x2*)(a.partial + (i64)2 * a.programs * BLOCK * D);
  float top = -__builtin_inff();
  for (int p = threadIdx.x; p < parts; p += 256) top = fmaxf(top, ml[(i64)wir::slot_of_part(slot, p) * BLOCK + row][0]);
  tops[threadIdx.x] = top;
  __syncthreads();
  for (int d = 128; d; d /= 2) {
    if (threadIdx.x < d) tops[threadIdx.x] = fmaxf(tops[threadIdx.x], tops[threadIdx.x + d]);
    __syncthreads();
  }
  top = tops[0];
  const float base = top == -__builtin_inff() ? 0.f : top;
  const int ch = threadIdx.x % CH, w = threadIdx.x / CH;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
#pragma unroll 4
  for (int p = w; p < parts; p += PER) {
    const i64 at = (i64)wir::slot_of_part(slot, p) * BLOCK + row;
    const f32x2 y = ml[at];
    const float f = __builtin_amdgcn_exp2f(y[0] - base);
    l += f * y[1];
    x += f * *(const f32x4*)(a.partial + at * D + 4 * ch);
  }
  sums[threadIdx.x] = x;
  if (ch == 0) ls[w] = l;
  __syncthreads();
  if (threadIdx.x >= D / 8) return;
  f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
  l = 0.f;
  for (int i = 0; i < PER; ++i) {
    lo += sums[i * CH + 2 * threadIdx.x];
    hi += sums[i * CH + 2 * threadIdx.x + 1];
    l += ls[i];
  }
  Program<D, BLOCK / 16, 1>::put(a, b, head, r, threadIdx.x, lo, hi, top, l);
}

}  // namespace

#define ATTN_KERNEL(NAME, D, NQ, WR, OCC)                                                                        \
  extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(256, 256), amdgpu_waves_per_eu(OCC, OCC))) \
  NAME(const attn_args args) {                                                                                   \
    __shared__ __attribute__((aligned(16))) Program<D, NQ, WR>::Shared shared;                                   \
    Program<D, NQ, WR>(args, shared).run();                                                                      \
  }
#define JOIN_KERNEL(NAME, D, BLOCK) \
  extern "C" __global__ void __launch_bounds__(256) NAME(const attn_args args) { join<D, BLOCK>(args); }

ATTN_KERNEL(wir_attn_cached_d64_r16, 64, 1, 1, 2)
ATTN_KERNEL(wir_attn_cached_d64_r32, 64, 2, 1, 2)
ATTN_KERNEL(wir_attn_cached_d64_r128, 64, 2, 4, 2)
ATTN_KERNEL(wir_attn_cached_d128_r16, 128, 1, 1, 2)
ATTN_KERNEL(wir_attn_cached_d128_r32, 128, 2, 1, 1)
ATTN_KERNEL(wir_attn_cached_d128_r128, 128, 2, 4, 1)
JOIN_KERNEL(wir_attn_join_d64_r16, 64, 16)
JOIN_KERNEL(wir_attn_join_d64_r32, 64, 32)
JOIN_KERNEL(wir_attn_join_d64_r128, 64, 128)
JOIN_KERNEL(wir_attn_join_d128_r16, 128, 16)
JOIN_KERNEL(wir_attn_join_d128_r32, 128, 32)
JOIN_KERNEL(wir_attn_join_d128_r128, 128, 128)
