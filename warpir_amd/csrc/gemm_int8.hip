// gemm_int8.hip -- tokens in 8-bit integers with a scale each, and the product
// of two matrices of such rows (warpir_amd.api.quantize_int8, gemm_int8).
//
//   scale_m = max(max_k |x_mk| * r, 2^-126) with r = 1 / 127 rounded to fp32 (torch
// divides a GPU tensor by a number like this, so amax(1) / 127 there has the same
// bits),  code_mk = the integer nearest to x_mk / scale_m, ties to even;
//   out_mn = bf16((float)(sum_k a_mk b_nk) * a_scale_m * b_scale_n), the sum
// exact in 32-bit integers.
#include "wir_cdna4.h"

namespace {

using wir::bf16;
using wir::bf16x8;

typedef long long i64;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) i32x4 lds_i32x4;
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef signed char i8x16 __attribute__((ext_vector_type(16)));

// ---------------------------------------------------------------------------
// codes and scales: one pass over a row, which stays in registers (up to 16384
// values; past that it is read again).  Bound by memory: 16384 x 8192 71 us, 5.6
// TB/s (reads are two thirds); 16 x 4096 2.9 us, a launch and two waits.

struct quantize_args {
  const bf16* x;       // [rows, width]
  signed char* codes;  // [rows, width]
  float* scale;        // [rows]
  i64 xs, cs;          // row strides
  int rows, width;
};

__device__ __forceinline__ unsigned larger(unsigned a, unsigned b) { return a > b ? a : b; }

// The largest magnitude of 16 bf16 values by their bits (infinity and NaN above every number).
__device__ __forceinline__ unsigned magnitude(const u16x8& u, const u16x8& v) {
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = larger(top, larger(u[i] & 0x7fffu, v[i] & 0x7fffu));
  return top;
}

// The integer nearest to x / scale, ties to even, where inv is 1 / scale within
// an ulp: the product is within 2^-16 of the quotient (which is at most 127.01),
// and what is left of x, exact in 32 bits, says which of two codes is nearer.
__device__ __forceinline__ int nearest(float x, float scale, float inv) {
  float n = __builtin_rintf(x * inv);
  const float rest = __builtin_fmaf(-n, scale, x), twice = 2.f * __builtin_fabsf(rest);
  if (twice > scale || (twice == scale && ((int)n & 1))) n += __builtin_copysignf(1.f, rest);
  return (int)n;
}

__device__ __forceinline__ i8x16 codes_of(const u16x8& u, const u16x8& v, float scale, float inv) {
  i8x16 c;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    c[i] = (signed char)nearest(__uint_as_float((unsigned)u[i] << 16), scale, inv);
    c[8 + i] = (signed char)nearest(__uint_as_float((unsigned)v[i] << 16), scale, inv);
  }
  return c;
}

// W waves a row; the row's values wait in registers where it has up to 1024 * W * N of them and are read again past that.
template <int W, int N>
__device__ __forceinline__ void quantize(const quantize_args& a) {
  constexpr int LANES = 64 * W, STEP = 16 * LANES;
  const int row = W == 1 ? blockIdx.x * 4 + threadIdx.x / 64 : blockIdx.x;
  if (row >= a.rows) return;   // (whole waves; with W > 1 no workgroup)
  const int lane = threadIdx.x % LANES;
  const u16x8* x = (const u16x8*)(a.x + row * a.xs);
  u16x8 u[N], v[N];
  unsigned top = 0;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int at = n * STEP + 16 * lane;
    u[n] = v[n] = u16x8{};
    if (at < a.width) u[n] = x[at / 8], v[n] = x[at / 8 + 1];
    top = larger(top, magnitude(u[n], v[n]));
  }
  for (int at = N * STEP + 16 * lane; at < a.width; at += STEP) top = larger(top, magnitude(x[at / 8], x[at / 8 + 1]));
#pragma unroll
  for (int d = 32; d; d /= 2) top = larger(top, __shfl_xor(top, d));
  if (W > 1) {
    __shared__ unsigned tops[W];
    if (lane % 64 == 0) tops[lane / 64] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) top = larger(top, tops[w]);
  }
  const bool finite = top < 0x7f80u;
  const float scale = fmaxf(__uint_as_float(top << 16) * (1.0f / 127.0f), 0x1p-126f);
  const float inv = finite ? 1.0f / scale : 0.f;
  i8x16* codes = (i8x16*)(a.codes + row * a.cs);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int at = n * STEP + 16 * lane;
    if (at < a.width) codes[at / 16] = finite ? codes_of(u[n], v[n], scale, inv) : i8x16{};
  }
  for (int at = N * STEP + 16 * lane; at < a.width; at += STEP)
    codes[at / 16] = finite ? codes_of(x[at / 8], x[at / 8 + 1], scale, inv) : i8x16{};
  if (lane == 0) a.scale[row] = finite ? scale : __builtin_nanf("");
}

// ---------------------------------------------------------------------------
// the product

struct gemm_args {
  const signed char* a;   // [M, K]
  const signed char* b;   // [N, K]
  const float* a_scale;   // [M]
  const float* b_scale;   // [N]
  bf16* out;              // [M, N]
  int* partial;           // [splits][tile][32 x 32 block][1024]: sums over a part of K
  i64 as, bs, os;         // row strides
  int m, n, k;
  int splits, each;       // parts of K, steps of 128 of one
};

// ROWS rows of a matrix of codes, 128 of each row's bytes a step, as a tile of 16-byte chunks in LDS.
template <int ROWS, int NW>
struct Codes {
  typedef wir::STile<ROWS, 64, wir::ROWREAD> T;   // (64 bf16 are 128 bytes)
  static constexpr int EACH = ROWS * 8 / 64 / NW;
  const signed char* base;
  unsigned off[EACH];   // of the lane's chunks from the base; rows past the matrix read its last row
  int chunk[EACH];

  __device__ __forceinline__ void init(const signed char* x, i64 stride, int row0, int rows, int wave) {
    base = x + row0 * stride;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const int p = (wave + j * NW) * 64 + wir::lane_id(), row = p / 8;
      chunk[j] = ((p % 8) ^ wir::swz<8, wir::ROWREAD>(row)) * 16;
      off[j] = (unsigned)min(row, rows - 1 - row0) * (unsigned)stride + chunk[j];
    }
  }

  // The wave's j-th load of the bytes from k on; whole: the rows hold 128 more (else those past their end read as zeros).
  __device__ __forceinline__ void load(char* tile, int k, int width, int wave, int j) const {
    const unsigned to = wir::lds_addr(tile + (wave + j * NW) * 1024);
    if (k + 128 <= width)
      wir::dma16_s(base + k, off[j], to);
    else
      wir::dma16_v(k + chunk[j] < width ? (const void*)(base + k + off[j]) : (const void*)wir::zero_page, to);
  }

  __device__ __forceinline__ void load(char* tile, int k, int width, int wave) const {
#pragma unroll
    for (int j = 0; j < EACH; ++j) load(tile, k, width, wave, j);
  }
};

__device__ __forceinline__ i32x16 mma(bf16x8 a, bf16x8 b, i32x16 c) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// float(acc) * a_scale * b_scale of four columns that follow one another
__device__ __forceinline__ f32x4 scales_at(const float* s, int at, int n) {
  f32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = s[min(at + i, n - 1)];
  return v;
}

// A wave's part of the output by way of `stage` in LDS, V values a store, the lanes next to one another.
template <int V, int R, int C>
__device__ __forceinline__ void store_narrow(const gemm_args& g, const wir::RTile<32, R, C>& t, int row0, int col0, char* stage) {
  typedef bf16 vec __attribute__((ext_vector_type(V)));
  typedef __attribute__((address_space(3))) vec lds_vec;
  typedef __attribute__((address_space(3))) wir::bf16x4 lds_bf16x4;
  constexpr int PITCH = C + 4, EACH = C / V;   // (rows are two banks apart)
  auto* s = (__attribute__((address_space(3))) bf16*)wir::lds(stage);
  const int lane = wir::lane_id(), lr = lane % 32, lh = lane / 32;
#pragma unroll
  for (int rb = 0; rb < R / 32; ++rb) {
#pragma unroll
    for (int cb = 0; cb < C / 32; ++cb)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        wir::bf16x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (bf16)t.f[cb][rb][4 * q + i];
        *(lds_bf16x4*)(s + lr * PITCH + cb * 32 + wir::ccol<32>(4 * q, lh)) = v;
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int it = 0; it < 32 * EACH / 64; ++it) {
      const int i = it * 64 + lane, row = row0 + rb * 32 + i / EACH, col = col0 + i % EACH * V;
      const vec v = *(lds_vec*)(s + i / EACH * PITCH + i % EACH * V);
      if (row < g.m && col < g.n) *(vec*)(g.out + (i64)row * g.os + col) = v;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// In the widest stores that the output's rows and the number of columns are whole multiples of.
template <int R, int C>
__device__ __forceinline__ void store_rows(const gemm_args& g, const wir::RTile<32, R, C>& t, int row0, int col0, char* stage) {
  const int whole = g.n | (int)g.os | (int)((size_t)g.out >> 1);   // (in values)
  if (((int)g.os | (int)((size_t)g.out >> 1)) % 8 == 0)
    wir::store_tile_staged<true>(wir::gl<bf16>{g.out, 1, 1, g.m, g.n, 0, 0, g.os}, t, 0, 0, row0, col0, stage);
  else if (whole % 4 == 0)
    store_narrow<4>(g, t, row0, col0, stage);
  else if (whole % 2 == 0)
    store_narrow<2>(g, t, row0, col0, stage);
  else
    store_narrow<1>(g, t, row0, col0, stage);
}

// Blocks of 32 x 32 sums from (row0, col0) on, the first OC x OR of acc, scaled and rounded, by way of `stage` in LDS.
template <int OC, int OR, int CB, int RB>
__device__ __forceinline__ void finish(const gemm_args& g, const i32x16 (&acc)[CB][RB], int row0, int col0, char* stage) {
  // a lane holds row lane % 32 of each block of rows, 16 columns of each block of columns
  const int lane = wir::lane_id();
  wir::RTile<32, 32 * OR, 32 * OC> out;
#pragma unroll
  for (int c = 0; c < OC; ++c)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 sb = scales_at(g.b_scale, col0 + c * 32 + wir::ccol<32>(4 * q, lane / 32), g.n);
#pragma unroll
      for (int r = 0; r < OR; ++r) {
        const float sa = g.a_scale[min(row0 + r * 32 + lane % 32, g.m - 1)];
#pragma unroll
        for (int i = 0; i < 4; ++i) out.f[c][r][4 * q + i] = (float)acc[c][r][4 * q + i] * sa * sb[i];
      }
    }
  store_rows(g, out, row0, col0, stage);
}

// Output tiles of BM x BN over a ring of S tiles of 128 bytes of each row.  A
// wave takes WM x WN of it, and of each row's bytes 1 / KW: KW waves have one
// part of the output, whose sums they share out and add at the end.
//
// Measured: 8192 x 8192 x 8192 in 451 to 464 us by the card (2370-2440 TOP/s, the library's product 512),
// where the clock is what the power leaves; 777 x 4100 x 4096 in 22.3 us.  Small tiles
// are bound by LDS, which takes 32 KB a step and reads 64 to 96: of 22 us without
// the loads 16, without the products 17, without the reads 19.  Two waves of 64 x
// 64 x K / 2 in place of 64 x 32 x K (KW = 2) read a third less: 128 x 128 tiles of 8192^3
// 684 -> 652 us, 64 x 64 (KW = 4) 939 -> 876.  Deeper rings change nothing.
//
// WHOLE: a wave's operands of the next tile are read while this one's products
// run, from registers.  Without (parts whose operands do not fit twice): a
// quarter of a tile ahead, and the last quarter's products run behind the
// barrier that the next tile needs, under the reads of its first operands.
//
// SPLIT: of few tiles, a workgroup each for a part of K, whose sums
// gemm_join adds (integers: in any order the same).
template <int BM, int BN, int WM, int WN, int KW, int S, bool WHOLE, bool SPLIT = false>
__device__ __forceinline__ void gemm_tiled(const gemm_args& g) {
  constexpr int PARTS = BM / WM * (BN / WN), NW = PARTS * KW, RB = WM / 32, CB = WN / 32, KS = 4 / KW;
  constexpr int OC = KW > 1 ? CB / 2 : CB, OR = KW > 2 ? RB / 2 : RB, GIVEN = CB * RB - OC * OR;   // blocks that a wave finishes, and gives
  static_assert(OC * OR * KW == CB * RB && (WHOLE || KW == 1), "the waves of a part finish it between them");
  typedef Codes<BM, NW> CA;
  typedef Codes<BN, NW> CBt;
  constexpr int SLOT = CA::T::BYTES + CBt::T::BYTES, EACH = CA::EACH + CBt::EACH;
  constexpr int STAGE = (OR > 1 ? OR * 32 * OC * 32 : 32 * (OC * 32 + 4)) * 2;   // bytes of a wave's output on its way
  static_assert(NW * STAGE <= S * SLOT && NW * GIVEN * 4096 <= S * SLOT, "the output goes through the tiles' LDS");
  __shared__ __attribute__((aligned(1024))) char smem[S * SLOT];
  const int nx = (g.n + BN - 1) / BN, ny = (g.m + BM - 1) / BM;
  int x, y;
  const int id = wir::remap_xcd(blockIdx.x, nx * ny * (SPLIT ? g.splits : 1)), split = SPLIT ? id / (nx * ny) : 0;
  wir::grouped_tile<8>(id - split * nx * ny, nx, ny, x, y);
  const int k0 = SPLIT ? split * g.each * 128 : 0, width = SPLIT ? min(g.k - k0, g.each * 128) : g.k;
  const int wave = wir::wave_id(), lane = wir::lane_id();
  const int part = wave % PARTS, kw = wave / PARTS, row0 = part / (BN / WN) * WM, col0 = part % (BN / WN) * WN;
  CA a;
  CBt b;
  a.init(g.a + k0, g.as, y * BM, g.m, wave);
  b.init(g.b + k0, g.bs, x * BN, g.n, wave);
  const int steps = (width + 127) / 128;
  auto load = [&](int t, int slot, int j) {
    char* at = smem + slot * SLOT;
    if (j < CA::EACH) a.load(at, t * 128, width, wave, j);
    else b.load(at + CA::T::BYTES, t * 128, width, wave, j - CA::EACH);
  };
  i32x16 acc[CB][RB];
#pragma unroll
  for (int c = 0; c < CB; ++c)
#pragma unroll
    for (int r = 0; r < RB; ++r) acc[c][r] = i32x16{};
  constexpr int SETS = WHOLE ? 2 * KS : 2;
  bf16x8 fa[SETS][RB], fb[SETS][CB];
  // (the swizzle repeats every 16 rows: a step along the row is an exclusive or, blocks of 32 rows are offsets)
  const unsigned a_at = wir::lds_addr(smem) + CA::T::chunk_off(row0 + lane % 32, kw * KS * 2 + lane / 32);
  const unsigned b_at = wir::lds_addr(smem) + CA::T::BYTES + CBt::T::chunk_off(col0 + lane % 32, kw * KS * 2 + lane / 32);
  typedef __attribute__((address_space(3))) bf16x8 lds_bf16x8;
  auto read = [&](int slot, int ks, int set) {
    const unsigned at = (a_at ^ ks * 32) + slot * SLOT, bt = (b_at ^ ks * 32) + slot * SLOT;
#pragma unroll
    for (int r = 0; r < RB; ++r) fa[set][r] = *(lds_bf16x8*)(at + r * 32 * 128);
#pragma unroll
    for (int c = 0; c < CB; ++c) fb[set][c] = *(lds_bf16x8*)(bt + c * 32 * 128);
  };
  // The products of a quarter of a tile; `between` them, the n-th of its calls behind the n-th.
  auto products = [&](int set, auto between) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        acc[c][r] = mma(fb[set][c], fa[set][r], acc[c][r]);
        between(c * RB + r);
      }
    __builtin_amdgcn_s_setprio(0);
  };
  // Tile t + 1 has come, t + 2 .. t + S - 1 may be on their way; nobody reads tile t's slot any more.
  auto settle = [&](int t) {
    if (t + S <= steps) wir::wait_vm_barrier<(S - 2) * EACH>();
    else wir::wait_vm_barrier<0>();
  };
  // Tile t + S goes to t's slot, in the shade of `all` products (a wave's loads queue: in a row before its products, they
  // hold those back): those behind the n-th of them.
  auto load_behind = [&](int t, int slot, int n, int all) {
    if (t + S >= steps) return;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < EACH; ++j)
      if (j * all / EACH == n) load(t + S, slot, j);
    __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll
  for (int t = 0; t < S; ++t)
    if (t < steps)
#pragma unroll
      for (int j = 0; j < EACH; ++j) load(t, t, j);
  if (steps >= S) wir::wait_vm_barrier<(S - 1) * EACH>();
  else wir::wait_vm_barrier<0>();
  int slot = 0;
  if (WHOLE) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) read(0, ks, ks);
    auto step = [&](int t, int set) {
      const int next = slot == S - 1 ? 0 : slot + 1;
      settle(t);
      if (t + 1 < steps) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) read(next, ks, (KS - set) + ks);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        products(set + ks, [&](int n) { load_behind(t, slot, ks * CB * RB + n, KS * CB * RB); });
      __builtin_amdgcn_sched_barrier(0);
      slot = next;
    };
    int t = 0;
    for (; t + 2 <= steps; t += 2) {
      step(t, 0);
      step(t + 1, KS);
    }
    if (t < steps) step(t, 0);
  } else {
    read(0, 0, 0);
    for (int t = 0; t < steps; ++t) {
      const int next = slot == S - 1 ? 0 : slot + 1;
#pragma unroll
      for (int ks = 0; ks < 3; ++ks) {
        read(slot, ks + 1, (ks + 1) % 2);
        __builtin_amdgcn_sched_barrier(0);
        products(ks % 2, [](int) {});
        __builtin_amdgcn_sched_barrier(0);
      }
      settle(t);
      if (t + 1 < steps) read(next, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      products(1, [&](int n) { load_behind(t, slot, n, CB * RB); });
      __builtin_amdgcn_sched_barrier(0);
      slot = next;
    }
  }
  if (WHOLE) wir::barrier();   // (the last tile's reads: the LDS takes the output)
  const int c0 = KW > 1 ? kw % 2 * OC : 0, r0 = KW > 2 ? kw / 2 * OR : 0;   // of the wave's own blocks
  if constexpr (KW > 1) {
    // block `at` of the wave's in a row of those that wave `by` gives: not its own ones, in order
    auto given = [&](int by, int c, int r) {
      const int bc = by % 2, br = KW > 2 ? by / 2 : 0, at = c * RB + r;
      const int before = KW > 2 ? at > bc * RB + br : c > bc ? RB : 0;   // its own ones before it
      return (lds_i32x4*)wir::lds(smem + ((part * KW + by) * GIVEN + at - before) * 4096) + lane;
    };
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        if (c / OC == kw % 2 && (KW == 2 || r / OR == kw / 2)) continue;
        auto* to = given(kw, c, r);
#pragma unroll
        for (int q = 0; q < 4; ++q) to[q * 64] = i32x4{acc[c][r][4 * q], acc[c][r][4 * q + 1], acc[c][r][4 * q + 2], acc[c][r][4 * q + 3]};
      }
    wir::barrier();
#pragma unroll
    for (int c = 0; c < OC; ++c)
#pragma unroll
      for (int r = 0; r < OR; ++r) {
        // (a wave's own blocks by selection: registers have no run-time index)
        i32x16 sum = acc[c][r];
#pragma unroll
        for (int w = 1; w < KW; ++w)
          if (kw == w) sum = acc[(w % 2) * OC + c][(KW > 2 ? w / 2 * OR : 0) + r];
#pragma unroll
        for (int w = 1; w < KW; ++w) {
          const auto* from = given((kw + w) % KW, c0 + c, r0 + r);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const i32x4 x = from[q * 64];
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[4 * q + i] += x[i];
          }
        }
        acc[c][r] = sum;
      }
    wir::barrier();
  }
  if constexpr (SPLIT) {
    static_assert(OC * OR == 1, "");
    auto* to = (i32x4*)(g.partial + ((i64)(split * ny * nx + y * nx + x) * NW + wave) * 1024) + lane;
#pragma unroll
    for (int q = 0; q < 4; ++q) to[q * 64] = i32x4{acc[0][0][4 * q], acc[0][0][4 * q + 1], acc[0][0][4 * q + 2], acc[0][0][4 * q + 3]};
    return;
  }
  finish<OC, OR>(g, acc, y * BM + row0 + r0 * 32, x * BN + col0 + c0 * 32, smem + wave * STAGE);
}

// The sums of a 64 x 64 tile over the parts of K, a wave's block as gemm_tiled<64, 64, 64, 64, 4, ..> left it: 3 us of a
// product's 10 to 14 that takes 14 to 45 undivided.
__device__ __forceinline__ void gemm_join(const gemm_args& g) {
  __shared__ __attribute__((aligned(1024))) char smem[4 * 32 * 36 * 2];
  const int nx = (g.n + 63) / 64, ny = (g.m + 63) / 64, wave = wir::wave_id(), lane = wir::lane_id();
  const auto* from = (const i32x4*)(g.partial + ((i64)blockIdx.x * 4 + wave) * 1024) + lane;
  i32x16 acc[1][1] = {};
  for (int split = 0; split < g.splits; ++split) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const i32x4 x = from[q * 64];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[0][0][4 * q + i] += x[i];
    }
    from += (i64)nx * ny * 1024;
  }
  finish<1, 1>(g, acc, (int)blockIdx.x / nx * 64 + wave / 2 * 32, (int)blockIdx.x % nx * 64 + wave % 2 * 32, smem + wave * 32 * 36 * 2);
}

// Few tokens, M <= 16 MT: a workgroup takes CH channels, its W waves every W-th
// 128 bytes of their rows and of the tokens' (each through a ring of S tiles of
// its own in LDS, without a barrier), and the waves' sums are added at the end.
// Bound by memory: 16 x 6144 x 4096 in 4.8-5.3 us (25.5 MB, 5 TB/s).
template <int MT, int CH, int W, int S>
__device__ __forceinline__ void gemm_few(const gemm_args& g) {
  constexpr int CT = (CH + 15) / 16;
  typedef Codes<CH, 1> CB;
  typedef Codes<16 * MT, 1> CA;
  typedef __attribute__((address_space(3))) int lds_int;
  constexpr int SLOT = CB::T::BYTES + CA::T::BYTES, EACH = CB::EACH + CA::EACH, SUMS = CT * MT * 1024;
  static_assert(CT * 16 * 128 <= SLOT && SUMS <= S * SLOT, "operands of channels past CH are read, and dropped");
  __shared__ __attribute__((aligned(1024))) char smem[W * S * SLOT];
  const int wave = wir::wave_id(), lane = wir::lane_id();
  const int channel0 = wir::remap_xcd(blockIdx.x, gridDim.x) * CH;
  char* own = smem + wave * S * SLOT;
  CB b;
  CA a;
  b.init(g.b, g.bs, channel0, g.n, 0);
  a.init(g.a, g.as, 0, g.m, 0);
  const int steps = (g.k + 127) / 128, mine = steps > wave ? (steps - wave + W - 1) / W : 0;
  auto load = [&](int t, int slot) {
    const int k = (wave + t * W) * 128;
    b.load(own + slot * SLOT, k, g.k, 0);
    a.load(own + slot * SLOT + CB::T::BYTES, k, g.k, 0);
  };
  i32x4 acc[CT][MT];
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[c][i] = i32x4{0, 0, 0, 0};
#pragma unroll
  for (int t = 0; t < S - 1; ++t)
    if (t < mine) load(t, t);
  // the lane's 16 bytes of a 16 x 64 operand (the swizzle repeats every 16 rows)
  const unsigned b_at = wir::lds_addr(own) + CB::T::chunk_off(lane % 16, lane / 16);
  const unsigned a_at = wir::lds_addr(own) + CB::T::BYTES + CA::T::chunk_off(lane % 16, lane / 16);
  int slot = 0;
  for (int t = 0; t < mine; ++t) {
    // (the slot that is loaded now was read in the step before: those reads have returned)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (t + S - 1 < mine) {
      load(t + S - 1, slot == 0 ? S - 1 : slot - 1);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 1) * EACH) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      i32x4 fb[CT], fa[MT];
#pragma unroll
      for (int c = 0; c < CT; ++c) fb[c] = *(lds_i32x4*)((b_at ^ h * 64) + slot * SLOT + c * 2048);
#pragma unroll
      for (int i = 0; i < MT; ++i) fa[i] = *(lds_i32x4*)((a_at ^ h * 64) + slot * SLOT + i * 2048);
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[c][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[c], fa[i], acc[c][i], 0, 0, 0);
    }
    slot = slot == S - 1 ? 0 : slot + 1;
  }
  // a lane holds token lane % 16, channels 4 (lane / 16) .. + 3
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int i = 0; i < MT; ++i) *((lds_i32x4*)wir::lds(own + (c * MT + i) * 1024) + lane) = acc[c][i];
  wir::barrier();
  for (int i = threadIdx.x; i < CT * MT * 256; i += 64 * W) {
    const int token = i / (16 * CT), channel = i % (16 * CT), n = channel0 + channel;
    if (token >= g.m || channel >= CH || n >= g.n) continue;
    const int tile = channel / 16 * MT + token / 16, at = (channel % 16 / 4 * 16 + token % 16) * 4 + channel % 4;
    int sum = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) sum += *((lds_int*)wir::lds(smem + w * S * SLOT + tile * 1024) + at);
    g.out[token * g.os + n] = (bf16)((float)sum * g.a_scale[token] * g.b_scale[n]);
  }
}

}  // namespace

#define QUANTIZE_KERNEL(NAME, W, N) \
  extern "C" __global__ void __launch_bounds__(256) NAME(const quantize_args args) { quantize<W, N>(args); }

QUANTIZE_KERNEL(wir_quantize_int8_w1, 1, 1)
QUANTIZE_KERNEL(wir_quantize_int8_w4, 4, 1)
QUANTIZE_KERNEL(wir_quantize_int8_w4_n2, 4, 2)
QUANTIZE_KERNEL(wir_quantize_int8_w4_n4, 4, 4)

#define GEMM_KERNEL(NAME, THREADS, WAVES_A_SIMD, ...)                                                   \
  extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(THREADS, THREADS),              \
                                            amdgpu_waves_per_eu(WAVES_A_SIMD, WAVES_A_SIMD)))           \
  NAME(const gemm_args args) { gemm_tiled<__VA_ARGS__>(args); }

GEMM_KERNEL(wir_gemm_int8_256, 512, 2, 256, 256, 128, 64, 1, 2, false)
GEMM_KERNEL(wir_gemm_int8_256x128, 512, 2, 256, 128, 64, 64, 1, 3, true)
GEMM_KERNEL(wir_gemm_int8_128_w4, 256, 2, 128, 128, 64, 64, 1, 2, false)
GEMM_KERNEL(wir_gemm_int8_128, 512, 2, 128, 128, 64, 64, 2, 3, true)
GEMM_KERNEL(wir_gemm_int8_128x64, 256, 2, 128, 64, 64, 64, 2, 3, true)
GEMM_KERNEL(wir_gemm_int8_64, 256, 2, 64, 64, 64, 64, 4, 4, true)
GEMM_KERNEL(wir_gemm_int8_64_split, 256, 2, 64, 64, 64, 64, 4, 4, true, true)

extern "C" __global__ void __launch_bounds__(256) wir_gemm_int8_join(const gemm_args args) { gemm_join(args); }

#define FEW_KERNEL(NAME, MT, CH, W, S) \
  extern "C" __global__ void __launch_bounds__(64 * W) NAME(const gemm_args args) { gemm_few<MT, CH, W, S>(args); }

FEW_KERNEL(wir_gemm_int8_few16_c16, 1, 16, 8, 4)
FEW_KERNEL(wir_gemm_int8_few16_c24, 1, 24, 8, 4)
FEW_KERNEL(wir_gemm_int8_few16_c32, 1, 32, 8, 2)
FEW_KERNEL(wir_gemm_int8_few16_c64, 1, 64, 8, 2)
FEW_KERNEL(wir_gemm_int8_few32_c16, 2, 16, 8, 3)
FEW_KERNEL(wir_gemm_int8_few32_c24, 2, 24, 8, 2)
FEW_KERNEL(wir_gemm_int8_few32_c32, 2, 32, 4, 2)
FEW_KERNEL(wir_gemm_int8_few64_c16, 4, 16, 4, 3)
FEW_KERNEL(wir_gemm_int8_few64_c32, 4, 32, 4, 3)
