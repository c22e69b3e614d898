// gemm_int8.hip -- tokens in 8-bit integers with a scale each, and the product
// of two matrices of such rows (warpir_amd.api.quantize_int8, gemm_int8).
//
//   scale_m = max(max_k |x_mk| / 127, 2^-126),  code_mk = the integer nearest to
//   x_mk / scale_m, ties to even;
//   out_mn = bf16((float)(sum_k a_mk b_nk) * a_scale_m * b_scale_n), the sum
// exact in 32-bit integers.
#include "wir_cdna4.h"

namespace {

using wir::bf16;
using wir::bf16x8;

typedef long long i64;
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef signed char i8x16 __attribute__((ext_vector_type(16)));

// ---------------------------------------------------------------------------
// codes and scales

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
  const float scale = fmaxf(__uint_as_float(top << 16) / 127.0f, 0x1p-126f);
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
  i64 as, bs, os;         // row strides
  int m, n, k;
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

  // The bytes from k on; whole: the row holds 128 more (else those past its end read as zeros).
  __device__ __forceinline__ void load(char* tile, int k, int width, int wave) const {
    const bool whole = k + 128 <= width;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const unsigned to = wir::lds_addr(tile + (wave + j * NW) * 1024);
      if (whole)
        wir::dma16_s(base + k, off[j], to);
      else
        wir::dma16_v(k + chunk[j] < width ? (const void*)(base + k + off[j]) : (const void*)wir::zero_page, to);
    }
  }
};

__device__ __forceinline__ i32x16 mma(bf16x8 a, bf16x8 b, i32x16 c) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// Output tiles of BM x BN, a wave's part WM x WN.
template <int BM, int BN, int WM, int WN>
__device__ __forceinline__ void gemm_tiled(const gemm_args& g) {
  constexpr int NW = BM / WM * (BN / WN), RB = WM / 32, CB = WN / 32;
  typedef Codes<BM, NW> CA;
  typedef Codes<BN, NW> CBt;
  constexpr int SLOT = CA::T::BYTES + CBt::T::BYTES;
  static_assert(NW * WM * WN * 2 <= 2 * SLOT, "the output goes through the tiles' LDS");
  __shared__ __attribute__((aligned(1024))) char smem[2 * SLOT];
  const int nx = (g.n + BN - 1) / BN, ny = (g.m + BM - 1) / BM;
  int x, y;
  wir::grouped_tile<8>(wir::remap_xcd(blockIdx.x, nx * ny), nx, ny, x, y);
  const int wave = wir::wave_id(), lane = wir::lane_id();
  const int row0 = wave / (BN / WN) * WM, col0 = wave % (BN / WN) * WN;
  CA a;
  CBt b;
  a.init(g.a, g.as, y * BM, g.m, wave);
  b.init(g.b, g.bs, x * BN, g.n, wave);
  const int steps = (g.k + 127) / 128;
  auto load = [&](int t) {
    char* at = smem + t % 2 * SLOT;
    a.load(at, t * 128, g.k, wave);
    b.load(at + CA::T::BYTES, t * 128, g.k, wave);
  };
  i32x16 acc[CB][RB];
#pragma unroll
  for (int c = 0; c < CB; ++c)
#pragma unroll
    for (int r = 0; r < RB; ++r) acc[c][r] = i32x16{};
  load(0);
  for (int t = 0; t < steps; ++t) {
    char *at = smem + t % 2 * SLOT, *bt = at + CA::T::BYTES;
    wir::wait_vm_barrier<0>();
    if (t + 1 < steps) load(t + 1);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      bf16x8 fa[RB], fb[CB];
#pragma unroll
      for (int r = 0; r < RB; ++r) fa[r] = wir::row_operand<typename CA::T, 32>(at, row0 + r * 32, ks);
#pragma unroll
      for (int c = 0; c < CB; ++c) fb[c] = wir::row_operand<typename CBt::T, 32>(bt, col0 + c * 32, ks);
#pragma unroll
      for (int c = 0; c < CB; ++c)
#pragma unroll
        for (int r = 0; r < RB; ++r) acc[c][r] = mma(fb[c], fa[r], acc[c][r]);
    }
  }
  wir::wait_vm_barrier<0>();
  // a lane holds row lane % 32 of each block of rows, 16 columns of each block of columns
  const int lh = lane / 32;
  wir::RTile<32, WM, WN> out;
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const float sa = g.a_scale[min(y * BM + row0 + r * 32 + lane % 32, g.m - 1)];
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float sb = g.b_scale[min(x * BN + col0 + c * 32 + wir::ccol<32>(i, lh), g.n - 1)];
        out.f[c][r][i] = (float)acc[c][r][i] * sa * sb;
      }
  }
  wir::store_tile_staged<true>(wir::gl<bf16>{g.out, 1, 1, g.m, g.n, 0, 0, g.os}, out, 0, 0, y * BM + row0, x * BN + col0,
                               smem + wave * WM * WN * 2);
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

GEMM_KERNEL(wir_gemm_int8_256, 256, 1, 256, 256, 128, 128)
GEMM_KERNEL(wir_gemm_int8_128, 256, 2, 128, 128, 64, 64)
GEMM_KERNEL(wir_gemm_int8_64, 256, 2, 64, 64, 32, 32)
