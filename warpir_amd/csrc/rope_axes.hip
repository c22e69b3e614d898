// rope_axes.hip -- the rotation of every query and key head by positions with
// several axes (warpir_amd.api.rope_axes, rope_axes_backward).
//
// A row is one head of one token, x of D values, of which the first 2 R turn in
// R pairs: (i, i + R), or (2i, 2i + 1) interleaved.  Pair i belongs to the axis
// whose section holds i and turns by the angle of that axis' position:
//   (a, b) -> (a c - b s, b c + a s),  c, s = cos, sin of the table's row
// pos[axis] and column i.  The gradient turns by minus the angle.  Values from
// 2 R on pass through.
//
// Everything is fp32 between one bf16 load and one bf16 store of each value.
//
// Bound by memory: 32768 tokens, 32/8 heads of 128, three axes 128-140 us a
// direction, 4.9 TB/s, the rate of a copy; 1369 tokens, 16/16 heads of 64 5.0 us,
// most of it a launch's.
#include <hip/hip_runtime.h>

namespace {

typedef __bf16 bf16;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct axes_side {
  const bf16* x;
  bf16* out;
  long long xb, xh, xs, ob, oh, os;   // strides: batch, head, token
};

struct axes_args {
  axes_side q, k;
  const float* cos;    // [table rows, R]
  const float* sin;
  const void* pos;     // [axes, (batch,) tokens]
  long long pa, pb, ps, cs, ss;
  int q_heads, k_heads, batch, seq, table_rows, pairs;
  int ends[3];         // first pair of axes 1, 2, 3
  int flags;           // 1: positions are 64-bit, 2: turn back, 4: an axis ends inside four pairs
};

// Cosines and sines of four pairs from `at` on, for the token at `token` of the positions; NaN outside the table.
__device__ __forceinline__ void angles(float* c, float* s, const axes_args& a, long long token, int at) {
  auto row_of = [&](int pair) {
    const int axis = (pair >= a.ends[0]) + (pair >= a.ends[1]) + (pair >= a.ends[2]);
    const long long i = token + axis * a.pa;
    const long long p = a.flags & 1 ? ((const long long*)a.pos)[i] : (long long)((const int*)a.pos)[i];
    return p >= 0 && p < a.table_rows ? p : -1;
  };
  const float bad = __builtin_nanf("");
  if (a.flags & 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long row = row_of(at + i), in = row < 0 ? 0 : row;
      const float x = a.cos[in * a.cs + at + i], y = a.sin[in * a.ss + at + i];
      c[i] = row < 0 ? bad : x, s[i] = row < 0 ? bad : y;
    }
  } else {
    const long long row = row_of(at), in = row < 0 ? 0 : row;
    const f32x4 x = *(const f32x4*)(a.cos + in * a.cs + at), y = *(const f32x4*)(a.sin + in * a.ss + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = row < 0 ? bad : x[i], s[i] = row < 0 ? bad : y[i];
  }
}

// Workgroup -> 256 / L rows of one sequence, the heads of a token first, q's
// and then k's, so that a token's angles are read together; a row's D / 16 = L
// lanes hold 16 values each: pairs 8j .. 8j + 7, or 16 values that pass through.
template <int D, bool INTER>
__device__ __forceinline__ void rotate(const axes_args& a) {
  constexpr int L = D / 16, ROWS = 256 / L;
  const unsigned heads = a.q_heads + a.k_heads;
  const unsigned rows = (unsigned)a.seq * heads, blocks = (rows + ROWS - 1) / ROWS;
  const unsigned b = blockIdx.x / blocks;
  const unsigned n = (blockIdx.x - b * blocks) * ROWS + threadIdx.x / L;
  if (n >= rows) return;
  const int j = threadIdx.x % L;
  const unsigned t = n / heads;
  int h = n - t * heads;
  const bool key = h >= a.q_heads;
  const axes_side& side = key ? a.k : a.q;
  if (key) h -= a.q_heads;
  const bool turns = 8 * j < a.pairs;
  const int lo = !turns || INTER ? 16 * j : 8 * j, hi = !turns || INTER ? 16 * j + 8 : a.pairs + 8 * j;
  const bf16* x = side.x + b * side.xb + h * side.xh + t * side.xs;
  bf16x8 u = *(const bf16x8*)(x + lo), v = *(const bf16x8*)(x + hi);
  if (turns) {
    float c[8], s[8];
    const long long token = b * a.pb + t * a.ps;
    angles(c, s, a, token, 8 * j);
    angles(c + 4, s + 4, a, token, 8 * j + 4);
    const float sign = a.flags & 2 ? -1.f : 1.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // pair i: (u[i], v[i]); interleaved: (2i, 2i + 1) of u for i < 4, of v past that
      const float y = INTER ? (float)(i < 4 ? u[2 * i & 7] : v[2 * i & 7]) : (float)u[i];
      const float z = INTER ? (float)(i < 4 ? u[(2 * i + 1) & 7] : v[(2 * i + 1) & 7]) : (float)v[i];
      const float sn = sign * s[i];
      const bf16 first = (bf16)(y * c[i] - z * sn), second = (bf16)(z * c[i] + y * sn);
      if (!INTER) u[i] = first, v[i] = second;
      else if (i < 4) u[2 * i & 7] = first, u[(2 * i + 1) & 7] = second;
      else v[2 * i & 7] = first, v[(2 * i + 1) & 7] = second;
    }
  }
  bf16* o = side.out + b * side.ob + h * side.oh + t * side.os;
  *(bf16x8*)(o + lo) = u;
  *(bf16x8*)(o + hi) = v;
}

}  // namespace

#define AXES_KERNEL(NAME, CALL) \
  extern "C" __global__ void __launch_bounds__(256) NAME(const axes_args args) { CALL(args); }

AXES_KERNEL(wir_rope_axes_d64, (rotate<64, false>))
AXES_KERNEL(wir_rope_axes_d64_inter, (rotate<64, true>))
AXES_KERNEL(wir_rope_axes_d128, (rotate<128, false>))
AXES_KERNEL(wir_rope_axes_d128_inter, (rotate<128, true>))
