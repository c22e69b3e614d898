// qk_norm_rope.hip -- the RMS norm of every query and key head with the
// rotation by its position in the same pass, and its gradients
// (warpir_amd.api.qk_norm_rope, qk_norm_rope_backward).
//
// A row is one head of one token, x of D values:
//   r = 1 / sqrt(mean(x^2) + eps),  y = x r w,
//   (a, b) -> (a c - b s, b c + a s) for the pairs (i, i + D/2), or
//   (2i, 2i + 1) interleaved, with c, s = cos, sin of pos * base^(-2i/D)
// from a table.  Backward, with gy the gradient turned back by -pos:
//   dw = sum over rows of gy x r,  dx = r (w gy - x r mean(w gy x r)).
//
// Everything is fp32 between one bf16 load and one bf16 store of each value.
// The pass is bound by memory (4 bytes a value forward, 6 backward).  A lane
// holds values 8j..8j+7 of both halves of its row, so loads and stores are 16
// bytes, both kinds of pairs are within a lane, and a row's sums take two or
// three lane steps of D/16 lanes.
//
// Measured (a 2 GiB copy moves 4.90 TB/s): 8 x 4096 tokens, 16/16 heads, D =
// 128: forward 110 us, 537 MB at 4.87 TB/s; backward 160 us, 805 MB at 5.03
// TB/s, and 4.6 us for the weights' sums.  Counters there: bytes written 1.00,
// read 1.07 and 1.04 of what the formula needs (the rest is the table).  3 x
// 1337 tokens, 24/8 heads, D = 64, interleaved: 8.5 us; 8 rows of one token: 3.4.
#include <hip/hip_runtime.h>

namespace {

typedef __bf16 bf16;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct rope_side {
  const bf16* x;
  const bf16* g;       // backward: the gradient of the output
  bf16* out;
  const void* w;
  long long xb, xh, xs, gb, gh, gs, ob, oh, os;   // strides: batch, head, token
  int heads;
  int blocks;          // backward: workgroups of this side
};

struct rope_args {
  rope_side q, k;
  const float* cos;    // [table rows, D / 2]
  const float* sin;
  const void* pos;     // null: 0, 1, ...
  float* partial;      // backward: [q.blocks + k.blocks, D]
  long long pb, ps, cs, ss;   // strides of pos (batch, token), row strides of cos and sin
  int batch, seq, table_rows;
  int flags;           // 1: weights are fp32 (else bf16), 2: positions are 64-bit
  float eps;
};

template <int L>
__device__ __forceinline__ float group_sum(float x) {   // over each L lanes, L = 4 or 8
  x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0xB1, 0xF, 0xF, true));    // lane ^ 1
  x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x4E, 0xF, 0xF, true));    // lane ^ 2
  if (L == 8) x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x141, 0xF, 0xF, true));   // 7 - lane
  return x;
}

__device__ __forceinline__ void widen(float (&o)[8], const bf16x8& v) {
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = (float)v[i];
}

__device__ __forceinline__ bf16x8 narrow(const float (&x)[8]) {
  bf16x8 v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (bf16)x[i];
  return v;
}

__device__ __forceinline__ void load_weights(float (&o)[8], const void* w, int at, bool wide) {
  if (wide) {
    const f32x4 a = *(const f32x4*)((const float*)w + at), b = *(const f32x4*)((const float*)w + at + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = a[i], o[4 + i] = b[i];
  } else {
    widen(o, *(const bf16x8*)((const bf16*)w + at));
  }
}

// The cosines and sines of this lane's eight pairs at a token; NaN for a
// position outside the table.
template <int D, bool INTER>
__device__ __forceinline__ void angles(float (&c)[8], float (&s)[8], const rope_args& a, int b, int t, int j) {
  long long p = t;
  if (a.pos) {
    const long long at = b * a.pb + t * a.ps;
    p = a.flags & 2 ? ((const long long*)a.pos)[at] : (long long)((const int*)a.pos)[at];
  }
  const bool in = p >= 0 && p < a.table_rows;
  const long long row = in ? p : 0;
  // half pairs: pair i of the row is value i of its halves; interleaved: a half holds D / 4 pairs
  const int lo = INTER ? 4 * j : 8 * j, hi = INTER ? D / 4 + 4 * j : 8 * j + 4;
  const f32x4 c0 = *(const f32x4*)(a.cos + row * a.cs + lo), c1 = *(const f32x4*)(a.cos + row * a.cs + hi);
  const f32x4 s0 = *(const f32x4*)(a.sin + row * a.ss + lo), s1 = *(const f32x4*)(a.sin + row * a.ss + hi);
  const float bad = __builtin_nanf("");
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c[i] = in ? c0[i] : bad, c[4 + i] = in ? c1[i] : bad;
    s[i] = in ? s0[i] : bad, s[4 + i] = in ? s1[i] : bad;
  }
}

// Turns a lane's pairs by the angle (SIGN = 1) or back (-1).
template <bool INTER, int SIGN>
__device__ __forceinline__ void turn(float (&lo)[8], float (&hi)[8], const float (&c)[8], const float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // pair i: (lo[i], hi[i]); interleaved: (x[2i], x[2i + 1]) of lo for i < 4, of hi past that
    float& a = INTER ? (i < 4 ? lo[2 * i & 7] : hi[2 * i & 7]) : lo[i];
    float& b = INTER ? (i < 4 ? lo[(2 * i + 1) & 7] : hi[(2 * i + 1) & 7]) : hi[i];
    const float u = a, v = b, sn = SIGN * s[i];
    a = u * c[i] - v * sn;
    b = v * c[i] + u * sn;
  }
}

// Workgroup -> 256 / L rows of one sequence; rows run over the heads of a
// token first, q's and then k's, so that a token's angles are read together.
// One row a lane group and no loop: the loads of 8 waves a SIMD hide one
// another.
template <int D, bool INTER>
__device__ __forceinline__ void forward(const rope_args& a) {
  constexpr int L = D / 16, ROWS = 256 / L;
  const unsigned heads = a.q.heads + a.k.heads;
  const unsigned rows = (unsigned)a.seq * heads, blocks = (rows + ROWS - 1) / ROWS;
  const unsigned b = blockIdx.x / blocks;
  const unsigned n = (blockIdx.x - b * blocks) * ROWS + threadIdx.x / L;
  if (n >= rows) return;
  const int j = threadIdx.x % L;
  const unsigned t = n / heads;
  int h = n - t * heads;
  const bool key = h >= a.q.heads;
  const rope_side& side = key ? a.k : a.q;
  if (key) h -= a.q.heads;
  const bf16* x = side.x + b * side.xb + h * side.xh + t * side.xs + 8 * j;
  float lo[8], hi[8], w0[8], w1[8], c[8], s[8];
  widen(lo, *(const bf16x8*)x);
  widen(hi, *(const bf16x8*)(x + D / 2));
  angles<D, INTER>(c, s, a, b, t, j);
  load_weights(w0, side.w, 8 * j, a.flags & 1);
  load_weights(w1, side.w, D / 2 + 8 * j, a.flags & 1);
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) sq += lo[i] * lo[i] + hi[i] * hi[i];
  const float r = 1.0f / sqrtf(group_sum<L>(sq) * (1.0f / D) + a.eps);
#pragma unroll
  for (int i = 0; i < 8; ++i) lo[i] = lo[i] * r * w0[i], hi[i] = hi[i] * r * w1[i];
  turn<INTER, 1>(lo, hi, c, s);
  bf16* o = side.out + b * side.ob + h * side.oh + t * side.os + 8 * j;
  *(bf16x8*)o = narrow(lo);
  *(bf16x8*)(o + D / 2) = narrow(hi);
}

// Workgroups [0, q.blocks) take q's rows, the others k's, 256 / L rows at a
// time in turn.  A lane adds up dw of its columns over its rows; the
// workgroup's sum goes to `partial` and `rope_weight_grad` adds those in
// order, so dw does not depend on when a workgroup runs.
template <int D, bool INTER>
__device__ __forceinline__ void backward(const rope_args& a) {
  constexpr int L = D / 16, ROWS = 256 / L;
  __shared__ float sums[ROWS * D];
  const bool key = blockIdx.x >= a.q.blocks;
  const rope_side& side = key ? a.k : a.q;
  const unsigned heads = side.heads, rows = (unsigned)a.batch * a.seq * heads;
  const int j = threadIdx.x % L;
  float w0[8], w1[8], d0[8], d1[8];
  load_weights(w0, side.w, 8 * j, a.flags & 1);
  load_weights(w1, side.w, D / 2 + 8 * j, a.flags & 1);
#pragma unroll
  for (int i = 0; i < 8; ++i) d0[i] = d1[i] = 0.f;
  const unsigned step = side.blocks * ROWS;
  for (unsigned n = (blockIdx.x - (key ? a.q.blocks : 0)) * ROWS + threadIdx.x / L; n < rows; n += step) {
    const unsigned token = n / heads, h = n - token * heads;
    const unsigned b = token / (unsigned)a.seq, t = token - b * a.seq;
    const bf16* x = side.x + b * side.xb + h * side.xh + t * side.xs + 8 * j;
    const bf16* g = side.g + b * side.gb + h * side.gh + t * side.gs + 8 * j;
    float x0[8], x1[8], g0[8], g1[8], c[8], s[8];
    widen(x0, *(const bf16x8*)x);
    widen(x1, *(const bf16x8*)(x + D / 2));
    widen(g0, *(const bf16x8*)g);
    widen(g1, *(const bf16x8*)(g + D / 2));
    angles<D, INTER>(c, s, a, b, t, j);
    turn<INTER, -1>(g0, g1, c, s);
    float sq = 0.f, dot = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sq += x0[i] * x0[i] + x1[i] * x1[i];
      dot += g0[i] * w0[i] * x0[i] + g1[i] * w1[i] * x1[i];
    }
    const float r = 1.0f / sqrtf(group_sum<L>(sq) * (1.0f / D) + a.eps);
    const float m = group_sum<L>(dot) * r * (1.0f / D);   // mean(w gy x r)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x0[i] *= r, x1[i] *= r;
      d0[i] += g0[i] * x0[i], d1[i] += g1[i] * x1[i];
      g0[i] = r * (g0[i] * w0[i] - x0[i] * m);
      g1[i] = r * (g1[i] * w1[i] - x1[i] * m);
    }
    bf16* o = side.out + b * side.ob + h * side.oh + t * side.os + 8 * j;
    *(bf16x8*)o = narrow(g0);
    *(bf16x8*)(o + D / 2) = narrow(g1);
  }
  float* own = sums + (threadIdx.x / L) * D + 8 * j;
#pragma unroll
  for (int i = 0; i < 8; ++i) own[i] = d0[i], own[D / 2 + i] = d1[i];
  __syncthreads();
  if (threadIdx.x < D) {
    float sum = 0.f;
#pragma unroll 8
    for (int i = 0; i < ROWS; ++i) sum += sums[i * D + threadIdx.x];
    a.partial[(long long)blockIdx.x * D + threadIdx.x] = sum;
  }
}

struct grad_args {
  const float* partial;   // [q_blocks + k_blocks, d]
  float* q;
  float* k;
  int q_blocks, k_blocks, d;
};

}  // namespace

#define ROPE_KERNEL(NAME, CALL) \
  extern "C" __global__ void __launch_bounds__(256) NAME(const rope_args args) { CALL(args); }

ROPE_KERNEL(wir_qk_norm_rope_d64, (forward<64, false>))
ROPE_KERNEL(wir_qk_norm_rope_d64_inter, (forward<64, true>))
ROPE_KERNEL(wir_qk_norm_rope_d128, (forward<128, false>))
ROPE_KERNEL(wir_qk_norm_rope_d128_inter, (forward<128, true>))
ROPE_KERNEL(wir_qk_norm_rope_bwd_d64, (backward<64, false>))
ROPE_KERNEL(wir_qk_norm_rope_bwd_d64_inter, (backward<64, true>))
ROPE_KERNEL(wir_qk_norm_rope_bwd_d128, (backward<128, false>))
ROPE_KERNEL(wir_qk_norm_rope_bwd_d128_inter, (backward<128, true>))

// Sums of the workgroups' partials: block (x, side) takes 32 columns, 32
// threads of each add every 32nd partial, then one another.
extern "C" __global__ void __launch_bounds__(256) wir_rope_weight_grad(const grad_args a) {
  __shared__ f32x4 sums[256];
  const bool key = blockIdx.y;
  const int at = blockIdx.x * 32 + (threadIdx.x % 8) * 4, blocks = key ? a.k_blocks : a.q_blocks;
  const float* p = a.partial + (long long)(key ? a.q_blocks : 0) * a.d + at;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = threadIdx.x / 8; i < blocks; i += 32) sum += *(const f32x4*)(p + (long long)i * a.d);
  sums[threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.x >= 8) return;
  for (int i = 1; i < 32; ++i) sum += sums[threadIdx.x + 8 * i];
  *(f32x4*)((key ? a.k : a.q) + at) = sum;
}
