// wir_packed_args.h -- arguments of the kernels over packed sequences
// (attn_packed.hip, attn_packed_bwd.hip, attn_packed_split.hip), and what they
// do with the tokens behind the last sequence.
#pragma once
#include "wir_packed.h"

namespace wir {

struct packed_fwd_args {
  const bf16* q;       // [H, T, D]
  const bf16* k;       // [H_kv, T, D]
  const bf16* v;
  bf16* out;           // [H, T, D]
  float* lse;          // [H, T]
  const int* offsets;  // [batch + 1]
  i64 qh, qt, kh, kt, vh, vt, oh, ot, lh, lt;
  int batch, tokens, heads, group, blocks;
  int flags;           // 1: rows behind the last sequence become 0 in out, 2: -inf in lse, 4: two heads a workgroup
};

struct packed_bwd_args {
  const bf16* q;       // [H, T, D], as o, d_o and dq
  const bf16* k;       // [H_kv, T, D], as v, dk and dv
  const bf16* v;
  const bf16* o;
  const bf16* d_o;
  const float* lse;    // [H, T]
  const int* offsets;  // [batch + 1]
  bf16* dq;
  bf16* dk;
  bf16* dv;
  float* stats;        // [2][H][T]: -LSE sqrt(D) and -D_p, what the scores of the dK/dV kernels begin with
  i64 qh, qt, kh, kt, vh, vt, oh, ot, gh, gt, lh, lt, dqh, dqt, dkh, dkt, dvh, dvt;
  int batch, tokens, heads, group, blocks;
  int flags;           // rows behind the last sequence become 0 in dq: 1, dk: 2, dv: 4
};

template <int D>
struct PackedScale {
  static constexpr double inv_sqrt = D == 64 ? 0.125 : 0.08838834764831845;
  static constexpr float root = D == 64 ? 8.0f : 11.313708498984761f, s = (float)inv_sqrt, c = (float)(1.4426950408889634 * inv_sqrt);
};

__device__ __forceinline__ void packed_fill_rest(const packed_fwd_args& a, const Rows& r, int head, int d, int most) {
  const int rows = min(r.len - r.row0, most);
  bf16* out = a.out + head * a.oh + (i64)(r.start + r.row0) * a.ot;
  if (a.flags & 1)
    for (int i = threadIdx.x; i < rows * (d / 8); i += blockDim.x)
      *(bf16x8*)(out + i / (d / 8) * a.ot + i % (d / 8) * 8) = bf16x8{};
  if ((a.flags & 2) && (int)threadIdx.x < rows)
    a.lse[head * a.lh + (r.start + r.row0 + (int)threadIdx.x) * a.lt] = -__builtin_inff();
}

__device__ __forceinline__ void packed_zero_rest(bf16* x, i64 head_stride, i64 row_stride, const Rows& r, int head, int d, int most) {
  const int rows = min(r.len - r.row0, most);
  x += head * head_stride + (i64)(r.start + r.row0) * row_stride;
  for (int i = threadIdx.x; i < rows * (d / 8); i += blockDim.x)
    *(bf16x8*)(x + i / (d / 8) * row_stride + i % (d / 8) * 8) = bf16x8{};
}

}  // namespace wir
