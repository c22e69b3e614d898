// attn_packed.hip -- attention over packed sequences of different lengths
// (warpir_amd.api.attention_packed).
//
// For query row p of a sequence, in 32 bits but for the operands of the two
// products (bf16):
//   s_j = q_p . k_j / sqrt(D) for j <= p (causal) or every j of the sequence,
//   O_p = sum_j softmax(s)_j v_j,  LSE_p = ln sum_j exp s_j.
#include "wir_packed.h"

namespace {

using wir::bf16;
using wir::i64;

struct fwd_args {
  const bf16* q;       // [H, T, D]
  const bf16* k;       // [H_kv, T, D]
  const bf16* v;
  bf16* out;           // [H, T, D]
  float* lse;          // [H, T]
  const int* offsets;  // [batch + 1]
  i64 qh, qt, kh, kt, vh, vt, oh, ot, lh, lt;
  int batch, tokens, heads, group, blocks;
  int flags;           // 1: rows behind the last sequence become 0 in out, 2: -inf in lse
};

constexpr int WAVES = wir::PACKED_WAVES, ROWS = wir::PACKED_ROWS, TILE = 64;

template <int D>
struct Scale {
  static constexpr double inv_sqrt = D == 64 ? 0.125 : 0.08838834764831845;
  static constexpr float c = (float)(1.4426950408889634 * inv_sqrt);
};

__device__ __forceinline__ void fill_rest(const fwd_args& a, const wir::Rows& r, int head, int d) {
  const int rows = min(r.len - r.row0, ROWS);
  bf16* out = a.out + head * a.oh + (i64)(r.start + r.row0) * a.ot;
  if (a.flags & 1)
    for (int i = threadIdx.x; i < rows * (d / 8); i += 256)
      *(wir::bf16x8*)(out + i / (d / 8) * a.ot + i % (d / 8) * 8) = wir::bf16x8{};
  if ((a.flags & 2) && (int)threadIdx.x < rows)
    a.lse[head * a.lh + (i64)(r.start + r.row0 + threadIdx.x) * a.lt] = -__builtin_inff();
}

// One block of 128 query rows, 32 a wave.  Returns whether a result is NaN (only then may CAREFUL give another).
template <int D, bool CAUSAL>
__device__ __forceinline__ bool forward_block(const fwd_args& a, const wir::Rows& r, int head, char* smem, bool careful) {
  typedef wir::STile<TILE, D, wir::ROWREAD> TK;
  typedef wir::STile<TILE, D, wir::TRREAD> TV;
  constexpr float c = Scale<D>::c;
  const int wave = wir::wave_id(), lane = wir::lane_id();
  const int row0 = r.row0 + wave * 32;
  const int kv = head / a.group;
  wir::HeadTiles<TK> K;
  wir::HeadTiles<TV> V;
  K.init(a.k + kv * a.kh + r.start * a.kt, a.kt, r.len);
  V.init(a.v + kv * a.vh + r.start * a.vt, a.vt, r.len);
  const int keys = CAUSAL ? min(r.len, r.row0 + ROWS) : r.len, tiles = (keys + TILE - 1) / TILE;
  auto load = [&](int t) {
    char* at = smem + t % 2 * TK::BYTES;
    K.load(at, t, wave);
    V.load(at + 2 * TK::BYTES, t, wave);
  };
  wir::RowFrags<32, 1, D / 16> q;
  wir::packed_rows(q, a.q + head * a.qh + r.start * a.qt, a.qt, row0, r.len);
  wir::RTile<32, 32, D> o;
  float m = -__builtin_inff(), l = 0.f;
  wir::fill(o, 0.f);
  auto* odd = (__attribute__((address_space(3))) wir::Odd<D>*)wir::lds(smem + 4 * TK::BYTES);
  if (careful) wir::no_odd<false, WAVES>(odd);
  load(0);
  for (int t = 0; t < tiles; ++t) {
    char *kt = smem + t % 2 * TK::BYTES, *vt = kt + 2 * TK::BYTES;
    const int col0 = t * TILE;
    wir::wait_vm_barrier<0>();
    if (t + 1 < tiles) load(t + 1);
    if (CAUSAL && !careful && col0 > row0 + 31) continue;   // no row of the wave sees the tile
    wir::RTile<32, 32, TILE> s;
    wir::mma_ABt_frags<32, 32, TILE, TK, D / 16>(s, q, kt, 0);
    const bool edge = CAUSAL ? col0 + TILE - 1 > row0 : col0 + TILE > r.len;
    if (edge) {
      wir::seldom();
      wir::packed_mask<CAUSAL>(s, row0, col0, r.len);
    }
    float top = s.f[0][0][0];
#pragma unroll
    for (int cb = 0; cb < 2; ++cb)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s.f[cb][0][i]);
    top = fmaxf(wir::lane_group_reduce<32>(top, wir::OpMax()) * c, m);
    wir::RVec<32, 32> corr;
    corr.v[0] = __builtin_amdgcn_exp2f(m - top);
    m = top;
    float sum[2] = {0.f, 0.f};
    wir::BTile<32, 32, TILE> p;
#pragma unroll
    for (int cb = 0; cb < 2; ++cb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s.f[cb][0][i], c, -m));
        sum[i % 2] += x;
        p.f[cb][0][i / 4][i % 4] = (bf16)x;   // (the product's operand; the sum has the value itself)
      }
    l = l * corr.v[0] + (sum[0] + sum[1]);
    wir::row_scale(o, o, corr);
    if (careful) {
      wir::barrier();
      wir::clear_odd<false, WAVES, TV>(vt, col0, odd);
      wir::barrier();
    }
    wir::mma_rAB<32, 32, TILE, D, TV>(o, p, vt, 0);
  }
  l = wir::lane_group_reduce<32>(l, wir::OpAdd());
  wir::RVec<32, 32> inv;
  inv.v[0] = 1.0f / l;
  wir::row_apply(o, o, inv, [](float x, float s) { return x * s; });
  if (!careful) {
    // an infinite or NaN value that not all of a tile's rows see
    int* flag = (int*)(smem + 4 * TK::BYTES);
    if (threadIdx.x == 0) *flag = 0;
    wir::wait_vm_barrier<0>();
    if (wir::has_nan(o, row0 + lane % 32 < r.len)) *flag = 1;
    wir::barrier();
    const bool odd = *flag;
    wir::barrier();
    if (odd) return true;
  } else {
    wir::wait_vm_barrier<0>();   // the tiles are read: their LDS takes the output
  }
  if (careful) {
    const int row = CAUSAL ? row0 + lane % 32 : r.len - 1;   // the last position that the row sees
#pragma unroll
    for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int d = cb * 32 + wir::ccol<32>(i, lane / 32);
        const bool nan = row >= odd->at[0][d], up = row >= odd->at[1][d], down = row >= odd->at[2][d];
        const float x = o.f[cb][0][i];
        o.f[cb][0][i] = nan || (up && down) ? __builtin_nanf("") : up ? x + __builtin_inff() : down ? x - __builtin_inff() : x;
      }
  }
  const auto O = wir::packed_head(a.out, a.oh, a.ot, head, r.start, r.len, D);
  wir::store_tile_staged<true>(O, o, 0, 0, row0, 0, smem + wave * 32 * D * 2);
  const int row = row0 + lane;
  if (lane < 32 && row < r.len)
    a.lse[head * a.lh + (i64)(r.start + row) * a.lt] = (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
  return false;
}

template <int D, bool CAUSAL>
__device__ __forceinline__ void forward(const fwd_args& a) {
  __shared__ __attribute__((aligned(1024))) char smem[4 * TILE * D * 2 + sizeof(wir::Odd<D>)];
  int x, head;
  wir::packed_program(a.blocks, a.heads, x, head);
  if (CAUSAL) x = a.blocks - 1 - x;   // a sequence's longest block first
  const wir::Rows r = wir::packed_block(a.offsets, a.batch, a.tokens, x);
  if (r.row0 < 0 || r.row0 >= r.len) return;   // (a number that no block has)
  if (r.rest) return fill_rest(a, r, head, D);
  bool careful = false;
  while (forward_block<D, CAUSAL>(a, r, head, smem, careful)) careful = true;
}

}  // namespace

#define PACKED_KERNEL(NAME, D, CAUSAL, WAVES_A_SIMD)                                                    \
  extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(256, 256),                      \
                                            amdgpu_waves_per_eu(WAVES_A_SIMD, WAVES_A_SIMD)))           \
  NAME(const fwd_args args) { forward<D, CAUSAL>(args); }

PACKED_KERNEL(wir_attn_packed_d64, 64, false, 3)
PACKED_KERNEL(wir_attn_packed_d64_causal, 64, true, 3)
PACKED_KERNEL(wir_attn_packed_d128, 128, false, 2)
PACKED_KERNEL(wir_attn_packed_d128_causal, 128, true, 2)
