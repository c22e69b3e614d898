// attn_packed_bwd.hip -- gradients of attention over packed sequences
// (warpir_amd.api.attention_packed_backward; attn_packed.hip is the forward).
//
// With P = exp(s - LSE) again from q, k and the forward's LSE, per sequence:
//   D_p = dO_p . O_p,  dS_pj = P_pj (dO_p . v_j - D_p),
//   dQ_p = sum_j dS_pj k_j / sqrt(D),
//   dK_j = sum_p dS_pj q_p / sqrt(D),  dV_j = sum_p P_pj dO_p,
// the last two over the query heads that share a key/value head as well.
#include "wir_packed.h"

namespace {

using wir::bf16;
using wir::i64;

struct bwd_args {
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
  float* stats;        // [2][H][T]: the LSE in log2 units, D_p
  i64 qh, qt, kh, kt, vh, vt, oh, ot, gh, gt, lh, lt, dqh, dqt, dkh, dkt, dvh, dvt;
  int batch, tokens, heads, group, blocks;
  int flags;           // rows behind the last sequence become 0 in dq: 1, dk: 2, dv: 4
};

constexpr int WAVES = wir::PACKED_WAVES, ROWS = wir::PACKED_ROWS;

template <int D>
struct Scale {
  static constexpr double inv_sqrt = D == 64 ? 0.125 : 0.08838834764831845;
  static constexpr float s = (float)inv_sqrt, c = (float)(1.4426950408889634 * inv_sqrt);
};

__device__ __forceinline__ void zero_rest(bf16* x, i64 head_stride, i64 row_stride, const wir::Rows& r, int head, int d) {
  const int rows = min(r.len - r.row0, ROWS);
  x += head * head_stride + (i64)(r.start + r.row0) * row_stride;
  for (int i = threadIdx.x; i < rows * (d / 8); i += 256)
    *(wir::bf16x8*)(x + i / (d / 8) * row_stride + i % (d / 8) * 8) = wir::bf16x8{};
}

// The workgroup's answer to "is there a NaN in a wave's results", after which the tiles' LDS is free.
__device__ __forceinline__ bool any_wave(bool mine, char* flag_at) {
  auto* flag = (__attribute__((address_space(3))) int*)wir::lds(flag_at);
  wir::wait_vm_barrier<0>();
  if (threadIdx.x == 0) *flag = 0;
  wir::barrier();
  if (mine) *flag = 1;
  wir::barrier();
  const bool any = *flag;
  wir::barrier();
  return any;
}

// dQ of one block of 128 query rows, 32 a wave.
template <int D, int KT, bool CAUSAL>
__device__ __forceinline__ bool dq_block(const bwd_args& a, const wir::Rows& r, int head, char* smem, bool careful) {
  typedef wir::STile<KT, D, wir::BOTH> TK;
  typedef wir::STile<KT, D, wir::ROWREAD> TV;
  constexpr float c = Scale<D>::c;
  const int wave = wir::wave_id(), lane = wir::lane_id();
  const int row0 = r.row0 + wave * 32, kv = head / a.group;
  const auto K = wir::packed_head(const_cast<bf16*>(a.k), a.kh, a.kt, kv, r.start, r.len, D);
  const auto V = wir::packed_head(const_cast<bf16*>(a.v), a.vh, a.vt, kv, r.start, r.len, D);
  const int keys = CAUSAL ? min(r.len, r.row0 + ROWS) : r.len, tiles = (keys + KT - 1) / KT;
  auto load = [&](int t) {
    char* at = smem + t % 2 * TK::BYTES;
    wir::Loader<TK, WAVES>::template load<false>(at, K, 0, 0, t * KT, 0, wave);
    wir::Loader<TV, WAVES>::template load<false>(at + 2 * TK::BYTES, V, 0, 0, t * KT, 0, wave);
  };
  auto* odd = (__attribute__((address_space(3))) wir::Odd<D>*)wir::lds(smem + 4 * TK::BYTES);
  if (CAUSAL && careful) wir::no_odd<false>(odd);
  wir::RowFrags<32, 1, D / 16> q, d_o, o;
  wir::load_row_frags_global(q, wir::packed_head(const_cast<bf16*>(a.q), a.qh, a.qt, head, r.start, r.len, D), 0, 0, row0, 0);
  wir::load_row_frags_global(d_o, wir::packed_head(const_cast<bf16*>(a.d_o), a.gh, a.gt, head, r.start, r.len, D), 0, 0,
                             row0, 0);
  wir::load_row_frags_global(o, wir::packed_head(const_cast<bf16*>(a.o), a.oh, a.ot, head, r.start, r.len, D), 0, 0, row0, 0);
  const int row = row0 + lane % 32;
  float lse = row < r.len ? a.lse[head * a.lh + (i64)(r.start + row) * a.lt] : 0.f;
  wir::RVec<32, 32> dots;
  wir::row_dot(dots, d_o, o);
  lse *= 1.4426950408889634f;
  if (lane < 32 && row < r.len) {
    float* to = a.stats + (i64)head * a.tokens + r.start + row;
    to[0] = lse;
    to[(i64)a.heads * a.tokens] = dots.v[0];
  }
  wir::RTile<32, 32, D> acc;
  wir::fill(acc, 0.f);
  load(0);
  for (int t = 0; t < tiles; ++t) {
    char *kt = smem + t % 2 * TK::BYTES, *vt = kt + 2 * TK::BYTES;
    const int col0 = t * KT;
    wir::wait_vm_barrier<0>();
    if (t + 1 < tiles) load(t + 1);
    if (CAUSAL && !careful && col0 > row0 + 31) continue;   // no row of the wave sees the tile
    wir::RTile<32, 32, KT> s, dp;
    wir::BTile<32, 32, KT> ds;
    wir::mma_ABt_frags<32, 32, KT, TK, D / 16>(s, q, kt, 0);
    const bool edge = CAUSAL ? col0 + KT - 1 > row0 : col0 + KT > r.len;
    if (edge) wir::packed_mask<CAUSAL, false>(s, row0, col0, r.len);
    wir::mma_ABt_frags<32, 32, KT, TV, D / 16>(dp, d_o, vt, 0);
#pragma unroll
    for (int cb = 0; cb < KT / 32; ++cb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s.f[cb][0][i], c, -lse));
        dp.f[cb][0][i] = p * (dp.f[cb][0][i] - dots.v[0]);
        s.f[cb][0][i] = p;
      }
    if (edge) {   // (a value that a row does not see may be NaN)
#pragma unroll
      for (int cb = 0; cb < KT / 32; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i) dp.f[cb][0][i] = s.f[cb][0][i] == 0.f ? 0.f : dp.f[cb][0][i];
    }
    wir::to_bf16(ds, dp);
    if (CAUSAL && careful) {
      wir::barrier();
      wir::clear_odd<false, TK>(kt, col0, odd);
      wir::barrier();
    }
    wir::mma_rAB<32, 32, KT, D, TK>(acc, ds, kt, 0);
  }
  if (CAUSAL && !careful) {
    if (any_wave(wir::has_nan(acc), smem + 4 * TK::BYTES)) return true;
  } else {
    wir::wait_vm_barrier<0>();
  }
#pragma unroll
  for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc.f[cb][0][i] *= Scale<D>::s;
  if (CAUSAL && careful) {
#pragma unroll
    for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int d = cb * 32 + wir::ccol<32>(i, lane / 32);
        const int first = min(odd->at[0][d], min(odd->at[1][d], odd->at[2][d]));
        acc.f[cb][0][i] = row >= first ? __builtin_nanf("") : acc.f[cb][0][i];
      }
  }
  wir::store_tile_staged<true>(wir::packed_head(a.dq, a.dqh, a.dqt, head, r.start, r.len, D), acc, 0, 0, row0, 0,
                               smem + wave * 32 * D * 2);
  return false;
}

template <int D, int KT, bool CAUSAL>
__device__ __forceinline__ void dq_kernel(const bwd_args& a) {
  constexpr int STAGE = WAVES * 32 * D * 2, TILES = 4 * KT * D * 2;
  static_assert(STAGE <= TILES, "the output goes through the tiles' LDS");
  __shared__ __attribute__((aligned(1024))) char smem[TILES + sizeof(wir::Odd<D>)];
  int x, head;
  wir::packed_program(a.blocks, a.heads, x, head);
  if (CAUSAL) x = a.blocks - 1 - x;   // a sequence's longest block first
  const wir::Rows r = wir::packed_block(a.offsets, a.batch, a.tokens, x);
  if (r.row0 < 0 || r.row0 >= r.len) return;   // (a number that no block has)
  if (r.rest) {
    if (a.flags & 1) zero_rest(a.dq, a.dqh, a.dqt, r, head, D);
    return;
  }
  bool careful = false;
  while (dq_block<D, KT, CAUSAL>(a, r, head, smem, careful)) careful = true;
}

// dK and dV of one block of 128 keys, 32 a wave, over the tiles of QT queries of the group's heads one after another.
template <int D, int QT, bool CAUSAL>
__device__ __forceinline__ bool dkdv_block(const bwd_args& a, const wir::Rows& r, int kv, char* smem, bool careful) {
  typedef wir::STile<QT, D, wir::BOTH> T;
  constexpr float c = Scale<D>::c;
  static_assert(WAVES * 32 * D * 2 <= 4 * T::BYTES, "the outputs go through the tiles' LDS");
  constexpr int VEC = 4 * T::BYTES, ODD = VEC + 4 * QT * 4;
  const int wave = wir::wave_id(), lane = wir::lane_id();
  const int row0 = r.row0 + wave * 32;
  const int first = CAUSAL ? r.row0 / QT : 0, tiles = (r.len + QT - 1) / QT;
  auto load = [&](int head, int t, int slot) {
    char* at = smem + slot * T::BYTES;
    const i64 stat = (i64)head * a.tokens + r.start;
    wir::Loader<T, WAVES>::template load<false>(
        at, wir::packed_head(const_cast<bf16*>(a.q), a.qh, a.qt, head, r.start, r.len, D), 0, 0, t * QT, 0, wave);
    wir::Loader<T, WAVES>::template load<false>(
        at + 2 * T::BYTES, wir::packed_head(const_cast<bf16*>(a.d_o), a.gh, a.gt, head, r.start, r.len, D), 0, 0, t * QT, 0,
        wave);
    wir::VecLoader<QT, WAVES>::template load<false>(
        smem + VEC + slot * QT * 4, wir::gl<float>{a.stats + stat, 1, 1, r.len, 1, 0, 0, 1}, 0, 0, t * QT, wave);
    wir::VecLoader<QT, WAVES>::template load<false>(
        smem + VEC + (2 + slot) * QT * 4,
        wir::gl<float>{a.stats + (i64)a.heads * a.tokens + stat, 1, 1, r.len, 1, 0, 0, 1}, 0, 0, t * QT, wave);
  };
  auto* odd = (__attribute__((address_space(3))) wir::Odd<D>*)wir::lds(smem + ODD);
  if (CAUSAL && careful) wir::no_odd<true>(odd), wir::no_odd<true>(odd + 1);
  wir::RowFrags<32, 1, D / 16> k, v;
  wir::load_row_frags_global(k, wir::packed_head(const_cast<bf16*>(a.k), a.kh, a.kt, kv, r.start, r.len, D), 0, 0, row0, 0);
  wir::load_row_frags_global(v, wir::packed_head(const_cast<bf16*>(a.v), a.vh, a.vt, kv, r.start, r.len, D), 0, 0, row0, 0);
  wir::RTile<32, 32, D> dk, dv;
  wir::fill(dk, 0.f);
  wir::fill(dv, 0.f);
  int head = kv * a.group, t = first, slot = 0;
  const int last = head + a.group;
  load(head, t, 0);
  while (head < last) {
    int head1 = head, t1 = t + 1;   // the next tile
    if (t1 == tiles) ++head1, t1 = first;
    char *qt = smem + slot * T::BYTES, *dot = qt + 2 * T::BYTES;
    const int col0 = t * QT;
    wir::wait_vm_barrier<0>();
    if (head1 < last) load(head1, t1, slot ^ 1);
    if (!CAUSAL || careful || col0 + QT - 1 >= row0) {   // (else no row of the wave is seen from the tile)
      wir::RTile<32, 32, QT> s, dp;
      wir::BTile<32, 32, QT> pb, ds;
      wir::CVec<32, QT> lse, dots;
      wir::load_cvec_lds(lse, smem + VEC + slot * QT * 4, 0);
      wir::load_cvec_lds(dots, smem + VEC + (2 + slot) * QT * 4, 0);
      wir::mma_ABt_frags<32, 32, QT, T, D / 16>(s, k, qt, 0);
      wir::mma_ABt_frags<32, 32, QT, T, D / 16>(dp, v, dot, 0);
#pragma unroll
      for (int cb = 0; cb < QT / 32; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s.f[cb][0][i], c, -lse.v[cb][i]));
          dp.f[cb][0][i] = p * (dp.f[cb][0][i] - dots.v[cb][i]);
          s.f[cb][0][i] = p;
        }
      if (CAUSAL && col0 < row0 + 31) {   // (a query that does not see the row may hold NaN)
#pragma unroll
        for (int cb = 0; cb < QT / 32; ++cb)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const bool seen = row0 + lane % 32 <= col0 + cb * 32 + wir::ccol<32>(i, lane / 32);
            s.f[cb][0][i] = seen ? s.f[cb][0][i] : 0.f;
            dp.f[cb][0][i] = seen ? dp.f[cb][0][i] : 0.f;
          }
      }
      wir::to_bf16(pb, s);
      wir::to_bf16(ds, dp);
      if (CAUSAL && careful) {
        wir::barrier();
        wir::clear_odd<true, T>(qt, col0, odd);
        wir::clear_odd<true, T>(dot, col0, odd + 1);
        wir::barrier();
      }
      wir::mma_rAB<32, 32, QT, D, T>(dv, pb, dot, 0);
      wir::mma_rAB<32, 32, QT, D, T>(dk, ds, qt, 0);
    }
    head = head1, t = t1, slot ^= 1;
  }
  if (CAUSAL && !careful) {
    const bool nan = wir::has_nan(dk) || wir::has_nan(dv);
    if (any_wave(nan, smem + ODD)) return true;
  } else {
    wir::wait_vm_barrier<0>();
  }
#pragma unroll
  for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
    for (int i = 0; i < 16; ++i) dk.f[cb][0][i] *= Scale<D>::s;
  if (CAUSAL && careful) {
    const int row = row0 + lane % 32;
#pragma unroll
    for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int d = cb * 32 + wir::ccol<32>(i, lane / 32);
        const int end_k = max(odd->at[0][d], max(odd->at[1][d], odd->at[2][d]));
        const int end_v = max(odd[1].at[0][d], max(odd[1].at[1][d], odd[1].at[2][d]));
        dk.f[cb][0][i] = row <= end_k ? __builtin_nanf("") : dk.f[cb][0][i];
        dv.f[cb][0][i] = row <= end_v ? __builtin_nanf("") : dv.f[cb][0][i];
      }
  }
  char* stage = smem + wave * 32 * D * 2;
  wir::store_tile_staged<true>(wir::packed_head(a.dk, a.dkh, a.dkt, kv, r.start, r.len, D), dk, 0, 0, row0, 0, stage);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (the wave's own part of the LDS: its reads are done)
  wir::store_tile_staged<true>(wir::packed_head(a.dv, a.dvh, a.dvt, kv, r.start, r.len, D), dv, 0, 0, row0, 0, stage);
  return false;
}

template <int D, int QT, bool CAUSAL>
__device__ __forceinline__ void dkdv_kernel(const bwd_args& a) {
  __shared__ __attribute__((aligned(1024))) char smem[4 * QT * D * 2 + 16 * QT + 2 * sizeof(wir::Odd<D>)];
  int x, kv;
  wir::packed_program(a.blocks, a.heads / a.group, x, kv);   // a sequence's longest block is its first
  const wir::Rows r = wir::packed_block(a.offsets, a.batch, a.tokens, x);
  if (r.row0 < 0 || r.row0 >= r.len) return;   // (a number that no block has)
  if (r.rest) {
    if (a.flags & 2) zero_rest(a.dk, a.dkh, a.dkt, r, kv, D);
    if (a.flags & 4) zero_rest(a.dv, a.dvh, a.dvt, r, kv, D);
    return;
  }
  bool careful = false;
  while (dkdv_block<D, QT, CAUSAL>(a, r, kv, smem, careful)) careful = true;
}

}  // namespace

#define PACKED_KERNEL(NAME, CALL, WAVES_A_SIMD)                                                         \
  extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(256, 256),                      \
                                            amdgpu_waves_per_eu(WAVES_A_SIMD, WAVES_A_SIMD)))           \
  NAME(const bwd_args args) { CALL(args); }

PACKED_KERNEL(wir_attn_packed_dq_d64, (dq_kernel<64, 32, false>), 3)
PACKED_KERNEL(wir_attn_packed_dq_d64_causal, (dq_kernel<64, 32, true>), 3)
PACKED_KERNEL(wir_attn_packed_dq_d128, (dq_kernel<128, 32, false>), 2)
PACKED_KERNEL(wir_attn_packed_dq_d128_causal, (dq_kernel<128, 32, true>), 2)
PACKED_KERNEL(wir_attn_packed_dkdv_d64, (dkdv_kernel<64, 32, false>), 2)
PACKED_KERNEL(wir_attn_packed_dkdv_d64_causal, (dkdv_kernel<64, 32, true>), 2)
PACKED_KERNEL(wir_attn_packed_dkdv_d128, (dkdv_kernel<128, 64, false>), 1)
PACKED_KERNEL(wir_attn_packed_dkdv_d128_causal, (dkdv_kernel<128, 64, true>), 1)
