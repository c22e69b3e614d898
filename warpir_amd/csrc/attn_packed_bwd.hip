// attn_packed_bwd.hip -- gradients of attention over packed sequences
// (warpir_amd.api.attention_packed_backward; attn_packed.hip is the forward).
//
// With P = exp(s - LSE) again from q, k and the forward's LSE, per sequence:
//   D_p = dO_p . O_p,  dS_pj = P_pj (dO_p . v_j - D_p),
//   dQ_p = sum_j dS_pj k_j / sqrt(D),
//   dK_j = sum_p dS_pj q_p / sqrt(D),  dV_j = sum_p P_pj dO_p,
// the last two over the query heads that share a key/value head as well.
#include "wir_packed_args.h"

namespace {

using wir::bf16;
using wir::i64;

constexpr int WAVES = wir::PACKED_WAVES, ROWS = wir::PACKED_ROWS;

// dQ of one block of 128 query rows, 32 a wave.  In the time of a tile of 32
// keys t a wave takes the product of dS(t - 1) with K(t - 1), the scores of t,
// q . k and dO . v in turn, and their exponentials; the operands of both are
// one stream of LDS reads that runs AHEAD products before their use.  dS is
// rounded to bf16 as the product's operand; P, dO . v and the sums are fp32.
//
// Measured: 8 x 4096 tokens, 16 heads of 128: 1.31 ms (its three products 1260
// TFLOP/s), causal 0.72; 64 x 512 tokens, 16 heads of 64: 0.14 ms (740).  At D =
// 128 LDS bounds it, as the forward: four SIMDs' three products, 96 cycles, ask for
// 128 of its cycles, and matrix instructions run in 69% of them.  Tiles of 32 keys,
// because three of K and two of V of 64 would leave room for one workgroup a CU.
template <int D, bool CAUSAL>
struct Dq {
  static constexpr int KT = 32, AHEAD = D == 64 ? 3 : 5, KS = D / 16, CB = D / 32;
  static constexpr int SCORES = 2 * KS, PRODUCTS = KT / 16 * CB;   // products of a wave for a tile
  typedef wir::STile<KT, D, wir::BOTH> TK;
  typedef wir::STile<KT, D, wir::ROWREAD> TV;
  typedef __attribute__((address_space(3))) wir::bf16x8 lds_bf16x8;
  typedef __attribute__((address_space(3))) wir::i16x4 lds_i16x4;
  typedef __attribute__((address_space(3))) wir::Odd<D> lds_odd;
  // LDS: three tiles of K, two of V, notes of what is odd
  static constexpr int VALUES = 3 * TK::BYTES, ODD = VALUES + 2 * TV::BYTES, BYTES = ODD + sizeof(wir::Odd<D>);
  static_assert(WAVES * 32 * D * 2 <= ODD, "the output goes through the tiles' LDS");

  const wir::packed_bwd_args& a;
  const wir::Rows& r;
  char* smem;
  int wave, lane, row0, tiles;
  wir::HeadTiles<TK> K;
  wir::HeadTiles<TV> V;
  unsigned k_at, v_at, tr_at;      // the lane's places in a tile, as operands of the scores and of the product
  wir::RowFrags<32, 1, KS> q, d_o;
  wir::RTile<32, 32, D> acc;
  wir::RTile<32, 32, KT> s, dp;
  wir::BTile<32, 32, KT> ds;
  wir::f32x16 dots;                // -D_p of the lane's row, what dO . v begins with
  float lse;                       // in log2 units

  __device__ __forceinline__ Dq(const wir::packed_bwd_args& args, const wir::Rows& rows, char* lds) : a(args), r(rows), smem(lds) {}

  __device__ __forceinline__ void product(const wir::bf16x8& b, int i) {
    const int g = 2 * (i / CB), cb = i % CB;
    acc.f[cb][0] = wir::MF<32>::mma(b, wir::cat(ds.f[0][0][g], ds.f[0][0][g + 1]), acc.f[cb][0]);
  }

  // The product of tile t - 1 (PRODUCT), whose keys are in slot `before`, and the scores of tile t (SCORE), in `slot`.
  template <bool PRODUCT, bool SCORE>
  __device__ __forceinline__ void stream(int t, int slot, int before) {
    constexpr int N0 = PRODUCT ? PRODUCTS : 0, N = N0 + (SCORE ? SCORES : 0);
    const unsigned from = tr_at + before * TK::BYTES, keys = k_at + slot * TK::BYTES, values = v_at + t % 2 * TV::BYTES;
    wir::bf16x8 ring[AHEAD + 1];
    auto read = [&](auto at) {
      constexpr int n = decltype(at)::value, i = n - N0;
      if constexpr (n < N0) {
        const unsigned tile = from ^ (n % CB * 64);
        constexpr int rows = n / CB * 16 * D * 2;   // (two groups of eight rows)
        const auto lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(tile + rows));
        const auto hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)((tile ^ 32) + rows + 8 * D * 2));
        ring[n % (AHEAD + 1)] = wir::cat(__builtin_bit_cast(wir::bf16x4, lo), __builtin_bit_cast(wir::bf16x4, hi));
      } else {
        ring[n % (AHEAD + 1)] = *(lds_bf16x8*)((i % 2 ? values : keys) ^ (i / 2 * 32));
      }
    };
    __builtin_amdgcn_s_setprio(1);
    wir::static_for<0, (AHEAD < N ? AHEAD : N)>(read);
    wir::static_for<0, N>([&](auto at) {
      constexpr int n = decltype(at)::value, i = n - N0;
      if constexpr (n + AHEAD < N) read(wir::ic<n + AHEAD>{});
      __builtin_amdgcn_sched_barrier(0);
      const wir::bf16x8& b = ring[n % (AHEAD + 1)];
      if constexpr (n < N0) product(b, n);
      else if constexpr (i % 2 == 0) s.f[0][0] = wir::MF<32>::mma(b, q.f[0][i / 2], i < 2 ? wir::f32x16{} : s.f[0][0]);
      else dp.f[0][0] = wir::MF<32>::mma(b, d_o.f[0][i / 2], i < 2 ? dots : dp.f[0][0]);
      __builtin_amdgcn_sched_barrier(0);
    });
    __builtin_amdgcn_s_setprio(0);
  }

  __device__ __forceinline__ void finish_scores(int t) {
    constexpr float c = wir::PackedScale<D>::c;
    const int col0 = t * KT;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s.f[0][0][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s.f[0][0][i], c, -lse));
      dp.f[0][0][i] *= s.f[0][0][i];
    }
    if (CAUSAL ? col0 + KT - 1 > row0 : col0 + KT > r.len) {   // (a value that a row does not see may be NaN)
      const int row = row0 + lane % 32, half = wir::seldom(lane / 32);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int col = col0 + wir::ccol<32>(i, half);
        dp.f[0][0][i] = (CAUSAL ? col <= row : col < r.len) ? dp.f[0][0][i] : 0.f;
      }
    }
    wir::to_bf16(ds, dp);
  }

  __device__ __forceinline__ bool run(int head, bool careful) {
    wave = wir::wave_id(), lane = wir::lane_id();
    row0 = r.row0 + wave * 32;
    const int kv = head / a.group, keys = CAUSAL ? min(r.len, r.row0 + ROWS) : r.len;
    tiles = (keys + KT - 1) / KT;
    const int mine = row0 >= r.len ? 0 : CAUSAL ? min(tiles, (row0 + 31) / KT + 1) : tiles;   // tiles that the wave's rows see
    K.init(a.k + kv * a.kh + r.start * a.kt, a.kt, r.len);
    V.init(a.v + kv * a.vh + r.start * a.vt, a.vt, r.len);
    const int part = lane % 16;   // of the transposed reads
    k_at = wir::lds_addr(smem) + TK::chunk_off(lane % 32, lane / 32);
    v_at = wir::lds_addr(smem) + VALUES + TV::chunk_off(lane % 32, lane / 32);
    tr_at = wir::lds_addr(smem) + TK::elem_off(lane / 32 * 4 + part / 4, lane % 32 / 16 * 16 + 4 * (part % 4));
    auto* odd = (lds_odd*)wir::lds(smem + ODD);
    if (careful) wir::no_odd<false, WAVES>(odd);
    K.load(smem, 0, wave);
    V.load(smem + VALUES, 0, wave);
    wir::packed_rows(q, a.q + head * a.qh + r.start * a.qt, a.qt, row0, r.len);
    wir::packed_rows(d_o, a.d_o + head * a.gh + r.start * a.gt, a.gt, row0, r.len);
    const int row = row0 + lane % 32;
    lse = a.lse[head * a.lh + (r.start + min(row, r.len - 1)) * a.lt];
    {
      wir::RowFrags<32, 1, KS> o;
      wir::packed_rows(o, a.o + head * a.oh + r.start * a.ot, a.ot, row0, r.len);
      wir::RVec<32, 32> sum;
      wir::row_dot(sum, d_o, o);
      dots = wir::f32x16{} - sum.v[0];
    }
    if (lane < 32 && row < r.len) {
      float* to = a.stats + (i64)head * a.tokens + r.start + row;
      to[0] = -lse * wir::PackedScale<D>::root;
      to[(i64)a.heads * a.tokens] = dots[0];
    }
    lse *= 1.4426950408889634f;
    wir::fill(acc, 0.f);
    int t = 0, slot = 0, before = 2;   // of tile t, of t - 1
    auto settle = [&]() {   // tile t has come, t + 1 is asked for
      wir::wait_vm_barrier<0>();
      const int next = slot == 2 ? 0 : slot + 1;
      if (t + 1 < tiles) {
        K.load(smem + next * TK::BYTES, t + 1, wave);
        V.load(smem + VALUES + (t + 1) % 2 * TV::BYTES, t + 1, wave);
      }
      if (careful && t > 0) {
        wir::clear_odd<false, WAVES, TK>(smem + before * TK::BYTES, (t - 1) * KT, odd);
        wir::barrier();
      }
    };
    auto advance = [&]() {
      ++t;
      before = slot;
      slot = slot == 2 ? 0 : slot + 1;
    };
    if (mine > 0) {
      settle();
      stream<false, true>(t, slot, before);
      finish_scores(t);
      advance();
      while (t < mine) {
        settle();
        stream<true, true>(t, slot, before);
        finish_scores(t);
        advance();
      }
      settle();
      stream<true, false>(t, slot, before);
      advance();
    }
    while (t <= tiles) {
      settle();
      advance();
    }
    if (!careful) {
      if (wir::any_wave(wir::has_nan(acc, row < r.len), smem + ODD)) return true;
    } else {
      wir::wait_vm_barrier<0>();
    }
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) acc.f[cb][0] *= wir::PackedScale<D>::s;
    if (careful) {
#pragma unroll
      for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int d = cb * 32 + wir::ccol<32>(i, lane / 32);
          const int first = min(odd->at[0][d], min(odd->at[1][d], odd->at[2][d]));
          acc.f[cb][0][i] = (CAUSAL ? row : r.len - 1) >= first ? __builtin_nanf("") : acc.f[cb][0][i];
        }
    }
    wir::store_tile_staged<true>(wir::packed_head(a.dq, a.dqh, a.dqt, head, r.start, r.len, D), acc, 0, 0, row0, 0,
                                 smem + wave * 32 * D * 2);
    return false;
  }
};

template <int D, bool CAUSAL>
__device__ __forceinline__ void dq_kernel(const wir::packed_bwd_args& a) {
  __shared__ __attribute__((aligned(1024))) char smem[Dq<D, CAUSAL>::BYTES];
  int x, head;
  wir::packed_program(a, a.heads, ROWS, x, head);
  if (CAUSAL) x = a.blocks - 1 - x;   // a sequence's longest block first
  const wir::Rows r = wir::packed_block(a.offsets, a.batch, a.tokens, x);
  if (r.row0 < 0 || r.row0 >= r.len) return;   // (a number that no block has)
  if (r.rest) {
    if (a.flags & 1) wir::packed_zero_rest(a.dq, a.dqh, a.dqt, r, head, D, ROWS);
    return;
  }
  Dq<D, CAUSAL> p(a, r, smem);
  bool careful = false;
  while (p.run(head, careful)) careful = true;
}

// dK and dV of one block of 128 keys, 32 a wave, over the tiles of QT queries of
// the group's heads one after another (so the sums over a group are in one wave's
// registers, in an order that the lengths fix).  In the time of a tile t a wave
// takes the products of P and dS of t - 1 with dO and Q, the scores of t, q . k
// and v . dO in turn, and their exponentials; the operands of both are one
// stream of LDS reads that runs AHEAD products before their use.  P and dS are
// rounded to bf16 as the products' operands.
//
// For D = 64, where both sums fit with two waves a SIMD.  8 x 4096 tokens, 32 heads:
// 1.94 ms (four products, 1130 TFLOP/s), causal 1.21; 64 x 512, 16 heads 0.17 (815).
// (Tiles of 32 queries 2.2, 1.39 and 0.18 ms; pairs of waves as below 1.70, causal.)
template <int D, int QT, bool CAUSAL>
struct Dkdv {
  static constexpr int AHEAD = 4, KS = D / 16, CB = D / 32, QB = QT / 32;
  static constexpr int SCORES = 2 * KS * QB, PRODUCTS = 2 * CB * (QT / 16);   // products of a wave for a tile
  typedef wir::STile<QT, D, wir::BOTH> T;
  typedef __attribute__((address_space(3))) wir::bf16x8 lds_bf16x8;
  typedef __attribute__((address_space(3))) wir::i16x4 lds_i16x4;
  typedef __attribute__((address_space(3))) wir::f32x4 lds_f32x4;
  typedef __attribute__((address_space(3))) wir::Odd<D> lds_odd;
  // LDS: three slots of a Q and a dO tile, the tiles' statistics, notes of what is odd
  static constexpr int SLOT = 2 * T::BYTES, VEC = 3 * SLOT, ODD = VEC + 3 * 2 * QT * 4, BYTES = ODD + 2 * sizeof(wir::Odd<D>);
  static_assert(WAVES * 32 * D * 2 <= VEC, "the outputs go through the tiles' LDS");

  struct At {
    int head, t;
  };

  const wir::packed_bwd_args& a;
  const wir::Rows& r;
  char* smem;
  int wave, lane, row0, first, tiles;
  wir::HeadTiles<T> Q, G;
  unsigned row_at, tr_at;          // the lane's places in a tile, as operands of the scores and of the products
  wir::RowFrags<32, 1, KS> k, v;
  wir::RTile<32, 32, D> dk, dv;
  wir::RTile<32, 32, QT> s, dp;
  wir::BTile<32, 32, QT> pb, ds;

  __device__ __forceinline__ Dkdv(const wir::packed_bwd_args& args, const wir::Rows& rows, char* lds) : a(args), r(rows), smem(lds) {}

  __device__ __forceinline__ At after(At i) const { return i.t + 1 < tiles ? At{i.head, i.t + 1} : At{i.head + 1, first}; }

  __device__ __forceinline__ void load(At i, int slot) {
    char* at = smem + slot * SLOT;
    Q.base = (const char*)(a.q + i.head * a.qh + r.start * a.qt);
    G.base = (const char*)(a.d_o + i.head * a.gh + r.start * a.gt);
    Q.load(at, i.t, wave);
    G.load(at + T::BYTES, i.t, wave);
    if (wave < 2 && lane < QT) {   // a wave each for the two statistics
      const float* from = a.stats + ((i64)(wave * a.heads + i.head) * a.tokens + r.start);
      wir::dma4_v(from + min(i.t * QT + lane, r.len - 1), wir::lds_addr(smem + VEC + (2 * slot + wave) * QT * 4));
    }
  }

  // The scores' sums begin with the statistics: p = exp2(c (q . k - LSE sqrt(D))), dP - D_p = dO . v - D_p.
  __device__ __forceinline__ void begin_scores(int slot) {
    const auto* vec = (lds_f32x4*)wir::lds(smem + VEC + 2 * slot * QT * 4 + lane / 32 * 16);
#pragma unroll
    for (int cb = 0; cb < QB; ++cb)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const wir::f32x4 x0 = vec[8 * cb + 2 * g], x1 = vec[QT / 4 + 8 * cb + 2 * g];
#pragma unroll
        for (int j = 0; j < 4; ++j) s.f[cb][0][4 * g + j] = x0[j], dp.f[cb][0][4 * g + j] = x1[j];
      }
  }

  // The products of the tile in `before` (PRODUCT) and the scores of that in `slot` (SCORE).
  template <bool PRODUCT, bool SCORE>
  __device__ __forceinline__ void stream(int slot, int before) {
    constexpr int N0 = PRODUCT ? PRODUCTS : 0, N = N0 + (SCORE ? SCORES : 0);
    const unsigned from = tr_at + before * SLOT, rows = row_at + slot * SLOT;
    wir::bf16x8 ring[AHEAD + 1];
    auto read = [&](auto at) {
      constexpr int n = decltype(at)::value, i = n - N0;
      if constexpr (n < N0) {   // dO for dV and Q for dK in turn
        constexpr int cb = n / 2 % CB, down = n / 2 / CB * 16 * D * 2;   // (two groups of eight rows)
        const unsigned tile = (from + (n % 2 ? 0 : T::BYTES)) ^ (cb * 64);
        const auto lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(tile + down));
        const auto hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)((tile ^ 32) + down + 8 * D * 2));
        ring[n % (AHEAD + 1)] = wir::cat(__builtin_bit_cast(wir::bf16x4, lo), __builtin_bit_cast(wir::bf16x4, hi));
      } else {                  // Q and dO in turn
        ring[n % (AHEAD + 1)] = *(lds_bf16x8*)((rows ^ (i / 2 % KS * 32)) + i % 2 * T::BYTES + i / 2 / KS * 32 * D * 2);
      }
    };
    if (SCORE) begin_scores(slot);
    __builtin_amdgcn_s_setprio(1);
    wir::static_for<0, AHEAD>(read);
    wir::static_for<0, N>([&](auto at) {
      constexpr int n = decltype(at)::value, i = n - N0;
      if constexpr (n + AHEAD < N) read(wir::ic<n + AHEAD>{});
      __builtin_amdgcn_sched_barrier(0);
      const wir::bf16x8& b = ring[n % (AHEAD + 1)];
      if constexpr (n < N0) {
        constexpr int cb = n / 2 % CB, g = 2 * (n / 2 / CB);
        auto& acc = n % 2 ? dk : dv;
        const auto& x = n % 2 ? ds : pb;
        acc.f[cb][0] = wir::MF<32>::mma(b, wir::cat(x.f[g / 4][0][g % 4], x.f[g / 4][0][g % 4 + 1]), acc.f[cb][0]);
      } else if constexpr (i % 2 == 0) {
        s.f[i / 2 / KS][0] = wir::MF<32>::mma(b, k.f[0][i / 2 % KS], s.f[i / 2 / KS][0]);
      } else {
        dp.f[i / 2 / KS][0] = wir::MF<32>::mma(b, v.f[0][i / 2 % KS], dp.f[i / 2 / KS][0]);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    __builtin_amdgcn_s_setprio(0);
  }

  __device__ __forceinline__ void finish_scores(int t) {
    constexpr float c = wir::PackedScale<D>::c;
    const int col0 = t * QT;
#pragma unroll
    for (int cb = 0; cb < QB; ++cb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s.f[cb][0][i] = __builtin_amdgcn_exp2f(s.f[cb][0][i] * c);
        dp.f[cb][0][i] *= s.f[cb][0][i];
      }
    // (a query that does not see the row may hold NaN; past the end the last one stands again)
    if ((CAUSAL && col0 < row0 + 31) || col0 + QT > r.len) {
      const int half = wir::seldom(lane / 32);
#pragma unroll
      for (int cb = 0; cb < QB; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int col = col0 + cb * 32 + wir::ccol<32>(i, half);
          const bool seen = (!CAUSAL || row0 + lane % 32 <= col) && col < r.len;
          s.f[cb][0][i] = seen ? s.f[cb][0][i] : 0.f;
          dp.f[cb][0][i] = seen ? dp.f[cb][0][i] : 0.f;
        }
    }
    wir::to_bf16(pb, s);
    wir::to_bf16(ds, dp);
  }

  __device__ __forceinline__ bool run(int kv, bool careful) {
    wave = wir::wave_id(), lane = wir::lane_id();
    row0 = r.row0 + wave * 32;
    first = CAUSAL ? r.row0 / QT : 0, tiles = (r.len + QT - 1) / QT;
    Q.init(a.q + r.start * a.qt, a.qt, r.len);
    G.init(a.d_o + r.start * a.gt, a.gt, r.len);
    const int part = lane % 16;   // of the transposed reads
    row_at = wir::lds_addr(smem) + T::chunk_off(lane % 32, lane / 32);
    tr_at = wir::lds_addr(smem) + T::elem_off(lane / 32 * 4 + part / 4, lane % 32 / 16 * 16 + 4 * (part % 4));
    auto* odd = (lds_odd*)wir::lds(smem + ODD);
    if (careful) wir::no_odd<true, WAVES>(odd), wir::no_odd<true, WAVES>(odd + 1);
    At now{kv * a.group, first};
    const int end = now.head + a.group;
    const int mine = row0 >= r.len ? tiles : CAUSAL ? row0 / QT : first;   // the first tile with queries that see the wave's rows
    load(now, 0);
    wir::packed_rows(k, a.k + kv * a.kh + r.start * a.kt, a.kt, row0, r.len);
    wir::packed_rows(v, a.v + kv * a.vh + r.start * a.vt, a.vt, row0, r.len);
    wir::fill(dk, 0.f);
    wir::fill(dv, 0.f);
    int slot = 0, before = 2;   // of the tile, of the one before
    auto settle = [&]() {       // the tile has come, the next one is asked for
      const At next = after(now);
      wir::wait_vm_barrier<0>();
      if (next.head < end) load(next, slot == 2 ? 0 : slot + 1);
    };
    auto step = [&]() {
      const int t = now.t;
      now = after(now), before = slot, slot = slot == 2 ? 0 : slot + 1;
      settle();
      if (careful) {
        wir::clear_odd<true, WAVES, T>(smem + before * SLOT, t * QT, odd);
        wir::clear_odd<true, WAVES, T>(smem + before * SLOT + T::BYTES, t * QT, odd + 1);
        wir::barrier();
      }
    };
    settle();
    while (now.head < end) {
      const int head = now.head;
      while (now.head == head && now.t < mine) step();
      if (now.head != head) continue;
      stream<false, true>(slot, before);
      finish_scores(now.t);
      for (step(); now.head == head; step()) {
        stream<true, true>(slot, before);
        finish_scores(now.t);
      }
      stream<true, false>(slot, before);
    }
    const int row = row0 + lane % 32;
    if (!careful) {
      const bool in = row < r.len, nan = wir::has_nan(dk, in) || wir::has_nan(dv, in);
      if (wir::any_wave(nan, smem + ODD)) return true;
    } else {
      wir::wait_vm_barrier<0>();
    }
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
      for (int i = 0; i < 16; ++i) dk.f[cb][0][i] *= wir::PackedScale<D>::s;
    if (careful) {
      // (the scores of an infinite query are no numbers, and dS with them; an infinite dO makes a sum of dV infinite)
      const int from = CAUSAL ? row : 0;   // the first query that sees the row
#pragma unroll
      for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int d = cb * 32 + wir::ccol<32>(i, lane / 32);
          const int end_k = max(odd->at[0][d], max(odd->at[1][d], odd->at[2][d]));
          dk.f[cb][0][i] = from <= end_k ? __builtin_nanf("") : dk.f[cb][0][i];
          dv.f[cb][0][i] = wir::with_odd<true>(odd + 1, d, from, dv.f[cb][0][i]);
        }
    }
    char* stage = smem + wave * 32 * D * 2;
    wir::store_tile_staged<true>(wir::packed_head(a.dk, a.dkh, a.dkt, kv, r.start, r.len, D), dk, 0, 0, row0, 0, stage);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (the wave's own part of the LDS: its reads are done)
    wir::store_tile_staged<true>(wir::packed_head(a.dv, a.dvh, a.dvt, kv, r.start, r.len, D), dv, 0, 0, row0, 0, stage);
    return false;
  }
};

// The same with eight waves, of which two share 32 keys: one takes the scores of
// a tile's first 32 queries and dV, the other those of its last 32 and dK.  A
// wave then has one sum of 64 registers instead of two, so that two waves a
// SIMD hide one another.  They hand each other the half of P and of dS that the
// other needs through LDS: in the time of one tile a wave takes the product of
// tile t and the scores of tile t + 1, in opposite orders.  The operands of both
// are one stream of LDS reads that runs AHEAD products before their use.
//
// For D = 128: 8 x 4096 tokens, 16 heads: 2.03 ms (four products, 1080 TFLOP/s),
// causal 1.21; 4 x 4096, 32/8 heads, causal 1.05 (all of it in a wave, one wave a
// SIMD, 1.56).  LDS bounds it: of a tile's operands the waves take 16 KB each as
// they lie, 16 KB transposed (at half the rate) and 4 KB that they hand on, which
// with the tile's writes are 3584 cycles for 2048 of products; matrix instructions
// run in 55% of the cycles, and without the tiles' loads it is 5% faster.  Tiles
// from the last one down, so that workgroups share them in L2, take a 28th of the
// bytes from memory and as long (D = 64: 10% longer).
template <int D, bool CAUSAL>
struct Paired {
  static constexpr int NW = 8, QT = 64, AHEAD = 5, KS = D / 16, CB = D / 32;
  static constexpr int SCORES = 2 * KS, PRODUCTS = QT / 16 * CB;   // products of a wave for a tile
  typedef wir::STile<QT, D, wir::BOTH> T;
  typedef __attribute__((address_space(3))) wir::bf16x8 lds_bf16x8;
  typedef __attribute__((address_space(3))) wir::bf16x4 lds_bf16x4;
  typedef __attribute__((address_space(3))) wir::i16x4 lds_i16x4;
  typedef __attribute__((address_space(3))) wir::f32x4 lds_f32x4;
  typedef __attribute__((address_space(3))) wir::Odd<D> lds_odd;
  // LDS: three slots of a Q and a dO tile, what the waves hand on (twice), the tiles' statistics, notes of what is odd
  static constexpr int SLOT = 2 * T::BYTES, HANDED = 3 * SLOT, VEC = HANDED + 2 * NW * 2048, ODD = VEC + 3 * 2 * QT * 4,
                       BYTES = ODD + 2 * sizeof(wir::Odd<D>);
  static_assert(D == 128, "the swizzle's addresses below are those of 16 chunks a row");

  struct At {
    int head, t;
  };

  const wir::packed_bwd_args& a;
  const wir::Rows& r;
  char* smem;
  int wave, lane, role, row0, first, tiles;
  wir::HeadTiles<T, NW> Q, G;
  unsigned row_at, tr_at;          // the lane's places in a tile, as operands of the scores and of the product
  wir::RowFrags<32, 1, KS> k, v;
  wir::RTile<32, 32, D> acc;       // dV or dK
  wir::RTile<32, 32, 32> s, dp;
  wir::BTile<32, 32, 32> keep;
  wir::BTile<32, 32, QT> x;

  __device__ __forceinline__ Paired(const wir::packed_bwd_args& args, const wir::Rows& rows, char* lds) : a(args), r(rows), smem(lds) {}

  __device__ __forceinline__ At after(At i) const { return i.t + 1 < tiles ? At{i.head, i.t + 1} : At{i.head + 1, first}; }

  __device__ __forceinline__ void load(At i, int slot) {
    char* at = smem + slot * SLOT;
    Q.base = (const char*)(a.q + i.head * a.qh + r.start * a.qt);
    G.base = (const char*)(a.d_o + i.head * a.gh + r.start * a.gt);
    Q.load(at, i.t, wave);
    G.load(at + T::BYTES, i.t, wave);
    if (wave < 2) {   // a wave each for the two statistics
      const float* from = a.stats + ((i64)(wave * a.heads + i.head) * a.tokens + r.start);
      wir::dma4_v(from + min(i.t * QT + lane, r.len - 1), wir::lds_addr(smem + VEC + (2 * slot + wave) * QT * 4));
    }
  }

  // The scores' sums begin with the statistics: p = exp2(c (q . k - LSE sqrt(D))), dP - D_p = dO . v - D_p.
  __device__ __forceinline__ void begin_scores(int slot) {
    const auto* vec = (lds_f32x4*)wir::lds(smem + VEC + 2 * slot * QT * 4 + role * 128 + lane / 32 * 16);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const wir::f32x4 x0 = vec[2 * g], x1 = vec[QT / 4 + 2 * g];
#pragma unroll
      for (int j = 0; j < 4; ++j) s.f[0][0][4 * g + j] = x0[j], dp.f[0][0][4 * g + j] = x1[j];
    }
  }

  __device__ __forceinline__ void begin_product(int turn) {
    const auto* from = (lds_bf16x4*)wir::lds(smem + HANDED + (turn * NW + (wave ^ 4)) * 2048) + lane;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const wir::bf16x4 other = from[g * 64];
      x.f[0][0][g] = role ? other : keep.f[0][0][g];
      x.f[1][0][g] = role ? keep.f[0][0][g] : other;
    }
  }

  __device__ __forceinline__ wir::bf16x8 score_operand(unsigned at, int i) const {
    return *(lds_bf16x8*)((at ^ (i / 2 * 32)) + i % 2 * T::BYTES);
  }
  __device__ __forceinline__ void score(const wir::bf16x8& b, int i) {
    if (i % 2 == 0) s.f[0][0] = wir::MF<32>::mma(b, k.f[0][i / 2], s.f[0][0]);
    else dp.f[0][0] = wir::MF<32>::mma(b, v.f[0][i / 2], dp.f[0][0]);
  }

  __device__ __forceinline__ wir::bf16x8 product_operand(unsigned at, int i) const {
    const int q = 2 * (i / CB), cb = i % CB, rows = q * 8 * D * 2;   // (two groups of eight rows)
    const auto lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)((at ^ (cb * 64)) + rows));
    const auto hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)((at ^ (cb * 64 + 32)) + rows + 8 * D * 2));
    return wir::cat(__builtin_bit_cast(wir::bf16x4, lo), __builtin_bit_cast(wir::bf16x4, hi));
  }
  __device__ __forceinline__ void product(const wir::bf16x8& b, int i) {
    const int q = 2 * (i / CB), cb = i % CB;
    acc.f[cb][0] = wir::MF<32>::mma(b, wir::cat(x.f[q / 4][0][q % 4], x.f[(q + 1) / 4][0][(q + 1) % 4]), acc.f[cb][0]);
  }

  // P and dS of the wave's half of a tile: one it keeps, one it hands on.
  __device__ __forceinline__ void finish_scores(At i, int turn) {
    constexpr float c = wir::PackedScale<D>::c;
    const int col0 = i.t * QT + role * 32;
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      s.f[0][0][n] = __builtin_amdgcn_exp2f(s.f[0][0][n] * c);
      dp.f[0][0][n] *= s.f[0][0][n];
    }
    // (a query that does not see the row may hold NaN; past the end the last one stands again)
    if ((CAUSAL && col0 < row0 + 31) || col0 + 32 > r.len) {
      const int half = wir::seldom(lane / 32);
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        const int col = col0 + wir::ccol<32>(n, half);
        const bool seen = (!CAUSAL || row0 + lane % 32 <= col) && col < r.len;
        s.f[0][0][n] = seen ? s.f[0][0][n] : 0.f;
        dp.f[0][0][n] = seen ? dp.f[0][0][n] : 0.f;
      }
    }
    wir::BTile<32, 32, 32> pb, ds;
    wir::to_bf16(pb, s);
    wir::to_bf16(ds, dp);
    auto* to = (lds_bf16x4*)wir::lds(smem + HANDED + (turn * NW + wave) * 2048) + lane;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      to[g * 64] = role ? pb.f[0][0][g] : ds.f[0][0][g];
      keep.f[0][0][g] = role ? ds.f[0][0][g] : pb.f[0][0][g];
    }
  }

  // The product of the tile in `slot` (PRODUCT) and the scores of tile i in `slot1` (SCORE), ROLE 1's scores first.
  template <int ROLE, bool PRODUCT, bool SCORE>
  __device__ __forceinline__ void stream(int slot, At i, int slot1, int turn) {
    constexpr int N0 = ROLE ? (SCORE ? SCORES : 0) : (PRODUCT ? PRODUCTS : 0);
    constexpr int N = N0 + (ROLE ? (PRODUCT ? PRODUCTS : 0) : (SCORE ? SCORES : 0));
    const unsigned product_at = tr_at + slot * SLOT, score_at = row_at + slot1 * SLOT;
    wir::bf16x8 ring[AHEAD + 1];
    auto read = [&](auto at) {
      constexpr int n = decltype(at)::value;
      if constexpr ((n >= N0) == (ROLE == 1)) ring[n % (AHEAD + 1)] = product_operand(product_at, n >= N0 ? n - N0 : n);
      else ring[n % (AHEAD + 1)] = score_operand(score_at, n >= N0 ? n - N0 : n);
    };
    if (PRODUCT) begin_product(turn);
    if (SCORE) begin_scores(slot1);
    __builtin_amdgcn_s_setprio(1);
    wir::static_for<0, AHEAD>(read);
    wir::static_for<0, N>([&](auto at) {
      constexpr int n = decltype(at)::value;
      if constexpr (n + AHEAD < N) read(wir::ic<n + AHEAD>{});
      __builtin_amdgcn_sched_barrier(0);
      if constexpr ((n >= N0) == (ROLE == 1)) product(ring[n % (AHEAD + 1)], n >= N0 ? n - N0 : n);
      else score(ring[n % (AHEAD + 1)], n >= N0 ? n - N0 : n);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (SCORE && n == (ROLE ? N0 : N) - 1) {
        __builtin_amdgcn_s_setprio(0);
        finish_scores(i, turn ^ 1);
        __builtin_amdgcn_s_setprio(1);
      }
    });
    __builtin_amdgcn_s_setprio(0);
  }

  // All tiles of a wave (a loop for each role: one with both in it moves the sums between registers).
  template <int ROLE>
  __device__ __forceinline__ void walk(At now, int end, bool careful, lds_odd* odd) {
    At next = after(now);
    load(now, 0);
    wir::wait_vm_barrier<0>();
    if (next.head < end) load(next, 1);
    stream<ROLE, false, true>(0, now, 0, 1);
    int slot = 0, turn = 0;
    auto settle = [&](At third, int slot2) {
      wir::wait_vm_barrier<0>();
      if (third.head < end) load(third, slot2);
      if (careful) {
        wir::clear_odd<true, NW, T>(smem + slot * SLOT, now.t * QT, odd);
        wir::clear_odd<true, NW, T>(smem + slot * SLOT + T::BYTES, now.t * QT, odd + 1);
        wir::barrier();
      }
    };
    while (next.head < end) {
      const At third = after(next);
      const int slot1 = slot == 2 ? 0 : slot + 1;
      settle(third, slot1 == 2 ? 0 : slot1 + 1);
      stream<ROLE, true, true>(slot, next, slot1, turn);
      now = next, next = third, slot = slot1, turn ^= 1;
    }
    settle(next, 0);
    stream<ROLE, true, false>(slot, next, 0, turn);
  }

  __device__ __forceinline__ bool run(int kv, bool careful) {
    wave = wir::wave_id(), lane = wir::lane_id();
    role = wave / 4;   // (waves w and w + 4 are on one SIMD)
    row0 = r.row0 + wave % 4 * 32;
    first = CAUSAL ? r.row0 / QT : 0, tiles = (r.len + QT - 1) / QT;
    Q.init(a.q + r.start * a.qt, a.qt, r.len);
    G.init(a.d_o + r.start * a.gt, a.gt, r.len);
    const int group = lane % 16;   // of the transposed reads
    row_at = wir::lds_addr(smem) + T::chunk_off(role * 32 + lane % 32, lane / 32);
    tr_at = wir::lds_addr(smem) + (role ? 0 : T::BYTES) + T::elem_off(lane / 32 * 4 + group / 4, lane % 32 / 16 * 16 + 4 * (group % 4));
    auto* odd = (lds_odd*)wir::lds(smem + ODD);
    if (careful) wir::no_odd<true, NW>(odd), wir::no_odd<true, NW>(odd + 1);
    wir::packed_rows(k, a.k + kv * a.kh + r.start * a.kt, a.kt, row0, r.len);
    wir::packed_rows(v, a.v + kv * a.vh + r.start * a.vt, a.vt, row0, r.len);
    wir::fill(acc, 0.f);
    const At now{kv * a.group, first};
    if (role == 0) walk<0>(now, now.head + a.group, careful, odd);
    else walk<1>(now, now.head + a.group, careful, odd);
    const int row = row0 + lane % 32;
    if (!careful) {
      if (wir::any_wave(wir::has_nan(acc, row < r.len), smem + ODD)) return true;
    } else {
      wir::wait_vm_barrier<0>();
    }
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
      for (int n = 0; n < 16; ++n) acc.f[cb][0][n] *= role ? wir::PackedScale<D>::s : 1.f;
    if (careful) {
      const int from = CAUSAL ? row : 0;   // as in Dkdv
      const auto* mine = odd + (role ? 0 : 1);
#pragma unroll
      for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          const int d = cb * 32 + wir::ccol<32>(n, lane / 32);
          const float x = acc.f[cb][0][n], y = wir::with_odd<true>(mine, d, from, x);
          acc.f[cb][0][n] = role && y != x ? __builtin_nanf("") : y;
        }
    }
    const auto out = role ? wir::packed_head(a.dk, a.dkh, a.dkt, kv, r.start, r.len, D)
                          : wir::packed_head(a.dv, a.dvh, a.dvt, kv, r.start, r.len, D);
    wir::store_tile_staged<true>(out, acc, 0, 0, row0, 0, smem + wave * 32 * D * 2);
    return false;
  }
};

template <int D, int QT, bool CAUSAL>
__device__ __forceinline__ void dkdv_kernel(const wir::packed_bwd_args& a) {
  __shared__ __attribute__((aligned(1024))) char smem[Dkdv<D, QT, CAUSAL>::BYTES];
  int x, kv;
  wir::packed_program(a, a.heads / a.group, ROWS, x, kv);   // a sequence's longest block is its first
  const wir::Rows r = wir::packed_block(a.offsets, a.batch, a.tokens, x);
  if (r.row0 < 0 || r.row0 >= r.len) return;   // (a number that no block has)
  if (r.rest) {
    if (a.flags & 2) wir::packed_zero_rest(a.dk, a.dkh, a.dkt, r, kv, D, ROWS);
    if (a.flags & 4) wir::packed_zero_rest(a.dv, a.dvh, a.dvt, r, kv, D, ROWS);
    return;
  }
  Dkdv<D, QT, CAUSAL> p(a, r, smem);
  bool careful = false;
  while (p.run(kv, careful)) careful = true;
}

template <int D, bool CAUSAL>
__device__ __forceinline__ void dkdv_kernel8(const wir::packed_bwd_args& a) {
  __shared__ __attribute__((aligned(1024))) char smem[Paired<D, CAUSAL>::BYTES];
  int x, kv;
  wir::packed_program(a, a.heads / a.group, ROWS, x, kv);   // a sequence's longest block is its first
  const wir::Rows r = wir::packed_block(a.offsets, a.batch, a.tokens, x);
  if (r.row0 < 0 || r.row0 >= r.len) return;   // (a number that no block has)
  if (r.rest) {
    if (a.flags & 2) wir::packed_zero_rest(a.dk, a.dkh, a.dkt, r, kv, D, ROWS);
    if (a.flags & 4) wir::packed_zero_rest(a.dv, a.dvh, a.dvt, r, kv, D, ROWS);
    return;
  }
  Paired<D, CAUSAL> p(a, r, smem);
  bool careful = false;
  while (p.run(kv, careful)) careful = true;
}

}  // namespace

#define PACKED_KERNEL8(NAME, CALL)                                                                             \
  extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(512, 512), amdgpu_waves_per_eu(2, 2))) \
  NAME(const wir::packed_bwd_args args) { CALL(args); }

#define PACKED_KERNEL(NAME, CALL, WAVES_A_SIMD)                                                         \
  extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(256, 256),                      \
                                            amdgpu_waves_per_eu(WAVES_A_SIMD, WAVES_A_SIMD)))           \
  NAME(const wir::packed_bwd_args args) { CALL(args); }

PACKED_KERNEL(wir_attn_packed_dq_d64, (dq_kernel<64, false>), 3)
PACKED_KERNEL(wir_attn_packed_dq_d64_causal, (dq_kernel<64, true>), 3)
PACKED_KERNEL(wir_attn_packed_dq_d128, (dq_kernel<128, false>), 2)
PACKED_KERNEL(wir_attn_packed_dq_d128_causal, (dq_kernel<128, true>), 2)
PACKED_KERNEL(wir_attn_packed_dkdv_d64, (dkdv_kernel<64, 64, false>), 2)
PACKED_KERNEL(wir_attn_packed_dkdv_d64_causal, (dkdv_kernel<64, 64, true>), 2)
PACKED_KERNEL8(wir_attn_packed_dkdv_d128, (dkdv_kernel8<128, false>))
PACKED_KERNEL8(wir_attn_packed_dkdv_d128_causal, (dkdv_kernel8<128, true>))
