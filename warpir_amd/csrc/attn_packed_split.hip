// attn_packed_split.hip -- attention over packed sequences and its gradients
// for launches too small to fill the chip: the counterparts of attn_packed.hip
// and attn_packed_bwd.hip, with their formulas and argument structures.
//
// Such a launch is bound by the walk of its longest block.  A workgroup takes 32
// query rows (or keys) and its waves every W-th tile of the other side (the
// gradients of keys: of the group's heads one after another), each through LDS
// of its own, without a barrier; the waves' results are joined in LDS, in the
// waves' order, in fp32.  Operands are rounded as there.
//
// Measured, this / 128 rows a workgroup: forward of 5 sequences of up to 150
// tokens, 16/4 heads of 128, causal 11.1 / 8.8 us, of 1 x 512, 8 heads of 64 7.4 /
// 11.2; dQ of 1 x 512, 8 heads of 128 13.0 / 19.0; dK/dV of 1 x 512, 16/4 heads of
// 64 18.2 / 44.9.  The rule is in packed.py.
#include "wir_packed_args.h"

namespace {

using wir::bf16;
using wir::bf16x8;
using wir::f32x4;
using wir::i64;

typedef __attribute__((address_space(3))) float lds_float;
typedef __attribute__((address_space(3))) f32x4 lds_f32x4;

constexpr int ROWS = 32;

// Floats from a row of a wave's partial result in LDS to the next: 16 rows land in 16 different 16-byte slots.
template <int D>
constexpr int PITCH = D + 4;

template <int D>
__device__ __forceinline__ void put_partial(lds_float* part, const wir::RTile<32, 32, D>& t) {
  const int lane = wir::lane_id(), lr = lane % 32, lh = lane / 32;
#pragma unroll
  for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = t.f[cb][0][4 * g + j];
      *(lds_f32x4*)(part + lr * PITCH<D> + cb * 32 + wir::ccol<32>(4 * g, lh)) = v;
    }
}

// The sum over W waves of weight(row, wave) times their partial results, a thread's chunks of 8 columns.
template <int D, int W>
struct Joined {
  static constexpr int CHUNKS = ROWS * (D / 8), EACH = (CHUNKS + 64 * W - 1) / (64 * W);
  float x[EACH][8];

  template <class Weight>
  __device__ __forceinline__ void read(const lds_float* part, Weight weight) {
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int i = min(e * 64 * W + (int)threadIdx.x, CHUNKS - 1), row = i / (D / 8), ch = i % (D / 8);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[e][j] = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const lds_float* p = part + (w * ROWS + row) * PITCH<D> + ch * 8;
        const f32x4 lo = *(const lds_f32x4*)p, hi = *(const lds_f32x4*)(p + 4);
        const float f = weight(row, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[e][j] += lo[j] * f, x[e][4 + j] += hi[j] * f;
      }
    }
  }

  // Whether the workgroup's first `rows` rows hold a NaN (the first time, clear_odd may give another).
  __device__ __forceinline__ bool nan(int rows) const {
    bool any = false;
#pragma unroll
    for (int e = 0; e < EACH; ++e)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        any |= x[e][j] != x[e][j] && min(e * 64 * W + (int)threadIdx.x, CHUNKS - 1) / (D / 8) < rows;
    return __builtin_amdgcn_ballot_w64(any) != 0;
  }

  // finish(row, column, value), rounded to bf16, to the first `rows` rows.
  template <class Finish>
  __device__ __forceinline__ void store(bf16* to, i64 row_stride, int rows, Finish finish) const {
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int i = e * 64 * W + threadIdx.x, row = i / (D / 8), ch = i % (D / 8);
      if (i >= CHUNKS || row >= rows) continue;
      bf16x8 v;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (bf16)finish(row, ch * 8 + j, x[e][j]);
      *(bf16x8*)(to + row * row_stride + ch * 8) = v;
    }
  }
};

// Waits for a wave's oldest tile, of EACH loads; `more`: another one is behind it.
template <int EACH>
__device__ __forceinline__ void wait_tile(bool more) {
  if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(EACH) : "memory");
  else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

template <int D, int KT, bool CAUSAL, int W>
struct ForwardSplit {
  typedef wir::STile<KT, D, wir::ROWREAD> TK;
  typedef wir::STile<KT, D, wir::TRREAD> TV;
  typedef __attribute__((address_space(3))) wir::Odd<D> lds_odd;
  static constexpr int SLOT = TK::BYTES + TV::BYTES, EACH = wir::HeadTiles<TK, 1>::LOADS + wir::HeadTiles<TV, 1>::LOADS;
  static constexpr int RING = W * 2 * SLOT, PART = W * ROWS * PITCH<D> * 4;
  static constexpr int STAT = RING > PART ? RING : PART, ODD = STAT + W * ROWS * 8, BYTES = ODD + sizeof(wir::Odd<D>);

  static __device__ __forceinline__ bool run(const wir::packed_fwd_args& a, const wir::Rows& r, int head, char* smem,
                                             bool careful) {
    constexpr float c = wir::PackedScale<D>::c;
    const int wave = wir::wave_id(), lane = wir::lane_id(), row0 = r.row0, kv = head / a.group;
    const int keys = CAUSAL ? min(r.len, row0 + ROWS) : r.len, tiles = (keys + KT - 1) / KT;
    wir::HeadTiles<TK, 1> K;
    wir::HeadTiles<TV, 1> V;
    K.init(a.k + kv * a.kh + r.start * a.kt, a.kt, r.len);
    V.init(a.v + kv * a.vh + r.start * a.vt, a.vt, r.len);
    char* own = smem + wave * 2 * SLOT;
    auto* odd = (lds_odd*)wir::lds(smem + ODD);
    if (careful) {
      wir::no_odd<false, W>(odd);
      wir::barrier();
    }
    auto load = [&](int t, int slot) {
      K.load(own + slot * SLOT, t, 0);
      V.load(own + slot * SLOT + TK::BYTES, t, 0);
    };
    if (wave < tiles) load(wave, 0);
    wir::RowFrags<32, 1, D / 16> q;
    wir::packed_rows(q, a.q + head * a.qh + r.start * a.qt, a.qt, row0, r.len);
    wir::RTile<32, 32, D> o;
    wir::fill(o, 0.f);
    float m = -__builtin_inff(), l = 0.f;
    int slot = 0;
    for (int t = wave; t < tiles; t += W, slot ^= 1) {
      char *kt = own + slot * SLOT, *vt = kt + TK::BYTES;
      const int col0 = t * KT;
      const bool more = t + W < tiles;
      if (more) load(t + W, slot ^ 1);
      wait_tile<EACH>(more);
      wir::RTile<32, 32, KT> s;
      wir::mma_ABt_frags<32, 32, KT, TK, D / 16>(s, q, kt, 0);
      if (CAUSAL ? col0 + KT - 1 > row0 : col0 + KT > r.len) wir::packed_mask<CAUSAL>(s, row0, col0, r.len);
      float top = s.f[0][0][0];
#pragma unroll
      for (int cb = 0; cb < KT / 32; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s.f[cb][0][i]);
      top = fmaxf(wir::lane_group_reduce<32>(top, wir::OpMax()) * c, m);
      const float base = top == -__builtin_inff() ? 0.f : top;   // (a row that sees nothing of the wave's tiles so far)
      wir::RVec<32, 32> corr;
      corr.v[0] = __builtin_amdgcn_exp2f(m - base);
      m = top;
      float sum = 0.f;
      wir::BTile<32, 32, KT> p;
#pragma unroll
      for (int cb = 0; cb < KT / 32; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s.f[cb][0][i], c, -base));
          sum += x;
          p.f[cb][0][i / 4][i % 4] = (bf16)x;   // (the product's operand; the sum has the value itself)
        }
      l = l * corr.v[0] + sum;
      wir::row_scale(o, o, corr);
      if (careful) wir::clear_odd<false, 1, TV>(vt, col0, odd);
      wir::mma_rAB<32, 32, KT, D, TV>(o, p, vt, 0);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (the slot is read: it may be loaded again)
    }
    l = wir::lane_group_reduce<32>(l, wir::OpAdd());
    wir::wait_vm_barrier<0>();
    lds_float* part = (lds_float*)wir::lds(smem);
    auto* stat = (__attribute__((address_space(3))) float*)wir::lds(smem + STAT);   // [wave][row][2]
    put_partial<D>(part + wave * ROWS * PITCH<D>, o);
    if (lane < 32) stat[(wave * ROWS + lane) * 2] = m, stat[(wave * ROWS + lane) * 2 + 1] = l;
    wir::barrier();
    const int rows = min(ROWS, r.len - row0);
    // each wave's maximum and sum become its weight, 2^(m - M) / sum
    if (wave == 0) {
      const int row = lane % 32;
      float most = stat[row * 2];
#pragma unroll
      for (int w = 1; w < W; ++w) most = fmaxf(most, stat[(w * ROWS + row) * 2]);
      float total = 0.f, f[W];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        f[w] = stat[(w * ROWS + row) * 2] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(stat[(w * ROWS + row) * 2] - most);
        const float lw = stat[(w * ROWS + row) * 2 + 1];
        total += lw != lw ? lw : lw * f[w];
      }
      if (lane < 32) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float lw = stat[(w * ROWS + row) * 2 + 1];
          stat[(w * ROWS + row) * 2] = lw != lw ? lw : f[w] / total;
        }
        if (row < rows)
          a.lse[head * a.lh + (r.start + row0 + row) * a.lt] = (most + __builtin_amdgcn_logf(total)) * 0.6931471805599453f;
      }
    }
    wir::barrier();
    auto weight = [&](int row, int w) { return stat[(w * ROWS + row) * 2]; };
    Joined<D, W> all;
    all.read(part, weight);
    if (!careful && wir::any_wave(all.nan(rows), smem + ODD)) return true;
    all.store(a.out + head * a.oh + (r.start + row0) * a.ot, a.ot, rows, [&](int row, int d, float x) {
      if (!careful) return x;
      const int last = CAUSAL ? row0 + row : r.len - 1;   // the last position that the row sees
      return wir::with_odd<false, D>(odd, d, last, x);
    });
    return false;
  }
};

template <int D, int KT, bool CAUSAL, int W>
struct DqSplit {
  typedef wir::STile<KT, D, wir::BOTH> TK;
  typedef wir::STile<KT, D, wir::ROWREAD> TV;
  typedef __attribute__((address_space(3))) wir::Odd<D> lds_odd;
  static constexpr int SLOT = TK::BYTES + TV::BYTES, EACH = wir::HeadTiles<TK, 1>::LOADS + wir::HeadTiles<TV, 1>::LOADS;
  static constexpr int RING = W * 2 * SLOT, PART = W * ROWS * PITCH<D> * 4;
  static constexpr int ODD = RING > PART ? RING : PART, BYTES = ODD + sizeof(wir::Odd<D>);

  static __device__ __forceinline__ bool run(const wir::packed_bwd_args& a, const wir::Rows& r, int head, char* smem,
                                             bool careful) {
    constexpr float c = wir::PackedScale<D>::c;
    const int wave = wir::wave_id(), lane = wir::lane_id(), row0 = r.row0, kv = head / a.group;
    const int keys = CAUSAL ? min(r.len, row0 + ROWS) : r.len, tiles = (keys + KT - 1) / KT;
    wir::HeadTiles<TK, 1> K;
    wir::HeadTiles<TV, 1> V;
    K.init(a.k + kv * a.kh + r.start * a.kt, a.kt, r.len);
    V.init(a.v + kv * a.vh + r.start * a.vt, a.vt, r.len);
    char* own = smem + wave * 2 * SLOT;
    auto* odd = (lds_odd*)wir::lds(smem + ODD);
    if (careful) {
      wir::no_odd<false, W>(odd);
      wir::barrier();
    }
    auto load = [&](int t, int slot) {
      K.load(own + slot * SLOT, t, 0);
      V.load(own + slot * SLOT + TK::BYTES, t, 0);
    };
    if (wave < tiles) load(wave, 0);
    wir::RowFrags<32, 1, D / 16> q, d_o, o;
    wir::packed_rows(q, a.q + head * a.qh + r.start * a.qt, a.qt, row0, r.len);
    wir::packed_rows(d_o, a.d_o + head * a.gh + r.start * a.gt, a.gt, row0, r.len);
    wir::packed_rows(o, a.o + head * a.oh + r.start * a.ot, a.ot, row0, r.len);
    const int row = row0 + lane % 32;
    float lse = a.lse[head * a.lh + (r.start + min(row, r.len - 1)) * a.lt];
    wir::RVec<32, 32> dots;
    wir::row_dot(dots, d_o, o);
    if (wave == 0 && lane < 32 && row < r.len) {
      float* to = a.stats + (i64)head * a.tokens + r.start + row;
      to[0] = -lse * wir::PackedScale<D>::root;
      to[(i64)a.heads * a.tokens] = -dots.v[0];
    }
    lse *= 1.4426950408889634f;
    wir::RTile<32, 32, D> acc;
    wir::fill(acc, 0.f);
    int slot = 0;
    for (int t = wave; t < tiles; t += W, slot ^= 1) {
      char *kt = own + slot * SLOT, *vt = kt + TK::BYTES;
      const int col0 = t * KT;
      const bool more = t + W < tiles;
      if (more) load(t + W, slot ^ 1);
      wait_tile<EACH>(more);
      wir::RTile<32, 32, KT> s, dp;
      wir::BTile<32, 32, KT> ds;
      wir::mma_ABt_frags<32, 32, KT, TK, D / 16>(s, q, kt, 0);
      wir::mma_ABt_frags<32, 32, KT, TV, D / 16>(dp, d_o, vt, 0);
#pragma unroll
      for (int cb = 0; cb < KT / 32; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          dp.f[cb][0][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s.f[cb][0][i], c, -lse)) * (dp.f[cb][0][i] - dots.v[0]);
      if (CAUSAL ? col0 + KT - 1 > row0 : col0 + KT > r.len) {   // (a value that a row does not see may be NaN)
        const int half = wir::seldom(lane / 32);
#pragma unroll
        for (int cb = 0; cb < KT / 32; ++cb)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int col = col0 + cb * 32 + wir::ccol<32>(i, half);
            dp.f[cb][0][i] = (CAUSAL ? col <= row : col < r.len) ? dp.f[cb][0][i] : 0.f;
          }
      }
      wir::to_bf16(ds, dp);
      if (careful) wir::clear_odd<false, 1, TK>(kt, col0, odd);
      wir::mma_rAB<32, 32, KT, D, TK>(acc, ds, kt, 0);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (the slot is read: it may be loaded again)
    }
    wir::wait_vm_barrier<0>();
    lds_float* part = (lds_float*)wir::lds(smem);
    put_partial<D>(part + wave * ROWS * PITCH<D>, acc);
    wir::barrier();
    const int rows = min(ROWS, r.len - row0);
    auto weight = [](int, int) { return wir::PackedScale<D>::s; };
    Joined<D, W> all;
    all.read(part, weight);
    if (!careful && wir::any_wave(all.nan(rows), smem + ODD)) return true;
    all.store(a.dq + head * a.dqh + (r.start + row0) * a.dqt, a.dqt, rows, [&](int at, int d, float x) {
      if (!careful) return x;
      const int first = min(odd->at[0][d], min(odd->at[1][d], odd->at[2][d]));
      return (CAUSAL ? row0 + at : r.len - 1) >= first ? __builtin_nanf("") : x;
    });
    return false;
  }
};

template <int D, bool CAUSAL, int W>
struct DkdvSplit {
  static constexpr int QT = 32;
  typedef wir::STile<QT, D, wir::BOTH> T;
  typedef __attribute__((address_space(3))) wir::Odd<D> lds_odd;
  static constexpr int SLOT = 2 * T::BYTES + 256, EACH = 2 * wir::HeadTiles<T, 1>::LOADS + 1;   // Q, dO, two statistics a query
  static constexpr int RING = W * 2 * SLOT, PART = W * ROWS * PITCH<D> * 4;
  static constexpr int ODD = RING > 2 * PART ? RING : 2 * PART, BYTES = ODD + 2 * sizeof(wir::Odd<D>);

  static __device__ __forceinline__ bool run(const wir::packed_bwd_args& a, const wir::Rows& r, int kv, char* smem,
                                             bool careful) {
    constexpr float c = wir::PackedScale<D>::c;
    const int wave = wir::wave_id(), lane = wir::lane_id(), row0 = r.row0;
    const int first = CAUSAL ? row0 / QT : 0, each = (r.len + QT - 1) / QT - first, items = each * a.group;
    wir::HeadTiles<T, 1> Q, G;
    Q.init(a.q, a.qt, r.len);
    G.init(a.d_o, a.gt, r.len);
    char* own = smem + wave * 2 * SLOT;
    auto* odd = (lds_odd*)wir::lds(smem + ODD);
    if (careful) {
      wir::no_odd<true, W>(odd), wir::no_odd<true, W>(odd + 1);
      wir::barrier();
    }
    auto load = [&](int i, int slot) {
      const int head = kv * a.group + i / each, t = first + i % each;
      char* at = own + slot * SLOT;
      Q.base = (const char*)(a.q + head * a.qh + r.start * a.qt);
      G.base = (const char*)(a.d_o + head * a.gh + r.start * a.gt);
      Q.load(at, t, 0);
      G.load(at + T::BYTES, t, 0);
      // half of the lanes each for the two statistics
      const float* from = a.stats + ((i64)(lane / 32 * a.heads + head) * a.tokens + r.start);
      wir::dma4_v(from + min(t * QT + lane % 32, r.len - 1), wir::lds_addr(at + 2 * T::BYTES));
    };
    if (wave < items) load(wave, 0);
    wir::RowFrags<32, 1, D / 16> k, v;
    wir::packed_rows(k, a.k + kv * a.kh + r.start * a.kt, a.kt, row0, r.len);
    wir::packed_rows(v, a.v + kv * a.vh + r.start * a.vt, a.vt, row0, r.len);
    wir::RTile<32, 32, D> dk, dv;
    wir::fill(dk, 0.f);
    wir::fill(dv, 0.f);
    int slot = 0;
    for (int i = wave; i < items; i += W, slot ^= 1) {
      char *qt = own + slot * SLOT, *dot = qt + T::BYTES;
      const int col0 = (first + i % each) * QT;
      const bool more = i + W < items;
      if (more) load(i + W, slot ^ 1);
      wait_tile<EACH>(more);
      wir::RTile<32, 32, QT> s, dp;
      wir::BTile<32, 32, QT> pb, ds;
      wir::CVec<32, QT> lse, dots;
      wir::load_cvec_lds(lse, qt + 2 * T::BYTES, 0);
      wir::load_cvec_lds(dots, qt + 2 * T::BYTES, QT);
      wir::mma_ABt_frags<32, 32, QT, T, D / 16>(s, k, qt, 0);
      wir::mma_ABt_frags<32, 32, QT, T, D / 16>(dp, v, dot, 0);
      const bool edge = (CAUSAL && col0 < row0 + 31) || col0 + QT > r.len;
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        float p = __builtin_amdgcn_exp2f((s.f[0][0][n] + lse.v[0][n]) * c);
        float x = p * (dp.f[0][0][n] + dots.v[0][n]);
        if (edge) {   // (a query that does not see the row may hold NaN; past the end the last one stands again)
          const int col = col0 + wir::ccol<32>(n, lane / 32);
          const bool seen = (!CAUSAL || row0 + lane % 32 <= col) && col < r.len;
          p = seen ? p : 0.f, x = seen ? x : 0.f;
        }
        pb.f[0][0][n / 4][n % 4] = (bf16)p;
        ds.f[0][0][n / 4][n % 4] = (bf16)x;
      }
      if (careful) {
        wir::clear_odd<true, 1, T>(qt, col0, odd);
        wir::clear_odd<true, 1, T>(dot, col0, odd + 1);
      }
      wir::mma_rAB<32, 32, QT, D, T>(dv, pb, dot, 0);
      wir::mma_rAB<32, 32, QT, D, T>(dk, ds, qt, 0);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (the slot is read: it may be loaded again)
    }
    wir::wait_vm_barrier<0>();
    lds_float* part = (lds_float*)wir::lds(smem);
    put_partial<D>(part + wave * ROWS * PITCH<D>, dk);
    put_partial<D>(part + PART / 4 + wave * ROWS * PITCH<D>, dv);
    wir::barrier();
    const int rows = min(ROWS, r.len - row0);
    auto scaled = [](int, int) { return wir::PackedScale<D>::s; };
    auto plain = [](int, int) { return 1.f; };
    Joined<D, W> keys, values;
    keys.read(part, scaled);
    values.read(part + PART / 4, plain);
    if (!careful) {
      const bool nan = keys.nan(rows) || values.nan(rows);
      if (wir::any_wave(nan, smem + ODD)) return true;
    }
    // (the scores of an infinite query are no numbers, and dS with them; an infinite dO makes a sum of dV infinite)
    keys.store(a.dk + kv * a.dkh + (r.start + row0) * a.dkt, a.dkt, rows, [=](int at, int d, float x) {
      if (!careful) return x;
      const int until = max(odd->at[0][d], max(odd->at[1][d], odd->at[2][d]));
      return (CAUSAL ? row0 + at : 0) <= until ? __builtin_nanf("") : x;
    });
    values.store(a.dv + kv * a.dvh + (r.start + row0) * a.dvt, a.dvt, rows, [=](int at, int d, float x) {
      return careful ? wir::with_odd<true, D>(odd + 1, d, CAUSAL ? row0 + at : 0, x) : x;
    });
    return false;
  }
};

template <class Split, int W, bool LONGEST_LAST, class Args, class Rest>
__device__ __forceinline__ void program(const Args& a, int heads, Rest rest) {
  __shared__ __attribute__((aligned(1024))) char smem[Split::BYTES];
  int x, head;
  wir::packed_program(a, heads, ROWS, x, head);
  if (LONGEST_LAST) x = a.blocks - 1 - x;   // a sequence's longest block first
  const wir::Rows r = wir::packed_block(a.offsets, a.batch, a.tokens, x, ROWS);
  if (r.row0 < 0 || r.row0 >= r.len) return;   // (a number that no block has)
  if (r.rest) return rest(r, head);
  bool careful = false;
  while (Split::run(a, r, head, smem, careful)) {
    careful = true;
    wir::barrier();
  }
}

}  // namespace

#define SPLIT_KERNELS(D, SUFFIX, CAUSAL, KT, FW, DW)                                                              \
  extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(64 * FW, 64 * FW), amdgpu_waves_per_eu(FW / 4, FW / 4))) \
  wir_attn_packed_d##D##_split##SUFFIX(const wir::packed_fwd_args args) {                                         \
    program<ForwardSplit<D, KT, CAUSAL, FW>, FW, CAUSAL>(                                                         \
        args, args.heads, [&](const wir::Rows& r, int head) { wir::packed_fill_rest(args, r, head, D, ROWS); });  \
  }                                                                                                               \
  extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(64 * FW, 64 * FW), amdgpu_waves_per_eu(FW / 4, FW / 4))) \
  wir_attn_packed_dq_d##D##_split##SUFFIX(const wir::packed_bwd_args args) {                                      \
    program<DqSplit<D, KT, CAUSAL, FW>, FW, CAUSAL>(args, args.heads, [&](const wir::Rows& r, int head) {         \
      if (args.flags & 1) wir::packed_zero_rest(args.dq, args.dqh, args.dqt, r, head, D, ROWS);                   \
    });                                                                                                           \
  }                                                                                                               \
  extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(64 * DW, 64 * DW), amdgpu_waves_per_eu(DW / 4, DW / 4))) \
  wir_attn_packed_dkdv_d##D##_split##SUFFIX(const wir::packed_bwd_args args) {                                    \
    program<DkdvSplit<D, CAUSAL, DW>, DW, false>(args, args.heads / args.group, [&](const wir::Rows& r, int kv) { \
      if (args.flags & 2) wir::packed_zero_rest(args.dk, args.dkh, args.dkt, r, kv, D, ROWS);                     \
      if (args.flags & 4) wir::packed_zero_rest(args.dv, args.dvh, args.dvt, r, kv, D, ROWS);                     \
    });                                                                                                           \
  }

SPLIT_KERNELS(64, , false, 64, 4, 8)
SPLIT_KERNELS(64, _causal, true, 64, 4, 8)
SPLIT_KERNELS(128, , false, 32, 4, 4)
SPLIT_KERNELS(128, _causal, true, 32, 4, 4)
