// attn_packed.hip -- attention over packed sequences of different lengths
// (warpir_amd.api.attention_packed).
//
// For query row p of a sequence, in 32 bits but for the operands of the two
// products (bf16):
//   s_j = q_p . k_j / sqrt(D) for j <= p (causal) or every j of the sequence,
//   O_p = sum_j softmax(s)_j v_j,  LSE_p = ln sum_j exp s_j.
#include "wir_packed_args.h"

namespace {

using wir::bf16;
using wir::i64;

// A workgroup: a group of four waves, 32 query rows a wave, that share tiles of
// 64 keys; in the time of one tile t a wave takes the products of P(t - 1) with
// V(t - 1) and of Q with K(t), and the softmax of t.
//
// NW = 8: two such groups with the same tiles, of two heads that share a
// key/value head where there are two (flags & 4), or else of 128 rows each one
// behind the other.  Waves w and w + 4 are on one SIMD and work in opposite
// phases, the second group's softmax is that of t - 1 before its products, so
// that one's matrix instructions run under the other's exponentials.
//
// The running maximum m of a row is kept until a tile's sum shows a score more
// than 16 above it (in log2 units): sums and results are fp32, and 2^(s - m) has
// the same relative error wherever it lies.  A probability is rounded to bf16 as
// the second product's operand; the row's sum has it unrounded.
//
// Measured: 8 x 4096 tokens, 32/8 heads of 128: 1.80 ms (1220 TFLOP/s), causal
// 1.00 ms (1100; with four waves 1.84 and 1.02); 16 heads of 64: 0.57 ms (970), 64
// x 512 tokens 97 us (700).  At D = 128 LDS bounds it: an operand of 1 KB serves
// the 32 rows of one wave, a product of 32 cycles, and takes LDS 8 cycles as it
// lies and 16 transposed, so that four SIMDs' products of both kinds, 64 cycles,
// ask for 96 of its cycles: matrix instructions run in 65% of them, causal.  Of 950
// us (16 heads of 128, 8 x 4096) the exponentials are 63, the tiles' loads 105, both 177.  At D = 64 the
// exponentials weigh twice as much (matrix instructions 38% of the cycles in 48
// sequences of up to 1024 tokens), and short sequences pay 5 us a round of
// workgroups for the first tile's way from memory and the last store.  Not faster:
// 64 rows a wave at D = 64 (0.53 ms, but 64 x 512 tokens causal 74 -> 90 us), a
// wave's exponentials between its own products (0.59 ms), three and four slots for
// tiles, the next tiles' loads between products (1.80 -> 1.92 ms).
template <int D, bool CAUSAL, int NW>
struct Forward {
  static constexpr int TILE = 64, AHEAD = 5, KS = D / 16, CB = D / 32;
  static constexpr int SCORES = 2 * KS, PRODUCTS = TILE / 16 * CB;   // products of a wave for a tile
  typedef wir::STile<TILE, D, wir::ROWREAD> TK;
  typedef wir::STile<TILE, D, wir::TRREAD> TV;
  typedef __attribute__((address_space(3))) wir::bf16x8 lds_bf16x8;
  typedef __attribute__((address_space(3))) wir::i16x4 lds_i16x4;
  typedef __attribute__((address_space(3))) wir::Odd<D> lds_odd;
  static constexpr int ODD = 4 * TK::BYTES, BYTES = ODD + sizeof(wir::Odd<D>);   // LDS: two tiles of K, two of V, notes
  // A row's probabilities are 2^(c s - m), m within 2^16 of its largest score so far: a sum past that asks for a new m.
  static constexpr float LIMIT = 65536.f;

  const wir::packed_fwd_args& a;
  const wir::Rows& r;
  char* smem;
  int wave, lane, head, row0, tiles, mine;
  wir::HeadTiles<TK, NW> K;
  wir::HeadTiles<TV, NW> V;
  unsigned row_at, tr_at;          // the lane's places in a tile, as operands of the scores and of the product
  wir::RowFrags<32, 1, KS> q;
  wir::RTile<32, 32, D> o;
  wir::RTile<32, 32, TILE> s;
  wir::BTile<32, 32, TILE> p;
  float m, l;                      // l: of the lane's half of the columns

  __device__ __forceinline__ Forward(const wir::packed_fwd_args& args, const wir::Rows& rows, char* lds) : a(args), r(rows), smem(lds) {}

  __device__ __forceinline__ wir::bf16x8 score_operand(unsigned at, int i) const {
    return *(lds_bf16x8*)((at ^ (i / 2 * 32)) + i % 2 * 32 * D * 2);
  }
  __device__ __forceinline__ void score(const wir::bf16x8& b, int i) {
    s.f[i % 2][0] = wir::MF<32>::mma(b, q.f[0][i / 2], i < 2 ? wir::f32x16{} : s.f[i % 2][0]);
  }
  __device__ __forceinline__ wir::bf16x8 product_operand(unsigned at, int i) const {
    const int rows = i / CB * 16 * D * 2, cb = i % CB;   // (two groups of eight rows)
    const auto lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)((at ^ (cb * 64)) + rows));
    const auto hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)((at ^ (cb * 64)) + rows + 8 * D * 2));
    return wir::cat(__builtin_bit_cast(wir::bf16x4, lo), __builtin_bit_cast(wir::bf16x4, hi));
  }
  __device__ __forceinline__ void product(const wir::bf16x8& b, int i) {
    const int g = 2 * (i / CB), cb = i % CB;
    o.f[cb][0] = wir::MF<32>::mma(b, wir::cat(p.f[g / 4][0][g % 4], p.f[g / 4][0][g % 4 + 1]), o.f[cb][0]);
  }

  // The product of tile t - 1 (PRODUCT) and the scores of tile t (SCORE): one stream of LDS reads, AHEAD products before
  // their use.
  template <bool PRODUCT, bool SCORE>
  __device__ __forceinline__ void stream(int t) {
    constexpr int N0 = PRODUCT ? PRODUCTS : 0, N = N0 + (SCORE ? SCORES : 0);
    const unsigned product_at = tr_at + (t + 1) % 2 * TV::BYTES, score_at = row_at + t % 2 * TK::BYTES;
    wir::bf16x8 ring[AHEAD + 1];
    auto read = [&](auto at) {
      constexpr int n = decltype(at)::value;
      if constexpr (n < N0) ring[n % (AHEAD + 1)] = product_operand(product_at, n);
      else ring[n % (AHEAD + 1)] = score_operand(score_at, n - N0);
    };
    __builtin_amdgcn_s_setprio(1);
    wir::static_for<0, AHEAD>(read);
    wir::static_for<0, N>([&](auto at) {
      constexpr int n = decltype(at)::value;
      if constexpr (n + AHEAD < N) read(wir::ic<n + AHEAD>{});
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (n < N0) product(ring[n % (AHEAD + 1)], n);
      else score(ring[n % (AHEAD + 1)], n - N0);
      __builtin_amdgcn_sched_barrier(0);
    });
    __builtin_amdgcn_s_setprio(0);
  }

  // p and the lane's sum of it, with m as it is.
  __device__ __forceinline__ float exponentials() {
    constexpr float c = wir::PackedScale<D>::c;
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int cb = 0; cb < 2; ++cb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s.f[cb][0][i], c, -m));
        sum[i % 2] += x;
        p.f[cb][0][i / 4][i % 4] = (bf16)x;   // (the product's operand; the sum has the value itself)
      }
    return sum[0] + sum[1];
  }

  __device__ __forceinline__ void softmax(int t) {
    constexpr float c = wir::PackedScale<D>::c;
    const int col0 = t * TILE;
    if (CAUSAL ? col0 + TILE - 1 > row0 : col0 + TILE > r.len) wir::packed_mask<CAUSAL>(s, row0, col0, r.len);
    float sum = exponentials();   // (infinite where the first scores are met that are not -inf)
    if (__builtin_amdgcn_ballot_w64(!(sum <= LIMIT)) != 0) {
      wir::seldom();
      float top = s.f[0][0][0];
#pragma unroll
      for (int cb = 0; cb < 2; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s.f[cb][0][i]);
      // (a row's results do not depend on what the wave's other rows ask for)
      const float asked = wir::lane_group_reduce<32>(sum <= LIMIT ? 0.f : 1.f, wir::OpMax());
      top = fmaxf(wir::lane_group_reduce<32>(top, wir::OpMax()) * c, m);
      top = asked != 0.f ? top : m;
      const float corr = __builtin_amdgcn_exp2f(m - top);
      m = top;
      l *= corr;
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) o.f[cb][0] *= corr;
      sum = exponentials();
    }
    l += sum;
  }

  // All tiles of a wave, its own `mine` and those that only others need.
  template <int ROLE>
  __device__ __forceinline__ void walk(bool careful, lds_odd* odd) {
    auto settle = [&](int t) {   // tile t of K and t - 1 of V have come; the next ones are asked for
      wir::wait_vm_barrier<0>();
      if (t + 1 < tiles) K.load(smem + (t + 1) % 2 * TK::BYTES, t + 1, wave);
      if (t < tiles) V.load(smem + (2 + t % 2) * TK::BYTES, t, wave);
      if (careful && t > 0) {
        wir::clear_odd<false, NW, TV>(smem + (2 + (t - 1) % 2) * TK::BYTES, (t - 1) * TILE, odd);
        wir::barrier();
      }
    };
    int t = 0;
    if (mine > 0) {
      settle(0);
      stream<false, true>(0);
      if (ROLE == 0) softmax(0);
      for (t = 1; t < mine; ++t) {
        settle(t);
        if (ROLE == 1) softmax(t - 1);
        stream<true, true>(t);
        if (ROLE == 0) softmax(t);
      }
      settle(t);
      if (ROLE == 1) softmax(t - 1);
      stream<true, false>(t);
      ++t;
    }
    for (; t <= tiles; ++t) settle(t);
  }

  // Returns whether a result is NaN the first time (only then may `careful` give another).
  __device__ __forceinline__ bool run(int head0, bool careful) {
    wave = wir::wave_id(), lane = wir::lane_id();
    const int second = wave / 4, two = NW == 4 || a.flags & 4;   // (the group; NW = 4: there is one)
    head = head0 + (two ? second : 0);
    row0 = r.row0 + wave % 4 * 32 + (two ? 0 : second * 128);
    const int kv = head0 / a.group, end = CAUSAL ? min(r.len, r.row0 + (two ? 128 : 256)) : r.len;
    tiles = (end + TILE - 1) / TILE;
    // (in the careful pass all waves clear all tiles, and so none stays behind)
    mine = row0 >= r.len ? 0 : CAUSAL ? min(tiles, (row0 + 31) / TILE + 1) : tiles;
    K.init(a.k + kv * a.kh + r.start * a.kt, a.kt, r.len);
    V.init(a.v + kv * a.vh + r.start * a.vt, a.vt, r.len);
    const int part = lane % 16;   // of the transposed reads
    row_at = wir::lds_addr(smem) + TK::chunk_off(lane % 32, lane / 32);
    tr_at = wir::lds_addr(smem) + 2 * TK::BYTES + TV::elem_off(lane / 32 * 4 + part / 4, lane % 32 / 16 * 16 + 4 * (part % 4));
    auto* odd = (lds_odd*)wir::lds(smem + ODD);
    if (careful) wir::no_odd<false, NW>(odd);
    K.load(smem, 0, wave);
    wir::packed_rows(q, a.q + head * a.qh + r.start * a.qt, a.qt, row0, r.len);
    // below every score but -inf, from which it differs by a number: a row whose scores are all -inf so far has sums of 0
    m = -3.4028234663852886e38f, l = 0.f;
    asm volatile("" : "+v"(m));   // (as a known number it and its negative would hold registers throughout: 1.5% more cycles)
    wir::fill(o, 0.f);
    if (NW == 4 || second == 0) walk<0>(careful, odd);
    else walk<1>(careful, odd);
    l = wir::lane_group_reduce<32>(l, wir::OpAdd());
    const float inv = 1.0f / l;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) o.f[cb][0] *= inv;
    if (!careful) {   // an infinite or NaN value that not all of a tile's rows see
      if (wir::any_wave(wir::has_nan(o, row0 + lane % 32 < r.len), smem + ODD)) return true;
    } else {
      wir::wait_vm_barrier<0>();   // the tiles are read: their LDS takes the output
      const int row = CAUSAL ? row0 + lane % 32 : r.len - 1;   // the last position that the row sees
#pragma unroll
      for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          o.f[cb][0][i] = wir::with_odd<false>(odd, cb * 32 + wir::ccol<32>(i, lane / 32), row, o.f[cb][0][i]);
    }
    const auto O = wir::packed_head(a.out, a.oh, a.ot, head, r.start, r.len, D);
    wir::store_tile_staged<true>(O, o, 0, 0, row0, 0, smem + wave * 32 * D * 2);
    const int row = row0 + lane;
    if (lane < 32 && row < r.len)
      a.lse[head * a.lh + (r.start + row) * a.lt] = (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
    return false;
  }
};

template <int D, bool CAUSAL, int NW>
__device__ __forceinline__ void forward(const wir::packed_fwd_args& a) {
  __shared__ __attribute__((aligned(1024))) char smem[Forward<D, CAUSAL, NW>::BYTES];
  int x, head;
  const int two = NW == 8 && a.flags & 4, rows = NW == 4 || two ? 128 : 256;
  wir::packed_program(a, two ? a.heads / 2 : a.heads, rows, x, head);
  if (two) head *= 2;
  if (CAUSAL) x = a.blocks - 1 - x;   // a sequence's longest block first
  const wir::Rows r = wir::packed_block(a.offsets, a.batch, a.tokens, x, rows);
  if (r.row0 < 0 || r.row0 >= r.len) return;   // (a number that no block has)
  if (r.rest) {
    wir::packed_fill_rest(a, r, head, D, rows);
    if (two) wir::packed_fill_rest(a, r, head + 1, D, 128);
    return;
  }
  Forward<D, CAUSAL, NW> f(a, r, smem);
  bool careful = false;
  while (f.run(head, careful)) careful = true;
}

}  // namespace

#define PACKED_KERNEL(NAME, D, CAUSAL, NW, WAVES_A_SIMD)                                                \
  extern "C" __global__ void __attribute__((amdgpu_flat_work_group_size(64 * NW, 64 * NW),              \
                                            amdgpu_waves_per_eu(WAVES_A_SIMD, WAVES_A_SIMD)))           \
  NAME(const wir::packed_fwd_args args) { forward<D, CAUSAL, NW>(args); }

PACKED_KERNEL(wir_attn_packed_d64, 64, false, 4, 3)
PACKED_KERNEL(wir_attn_packed_d64_causal, 64, true, 4, 3)
PACKED_KERNEL(wir_attn_packed_d128, 128, false, 4, 2)
PACKED_KERNEL(wir_attn_packed_d128_causal, 128, true, 4, 2)
PACKED_KERNEL(wir_attn_packed_d128_w8, 128, false, 8, 2)
PACKED_KERNEL(wir_attn_packed_d128_w8_causal, 128, true, 8, 2)
