// wir_packed.h -- what the kernels over packed sequences (attn_packed.hip,
// attn_packed_bwd.hip) share: which rows a workgroup takes, and products whose
// tile may hold infinities or NaN in places that not all rows see.
#pragma once
#include "wir_cdna4.h"

namespace wir {

typedef long long i64;

// Rows of a workgroup, and of one of its four waves.
constexpr int PACKED_WAVES = 4, PACKED_ROWS = 128;

// A workgroup's rows: row0 .. of the sequence of `len` tokens from token `start`
// on.  `rest`: of the tokens behind the last sequence instead.
struct Rows {
  int start, len, row0;
  bool rest;
};

// offsets[i], within the tokens.  Every index that follows from the offsets is
// bounded: offsets that do not ascend give wrong rows, no more.
__device__ __forceinline__ int packed_offset(const int* offsets, int i, int batch, int tokens) {
  return i > batch ? tokens : min(max(offsets[i], 0), tokens);
}

// Block x of all sequences' blocks of `rows` rows (a power of two).  Sequence
// i's blocks are numbered from offsets[i] / rows + i on: that leaves each at
// least as many numbers as it has blocks, needs no sum over the sequences'
// blocks and no length on the host; tokens / rows + batch + 1 numbers hold all,
// the last ones those of the tokens behind the last sequence (i = batch).  The lanes look
// at 64 sequences at a time: one round of loads up to 63 sequences, two up to 4095.
__device__ __forceinline__ Rows packed_block(const int* offsets, int batch, int tokens, int x, int rows = PACKED_ROWS) {
  const int lane = lane_id();
  int lo = 0, n = batch + 1;   // the sequence is one of lo .. lo + n - 1
  for (;;) {
    const int step = (n + 63) / 64, i = lo + lane * step;
    const int from = packed_offset(offsets, min(i, batch), batch, tokens);
    const int to = packed_offset(offsets, min(i, batch) + 1, batch, tokens);
    const bool here = lane * step < n && from / rows + i <= x;
    const int last = max(63 - __builtin_clzll(__builtin_amdgcn_ballot_w64(here) | 1), 0);
    if (step > 1) {
      lo += last * step;
      n = min(step, n - last * step);
      continue;
    }
    Rows r;
    r.start = __builtin_amdgcn_readlane(from, last);
    r.len = __builtin_amdgcn_readlane(to, last) - r.start;
    const int seq = lo + last;
    r.row0 = (x - r.start / rows - seq) * rows;
    r.rest = seq == batch;
    return r;
  }
}

// Program -> (block, head).  The programs of one XCD are of few heads, so that
// a head's keys and values stay in its L2.
//
// Where sequences are about as long as a block, every second number is no
// block's, and programs go to the XCD's 32 CUs in turn: half of the CUs would get only
// those.  There the even ones of 64 blocks come first (256 x 128 tokens, 32/8 heads
// of 128, causal: forward 285 -> 199 us, backward 856 -> 542; other lengths would be 2 to 7% slower).
template <class Args>
__device__ __forceinline__ void packed_program(const Args& a, int heads, int rows, int& x, int& head) {
  const int id = remap_xcd(blockIdx.x, a.blocks * heads);
  head = id / a.blocks;
  x = id - head * a.blocks;
  const i64 tokens = a.tokens, one = (i64)rows * a.batch;   // (of one block a sequence)
  if (4 * tokens > 3 * one && 2 * tokens < 3 * one && (x | 63) < a.blocks) x = (x & ~63) | (x & 31) << 1 | (x >> 5 & 1);
}

// One head of one sequence as a tensor of its own: rows past its end read as zeros and are not stored.
template <typename T>
__device__ __forceinline__ gl<T> packed_head(T* data, i64 head_stride, i64 row_stride, int head, int start, int len,
                                             int cols) {
  return gl<T>{data + head * head_stride + (i64)start * row_stride, 1, 1, len, cols, 0, 0, row_stride};
}

// The tiles of one head of one sequence, loaded into LDS by NW waves.
// A lane's j-th load moves a 16-byte chunk of row row + j * EVERY (row < EVERY, a
// power of two, and the swizzles are exclusive ors of a row's bits, so that
// the two parts' swizzles are taken one after the other).  Rows past the sequence's end read its last row (no branch,
// no address of another sequence): whoever uses the tile masks them.
template <class Tile, int NW = PACKED_WAVES>
struct HeadTiles {
  static constexpr int LOADS = Tile::ROWS * Tile::CPR / 64 / NW, EVERY = Tile::ROWS / LOADS;
  static_assert((EVERY & (EVERY - 1)) == 0, "");
  const char* base;
  unsigned row, chunk, pitch;   // the lane's row and bytes in it, bytes from a row to the next
  int len;

  __device__ __forceinline__ void init(const bf16* x, i64 row_stride, int rows) {
    const int p = NW == 1 ? lane_id() : threadIdx.x, c = p % Tile::CPR;   // (wave w's chunks start at 64 w)
    row = p / Tile::CPR;
    chunk = (c ^ swz<Tile::CPR, Tile::ROLE>(row)) * 16;
    pitch = (unsigned)row_stride * 2;
    base = (const char*)x;
    len = rows;
  }

  __device__ __forceinline__ void load(char* tile, int t, int wave) const {
    const char* from = base + (i64)(t * Tile::ROWS) * pitch;
    const unsigned end = (unsigned)min(len - 1 - t * Tile::ROWS, Tile::ROWS - 1);
#pragma unroll
    for (int j = 0; j < LOADS; ++j)
      dma16_s(from, min(row + j * EVERY, end) * pitch + (chunk ^ swz<Tile::CPR, Tile::ROLE>(j * EVERY) * 16), lds_addr(tile + (wave + j * NW) * 1024));
  }
};

// A wave's 32 rows from row0 on of one head of one sequence as operands; past the sequence's end its last row.
template <int KS>
__device__ __forceinline__ void packed_rows(RowFrags<32, 1, KS>& fr, const bf16* x, i64 row_stride, int row0, int len) {
  const int lane = lane_id();
  const bf16* from = x + (i64)min(row0 + lane % 32, len - 1) * row_stride + lane / 32 * 8;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) fr.f[0][ks] = *(const bf16x8*)(from + ks * 16);
}

// In a branch that few tiles take: keeps the compiler from computing it for all of them and selecting.
__device__ __forceinline__ void seldom() { asm volatile(""); }
// The same, and what follows from x is computed in that branch, not kept in registers from before a loop.
__device__ __forceinline__ int seldom(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Keep (row, col) for col <= row (CAUSAL), or for col < cols; elsewhere -inf.
template <bool CAUSAL, int MS, int R, int C>
__device__ __forceinline__ void packed_mask(RTile<MS, R, C>& t, int row0, int col0, int cols) {
  const int lane = lane_id(), lr = lane % MS, lh = seldom(lane / MS);
#pragma unroll
  for (int cb = 0; cb < t.CB; ++cb)
#pragma unroll
    for (int rb = 0; rb < t.RB; ++rb)
#pragma unroll
      for (int i = 0; i < MF<MS>::CREGS; ++i) {
        const int row = row0 + rb * MS + lr, col = col0 + cb * MS + ccol<MS>(i, lh);
        t.f[cb][rb][i] = (CAUSAL ? col <= row : col < cols) ? t.f[cb][rb][i] : -__builtin_inff();
      }
}

// Whether a wave's tile holds a NaN, in the lanes whose row is `in`.
template <int MS, int R, int C>
__device__ __forceinline__ bool has_nan(const RTile<MS, R, C>& t, bool in) {
  bool any = false;
#pragma unroll
  for (int cb = 0; cb < t.CB; ++cb)
#pragma unroll
    for (int rb = 0; rb < t.RB; ++rb)
#pragma unroll
      for (int i = 0; i < MF<MS>::CREGS; ++i) any |= t.f[cb][rb][i] != t.f[cb][rb][i];
  return __builtin_amdgcn_ballot_w64(any && in) != 0;
}

// The workgroup's answer to "is there a NaN in a wave's results", after which the tiles' LDS is free.
__device__ __forceinline__ bool any_wave(bool mine, char* flag_at) {
  auto* flag = (__attribute__((address_space(3))) int*)lds(flag_at);
  wait_vm_barrier<0>();
  if (threadIdx.x == 0) *flag = 0;
  barrier();
  if (mine) *flag = 1;
  barrier();
  const bool any = *flag;
  barrier();
  return any;
}

// A product a @ b over a tile b (K rows, C columns) whose rows not all rows of
// `a` see: a is 0 where it does not see, but 0 times an infinity or NaN is NaN.
// clear_odd makes those values of b 0 for the product and notes for each of its
// columns the first (LAST: the last) position that holds one: they rule the
// results of the rows that see that position.
template <int D>
struct Odd {
  int at[3][D];   // NaN, +infinity, -infinity
};

constexpr int NOWHERE = 0x7fffffff;

template <bool LAST, int NW, int D>
__device__ __forceinline__ void no_odd(__attribute__((address_space(3))) Odd<D>* odd) {
  for (int i = threadIdx.x; i < 3 * D; i += 64 * NW) (&odd->at[0][0])[i] = LAST ? -1 : NOWHERE;
}

template <bool LAST, int NW, class TB>
__device__ __forceinline__ void clear_odd(char* b_base, int pos0, __attribute__((address_space(3))) Odd<TB::COLS>* odd) {
  typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
#pragma unroll 1
  for (int i = NW == 1 ? lane_id() : threadIdx.x; i < TB::ROWS * TB::CPR; i += 64 * NW) {
    const int row = i / TB::CPR, chunk = i % TB::CPR;
    auto* p = (__attribute__((address_space(3))) u16x8*)(lds(b_base) + TB::chunk_off(row, chunk));
    u16x8 w = *p;
    bool any = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) any |= (w[j] & 0x7f80) == 0x7f80;
    if (!any) continue;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if ((w[j] & 0x7f80) != 0x7f80) continue;
      int* at = (int*)&odd->at[w[j] & 0x7f ? 0 : w[j] & 0x8000 ? 2 : 1][chunk * 8 + j];
      if (LAST) atomicMax(at, pos0 + row);
      else atomicMin(at, pos0 + row);
      w[j] = 0;
    }
    *p = w;
  }
  if (NW == 1) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (other waves have nothing to do with the tile)
}

// x, a sum over column d without its odd values, with those that `row` sees: positions up to it (LAST: from it on).
template <bool LAST, int D>
__device__ __forceinline__ float with_odd(const __attribute__((address_space(3))) Odd<D>* odd, int d, int row, float x) {
  auto sees = [&](int i) { return LAST ? row <= odd->at[i][d] : row >= odd->at[i][d]; };
  const bool nan = sees(0), up = sees(1), down = sees(2);
  return nan || (up && down) ? __builtin_nanf("") : up ? x + __builtin_inff() : down ? x - __builtin_inff() : x;
}

}  // namespace wir
