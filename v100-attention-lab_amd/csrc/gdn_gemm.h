// Shared parts of the matrix products of the head's loss and of the 8-bit
// product: how tiles of the two operands come to LDS, and the loop over the
// contraction.
//
// A workgroup takes a tile of BM x BN outputs, M being the dimension that lies
// contiguous in the result, and goes over the contraction in slabs of 128 bytes
// of each row (64 elements of 16 bits, 128 of 8).  A ring of S slabs of both
// operands lies in LDS, 2 or 3; slab k + S is copied (LDS-DMA) over slab k once
// every wave has its last operands of k in registers, so a copy has as long as the
// products of S - 1 slabs, and there is one barrier a slab.  Operands of a step are
// read from LDS while the step before it is in the matrix unit.
//
// Large tiles are 256 x 256, 8 waves of 128 x 64: 64 KB a slab for 4 times the
// products of a 128 x 128 tile at twice its reading.  8192 x 4096 x 32000 in bf16: 1.27
// PFLOP/s, the card at about 2.0 of its 2.4 GHz, its matrix units busy for 67 % of the
// cycles.  Tried: slabs of 64 bytes in a ring of 4 (5 % slower: twice the barriers), 4
// waves of 128 x 128 (17 %: one wave a SIMD, with spills), copies spread between the
// products (no change).
//
// An operand is `Plain` where its rows are contiguous along the contraction and
// `Turned` where they are contiguous along M or N (16 bits only: the transposing
// LDS read takes it from there).
#pragma once

#include "gdn_attn.h"

namespace gdn {
namespace gemm {

using attn::dma16;
using attn::dma4;
using attn::dma_wait;
using attn::f32x16;
using attn::lds_addr;
using attn::lds_s16x4;
using attn::lds_f32;
using attn::lds_u32x4;
using attn::s16x4;
using attn::u32x4;
using attn::uniform64;
typedef __attribute__((address_space(3))) uint8_t lds_u8;

constexpr int kSlab = 128;      // bytes of a row of a slab

// MT x NT products of 32 x 32 a wave, WM x WN waves, STAGES slabs in LDS.
template <int MT_, int NT_, int WM_, int WN_, int STAGES_ = 2>
struct Shape {
  static constexpr int MT = MT_, NT = NT_, WM = WM_, WN = WN_, kStages = STAGES_;
  static constexpr int BM = 32 * MT * WM, BN = 32 * NT * WN, kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr uint32_t kA = kSlab * BM, kB = kSlab * BN, kStage = kA + kB, kLds = kStages * kStage;
  static constexpr int kCopies = kStage / 1024 / kWaves;      // of a wave for a slab
};

// What copies read where an operand has no row or column: zeros.
__device__ __attribute__((aligned(16))) const uint32_t kNothing[4] = {0, 0, 0, 0};

__device__ __forceinline__ const uint8_t* uniform_bytes(const void* p) {
  return (const uint8_t*)(uintptr_t)uniform64((int64_t)(uintptr_t)p);
}

// R rows, each contiguous along the contraction.  Row r of a slab lies at 128 r
// in 16-byte pieces, piece c at place c ^ ((r >> 1) & 7): 16 rows at one piece
// cover all banks once.  Rows past the last are copies of it; pieces past the
// end of the contraction are zeros.
template <int R, int WAVES>
struct PlainCopy {
  static constexpr int kPasses = R / (8 * WAVES);
  static_assert(R % (8 * WAVES) == 0, "whole passes");
  const uint8_t* base;     // of the tile's first row
  uint32_t ofs[kPasses];
  int piece, bytes;        // the lane's piece of a slab; the contraction's bytes
  uint32_t wave;
  __device__ __forceinline__ PlainCopy(const void* p, int64_t ld, int row0, int rows, int bytes_) : bytes(bytes_) {
    const int lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) % WAVES);
    base = uniform_bytes((const uint8_t*)p + (int64_t)row0 * ld);
    const int r = (int)wave * 8 + lane / 8;
    piece = (lane % 8) ^ ((r >> 1) & 7);     // (8 WAVES rows further on: the same)
    static_assert((8 * WAVES) % 16 == 0, "one piece for all passes");
#pragma unroll
    for (int i = 0; i < kPasses; ++i)
      ofs[i] = (uint32_t)min(r + i * 8 * WAVES, rows - 1 - row0) * (uint32_t)ld + 16u * piece;
  }
  __device__ __forceinline__ void copy(int slab, uint32_t at) const {
    const uint8_t* src = base + (int64_t)slab * kSlab;
    if ((slab + 1) * kSlab <= bytes) {
#pragma unroll
      for (int i = 0; i < kPasses; ++i) dma16(src, ofs[i], at + (i * WAVES + wave) * 1024);
    } else {
      const bool some = slab * kSlab + 16 * piece < bytes;
#pragma unroll
      for (int i = 0; i < kPasses; ++i)
        dma16(some ? src + ofs[i] : (const uint8_t*)kNothing, at + (i * WAVES + wave) * 1024);
    }
  }
};

// R columns of 16 bits that are contiguous, 64 rows of the contraction a slab.
// Row k lies at 2 R k, piece c at place c ^ ((k & 3) << 2): 4 rows at 64
// neighbouring bytes (a transposing read) cover all banks once.  Columns past
// the last are copies of the last 8; rows that are not in `live` are zeros.
template <int R, int WAVES>
struct TurnedCopy {
  static constexpr int kPieces = R / 8, kRows = 64 / kPieces, kPasses = 64 / (kRows * WAVES);
  static_assert(R >= 128 && 64 % (kRows * WAVES) == 0 && (kRows * WAVES) % 4 == 0, "whole passes");
  const uint8_t* base;
  int64_t ld;
  uint32_t ofs;
  int row;                 // of the lane in the first pass
  uint32_t wave;
  __device__ __forceinline__ TurnedCopy(const void* p, int64_t ld_, int col0, int cols) : ld(ld_) {
    const int lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    base = uniform_bytes(p);
    row = (int)wave * kRows + lane / kPieces;
    const int piece = (lane % kPieces) ^ ((row & 3) << 2);
    ofs = (uint32_t)row * (uint32_t)ld + 2u * (uint32_t)min(col0 + 8 * piece, cols - 8);
  }
  __device__ __forceinline__ void copy(int slab, uint32_t at, uint64_t live) const {
    const uint8_t* src = base + (int64_t)slab * 64 * ld;
    if (live == ~0ull) {
#pragma unroll
      for (int i = 0; i < kPasses; ++i)
        dma16(src + (int64_t)(i * kRows * WAVES) * ld, ofs, at + (i * WAVES + wave) * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const bool some = (live >> (row + i * kRows * WAVES)) & 1;
        dma16(some ? src + (int64_t)(i * kRows * WAVES) * ld + ofs : (const uint8_t*)kNothing,
              at + (i * WAVES + wave) * 1024);
      }
    }
  }
};

// Rows of a slab that lie before the end.
__device__ __forceinline__ uint64_t rows_left(int64_t slab, int64_t rows) {
  const int64_t n = rows - slab * 64;
  return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
}

// Operands of a step of 16 elements of 16 bits: row (or column) 32 i + l % 32
// from the wave's first, elements 16 s + 8 (l / 32) .. + 7 of the slab.
struct PlainRead {
  uint32_t ofs;
  __device__ __forceinline__ PlainRead(int lane, int first) {
    const int r = lane & 31;      // (first: a multiple of 32)
    ofs = (uint32_t)(first + r) * kSlab + 16 * ((lane >> 5) ^ ((r >> 1) & 7));
  }
  __device__ __forceinline__ uint4 operator()(uint32_t tile, int i, int s) const {
    const u32x4 v = *(const lds_u32x4*)(tile + (ofs ^ (32 * s)) + 32 * kSlab * i);
    return make_uint4(v[0], v[1], v[2], v[3]);
  }
};
template <int R>
struct TurnedRead {
  uint32_t ofs;
  __device__ __forceinline__ TurnedRead(int lane, int first) {
    const int a = lane & 15, k = 8 * (lane >> 5) + (a >> 2);
    const int piece = first / 8 + 2 * ((lane >> 4) & 1) + ((a & 3) >> 1);
    ofs = (uint32_t)k * (2 * R) + 16 * (piece ^ ((k & 3) << 2)) + 8 * (a & 1);
  }
  // (first is a multiple of 32 MT, so i is apart from its bits)
  __device__ __forceinline__ uint4 operator()(uint32_t tile, int i, int s) const {
    union {
      s16x4 h[2];
      uint4 v;
    } u;
    const uint32_t at = tile + (ofs ^ (64 * i)) + 16 * s * 2 * R;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 4 * 2 * R));
    return u.v;
  }
};

// All but the last N loads of this wave from memory, and all from LDS, are done.
template <int N>
__device__ __forceinline__ void dma_wait_but() {
  static_assert(N < 64, "6 bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | ((N >> 4) << 14));
  asm volatile("" ::: "memory");
}

// acc += A B^T over `slabs` slabs of 16-bit elements.  copy(slab, at): the
// workgroup's copies of both operands of a slab to `at`; every thread of the
// workgroup calls this, and LDS is free again behind it.
template <typename T, typename S, typename ReadA, typename ReadB, typename Copy>
__device__ __forceinline__ void product16(f32x16 (&acc)[S::MT][S::NT], int slabs, uint32_t lds, const ReadA& ra,
                                          const ReadB& rb, Copy copy) {
  using O = attn::Ops<T>;
  constexpr int MT = S::MT, NT = S::NT, N = MT * NT, F = MT + NT, ST = S::kStages;
  if (slabs <= 0) return;
  uint4 f[2][F];        // operands of two steps: NT of B, MT of A
  auto read = [&](uint32_t stage, int s, int e) {
    f[s & 1][e] = e < NT ? rb(stage + S::kA, e, s) : ra(stage, e - NT, s);
  };
  // products of step s, an operand of the next one read beside each (behind the
  // last slab from the other stage, for nobody)
  auto step = [&](int s, uint32_t stage, int next) {
#pragma unroll
    for (int e = 0; e < (N > F ? N : F); ++e) {
      if (e < N) {
        const int i = e / NT, j = e % NT;
        acc[i][j] = O::mfma(attn::as_vec<T>(f[s & 1][NT + i]), attn::as_vec<T>(f[s & 1][j]), acc[i][j]);
      }
      if (e < F) read(stage, next, e);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  for (int k = 0; k < ST && k < slabs; ++k) copy(k, lds + k * S::kStage);
  if (slabs >= ST) dma_wait_but<(ST - 1) * S::kCopies>();
  else dma_wait();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int e = 0; e < F; ++e) read(lds, 0, e);
  uint32_t here = lds;
  for (int k = 0; k < slabs; ++k) {
    const uint32_t other = here + S::kStage < lds + S::kLds ? here + S::kStage : lds;
#pragma unroll
    for (int s = 0; s < 3; ++s) step(s, here, s + 1);
    // every operand of this slab is in registers, and the next slab in LDS
    if (k + ST <= slabs) dma_wait_but<(ST - 2) * S::kCopies>();
    else dma_wait();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (k + ST < slabs) copy(k + ST, here);
    step(3, other, 0);
    here = other;
  }
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Tile of a workgroup, tm x tn of them for each part of the contraction.  Workgroups
// go round the 8 dies one by one: each die gets neighbouring tiles of as few parts as
// may be, 8 of N at a time, that share rows in its L2.
struct TileAt {
  int m, n, split;
  __device__ __forceinline__ TileAt(uint32_t id, uint32_t tm, uint32_t tn, uint32_t splits = 1) {
    const uint32_t tiles = tm * tn, total = tiles * splits, per = total / 8, left = total % 8, die = id % 8;
    uint32_t at = die * per + min(die, left) + id / 8;
    split = (int)(at / tiles);
    at %= tiles;
    const uint32_t group = at / (8 * tm), in = at % (8 * tm), width = min(8u, tn - 8 * group);
    n = (int)(8 * group + in % width);
    m = (int)(in / width);
  }
};

}  // namespace gemm
}  // namespace gdn
