// Product of e4m3 rows with an e4m3 weight, with scales along the contraction,
// and the quantisers that make its operands:
//     y_mn = sum_b xs_mb ws_{n / 128, b} sum_{k in block b} x_mk w_nk
// (blocks of 128 columns; a row's scale may also be one for all blocks).
//
// Matrix instructions take 128 products deep blocks at a time; each block's sums
// start at zero and enter the result times their scales, in fp32, which costs
// one multiply-add for every 32 multiply-adds' time of the matrix unit and runs
// beside it.  The matrix unit adds 8-bit products in groups of 8, each cut (towards
// zero) at 2^-13 of the largest of its group (found by products of chosen sizes):
// about 1.4e-5 of a result of normally distributed terms, under what 16-bit results
// show and far under e4m3's own steps; up to 2^-10 of the sum of the terms' sizes, which
// a 16-bit result does show where they cancel.  fp32 results are made of the same bytes
// as fp16 operands instead, whose products are summed in fp32, at less than half the rate.
//   - up to 32 rows: the weight is read once from memory straight into the
//     operands' registers, the contraction dealt to the waves of a workgroup,
//     whose sums are joined in LDS in order: bound by that reading and its start,
//     1 x 2048 x 2048 3.8 us, 16 x 2048 x 6176 7.2 us (1.8 TB/s);
//   - more: tiles through LDS (gdn_gemm.h), a slab being one block of 128: bound by
//     the products and, where the card is full, by its power: 8192 x 4096 x 8192 265 us,
//     2.07 PFLOP/s of the 2.74 that a product with one scale for each operand reaches
//     there.  The products alone take 189 us, without the copies of later slabs 207,
//     the copies alone 172; beside each other the clock falls to 2.04 GHz.
// The quantisers are bound by memory (777 x 2048 4.6 us, mostly the launch).
#include <algorithm>

#include "gdn_fp8.h"
#include "gdn_gemm.h"

namespace gdn {
namespace fp8 {

using namespace gemm;
using rowio::Pack;
typedef int i32x8 __attribute__((ext_vector_type(8)));

struct LArgs {
  const uint8_t* x;
  const float* xs;
  const uint8_t* w;
  const float* ws;
  void* y;
  int64_t xld, wld, xsld, wsld;   // bytes; scales a row
  int M, N, K;
  int xstep;                      // 1: a scale a block, 0: a scale a row
  int y_dtype;
  int tm, tn;
};

// 8 e4m3 numbers as fp16 (exact).
__device__ __forceinline__ f16x8 widen(int lo, int hi) {
  typedef f16 f16x2 __attribute__((ext_vector_type(2)));
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false);
  const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false);
  const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Products of a block of 128.  EXACT: summed in fp32.
template <bool EXACT>
__device__ __forceinline__ f32x4 mfma128(const i32x8& a, const i32x8& b) {
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  if constexpr (EXACT) {
#pragma unroll
    for (int s = 0; s < 8; s += 2)
      sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen(a[s], a[s + 1]), widen(b[s], b[s + 1]), sum, 0, 0, 0);
    return sum;
  } else {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, sum, 0, 0, 0, 0, 0, 0);
  }
}
__device__ __forceinline__ i32x8 join16(const uint4& a, const uint4& b) {
  return i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}

// 4 neighbouring outputs n .. n + 3 of a row of N.
__device__ __forceinline__ void store_y(const LArgs& a, int64_t m, int n, const f32x4& v) {
  const int64_t at = m * a.N + n;
  if (a.N % 4 == 0) {
    if (n >= a.N) return;
    if (a.y_dtype == GDN_DTYPE_F32) {
      *reinterpret_cast<f32x4*>(static_cast<float*>(a.y) + at) = v;
    } else {
      const bool h = a.y_dtype == GDN_DTYPE_F16;
      uint2 p;
      p.x = h ? attn::Ops<f16>::pack(v[0], v[1]) : attn::Ops<bf16_t>::pack(v[0], v[1]);
      p.y = h ? attn::Ops<f16>::pack(v[2], v[3]) : attn::Ops<bf16_t>::pack(v[2], v[3]);
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.y) + at) = p;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < a.N) store_scalar(a.y, at + e, a.y_dtype, v[e]);
  }
}

// ---------------------------------------------------------------------------
// few rows
// ---------------------------------------------------------------------------

constexpr int kFewWaves = 8;

// 16 outputs of up to 16 NB rows; wave w takes blocks w, w + 8, ...  Lane l holds row
// l % 16 of an operand, bytes 32 (l / 16) .. + 31 of the block.
template <int NB, bool EXACT>
__global__ __launch_bounds__(64 * kFewWaves) void few_kernel(const LArgs a) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, part = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16;
  const uint8_t* w = a.w + (int64_t)min(n0 + l16, a.N - 1) * a.wld + 32 * part;
  const uint8_t* x[NB];
  const float* xs[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int64_t m = min(16 * j + l16, a.M - 1);
    x[j] = a.x + m * a.xld + 32 * part;
    xs[j] = a.xs + m * a.xsld;
  }
  const float* ws = a.ws + (int64_t)(n0 / 128) * a.wsld;
  f32x4 acc[NB] = {};
  const int blocks = a.K / 128;
  struct Block {
    uint4 w[2], x[NB][2];
    float xs[NB], ws;
  };
  auto load = [&](Block& f, int b) {
#pragma unroll
    for (int h = 0; h < 2; ++h) f.w[h] = *reinterpret_cast<const uint4*>(w + (int64_t)b * 128 + 16 * h);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
#pragma unroll
      for (int h = 0; h < 2; ++h) f.x[j][h] = *reinterpret_cast<const uint4*>(x[j] + (int64_t)b * 128 + 16 * h);
      f.xs[j] = xs[j][b * a.xstep];
    }
    f.ws = ws[b];
  };
  auto use = [&](const Block& f) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const float s = f.xs[j] * f.ws;
      const f32x4 p = mfma128<EXACT>(join16(f.w[0], f.w[1]), join16(f.x[j][0], f.x[j][1]));
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[j][r] = __builtin_fmaf(p[r], s, acc[j][r]);
    }
  };
  for (int b = wv; b < blocks; b += 2 * kFewWaves) {
    Block f[2];
    load(f[0], b);
    const bool two = b + kFewWaves < blocks;
    if (two) load(f[1], b + kFewWaves);
    use(f[0]);
    if (two) use(f[1]);
  }
  __shared__ f32x4 sums[kFewWaves][NB][64];
#pragma unroll
  for (int j = 0; j < NB; ++j) sums[wv][j][lane] = acc[j];
  __syncthreads();
  for (int j = wv; j < NB; j += kFewWaves) {
    f32x4 v = sums[0][j][lane];
#pragma unroll
    for (int k = 1; k < kFewWaves; ++k) v += sums[k][j][lane];
    const int m = 16 * j + l16;
    if (m < a.M) store_y(a, m, n0 + 4 * part, v);
  }
}

// ---------------------------------------------------------------------------
// tiles
// ---------------------------------------------------------------------------

// MT x NT products of 16 x 16 a wave, WM x WN waves, STAGES slabs in LDS; GROUPS of
// such waves take every GROUPS-th slab each.  A stage holds the slabs of both operands
// and a line of 64 scales from each wave: of 64 rows each, then of the tile's
// 128-output blocks.
template <int MT_, int NT_, int WM_, int WN_, int STAGES_, int GROUPS_ = 1>
struct Shape8 {
  static constexpr int MT = MT_, NT = NT_, WM = WM_, WN = WN_, kStages = STAGES_, kGroups = GROUPS_;
  static constexpr int BM = 16 * MT * WM, BN = 16 * NT * WN, kWaves = WM * WN, kThreads = 64 * kWaves * kGroups;
  static constexpr uint32_t kA = kSlab * BM, kB = kSlab * BN, kStage = kA + kB + 256 * kWaves, kRing = kStages * kStage;
  static constexpr uint32_t kLds = kGroups * kRing;
  static constexpr int kCopies = (kA + kB) / 1024 / kWaves + 1;       // of a wave for a slab
  static_assert(MT % 4 == 0 && BN / 64 < kWaves, "4 operands in turn; a wave for each 64 rows' scales and one more");
};
typedef Shape8<8, 4, 2, 4, 2> Big8;      // 256 outputs x 256 rows, one workgroup a CU
typedef Shape8<4, 4, 2, 2, 2> Mid8;      // 128 x 128, two
typedef Shape8<4, 2, 2, 2, 2> Low8;      // 128 x 64, three
typedef Shape8<4, 2, 2, 2, 3, 2> Low8x2; // the same, one: two groups that share the contraction
typedef Shape8<4, 1, 1, 4, 2, 4> Tiny8;  // 64 x 64, one: four groups

// Operand of a block: row 16 i + l % 16 from the wave's first, and of it the pieces
// l / 16 and l / 16 + 4 (any two, as long as both operands have the same; these leave
// the banks free of conflicts, pieces 2 (l / 16) and 2 (l / 16) + 1 took twice as long).
struct Read8 {
  uint32_t ofs;
  __device__ __forceinline__ Read8(int lane, int first) {
    const int r = lane & 15;      // (first: a multiple of 16)
    ofs = (uint32_t)(first + r) * kSlab + 16 * ((lane >> 4) ^ ((r >> 1) & 7));
  }
  __device__ __forceinline__ i32x8 operator()(uint32_t tile, int i) const {
    const u32x4 a = *(const lds_u32x4*)(tile + ofs + 16 * kSlab * i);
    const u32x4 b = *(const lds_u32x4*)(tile + (ofs ^ 64) + 16 * kSlab * i);
    return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
  }
};

// Rows m0 .. m0 + 15, columns n0 .. of a wave's tile (products 16 j .. + 15 of its
// rows).  A lane has 4 neighbouring columns of one row: they go through the wave's own
// share of LDS, so that rows leave in whole lines.
template <typename E, typename S>
__device__ __forceinline__ void store_rows(const f32x4 (&acc)[S::MT][S::NT], int j, const LArgs& a, uint8_t* mem, int m0,
                                           int n0) {
  constexpr int kCols = 16 * S::MT, kPitch = kCols * (int)sizeof(E) + 16, kPer = 16 / (int)sizeof(E);
  static_assert(16 * kPitch * S::kWaves <= (int)S::kLds, "a share for every wave");
  const int lane = threadIdx.x & 63;
  uint8_t* mine = mem + (threadIdx.x >> 6) * 16 * kPitch;
#pragma unroll
  for (int i = 0; i < S::MT; ++i) {
    Pack<E, 4> p;
    const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
    p.set(v);
    p.store(reinterpret_cast<E*>(mine + (lane & 15) * kPitch) + 16 * i + 4 * (lane >> 4));
  }
  E* y = static_cast<E*>(a.y) + (int64_t)m0 * a.N + n0;
  const int rows = a.M - m0, cols = a.N - n0;
  if (a.N % kPer == 0) {
    constexpr int kLanes = kCols / kPer;      // a row
#pragma unroll
    for (int i = 0; i < 16 * kLanes / 64; ++i) {
      const int r = lane / kLanes + i * (64 / kLanes), c = lane % kLanes * kPer;
      const uint4 v = *reinterpret_cast<const uint4*>(mine + r * kPitch + c * (int)sizeof(E));
      if (r < rows && c < cols) *reinterpret_cast<uint4*>(y + (int64_t)r * a.N + c) = v;
    }
  } else {
    for (int e = lane; e < 16 * kCols; e += 64) {
      const int r = e / kCols, c = e % kCols;
      const E v = reinterpret_cast<const E*>(mine + r * kPitch)[c];
      if (r < rows && c < cols) y[(int64_t)r * a.N + c] = v;
    }
  }
}

// The operands of 4 rows of products are in registers at a time, read up to 3 rows
// ahead.  The barrier of a slab stands before its last two rows, which go column by
// column: the next slab's operands are read beside them, each column's over the one
// that has just been used.
template <typename S, bool EXACT>
__global__ __launch_bounds__(S::kThreads) void tile_kernel(const LArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t mem[S::kLds];
  constexpr int MT = S::MT, NT = S::NT;
  const TileAt t(blockIdx.x, a.tm, a.tn);
  const int lane = threadIdx.x & 63, l16 = lane & 15;
  const int group = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) / S::kWaves);
  const int wv = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) % S::kWaves), wm = wv % S::WM, wn = wv / S::WM;
  const uint32_t lds = lds_addr(mem) + group * S::kRing;
  const PlainCopy<S::BM, S::kWaves> ca(a.w, a.wld, t.m * S::BM, a.N, a.K);
  const PlainCopy<S::BN, S::kWaves> cb(a.x, a.xld, t.n * S::BN, a.M, a.K);
  const Read8 ra(lane, 16 * MT * wm), rb(lane, 16 * NT * wn);
  // wave w < BN / 64 brings the scales of rows 64 w .., the others those of the outputs
  const bool rows = wv < S::BN / 64;
  const float* sp = rows ? a.xs + (int64_t)min(t.n * S::BN + 64 * wv + lane, a.M - 1) * a.xsld
                         : a.ws + (int64_t)min(t.m * S::BM / 128 + lane, (a.N - 1) / 128) * a.wsld;
  const int step = rows ? a.xstep : 1;
  // the group's k-th slab (the last ones again where the groups' shares differ)
  const int all = a.K / 128, slabs = (all + S::kGroups - 1) / S::kGroups;
  auto copy = [&](int k, uint32_t at) {
    const int b = min(k * S::kGroups + group, all - 1);
    dma4(sp + b * step, at + S::kA + S::kB + 256 * wv);
    ca.copy(b, at);
    cb.copy(b, at + S::kA);
  };
  const uint32_t sx = S::kA + S::kB + 4 * (16 * NT * wn + l16), sw = S::kA + S::kB + 4 * S::BN + 4 * (16 * MT * wm / 128);
  constexpr int ST = S::kStages;
  f32x4 acc[MT][NT] = {};
  for (int k = 0; k < ST && k < slabs; ++k) copy(k, lds + k * S::kStage);
  if (slabs >= ST) dma_wait_but<(ST - 1) * S::kCopies>();
  else dma_wait();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  i32x8 fb[NT], fa[4];
  float f[NT], x[NT], w;
  auto scales = [&](uint32_t stage) {
    w = *(const lds_f32*)(stage + sw);
#pragma unroll
    for (int j = 0; j < NT; ++j) x[j] = *(const lds_f32*)(stage + sx + 64 * j);
  };
  scales(lds);
#pragma unroll
  for (int j = 0; j < NT; ++j) fb[j] = rb(lds + S::kA, j);
  fa[0] = ra(lds, 0);
  fa[1] = ra(lds, 1);
  uint32_t here = lds;
  for (int k = 0; k < slabs; ++k) {
    const uint32_t other = here + S::kStage < lds + S::kRing ? here + S::kStage : lds;
    const bool ours = S::kGroups == 1 || k * S::kGroups + group < all;
#pragma unroll
    for (int j = 0; j < NT; ++j) f[j] = ours ? x[j] * w : 0.f;
    // a product enters its sum when the fourth one behind it starts (or with the
    // slab's last)
    f32x4 p[4];
    auto row = [](int e) { return e < (MT - 2) * NT ? e / NT : MT - 2 + ((e - (MT - 2) * NT) & 1); };
    auto col = [](int e) { return e < (MT - 2) * NT ? e % NT : (e - (MT - 2) * NT) >> 1; };
    auto add = [&](int e) {
      const int i = row(e), j = col(e);
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_fmaf(p[e & 3][r], f[j], acc[i][j][r]);
      asm volatile("" : "+v"(acc[i][j]));     // (here, not at the slab's end with all products kept)
    };
#pragma unroll
    for (int e = 0; e < MT * NT; ++e) {
      const int i = row(e), j = col(e);
      if (e == (MT - 2) * NT) {
        // every operand of this slab is in registers, and the next slab in LDS
        if (k + ST <= slabs) dma_wait_but<(ST - 2) * S::kCopies>();
        else dma_wait();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (k + ST < slabs) copy(k + ST, here);
      }
      if (e >= 4) add(e - 4);
      p[e & 3] = mfma128<EXACT>(fa[i & 3], fb[j]);
      if (i < MT - 2) {
        if (e == 0) fa[2] = ra(here, 2);
        if (j == (e < NT ? NT - 1 : 0) && i + 3 < MT) fa[(i + 3) & 3] = ra(here, i + 3);
      } else if (i == MT - 1) {
        // (behind the last slab from the other stage, for nobody)
        fb[j] = rb(other + S::kA, j);
        if (j == 0) scales(other);
        if (j == 0) fa[0] = ra(other, 0);
        if (j == std::min(1, NT - 1)) fa[1] = ra(other, 1);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int e = MT * NT - 4; e < MT * NT; ++e) add(e);
    here = other;
  }
  __syncthreads();      // (LDS is free)
  if constexpr (S::kGroups > 1) {
    // the groups' sums, added in order (behind the places that the rows go through)
    constexpr int kRows = S::kWaves * 16 * (64 * MT + 16);
    static_assert(kRows + (S::kGroups - 1) * S::BM * S::BN * 4 <= (int)S::kLds, "room for both");
    f32x4* sums = reinterpret_cast<f32x4*>(mem + kRows) + wv * 64 + lane;
    if (group > 0) {
#pragma unroll
      for (int e = 0; e < MT * NT; ++e)
        sums[((group - 1) * MT * NT + e) * S::kWaves * 64] = acc[e / NT][e % NT];
    }
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int g = 1; g < S::kGroups; ++g)
#pragma unroll
      for (int e = 0; e < MT * NT; ++e) acc[e / NT][e % NT] += sums[((g - 1) * MT * NT + e) * S::kWaves * 64];
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int m0 = t.n * S::BN + 16 * (NT * wn + j), n0 = t.m * S::BM + 16 * MT * wm;
    if (a.y_dtype == GDN_DTYPE_F32) {
      if constexpr (EXACT) store_rows<float, S>(acc, j, a, mem, m0, n0);
    } else if (a.y_dtype == GDN_DTYPE_F16) {
      store_rows<f16, S>(acc, j, a, mem, m0, n0);
    } else {
      store_rows<bf16_t, S>(acc, j, a, mem, m0, n0);
    }
  }
}

// ---------------------------------------------------------------------------
// quantisers
// ---------------------------------------------------------------------------

struct QArgs {
  const void* x;
  uint8_t* q;
  float* scale;
  int64_t ld;        // elements between rows
  int rows, D;
  uint32_t groups;   // of all rows
  uint32_t first;    // workgroup of a launch
};

constexpr int kQ = 256;

// A group of 128 columns: 16 lanes.
template <typename T>
__global__ __launch_bounds__(kQ) void quant_groups_kernel(const QArgs a) {
  const uint32_t g = (a.first + blockIdx.x) * (kQ / 16) + threadIdx.x / 16, per = a.D / 128;
  const bool ok = g < a.groups;
  const uint32_t row = ok ? g / per : 0, c = (ok ? g - row * per : 0) * 128 + threadIdx.x % 16 * 8;
  Pack<T, 8> x;
  x.load(static_cast<const T*>(a.x) + (int64_t)row * a.ld + c);
  float v[8], m = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = x.get(e);
    m = nan_max(m, fabsf(v[e]));
  }
  m = lanes_max<16>(m) / kFp8Max;
  if (!ok) return;
  if (threadIdx.x % 16 == 0) a.scale[g] = m;
  const Quant quant(m);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = quant(v[e]);
  store_fp8<8>(a.q + (int64_t)row * a.D + c, v);
}

// A whole row, read twice: a workgroup.  (Columns are counted past the last one, which
// 31 bits need not hold.)
template <typename T>
__global__ __launch_bounds__(kQ) void quant_rows_kernel(const QArgs a) {
  const int64_t row = a.first + blockIdx.x;
  const uint32_t D = a.D;
  const T* x = static_cast<const T*>(a.x) + row * a.ld;
  float m = 0.f;
  for (uint32_t c = threadIdx.x * 8; c < D; c += kQ * 8) {
    Pack<T, 8> p;
    p.load(x + c);
#pragma unroll
    for (int e = 0; e < 8; ++e) m = nan_max(m, fabsf(p.get(e)));
  }
  __shared__ float slots[kQ / 64];
  m = lanes_max<64>(m);
  if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kQ / 64; ++w) m = nan_max(m, slots[w]);
  m = m / kFp8Max;
  if (threadIdx.x == 0) a.scale[row] = m;
  const Quant quant(m);
  for (uint32_t c = threadIdx.x * 8; c < D; c += kQ * 8) {
    Pack<T, 8> p;
    p.load(x + c);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = quant(p.get(e));
    store_fp8<8>(a.q + row * a.D + c, v);
  }
}

// A block of 128 x 128 of a weight: 16 lanes a row, 8 rows a thread.
template <typename T>
__global__ __launch_bounds__(kQ) void quant_blocks_kernel(const QArgs a) {
  const uint32_t block = a.first + blockIdx.x, per = a.D / 128, br = block / per, bc = block - br * per;
  const int c = bc * 128 + threadIdx.x % 16 * 8, r0 = br * 128 + threadIdx.x / 16;
  Pack<T, 8> x[8];
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i].zero();
    if (r0 + 16 * i < a.rows) x[i].load(static_cast<const T*>(a.x) + (int64_t)(r0 + 16 * i) * a.ld + c);
#pragma unroll
    for (int e = 0; e < 8; ++e) m = nan_max(m, fabsf(x[i].get(e)));
  }
  __shared__ float slots[kQ / 64];
  m = lanes_max<64>(m);
  if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kQ / 64; ++w) m = nan_max(m, slots[w]);
  m = m / kFp8Max;
  if (threadIdx.x == 0) a.scale[block] = m;
  const Quant quant(m);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = quant(x[i].get(e));
    if (r0 + 16 * i < a.rows) store_fp8<8>(a.q + (int64_t)(r0 + 16 * i) * a.D + c, v);
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

inline int64_t tiles_of(int64_t m, int64_t n, int bm, int bn) { return (m + bm - 1) / bm * ((n + bn - 1) / bn); }

template <typename S, bool EXACT>
void launch_tiles(LArgs& a, hipStream_t s) {
  a.tm = (a.N + S::BM - 1) / S::BM;
  a.tn = (a.M + S::BN - 1) / S::BN;
  hipLaunchKernelGGL((tile_kernel<S, EXACT>), dim3((uint32_t)a.tm * a.tn), dim3(S::kThreads), 0, s, a);
}
template <int NB, bool EXACT>
void launch_few(const LArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((few_kernel<NB, EXACT>), dim3((a.N + 15) / 16), dim3(64 * kFewWaves), 0, s, a);
}

// Which kernel (us in a graph, rows x K x N, 16-bit results):
//   - up to 32 rows the weight goes straight into registers (1 x 4096 x 11008 10.8, by
//     tiles 12.8; 17 x 4096 x 8192 12.7 either way; 40 x 4096 x 8192 15.2 and 13.4);
//   - up to 256 tiles of 64 x 64 (a CU each) four groups share the contraction
//     (256 x 2048 x 2048 7.0, Low8x2 8.9), up to 256 tiles of 128 x 64 two (512 x 4096
//     x 4096 16.5, Low8 22.3, Tiny8 24.4);
//   - then larger tiles as they fill the card: 256 x 256 from 192 of them (3000 x 2048 x
//     4096 34.5, Mid8 34.7; 4096 x 4096 x 4096 70.5 and 78.8), 128 x 128 from 256 (1024 x
//     2048 x 6176 21.3, Low8 27.4) unless few outputs leave it to the reading of x
//     (34486 x 2304 x 77 Low8 22.1, Mid8 25.3).
template <bool EXACT>
void launch_linear(LArgs& a, hipStream_t s) {
  if (a.M <= 16) return launch_few<1, EXACT>(a, s);
  if (a.M <= 32) return launch_few<2, EXACT>(a, s);
  if (tiles_of(a.N, a.M, 64, 64) <= 256) return launch_tiles<Tiny8, EXACT>(a, s);
  if (tiles_of(a.N, a.M, 128, 64) <= 256) return launch_tiles<Low8x2, EXACT>(a, s);
  if constexpr (!EXACT) {
    if (tiles_of(a.N, a.M, 256, 256) >= 192) return launch_tiles<Big8, EXACT>(a, s);
  }
  if (a.N > 128 && tiles_of(a.N, a.M, 128, 128) >= 256) return launch_tiles<Mid8, EXACT>(a, s);
  launch_tiles<Low8, EXACT>(a, s);
}

// As many launches as the workgroups take (see grid_fits).
template <typename T>
int launch_quant(QArgs a, int mode, hipStream_t s) {
  constexpr uint32_t kMost = 1 << 23;
  static_assert(kMost <= 0xffffffffu / kQ, "one launch holds them");
  const uint32_t all = mode == GDN_FP8_GROUPS ? (a.groups + kQ / 16 - 1) / (kQ / 16)
                       : mode == GDN_FP8_ROWS ? (uint32_t)a.rows
                                              : ((uint32_t)a.rows + 127) / 128 * (a.D / 128);
  for (; a.first < all; a.first += kMost) {
    const dim3 grid(std::min(kMost, all - a.first));
    if (mode == GDN_FP8_GROUPS) hipLaunchKernelGGL((quant_groups_kernel<T>), grid, dim3(kQ), 0, s, a);
    else if (mode == GDN_FP8_ROWS) hipLaunchKernelGGL((quant_rows_kernel<T>), grid, dim3(kQ), 0, s, a);
    else hipLaunchKernelGGL((quant_blocks_kernel<T>), grid, dim3(kQ), 0, s, a);
    if (const int st = (int)hipGetLastError()) return st;
  }
  return GDN_OK;
}

}  // namespace fp8
}  // namespace gdn

using namespace gdn;
using namespace gdn::fp8;

extern "C" {

int gdn_fp8_quant_launch(const GdnFp8QuantParams* prm, void* stream) {
  if (prm == nullptr) return GDN_ERR_NULL_POINTER;
  const GdnFp8QuantParams& P = *prm;
  if (P.rows < 0 || P.D < 128 || P.x_stride < 0) return GDN_ERR_BAD_SHAPE;
  if (P.D % 128 != 0 || P.mode < GDN_FP8_GROUPS || P.mode > GDN_FP8_BLOCKS) return GDN_ERR_UNSUPPORTED;
  if (!scan_dtype_ok(P.x_dtype)) return GDN_ERR_BAD_DTYPE;
  if (P.rows == 0) return GDN_OK;
  if (P.x == nullptr || P.q == nullptr || P.scale == nullptr) return GDN_ERR_NULL_POINTER;
  if (reinterpret_cast<uintptr_t>(P.x) % 16 != 0 || (P.rows > 1 && P.x_stride * dtype_bytes(P.x_dtype) % 16 != 0) ||
      reinterpret_cast<uintptr_t>(P.q) % 8 != 0)
    return GDN_ERR_MISALIGNED;
  const int64_t groups = (int64_t)P.rows * (P.D / 128);
  if (groups > 0x7fffffff) return GDN_ERR_BAD_SHAPE;      // they are counted in 32 bits
  QArgs a = {};
  a.x = P.x;
  a.q = static_cast<uint8_t*>(P.q);
  a.scale = P.scale;
  a.ld = P.rows > 1 ? P.x_stride : 0;
  a.rows = P.rows;
  a.D = P.D;
  a.groups = (uint32_t)groups;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (P.x_dtype == GDN_DTYPE_F16) return launch_quant<f16>(a, P.mode, s);
  if (P.x_dtype == GDN_DTYPE_BF16) return launch_quant<bf16_t>(a, P.mode, s);
  return launch_quant<float>(a, P.mode, s);
}

int gdn_fp8_linear_launch(const GdnFp8LinearParams* prm, void* stream) {
  if (prm == nullptr) return GDN_ERR_NULL_POINTER;
  const GdnFp8LinearParams& P = *prm;
  if (P.M < 0 || P.N < 1 || P.K < 128) return GDN_ERR_BAD_SHAPE;
  if (P.K % 128 != 0 || (P.group != 0 && P.group != 128)) return GDN_ERR_UNSUPPORTED;
  if (!scan_dtype_ok(P.y_dtype)) return GDN_ERR_BAD_DTYPE;
  if (P.M > 1 << 28 || P.N > 1 << 28) return GDN_ERR_BAD_SHAPE;
  // rows of a tile lie within 31 bits
  if ((P.M > 1 && (P.x_stride < 0 || P.x_stride > 1 << 23)) || (P.N > 1 && (P.w_stride < 0 || P.w_stride > 1 << 23)) ||
      P.K > 1 << 23)
    return GDN_ERR_UNSUPPORTED;
  if (P.M == 0) return GDN_OK;
  if (P.x == nullptr || P.x_scale == nullptr || P.w == nullptr || P.w_scale == nullptr || P.y == nullptr)
    return GDN_ERR_NULL_POINTER;
  if (reinterpret_cast<uintptr_t>(P.x) % 16 != 0 || (P.M > 1 && P.x_stride % 16 != 0) ||
      reinterpret_cast<uintptr_t>(P.w) % 16 != 0 || (P.N > 1 && P.w_stride % 16 != 0) ||
      reinterpret_cast<uintptr_t>(P.y) % 16 != 0)
    return GDN_ERR_MISALIGNED;
  if (!(P.M <= 32 ? grid_fits((P.N + 15) / 16, 64 * kFewWaves) : grid_fits(tiles_of(P.N, P.M, 128, 64), 256)))
    return GDN_ERR_BAD_SHAPE;
  LArgs a = {};
  a.x = static_cast<const uint8_t*>(P.x);
  a.xs = P.x_scale;
  a.w = static_cast<const uint8_t*>(P.w);
  a.ws = P.w_scale;
  a.y = P.y;
  a.xld = P.M > 1 ? P.x_stride : P.K;
  a.wld = P.N > 1 ? P.w_stride : P.K;
  a.M = P.M;
  a.N = P.N;
  a.K = P.K;
  a.wsld = P.K / 128;
  a.xsld = P.group != 0 ? P.K / 128 : 1;
  a.xstep = P.group != 0 ? 1 : 0;
  a.y_dtype = P.y_dtype;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (P.y_dtype == GDN_DTYPE_F32) launch_linear<true>(a, s);
  else launch_linear<false>(a, s);
  return (int)hipGetLastError();
}

}  // extern "C"
