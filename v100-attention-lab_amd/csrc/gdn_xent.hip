// Softmax cross entropy of a linear head, logits made in pieces and never kept:
//     l = X W^T,  lse_n = log sum_v e^{l_nv},  loss_n = lse_n - l_{n, t_n}
//     G = dloss_n (e^{l - lse} - [v = t_n]),  dX = G W,  dW = G^T X
//
// Forward: tiles of logits (vocabulary x rows) on matrix instructions; each
// leaves the maximum m and the sum s of e^{l - m} of its vocabulary for its rows,
// and a second kernel joins them in order.  m stays a logit and s is 1 or more, so
// the loss (m - l_t) + ln s has no rounding of the logits' size and is never below 0
// (targets 18 to 40 above 10240 words: off by 6e-9 on average; as lse - l_t, through
// powers of 2, by 4e-7, an eighth of the rows below 0).
// Backward: piece by piece of the vocabulary the logits are made again by the
// same loop (so that e^{l - lse} fits its lse), G of the piece is rounded once to
// the operands' type into the workspace, dW of the piece is one product over all
// rows and dX a sum over the pieces, kept in fp32 in the order of the
// accumulators.  Where dX has few tiles the piece's vocabulary is cut into parts
// that have sums of their own, joined in order at the end.
//
// Bound by the products: 2 N D V forward, 6 N D V backward (the logits a second time;
// keeping them would take 2 N V bytes and their reading).  bf16 on a card whose large
// matrix product reaches 1.41 PFLOP/s: 8192 x 4096, 128000 words forward 6.7 ms (1.28
// PFLOP/s), backward 21 ms (1.23); a piece of 8192 words G 0.44, dW 0.44 and dX 0.47
// ms, dX with its fp32 sums read and written.  48 rows of 2048 against 50257 words are
// bound by reading the weight, 32 us at 6.5 TB/s where the last-level cache holds it.
//
// G is kept in a unit that makes the largest finite |dloss| a power of 2.  A mean gives all
// rows the same dloss, and the target's G, close to -dloss, outweighs the others: it
// is then rounded not at all where the target is improbable, and else by the row and
// not for all alike (511 x 1024 x 4000, dloss 1/511, bf16: dX 0.0024 -> 0.0017 off).  In fp16 the
// power is 2^13, so that probabilities of a large vocabulary over many rows stay normal
// numbers; bf16 has the range and keeps its power.
#include <algorithm>

#include "gdn_gemm.h"

namespace gdn {
namespace xent {

using namespace gemm;
using attn::exp2_fast;
using attn::kLn2;
using attn::kLog2e;
using attn::max_halves;
using attn::Ops;
using attn::swap_halves;

// Where there are few of them, a third slab on the way pays more than another
// workgroup beside: 128 rows, 16000 words of 2048 32 -> 26 us (Wide for Mid), 48 rows,
// 50257 words 56 -> 53 (Narrow with 3 slabs for 2; with 4 and one workgroup 58).
typedef Shape<4, 2, 2, 4> Big;         // 256 x 256, one workgroup a CU
static_assert(Big::BM == 256 && Big::BN == 256 && Big::kThreads == 512, "as check() counts them");
typedef Shape<2, 2, 2, 2> Mid;         // 128 x 128, two
typedef Shape<2, 2, 2, 2, 3> Wide;     // the same, one
typedef Shape<2, 1, 2, 2, 3> Narrow;   // 128 x 64 (vocabulary x rows), two

struct Row {
  float lse, g;       // g: dloss in the unit of G, 0 for rows that do not count
};

struct Args {
  const void* x;
  const void* w;
  const int64_t* target;
  float* loss;
  float* lse;              // written by the forward, read by the backward
  const float* dloss;
  void* dx;
  void* dw;
  int64_t xld, wld;        // bytes between rows
  int64_t dloss_step;
  int N, D, V;
  // workspace
  float2* part;            // forward: (maximum, sum) [tiles of V][N]
  float* hit;              // the target's logit [N]
  Row* rows;               // backward: [N up to 256]
  int32_t* tgt;            // the row's target, -1 without
  uint64_t* live;          // a bit for each row that counts
  float* unit;             // 1 / unit of G
  uint16_t* g;             // [N up to 256][ldg]
  float4* sums;            // of dX, or of dW's parts, in the order of the accumulators
  int ldg;
  int v0, vn;              // the piece: first of V, how many
  int tm, tn, splits, first, last;
};

// ---------------------------------------------------------------------------
// logits
// ---------------------------------------------------------------------------

// Tile of logits: M the vocabulary, N the rows.
template <typename T, typename S>
__device__ __forceinline__ void logits(const Args& a, f32x16 (&acc)[S::MT][S::NT], const TileAt& t, uint32_t lds, int wm,
                                       int wn) {
  const int lane = threadIdx.x & 63;
  const PlainCopy<S::BM, S::kWaves> ca((const uint8_t*)a.w + (int64_t)a.v0 * a.wld, a.wld, t.m * S::BM, a.vn, 2 * a.D);
  const PlainCopy<S::BN, S::kWaves> cb(a.x, a.xld, t.n * S::BN, a.N, 2 * a.D);
  const PlainRead ra(lane, 32 * S::MT * wm), rb(lane, 32 * S::NT * wn);
  product16<T, S>(acc, (a.D + 63) / 64, lds, ra, rb, [&](int k, uint32_t at) {
    ca.copy(k, at);
    cb.copy(k, at + S::kA);
  });
}

template <typename T, typename S>
__global__ __launch_bounds__(S::kThreads) void fwd_kernel(const Args a) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[S::kLds];
  const TileAt t(blockIdx.x, a.tm, a.tn);
  const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wv % S::WM, wn = wv / S::WM;
  f32x16 acc[S::MT][S::NT] = {};
  logits<T, S>(a, acc, t, lds_addr(lds), wm, wn);

  const int v0 = t.m * S::BM + 32 * S::MT * wm, left = a.V - v0;     // of the wave's vocabulary
  float* sm = reinterpret_cast<float*>(lds);                        // [WM][BN]
  float* ss = sm + S::WM * S::BN;
#pragma unroll
  for (int j = 0; j < S::NT; ++j) {
    const int c = 32 * (S::NT * wn + j) + l32, n = t.n * S::BN + c;
    const int64_t hit = n < a.N ? a.target[n] - v0 : -1;
    const bool here = hit >= 0 && hit < min(32 * S::MT, left);
    if (__any(here)) {
#pragma unroll
      for (int i = 0; i < S::MT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (here && hit == 32 * i + attn::acc_row(r, half)) a.hit[n] = acc[i][j][r];
    }
    if (left < 32 * S::MT) {
#pragma unroll
      for (int i = 0; i < S::MT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          acc[i][j][r] = 32 * i + attn::acc_row(r, half) < left ? acc[i][j][r] : -__builtin_inff();
    }
    float m = acc[0][j][0];
#pragma unroll
    for (int i = 0; i < S::MT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) m = fmaxf(m, acc[i][j][r]);
    m = max_halves(m);
    const float mb = m == -__builtin_inff() ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < S::MT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) s += exp2_fast((acc[i][j][r] - mb) * kLog2e);
    s += swap_halves(s);
    if (half == 0) {
      sm[wm * S::BN + c] = m;
      ss[wm * S::BN + c] = s;
    }
  }
  __syncthreads();
  const int c = threadIdx.x, n = t.n * S::BN + c;
  if (c >= S::BN || n >= a.N) return;
  float m = sm[c], s = 0.f;
#pragma unroll
  for (int w = 1; w < S::WM; ++w) m = fmaxf(m, sm[w * S::BN + c]);
#pragma unroll
  for (int w = 0; w < S::WM; ++w) {
    const float x = sm[w * S::BN + c];
    s += ss[w * S::BN + c] * (x == m ? 1.f : exp2_fast((x - m) * kLog2e));
  }
  a.part[(int64_t)t.m * a.N + n] = make_float2(m, s);
}

// (maximum, sum) pairs of parts of the vocabulary.
__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float top = fmaxf(a.x, b.x);
  // (a sum is 0, or NaN, only where all logits are -inf or NaN)
  if (top == -__builtin_inff()) return make_float2(top, a.y + b.y);
  return make_float2(top, a.y * (a.x == top ? 1.f : exp2_fast((a.x - top) * kLog2e)) +
                              b.y * (b.x == top ? 1.f : exp2_fast((b.x - top) * kLog2e)));
}

// lse and loss: 16 rows a workgroup, 64 threads a row (one of 4 in each wave).
constexpr int kJoin = 1024;
__global__ __launch_bounds__(kJoin) void join_kernel(const Args a) {
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
  const int n = blockIdx.x * 16 + c;
  float2 p = make_float2(-__builtin_inff(), 0.f);
  if (n < a.N) {
#pragma unroll 4
    for (int t = g; t < a.tm; t += kJoin / 16) p = join(p, a.part[(int64_t)t * a.N + n]);
  }
#pragma unroll
  for (int o = 16; o <= 32; o *= 2) p = join(p, make_float2(__shfl_xor(p.x, o, 64), __shfl_xor(p.y, o, 64)));
  __shared__ float2 all[kJoin / 64][16];
  if ((threadIdx.x & 63) < 16) all[threadIdx.x >> 6][c] = p;
  __syncthreads();
  if (g != 0 || n >= a.N) return;
#pragma unroll
  for (int k = 1; k < kJoin / 64; ++k) p = join(p, all[k][c]);
  const int64_t t = a.target[n];
  const bool counts = t >= 0 && t < a.V;
  const float ln = __builtin_amdgcn_logf(p.y) * kLn2;
  a.lse[n] = counts ? p.x + ln : 0.f;
  a.loss[n] = 0.f;
  if (counts) a.loss[n] = (p.x - a.hit[n]) + ln;
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------

__device__ __forceinline__ bool row_counts(const Args& a, int n) {
  const int64_t t = n < a.N ? a.target[n] : -1;
  return t >= 0 && t < a.V;
}

// What the pieces need of each row, and the unit of G (every workgroup finds it
// for itself).
constexpr int kRowsNT = 1024;
template <bool F16>
__global__ __launch_bounds__(kRowsNT) void rows_kernel(const Args a) {
  float top = 0.f;
  if (a.dloss_step == 0) {
    top = fabsf(a.dloss[0]);
  } else {
    for (int64_t n0 = threadIdx.x; n0 < a.N; n0 += 4 * kRowsNT) {
      int64_t t[4];
      float d[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {      // (the last row again past the end)
        const int64_t n = min(n0 + i * kRowsNT, (int64_t)a.N - 1);
        t[i] = a.target[n];
        d[i] = fabsf(a.dloss[n * a.dloss_step]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)      // (of the finite ones: one that is not is its row's alone)
        top = t[i] >= 0 && t[i] < a.V && d[i] < __builtin_inff() ? fmaxf(top, d[i]) : top;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    __shared__ float tops[kRowsNT / 64];
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kRowsNT / 64; ++w) top = fmaxf(top, tops[w]);
  }
  float unit = 1.f;
  if (top > 0.f && top < __builtin_inff()) {
    const int e = ilogbf(top);
    unit = ldexpf(1.f / ldexpf(top, -e), F16 ? max(-100, min(100, 13 - e)) : 0);
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.unit = 1.f / unit;
  const int all = (a.N + 255) / 256 * 256;
  for (int n = blockIdx.x * kRowsNT + threadIdx.x; n < all; n += gridDim.x * kRowsNT) {
    const bool c = row_counts(a, n);
    Row r = {0.f, 0.f};
    if (c) r = Row{a.lse[n], a.dloss[n * a.dloss_step] * unit};
    a.rows[n] = r;
    a.tgt[n] = c ? (int32_t)a.target[n] : -1;
    const uint64_t m = __ballot(c);
    if ((threadIdx.x & 63) == 0) a.live[n / 64] = m;
  }
}

// Columns 32 j .. of a wave's tile, times f, as rows n0 .. of `out` (ld elements
// apart, below `rows`), columns m0 .. (below `cols`, a multiple of 8).  A lane has 4
// neighbouring M of one row: they go through the wave's own share of LDS, so that the
// rows leave in whole lines (8-byte stores of 32 rows at a time: 2.5 times as long
// where the sums are short).
template <typename T, typename S>
__device__ __forceinline__ void store_columns(const f32x16 (&acc)[S::MT][S::NT], int j, float f, uint8_t* lds, void* out,
                                              int64_t ld, int n0, int rows, int m0, int cols) {
  using O = Ops<T>;
  constexpr int kRow = 64 * S::MT, kPitch = kRow + 16, kLanes = kRow / 16;      // bytes; lanes a row
  static_assert(32 * kPitch * S::kWaves <= (int)S::kLds, "a share for every wave");
  const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
  uint8_t* mine = lds + (threadIdx.x >> 6) * 32 * kPitch;
#pragma unroll
  for (int i = 0; i < S::MT; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<uint2*>(mine + l32 * kPitch + 64 * i + 16 * q + 8 * half) =
          make_uint2(O::pack(acc[i][j][4 * q] * f, acc[i][j][4 * q + 1] * f),
                     O::pack(acc[i][j][4 * q + 2] * f, acc[i][j][4 * q + 3] * f));
  const int col = m0 + lane % kLanes * 8;
#pragma unroll
  for (int i = 0; i < 32 * kLanes / 64; ++i) {
    const int r = lane / kLanes + i * (64 / kLanes);
    const uint4 v = *reinterpret_cast<const uint4*>(mine + r * kPitch + lane % kLanes * 16);
    if (n0 + r < rows && col < cols)
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + (int64_t)(n0 + r) * ld + col) = v;
  }
}

// G of a tile of the piece.
template <typename T, typename S>
__global__ __launch_bounds__(S::kThreads) void grad_kernel(const Args a) {
  using O = Ops<T>;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[S::kLds];
  const TileAt t(blockIdx.x, a.tm, a.tn);
  const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wv % S::WM, wn = wv / S::WM;
  f32x16 acc[S::MT][S::NT] = {};
  logits<T, S>(a, acc, t, lds_addr(lds), wm, wn);

  const int v0 = t.m * S::BM + 32 * S::MT * wm, left = a.vn - v0;    // in the piece
#pragma unroll
  for (int j = 0; j < S::NT; ++j) {
    const int n = t.n * S::BN + 32 * (S::NT * wn + j) + l32;
    const Row row = a.rows[n];
    const int hit = a.tgt[n] - a.v0 - v0;
    const bool counts = a.tgt[n] >= 0;
#pragma unroll
    for (int i = 0; i < S::MT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = exp2_fast((acc[i][j][r] - row.lse) * kLog2e) * row.g;
        acc[i][j][r] = counts ? p : 0.f;
      }
    if (__any(counts && hit >= 0 && hit < 32 * S::MT)) {
#pragma unroll
      for (int i = 0; i < S::MT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (counts && hit == 32 * i + attn::acc_row(r, half)) acc[i][j][r] -= row.g;
    }
    if (left < 32 * S::MT) {
#pragma unroll
      for (int i = 0; i < S::MT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 32 * i + attn::acc_row(r, half) < left ? acc[i][j][r] : 0.f;
    }
    store_columns<T, S>(acc, j, 1.f, lds, a.g, a.ldg, t.n * S::BN + 32 * (S::NT * wn + j), 1 << 30, v0, a.ldg);
  }
}

// dX += G W over the piece, M the columns of X.
template <typename T, typename S>
__global__ __launch_bounds__(S::kThreads) void dx_kernel(const Args a) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[S::kLds];
  const TileAt t(blockIdx.x, a.tm, a.tn, a.splits);
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wv % S::WM, wn = wv / S::WM;
  const int slabs = (a.vn + 63) / 64, per = (slabs + a.splits - 1) / a.splits;
  const int s0 = min(t.split * per, slabs), s1 = min(s0 + per, slabs);
  f32x16 acc[S::MT][S::NT] = {};
  {
    const TurnedCopy<S::BM, S::kWaves> ca((const uint8_t*)a.w + (int64_t)a.v0 * a.wld, a.wld, t.m * S::BM, a.D);
    const PlainCopy<S::BN, S::kWaves> cb(a.g, 2 * (int64_t)a.ldg, t.n * S::BN, (a.N + 255) / 256 * 256, 2 * a.ldg);
    const TurnedRead<S::BM> ra(lane, 32 * S::MT * wm);
    const PlainRead rb(lane, 32 * S::NT * wn);
    product16<T, S>(acc, s1 - s0, lds_addr(lds), ra, rb, [&](int k, uint32_t at) {
      ca.copy(s0 + k, at, rows_left(s0 + k, a.vn));
      cb.copy(s0 + k, at + S::kA);
    });
  }
  const bool whole = a.last && a.splits == 1;
  float4* sums = a.sums + ((int64_t)(t.split * a.tm + t.m) * a.tn + t.n) * (S::BM * S::BN / 4) + threadIdx.x;
  if (!a.first || !whole) {
#pragma unroll
    for (int j = 0; j < S::NT; ++j)
#pragma unroll
      for (int i = 0; i < S::MT; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float4* at = sums + ((j * S::MT + i) * 4 + q) * S::kThreads;
          if (!a.first) {
            const float4 o = *at;
            acc[i][j][4 * q] += o.x;
            acc[i][j][4 * q + 1] += o.y;
            acc[i][j][4 * q + 2] += o.z;
            acc[i][j][4 * q + 3] += o.w;
          }
          if (!whole)
            *at = make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
        }
  }
  if (whole) {
#pragma unroll
    for (int j = 0; j < S::NT; ++j)
      store_columns<T, S>(acc, j, *a.unit, lds, a.dx, a.D, t.n * S::BN + 32 * (S::NT * wn + j), a.N,
                          t.m * S::BM + 32 * S::MT * wm, a.D);
  }
}

// Parts of dX or of a piece of dW (`rows` rows of D), added in order.
template <typename T, typename S>
__global__ __launch_bounds__(S::kThreads) void parts_kernel(const Args a, uint16_t* out, int rows) {
  constexpr int kPer = S::MT * S::NT * 4;
  const uint32_t tile = blockIdx.x / kPer, e = blockIdx.x % kPer, tiles = a.tm * a.tn;
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, wm = wv % S::WM, wn = wv / S::WM;
  const int q = e % 4, i = e / 4 % S::MT, j = e / 4 / S::MT;
  const int m = tile / a.tn * S::BM + 32 * (S::MT * wm + i) + 8 * q + 4 * (lane >> 5);
  const int n = tile % a.tn * S::BN + 32 * (S::NT * wn + j) + (lane & 31);
  const float4* p = a.sums + ((int64_t)tile * kPer + e) * S::kThreads + threadIdx.x;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const float4 o = p[(int64_t)s * tiles * kPer * S::kThreads];
    v = make_float4(v.x + o.x, v.y + o.y, v.z + o.z, v.w + o.w);
  }
  const float f = *a.unit;
  if (n < rows && m < a.D)      // (D: a multiple of 8)
    *reinterpret_cast<uint2*>(out + (int64_t)n * a.D + m) =
        make_uint2(Ops<T>::pack(v.x * f, v.y * f), Ops<T>::pack(v.z * f, v.w * f));
}

// dW of the piece = G^T X, M the columns of X, N the vocabulary.
template <typename T, typename S>
__global__ __launch_bounds__(S::kThreads) void dw_kernel(const Args a) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[S::kLds];
  const TileAt t(blockIdx.x, a.tm, a.tn, a.splits);
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wv % S::WM, wn = wv / S::WM;
  const int slabs = (a.N + 63) / 64, per = (slabs + a.splits - 1) / a.splits;
  const int s0 = min(t.split * per, slabs), s1 = min(s0 + per, slabs);
  f32x16 acc[S::MT][S::NT] = {};
  {
    const TurnedCopy<S::BM, S::kWaves> ca(a.x, a.xld, t.m * S::BM, a.D);
    const TurnedCopy<S::BN, S::kWaves> cb(a.g, 2 * (int64_t)a.ldg, t.n * S::BN, a.ldg);
    const TurnedRead<S::BM> ra(lane, 32 * S::MT * wm);
    const TurnedRead<S::BN> rb(lane, 32 * S::NT * wn);
    // a row that does not count may hold anything; which do is read a slab ahead
    const auto* live = (const __attribute__((address_space(4))) uint64_t*)(uintptr_t)uniform64((int64_t)(uintptr_t)a.live);
    uint64_t now = live[min(s0, slabs - 1)];
    product16<T, S>(acc, s1 - s0, lds_addr(lds), ra, rb, [&](int k, uint32_t at) {
      const uint64_t rows = now;
      now = live[min(s0 + k + 1, slabs - 1)];
      ca.copy(s0 + k, at, rows);
      cb.copy(s0 + k, at + S::kA, ~0ull);
    });
  }
  if (a.splits > 1) {
    float4* sums = a.sums + ((int64_t)(t.split * a.tm + t.m) * a.tn + t.n) * (S::BM * S::BN / 4) + threadIdx.x;
#pragma unroll
    for (int j = 0; j < S::NT; ++j)
#pragma unroll
      for (int i = 0; i < S::MT; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          sums[((j * S::MT + i) * 4 + q) * S::kThreads] =
              make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
    return;
  }
#pragma unroll
  for (int j = 0; j < S::NT; ++j)
    store_columns<T, S>(acc, j, *a.unit, lds, (uint16_t*)a.dw + (int64_t)a.v0 * a.D, a.D,
                        t.n * S::BN + 32 * (S::NT * wn + j), a.vn, t.m * S::BM + 32 * S::MT * wm, a.D);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

inline int64_t ceil_to(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
inline int64_t tiles_of(int64_t m, int64_t n, int bm, int bn) { return (m + bm - 1) / bm * ((n + bn - 1) / bn); }

// Tiles of 256 x 256 or of 128 x 128, by the rounds that they make of the card: 256 at
// a time take about 13 parts of time, 512 small ones 8.  So small ones up to 512, and
// where the big ones leave much of their second round idle: logits of 1024 rows of 2048
// in us, small and big, 8000 words 40 and 51, 10240 59 and 51, 17408 88 and 104,
// 26624 118 and 107, 65536 279 and 237 (40960 words, 640 big tiles, 167 and 160).
enum Kind { kBig, kMid, kWide, kNarrow };
Kind kind_of(int64_t m, int64_t n) {
  return 13 * ((tiles_of(m, n, 256, 256) + 255) / 256) <= 8 * ((tiles_of(m, n, 128, 128) + 511) / 512) ? kBig : kMid;
}
// Of logits: vocabulary x rows.
Kind logits_kind(int64_t v, int64_t rows) {
  if (rows <= 64) return kNarrow;
  const Kind k = kind_of(v, rows);
  return k == kMid && tiles_of(v, rows, 128, 128) <= 256 ? kWide : k;
}

int check(const GdnXentParams& P) {
  if (P.N < 0 || P.D < 8 || P.V < 1) return GDN_ERR_BAD_SHAPE;
  if (P.D % 8 != 0) return GDN_ERR_UNSUPPORTED;
  if (P.dtype != GDN_DTYPE_F16 && P.dtype != GDN_DTYPE_BF16) return GDN_ERR_BAD_DTYPE;
  // rows of a tile lie within 31 bits
  if ((P.N > 1 && (P.x_stride < 0 || P.x_stride > 1 << 22)) || (P.V > 1 && (P.w_stride < 0 || P.w_stride > 1 << 22)) ||
      P.D > 1 << 22)
    return GDN_ERR_UNSUPPORTED;
  if (P.N >= 1 << 26 || P.V > 1 << 28) return GDN_ERR_BAD_SHAPE;      // (the join has 64 threads a row)
  // one launch each: the logits in the tiles that they are made in (512 threads for 256 x
  // 256; else 256 for 128 x 64 at the least, which only sizes that fit take: with more
  // than 384 rows and words the rule comes to the large ones), the gradients in 128 x 128
  const bool big = logits_kind(P.V, P.N) == kBig;
  if (!(big ? grid_fits(tiles_of(P.V, P.N, 256, 256), 512) : grid_fits(tiles_of(P.V, P.N, 128, 64), 256)) ||
      !grid_fits(tiles_of(P.D, std::max(P.N, P.V), 128, 128), 256))
    return GDN_ERR_BAD_SHAPE;
  return GDN_OK;
}

// Vocabulary of a piece: G takes about 128 MiB.  (Larger pieces gave 0 to 1.6 % at 8192
// rows.  More rows make a piece of fewer words, and dX's sums are read and written for
// each: rows of 4096 against 128000 words backward, in 6 N D V operations, 1.24 PFLOP/s
// at 8192 rows, 1.04 at 32768, 0.87 at 65536.)
int piece_of(const GdnXentParams& P) {
  const int64_t rows = ceil_to(std::max(P.N, 1), 256);
  const int64_t most = std::max<int64_t>((128ll << 20) / (2 * rows) / 256 * 256, 256);
  return (int)std::min(most, ceil_to(P.V, 256));
}

// A gradient's product of m columns and n rows over k: shape, parts of its
// contraction where its tiles do not fill the card, and fp32 sums that it keeps.
struct GradPlan {
  Kind kind;
  int splits;
  int64_t tiles, floats;
  GradPlan(int64_t m, int64_t n, int64_t k, bool kept) {
    kind = kind_of(m, n);
    const int b = kind == kBig ? 256 : 128;
    tiles = tiles_of(m, n, b, b);
    const int64_t slabs = (k + 63) / 64, places = kind == kBig ? 256 : 512;
    splits = (int)std::max<int64_t>(1, std::min(places / tiles, slabs / 8));
    floats = kept || splits > 1 ? tiles * splits * b * b : 0;
  }
};
// dX: rows of X, the contraction is the piece's vocabulary; kept from piece to piece.
GradPlan dx_plan(const GdnXentParams& P) {
  return GradPlan(P.D, std::max(P.N, 1), piece_of(P), piece_of(P) < P.V);
}
// dW of a piece: rows of its vocabulary, the contraction is X's rows.
GradPlan dw_plan(const GdnXentParams& P, int vn) { return GradPlan(P.D, vn, std::max(P.N, 1), false); }

struct BwdLayout {
  int64_t rows, tgt, live, unit, g, dx, dw, bytes;
  explicit BwdLayout(const GdnXentParams& P) {
    const int64_t n = ceil_to(std::max(P.N, 1), 256);
    rows = 0;
    tgt = rows + n * (int64_t)sizeof(Row);
    live = tgt + n * 4;
    unit = ceil_to(live + n / 8, 256);
    g = unit + 256;
    dx = g + n * piece_of(P) * 2;
    dw = dx + dx_plan(P).floats * 4;
    // (the last piece may be cut into more parts than the others)
    const int piece = piece_of(P), last = P.V - (P.V - 1) / piece * piece;
    bytes = dw + 4 * std::max(dw_plan(P, std::min(piece, P.V)).floats, dw_plan(P, last).floats);
  }
};

// Pairs that the forward leaves for a row: one a tile.
int64_t fwd_tiles(const GdnXentParams& P) {
  const int bm = logits_kind(P.V, P.N) == kBig ? 256 : 128;
  return (P.V + bm - 1) / bm;
}

Args args_of(const GdnXentParams& P) {
  Args a = {};
  a.x = P.x;
  a.w = P.w;
  a.target = P.target;
  a.loss = P.loss;
  a.lse = P.lse;
  a.dloss = P.dloss;
  a.dx = P.dx;
  a.dw = P.dw;
  a.xld = 2 * (P.N > 1 ? P.x_stride : (int64_t)P.D);
  a.wld = 2 * (P.V > 1 ? P.w_stride : (int64_t)P.D);
  a.dloss_step = P.dloss_stride;
  a.N = P.N;
  a.D = P.D;
  a.V = P.V;
  return a;
}

// kernel<T, S> by kind: of logits, of gradients.
#define GDN_XENT_LOGITS(kernel, T, kind, grid, s, a)                                                         \
  switch (kind) {                                                                                            \
    case kBig: hipLaunchKernelGGL((kernel<T, Big>), dim3(grid), dim3(Big::kThreads), 0, s, a); break;        \
    case kMid: hipLaunchKernelGGL((kernel<T, Mid>), dim3(grid), dim3(Mid::kThreads), 0, s, a); break;        \
    case kWide: hipLaunchKernelGGL((kernel<T, Wide>), dim3(grid), dim3(Wide::kThreads), 0, s, a); break;     \
    default: hipLaunchKernelGGL((kernel<T, Narrow>), dim3(grid), dim3(Narrow::kThreads), 0, s, a); break;    \
  }
#define GDN_XENT_GRADIENT(kernel, T, kind, grid, s, a)                                                        \
  switch (kind) {                                                                                            \
    case kBig: hipLaunchKernelGGL((kernel<T, Big>), dim3(grid), dim3(Big::kThreads), 0, s, a); break;        \
    default: hipLaunchKernelGGL((kernel<T, Mid>), dim3(grid), dim3(Mid::kThreads), 0, s, a); break;          \
  }

void set_tiles(Args& a, Kind k, int64_t m, int64_t n) {
  const int bm = k == kBig ? 256 : 128, bn = k == kBig ? 256 : k == kNarrow ? 64 : 128;
  a.tm = (int)((m + bm - 1) / bm);
  a.tn = (int)((n + bn - 1) / bn);
}

template <typename T>
int launch_fwd(Args a, hipStream_t s) {
  const Kind kind = logits_kind(a.V, a.N);
  a.v0 = 0;
  a.vn = a.V;
  set_tiles(a, kind, a.V, a.N);
  const uint32_t grid = (uint32_t)a.tm * a.tn;
  GDN_XENT_LOGITS(fwd_kernel, T, kind, grid, s, a);
  hipLaunchKernelGGL(join_kernel, dim3((a.N + 15) / 16), dim3(kJoin), 0, s, a);
  return (int)hipGetLastError();
}

template <typename T>
int launch_bwd(Args a, const GdnXentParams& P, const BwdLayout& l, hipStream_t s) {
  char* ws = static_cast<char*>(P.workspace);
  const GradPlan dx = dx_plan(P);
  const int piece = piece_of(P);
  a.ldg = piece;
  const int blocks = std::min<int>((a.N + kRowsNT - 1) / kRowsNT, 64);      // (each goes over all rows)
  hipLaunchKernelGGL((rows_kernel<std::is_same<T, f16>::value>), dim3(blocks), dim3(kRowsNT), 0, s, a);
  auto parts = [&](const GradPlan& p, void* out, int rows) {
    const uint32_t grid = (uint32_t)(p.tiles * (p.kind == kBig ? 32 : 16));
    if (p.kind == kBig) hipLaunchKernelGGL((parts_kernel<T, Big>), dim3(grid), dim3(Big::kThreads), 0, s, a, (uint16_t*)out, rows);
    else hipLaunchKernelGGL((parts_kernel<T, Mid>), dim3(grid), dim3(Mid::kThreads), 0, s, a, (uint16_t*)out, rows);
  };
  for (int64_t v = 0; v < a.V; v += piece) {
    a.v0 = (int)v;
    a.vn = std::min(piece, a.V - a.v0);
    a.first = v == 0;
    a.last = v + piece >= a.V;
    const Kind kl = logits_kind(a.vn, a.N);
    set_tiles(a, kl, a.vn, a.N);
    const uint32_t grid = (uint32_t)a.tm * a.tn;
    GDN_XENT_LOGITS(grad_kernel, T, kl, grid, s, a);
    const GradPlan dw = dw_plan(P, a.vn);
    set_tiles(a, dw.kind, a.D, a.vn);
    a.splits = dw.splits;
    a.sums = reinterpret_cast<float4*>(ws + l.dw);
    GDN_XENT_GRADIENT(dw_kernel, T, dw.kind, (uint32_t)(dw.tiles * dw.splits), s, a);
    if (dw.splits > 1) parts(dw, (uint16_t*)a.dw + v * a.D, a.vn);
    set_tiles(a, dx.kind, a.D, a.N);
    a.splits = dx.splits;
    a.sums = reinterpret_cast<float4*>(ws + l.dx);
    GDN_XENT_GRADIENT(dx_kernel, T, dx.kind, (uint32_t)(dx.tiles * dx.splits), s, a);
  }
  if (dx.splits > 1) parts(dx, a.dx, a.N);
  return (int)hipGetLastError();
}

bool rows_ok(const void* p, int64_t stride, int64_t n) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (n <= 1 || stride % 8 == 0);
}

}  // namespace xent
}  // namespace gdn

using namespace gdn;
using namespace gdn::xent;

extern "C" {

int64_t gdn_xent_workspace_size(const GdnXentParams* prm) {
  if (prm == nullptr || check(*prm) != GDN_OK) return -1;
  return (int64_t)prm->N * (fwd_tiles(*prm) * 8 + 4);
}

int64_t gdn_xent_bwd_workspace_size(const GdnXentParams* prm) {
  if (prm == nullptr || check(*prm) != GDN_OK) return -1;
  return BwdLayout(*prm).bytes;
}

static int check_call(const GdnXentParams& P, int64_t need) {
  const int st = check(P);
  if (st != GDN_OK) return st;
  if ((P.N > 0 && (P.x == nullptr || P.target == nullptr || P.lse == nullptr)) || P.w == nullptr) return GDN_ERR_NULL_POINTER;
  if (!rows_ok(P.x, P.x_stride, P.N) || !rows_ok(P.w, P.w_stride, P.V)) return GDN_ERR_MISALIGNED;
  if (need > 0 && (P.workspace == nullptr || P.workspace_bytes < need ||
                   reinterpret_cast<uintptr_t>(P.workspace) % 256 != 0))
    return GDN_ERR_WORKSPACE;
  return GDN_OK;
}

int gdn_xent_launch(const GdnXentParams* prm, void* stream) {
  if (prm == nullptr) return GDN_ERR_NULL_POINTER;
  const GdnXentParams& P = *prm;
  if (const int st = check_call(P, gdn_xent_workspace_size(prm))) return st;
  if (P.N == 0) return GDN_OK;
  if (P.loss == nullptr) return GDN_ERR_NULL_POINTER;
  Args a = args_of(P);
  a.part = static_cast<float2*>(P.workspace);
  a.hit = reinterpret_cast<float*>(a.part + fwd_tiles(P) * P.N);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return P.dtype == GDN_DTYPE_F16 ? launch_fwd<f16>(a, s) : launch_fwd<bf16_t>(a, s);
}

int gdn_xent_bwd_launch(const GdnXentParams* prm, void* stream) {
  if (prm == nullptr) return GDN_ERR_NULL_POINTER;
  const GdnXentParams& P = *prm;
  if (const int st = check_call(P, gdn_xent_bwd_workspace_size(prm))) return st;
  if (P.N < 1) return GDN_ERR_BAD_SHAPE;
  if (P.dloss == nullptr || P.dx == nullptr || P.dw == nullptr) return GDN_ERR_NULL_POINTER;
  if (!rows_ok(P.dx, 0, 1) || !rows_ok(P.dw, 0, 1)) return GDN_ERR_MISALIGNED;
  const BwdLayout l(P);
  Args a = args_of(P);
  char* ws = static_cast<char*>(P.workspace);
  a.rows = reinterpret_cast<Row*>(ws + l.rows);
  a.tgt = reinterpret_cast<int32_t*>(ws + l.tgt);
  a.live = reinterpret_cast<uint64_t*>(ws + l.live);
  a.unit = reinterpret_cast<float*>(ws + l.unit);
  a.g = reinterpret_cast<uint16_t*>(ws + l.g);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return P.dtype == GDN_DTYPE_F16 ? launch_bwd<f16>(a, P, l, s) : launch_bwd<bf16_t>(a, P, l, s);
}

}  // extern "C"
