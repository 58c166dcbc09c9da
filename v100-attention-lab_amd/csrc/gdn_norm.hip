// Root-mean-square norm with the residual's addition, its gradient, and the
// same norm with an 8-bit output:
//     r = x + res,  n = r rstd,  rstd = 1 / sqrt(mean(r^2) + eps),  y = n w
//     dr = dr_in + rstd (w dy - n mean(w dy n)),  dw = sum_rows dy n
//
// A row is read once, held in registers in fp32 and written once: a team of
// 8 to 256 threads takes a row, each thread P pieces of V columns.  Rows
// that do not fit the registers, and 128-column scales of rows without
// 16-byte alignment, are read a second time (long kernels).
// dw: every workgroup sums its rows' dy n in registers, in row order, and
// writes one partial row; a second kernel adds the partial rows in order.
//
// Bound by memory.  16384 rows of 2048, bf16 with an fp32 residual stream:
// forward 71 us (403 MB, 5.7 TB/s), backward 98 us (470 MB, 4.8 TB/s) and 5 us
// for dw's partial rows; 8192 rows of 4096 to 8 bits with 128-column scales 47 us
// with the call (235 MB, 5.0 TB/s).  A large copy: 4.9 TB/s.

#include <algorithm>

#include "gdn_fp8.h"

namespace gdn {
namespace norm {

using namespace rowio;
using namespace fp8;

constexpr int kBlock = 256;
constexpr int kMaxPartials = 512;    // partial rows of dw

struct Args {
  const void* x;
  const void* res;
  const void* w;
  void* y;
  void* r_out;
  float* scale;
  const void* r;
  const void* dy;
  const void* dr_in;
  void* dr;
  void* dx;
  void* dw;
  float* part;      // [parts, D] partial sums of dw
  float* rstd;      // [rows] (long rows' backward)
  int64_t xs[2], ress[2], ys[2], ros[2], rs[2], dys[2], dris[2], drs[2], dxs[2];
  uint32_t rows, n_inner, row0;   // row0: first row of a launch (forward, long rows' backward)
  int D, group, parts;
  float eps;
  int w_f32;
};

__device__ __forceinline__ int64_t row_at(const Args& p, uint32_t row, const int64_t* s) {
  const uint32_t o = row / p.n_inner, i = row - o * p.n_inner;
  return (int64_t)o * s[0] + (int64_t)i * s[1];
}

template <int W>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = W / 2; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// Sum over a team of TEAM threads (a wave or less, or the block's waves through LDS;
// each use has a slot of its own, so no wait is needed after the read).
template <int TEAM, bool MAX>
__device__ __forceinline__ float team_reduce(float v, float* slot) {
  constexpr int W = TEAM < 64 ? TEAM : 64;
  v = MAX ? lanes_max<W>(v) : lanes_sum<W>(v);
  if constexpr (TEAM > 64) {
    constexpr int NW = TEAM / 64;
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
    __syncthreads();
    v = slot[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) v = MAX ? nan_max(v, slot[i]) : v + slot[i];
  }
  return v;
}

// Weights of V columns, from either type (p.w_f32 is uniform).
template <typename TX, int V>
__device__ __forceinline__ void load_w(const Args& p, int c, float (&w)[V]) {
  if (p.w_f32) {
    Pack<float, V> k;
    k.load(static_cast<const float*>(p.w) + c);
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] = k.get(e);
  } else {
    Pack<TX, V> k;
    k.load(static_cast<const TX*>(p.w) + c);
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] = k.get(e);
  }
}

// Forward, the row in registers.  FP8: 0 none, 1 a scale per row, 2 per 128
// columns (V = 8: 16 neighbouring lanes).
template <typename TX, typename TR, int V, int P, int TEAM, int FP8>
__global__ __launch_bounds__(kBlock) void fwd_kernel(const Args p) {
  constexpr int ROWS = kBlock / TEAM;
  const int t = threadIdx.x % TEAM;
  const uint32_t row = p.row0 + blockIdx.x * ROWS + threadIdx.x / TEAM;
  if (TEAM <= 64 && row >= p.rows) return;   // no barrier below for these
  const TX* x = static_cast<const TX*>(p.x) + row_at(p, row, p.xs);
  Pack<TX, V> xr[P];
  Pack<TR, V> rr[P];
  const bool has_res = p.res != nullptr;
  const TR* res = has_res ? static_cast<const TR*>(p.res) + row_at(p, row, p.ress) : nullptr;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = (i * TEAM + t) * V;
    xr[i].zero();
    rr[i].zero();
    if (c < p.D) {
      xr[i].load(x + c);
      if (has_res) rr[i].load(res + c);
    }
  }
  float r[P][V], ss = 0.f;
#pragma unroll
  for (int i = 0; i < P; ++i) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      r[i][e] = has_res ? xr[i].get(e) + rr[i].get(e) : xr[i].get(e);
      ss = __builtin_fmaf(r[i][e], r[i][e], ss);
    }
  }
  __shared__ float slots[2][kBlock / 64];
  ss = team_reduce<TEAM, false>(ss, slots[0]);
  const float rstd = 1.f / sqrtf(ss / (float)p.D + p.eps);
  if (has_res) {
    TR* ro = static_cast<TR*>(p.r_out) + row_at(p, row, p.ros);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = (i * TEAM + t) * V;
      Pack<TR, V> o;
      o.set(r[i]);
      if (c < p.D) o.store(ro + c);
    }
  }
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = (i * TEAM + t) * V;
    float w[V];
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] = 0.f;
    if (c < p.D) load_w<TX, V>(p, c, w);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      r[i][e] = r[i][e] * rstd * w[e];
      if constexpr (FP8 == 1) amax = nan_max(amax, fabsf(r[i][e]));
    }
  }
  if constexpr (FP8 == 0) {
    TX* y = static_cast<TX*>(p.y) + row_at(p, row, p.ys);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = (i * TEAM + t) * V;
      Pack<TX, V> o;
      o.set(r[i]);
      if (c < p.D) o.store(y + c);
    }
  } else {
    uint8_t* y = static_cast<uint8_t*>(p.y) + row_at(p, row, p.ys);
    if constexpr (FP8 == 1) {
      amax = team_reduce<TEAM, true>(amax, slots[1]) / kFp8Max;
      if (t == 0) p.scale[row] = amax;
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = (i * TEAM + t) * V;
      float m = amax;
      if constexpr (FP8 == 2) {
        m = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) m = nan_max(m, fabsf(r[i][e]));
        m = lanes_max<16>(m) / kFp8Max;
        if (c < p.D && (c & 127) == 0) p.scale[(int64_t)row * (p.D / 128) + c / 128] = m;
      }
      const Quant quant(m);      // (amax, m: the scale by now)
      float q[V];
#pragma unroll
      for (int e = 0; e < V; ++e) q[e] = quant(r[i][e]);
      if (c < p.D) store_fp8<V>(y + c, q);
    }
  }
}

// Forward of any row: one workgroup a row, the row read again for each step.
template <typename TX, typename TR, int FP8>
__global__ __launch_bounds__(kBlock) void fwd_long_kernel(const Args p) {
  const uint32_t row = p.row0 + blockIdx.x;
  const int t = threadIdx.x;
  const bool has_res = p.res != nullptr;
  const TX* x = static_cast<const TX*>(p.x) + row_at(p, row, p.xs);
  const TR* res = has_res ? static_cast<const TR*>(p.res) + row_at(p, row, p.ress) : nullptr;
  auto value = [&](int c) { return to_f32<TX>(x[c]) + (has_res ? to_f32<TR>(res[c]) : 0.f); };
  auto weight = [&](int c) {
    return p.w_f32 ? static_cast<const float*>(p.w)[c] : to_f32<TX>(static_cast<const TX*>(p.w)[c]);
  };
  __shared__ float slots[2][kBlock / 64];
  float ss = 0.f;
  for (int c = t; c < p.D; c += kBlock) {
    const float v = value(c);
    ss = __builtin_fmaf(v, v, ss);
  }
  ss = team_reduce<kBlock, false>(ss, slots[0]);
  const float rstd = 1.f / sqrtf(ss / (float)p.D + p.eps);
  TR* ro = has_res ? static_cast<TR*>(p.r_out) + row_at(p, row, p.ros) : nullptr;
  if constexpr (FP8 == 0) {
    TX* y = static_cast<TX*>(p.y) + row_at(p, row, p.ys);
    for (int c = t; c < p.D; c += kBlock) {
      const float v = value(c);
      if (has_res) ro[c] = from_f32<TR>(v);
      y[c] = from_f32<TX>(v * rstd * weight(c));
    }
  } else {
    uint8_t* y = static_cast<uint8_t*>(p.y) + row_at(p, row, p.ys);
    if constexpr (FP8 == 1) {
      float amax = 0.f;
      for (int c = t; c < p.D; c += kBlock) {
        const float v = value(c) * rstd * weight(c);
        amax = nan_max(amax, fabsf(v));
      }
      const float scale = team_reduce<kBlock, true>(amax, slots[1]) / kFp8Max;
      if (t == 0) p.scale[row] = scale;
      const Quant quant(scale);
      for (int c = t; c < p.D; c += kBlock) {
        const float v = value(c);
        if (has_res) ro[c] = from_f32<TR>(v);
        const float q[1] = {quant(v * rstd * weight(c))};
        store_fp8<1>(y + c, q);
      }
    } else {
      // a wave takes 128 columns, two a lane
      const int lane = t & 63;
      for (int g = t >> 6; g < p.D / 128; g += kBlock / 64) {
        float v[2], m = 0.f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = g * 128 + 64 * e + lane;
          v[e] = value(c);
          if (has_res) ro[c] = from_f32<TR>(v[e]);
          v[e] = v[e] * rstd * weight(c);
          m = nan_max(m, fabsf(v[e]));
        }
        m = lanes_max<64>(m) / kFp8Max;
        if (lane == 0) p.scale[(int64_t)row * (p.D / 128) + g] = m;
        const Quant quant(m);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float q[1] = {quant(v[e])};
          store_fp8<1>(y + g * 128 + 64 * e + lane, q);
        }
      }
    }
  }
}

// Backward, the row in registers; a workgroup takes rows blockIdx.x + k parts
// (ROWS at a time) and leaves one partial row of dw.
template <typename TX, typename TR, int V, int P, int TEAM>
__global__ __launch_bounds__(kBlock) void bwd_kernel(const Args p) {
  constexpr int ROWS = kBlock / TEAM;
  const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
  float dw[P][V], w[P][V];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = (i * TEAM + t) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) dw[i][e] = w[i][e] = 0.f;
    if (c < p.D) load_w<TX, V>(p, c, w[i]);
  }
  __shared__ float slots[2][2][kBlock / 64];
  int turn = 0;
  for (uint32_t row = blockIdx.x * ROWS + team; row - team < p.rows; row += p.parts * ROWS, turn ^= 1) {
    // a block's teams leave the loop together; a team without a row sums zeros
    const bool live = row < p.rows;
    const TR* r = static_cast<const TR*>(p.r) + (live ? row_at(p, row, p.rs) : 0);
    const TX* dy = static_cast<const TX*>(p.dy) + (live ? row_at(p, row, p.dys) : 0);
    const TR* di = p.dr_in != nullptr && live ? static_cast<const TR*>(p.dr_in) + row_at(p, row, p.dris) : nullptr;
    Pack<TR, V> rr[P], ir[P];
    Pack<TX, V> yr[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = (i * TEAM + t) * V;
      rr[i].zero();
      yr[i].zero();
      ir[i].zero();
      if (live && c < p.D) {
        rr[i].load(r + c);
        yr[i].load(dy + c);
        if (di != nullptr) ir[i].load(di + c);
      }
    }
    float ss = 0.f, sd = 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float v = rr[i].get(e);
        ss = __builtin_fmaf(v, v, ss);
        sd = __builtin_fmaf(w[i][e] * yr[i].get(e), v, sd);
      }
    }
    constexpr int W = TEAM < 64 ? TEAM : 64;
    ss = lanes_sum<W>(ss);
    sd = lanes_sum<W>(sd);
    if constexpr (TEAM > 64) {
      // two sums behind one barrier; the slots alternate between rows
      if ((threadIdx.x & 63) == 0) {
        slots[turn][0][threadIdx.x >> 6] = ss;
        slots[turn][1][threadIdx.x >> 6] = sd;
      }
      __syncthreads();
      ss = slots[turn][0][0];
      sd = slots[turn][1][0];
#pragma unroll
      for (int k = 1; k < kBlock / 64; ++k) {
        ss += slots[turn][0][k];
        sd += slots[turn][1][k];
      }
    }
    const float rstd = 1.f / sqrtf(ss / (float)p.D + p.eps);
    const float mean = sd * rstd / (float)p.D;   // mean of w dy n
    if (live) {
      TR* dr = static_cast<TR*>(p.dr) + row_at(p, row, p.drs);
      TX* dx = p.dx != nullptr ? static_cast<TX*>(p.dx) + row_at(p, row, p.dxs) : nullptr;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int c = (i * TEAM + t) * V;
        float d[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float n = rr[i].get(e) * rstd, y = yr[i].get(e);
          d[e] = __builtin_fmaf(rstd, w[i][e] * y - n * mean, ir[i].get(e));
          dw[i][e] = __builtin_fmaf(y, n, dw[i][e]);
        }
        if (c < p.D) {
          Pack<TR, V> o;
          o.set(d);
          o.store(dr + c);
          if (dx != nullptr) {
            Pack<TX, V> ox;
            ox.set(d);
            ox.store(dx + c);
          }
        }
      }
    }
  }
  // the teams' sums of dw, added in order
  if constexpr (ROWS > 1) {
    __shared__ float sh[ROWS - 1][TEAM * V];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      __syncthreads();
      if (team > 0) {
#pragma unroll
        for (int e = 0; e < V; ++e) sh[team - 1][t * V + e] = dw[i][e];
      }
      __syncthreads();
      if (team == 0) {
#pragma unroll
        for (int k = 0; k < ROWS - 1; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) dw[i][e] += sh[k][t * V + e];
      }
    }
  }
  if (team == 0) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = (i * TEAM + t) * V;
      if (c < p.D) {
#pragma unroll
        for (int e = 0; e < V; ++e) p.part[(int64_t)blockIdx.x * p.D + c + e] = dw[i][e];
      }
    }
  }
}

// Backward of any row: dr (and dx), and rstd for the columns' kernel.
template <typename TX, typename TR>
__global__ __launch_bounds__(kBlock) void bwd_long_kernel(const Args p) {
  const uint32_t row = p.row0 + blockIdx.x;
  const int t = threadIdx.x;
  const TR* r = static_cast<const TR*>(p.r) + row_at(p, row, p.rs);
  const TX* dy = static_cast<const TX*>(p.dy) + row_at(p, row, p.dys);
  const TR* di = p.dr_in != nullptr ? static_cast<const TR*>(p.dr_in) + row_at(p, row, p.dris) : nullptr;
  auto weight = [&](int c) {
    return p.w_f32 ? static_cast<const float*>(p.w)[c] : to_f32<TX>(static_cast<const TX*>(p.w)[c]);
  };
  __shared__ float slots[2][kBlock / 64];
  float ss = 0.f, sd = 0.f;
  for (int c = t; c < p.D; c += kBlock) {
    const float v = to_f32<TR>(r[c]);
    ss = __builtin_fmaf(v, v, ss);
    sd = __builtin_fmaf(weight(c) * to_f32<TX>(dy[c]), v, sd);
  }
  ss = team_reduce<kBlock, false>(ss, slots[0]);
  sd = team_reduce<kBlock, false>(sd, slots[1]);
  const float rstd = 1.f / sqrtf(ss / (float)p.D + p.eps);
  const float mean = sd * rstd / (float)p.D;
  if (t == 0) p.rstd[row] = rstd;
  TR* dr = static_cast<TR*>(p.dr) + row_at(p, row, p.drs);
  TX* dx = p.dx != nullptr ? static_cast<TX*>(p.dx) + row_at(p, row, p.dxs) : nullptr;
  for (int c = t; c < p.D; c += kBlock) {
    const float n = to_f32<TR>(r[c]) * rstd;
    const float d = __builtin_fmaf(rstd, weight(c) * to_f32<TX>(dy[c]) - n * mean, di != nullptr ? to_f32<TR>(di[c]) : 0.f);
    dr[c] = from_f32<TR>(d);
    if (dx != nullptr) dx[c] = from_f32<TX>(d);
  }
}

// Partial rows of dw of any rows: a thread a column, rows of a part in order.
template <typename TX, typename TR>
__global__ __launch_bounds__(kBlock) void dw_cols_kernel(const Args p) {
  const int c = blockIdx.x * kBlock + threadIdx.x;
  if (c >= p.D) return;
  float s = 0.f;
  for (uint32_t row = blockIdx.y; row < p.rows; row += p.parts) {
    const float n = to_f32<TR>((static_cast<const TR*>(p.r) + row_at(p, row, p.rs))[c]) * p.rstd[row];
    s = __builtin_fmaf(to_f32<TX>((static_cast<const TX*>(p.dy) + row_at(p, row, p.dys))[c]), n, s);
  }
  p.part[(int64_t)blockIdx.y * p.D + c] = s;
}

// dw: 64 columns a workgroup, the partial rows split over 16 waves, each in
// order, then the waves in order.
template <typename TX>
__global__ __launch_bounds__(1024) void dw_sum_kernel(const Args p) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane;
  float s = 0.f;
  if (c < p.D) {
#pragma unroll 8
    for (int k = w; k < p.parts; k += 16) s += p.part[(int64_t)k * p.D + c];
  }
  __shared__ float sh[16][64];
  sh[w][lane] = s;
  __syncthreads();
  if (w == 0 && c < p.D) {
    s = sh[0][lane];
#pragma unroll
    for (int k = 1; k < 16; ++k) s += sh[k][lane];
    if (p.w_f32) static_cast<float*>(p.dw)[c] = s;
    else static_cast<TX*>(p.dw)[c] = from_f32<TX>(s);
  }
}

// The team and pieces that hold a row, or 0 pieces: it does not fit.  The
// smallest team whose threads hold the row in 4 pieces of 8 columns (1 or 2 of
// the shortest rows) or 16 of one: fewer steps between lanes, no barrier up to a
// wave, and enough bytes in flight for the backward's 512 workgroups.  bf16, 2^25
// columns in all, forward / backward in us:
//   8 columns: D 64 8 lanes 41 / 47, 64 lanes 157 / 301; D 256 16 lanes 41 / 41,
//     64 lanes 46 / 82; D 1024 32 lanes 42 / 39, 64 lanes 41 / 41, 256 lanes
//     52 / 102; D 2048 64 lanes 43 / 38, 256 lanes 41 / 58; D 4096 256 lanes
//     41 / 41, 64 lanes of 8 pieces 46 / 53; no registers (long) 76 / 114;
//   one column: D 63 16 lanes 58 / 129, 256 lanes 506 / 1275; D 255 16 lanes
//     58 / 103, 256 lanes 138 / 349; D 1001 64 lanes 53 / 118, 256 lanes 66 / 153;
//     D 2047 256 lanes 59 / 137, 64 lanes 72 / 117.
struct Shape {
  int v, p, team;
};
Shape shape_of(int D, bool wide) {
  if (wide) {
    if (D <= 64) return {8, 1, 8};
    if (D <= 128) return {8, 1, 16};
    if (D <= 256) return {8, 2, 16};
    if (D <= 512) return {8, 4, 16};
    if (D <= 1024) return {8, 4, 32};
    if (D <= 2048) return {8, 4, 64};
    if (D <= 4096) return {8, 2, 256};
    if (D <= 8192) return {8, 4, 256};
    if (D <= 16384) return {8, 8, 256};
    return {0, 0, 0};
  }
  if (D <= 64) return {1, 4, 16};
  if (D <= 128) return {1, 8, 16};
  if (D <= 256) return {1, 16, 16};
  if (D <= 512) return {1, 16, 32};
  if (D <= 1024) return {1, 16, 64};
  if (D <= 4096) return {1, 16, 256};
  if (D <= 8192) return {1, 32, 256};
  return {0, 0, 0};
}

// launch(args, grid) for all rows, `per` a workgroup, as many launches as they take.
template <typename F>
int by_rows(Args a, uint32_t per, F launch) {
  constexpr uint32_t kMost = 1 << 23;
  static_assert(kMost <= 0xffffffffu / kBlock, "one launch holds them (see grid_fits)");
  for (; a.row0 < a.rows; a.row0 += kMost * per) {
    launch(a, dim3((uint32_t)std::min<uint64_t>(kMost, ((uint64_t)a.rows - a.row0 + per - 1) / per)));
    const int st = (int)hipGetLastError();
    if (st != 0) return st;
  }
  return 0;
}

template <typename TX, typename TR, int V, int P, int TEAM>
int fwd_shape(const Args& a, hipStream_t s) {
  return by_rows(a, kBlock / TEAM, [&](const Args& b, dim3 grid) {
    if (b.scale == nullptr) hipLaunchKernelGGL((fwd_kernel<TX, TR, V, P, TEAM, 0>), grid, dim3(kBlock), 0, s, b);
    else if (b.group == 0) hipLaunchKernelGGL((fwd_kernel<TX, TR, V, P, TEAM, 1>), grid, dim3(kBlock), 0, s, b);
    else if constexpr (V == 8 && TEAM >= 16) hipLaunchKernelGGL((fwd_kernel<TX, TR, V, P, TEAM, 2>), grid, dim3(kBlock), 0, s, b);
  });
}

template <typename TX, typename TR>
int fwd_typed(const Args& a, bool wide, hipStream_t s) {
  Shape sh = shape_of(a.D, wide);
  if (!wide && a.scale != nullptr && a.group != 0) sh.p = 0;   // 128 columns are not a lane group there
  switch (sh.p * 1000 + sh.team) {
    case 1008: return fwd_shape<TX, TR, 8, 1, 8>(a, s);
    case 1016: return fwd_shape<TX, TR, 8, 1, 16>(a, s);
    case 2016: return fwd_shape<TX, TR, 8, 2, 16>(a, s);
    case 4016: return sh.v == 8 ? fwd_shape<TX, TR, 8, 4, 16>(a, s) : fwd_shape<TX, TR, 1, 4, 16>(a, s);
    case 4032: return fwd_shape<TX, TR, 8, 4, 32>(a, s);
    case 4064: return fwd_shape<TX, TR, 8, 4, 64>(a, s);
    case 8016: return fwd_shape<TX, TR, 1, 8, 16>(a, s);
    case 16016: return fwd_shape<TX, TR, 1, 16, 16>(a, s);
    case 16032: return fwd_shape<TX, TR, 1, 16, 32>(a, s);
    case 16064: return fwd_shape<TX, TR, 1, 16, 64>(a, s);
    case 2256: return fwd_shape<TX, TR, 8, 2, 256>(a, s);
    case 4256: return fwd_shape<TX, TR, 8, 4, 256>(a, s);
    case 8256: return fwd_shape<TX, TR, 8, 8, 256>(a, s);
    case 16256: return fwd_shape<TX, TR, 1, 16, 256>(a, s);
    case 32256: return fwd_shape<TX, TR, 1, 32, 256>(a, s);
    default: break;
  }
  return by_rows(a, 1, [&](const Args& b, dim3 grid) {
    if (b.scale == nullptr) hipLaunchKernelGGL((fwd_long_kernel<TX, TR, 0>), grid, dim3(kBlock), 0, s, b);
    else if (b.group == 0) hipLaunchKernelGGL((fwd_long_kernel<TX, TR, 1>), grid, dim3(kBlock), 0, s, b);
    else hipLaunchKernelGGL((fwd_long_kernel<TX, TR, 2>), grid, dim3(kBlock), 0, s, b);
  });
}

template <typename TX, typename TR, int V, int P, int TEAM>
void bwd_shape(const Args& a, hipStream_t s) {
  hipLaunchKernelGGL((bwd_kernel<TX, TR, V, P, TEAM>), dim3(a.parts), dim3(kBlock), 0, s, a);
}

template <typename TX, typename TR>
int bwd_typed(const Args& a, bool wide, hipStream_t s) {
  const Shape sh = shape_of(a.D, wide);
  switch (sh.p * 1000 + sh.team) {
    case 1008: bwd_shape<TX, TR, 8, 1, 8>(a, s); break;
    case 1016: bwd_shape<TX, TR, 8, 1, 16>(a, s); break;
    case 2016: bwd_shape<TX, TR, 8, 2, 16>(a, s); break;
    case 4016: sh.v == 8 ? bwd_shape<TX, TR, 8, 4, 16>(a, s) : bwd_shape<TX, TR, 1, 4, 16>(a, s); break;
    case 4032: bwd_shape<TX, TR, 8, 4, 32>(a, s); break;
    case 4064: bwd_shape<TX, TR, 8, 4, 64>(a, s); break;
    case 8016: bwd_shape<TX, TR, 1, 8, 16>(a, s); break;
    case 16016: bwd_shape<TX, TR, 1, 16, 16>(a, s); break;
    case 16032: bwd_shape<TX, TR, 1, 16, 32>(a, s); break;
    case 16064: bwd_shape<TX, TR, 1, 16, 64>(a, s); break;
    case 2256: bwd_shape<TX, TR, 8, 2, 256>(a, s); break;
    case 4256: bwd_shape<TX, TR, 8, 4, 256>(a, s); break;
    case 8256: bwd_shape<TX, TR, 8, 8, 256>(a, s); break;
    case 16256: bwd_shape<TX, TR, 1, 16, 256>(a, s); break;
    case 32256: bwd_shape<TX, TR, 1, 32, 256>(a, s); break;
    default:
      by_rows(a, 1, [&](const Args& b, dim3 grid) {
        hipLaunchKernelGGL((bwd_long_kernel<TX, TR>), grid, dim3(kBlock), 0, s, b);
      });
      hipLaunchKernelGGL((dw_cols_kernel<TX, TR>), dim3((a.D + kBlock - 1) / kBlock, a.parts), dim3(kBlock), 0, s, a);
  }
  hipLaunchKernelGGL((dw_sum_kernel<TX>), dim3((a.D + 63) / 64), dim3(1024), 0, s, a);
  return (int)hipGetLastError();
}

template <typename F>
int by_type(int xt, int rt, F f) {
  const bool wide_r = rt == GDN_DTYPE_F32;
  if (xt == GDN_DTYPE_F32) return f.template operator()<float, float>();
  if (xt == GDN_DTYPE_F16) return wide_r ? f.template operator()<f16, float>() : f.template operator()<f16, f16>();
  return wide_r ? f.template operator()<bf16_t, float>() : f.template operator()<bf16_t, bf16_t>();
}
struct Fwd {
  const Args& a;
  bool wide;
  hipStream_t s;
  template <typename TX, typename TR>
  int operator()() {
    return fwd_typed<TX, TR>(a, wide, s);
  }
};
struct Bwd {
  const Args& a;
  bool wide;
  hipStream_t s;
  template <typename TX, typename TR>
  int operator()() {
    return bwd_typed<TX, TR>(a, wide, s);
  }
};

int check(const GdnNormParams& P) {
  // (columns are counted in 32 bits, a workgroup's past the last)
  if (P.n_outer < 0 || P.n_inner < 0 || P.D <= 0 || P.D > 0x7fffffff - 1024 ||
      (int64_t)P.n_outer * P.n_inner > 0x3fffffffLL)
    return GDN_ERR_BAD_SHAPE;
  if (!scan_dtype_ok(P.x_dtype) || !(P.r_dtype == P.x_dtype || P.r_dtype == GDN_DTYPE_F32) ||
      !(P.w_dtype == P.x_dtype || P.w_dtype == GDN_DTYPE_F32))
    return GDN_ERR_BAD_DTYPE;
  return GDN_OK;
}

// The gradient's too: dw's sum takes 1024 threads for 64 columns.
int check_bwd(const GdnNormParams& P) {
  const int st = check(P);
  return st == GDN_OK && !grid_fits((P.D + 63) / 64, 1024) ? GDN_ERR_BAD_SHAPE : st;
}

// Whether 8 columns at a time fit these rows: 16-byte aligned (8 for e4m3).
bool rows_ok(const void* p, const int64_t* s, int eb) {
  const int al = eb == 1 ? 8 : 16;
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % al == 0 && (s[0] * eb) % al == 0 && (s[1] * eb) % al == 0);
}

int parts_of(int64_t rows, int D, bool wide) {
  const Shape sh = shape_of(D, wide);
  const int64_t per = sh.p > 0 ? kBlock / sh.team : 1;
  return (int)std::min<int64_t>(std::max<int64_t>(1, (rows + per - 1) / per), kMaxPartials);
}

int64_t up256(int64_t n) { return (n + 255) & ~(int64_t)255; }

void copy2(int64_t* d, const int64_t* s) {
  d[0] = s[0];
  d[1] = s[1];
}

}  // namespace norm
}  // namespace gdn

using namespace gdn;
using namespace gdn::norm;

extern "C" {

int gdn_norm_launch(const GdnNormParams* prm, void* stream) {
  if (prm == nullptr) return GDN_ERR_NULL_POINTER;
  const GdnNormParams& P = *prm;
  const int st = check(P);
  if (st != GDN_OK) return st;
  if (P.group != 0 && (P.group != 128 || P.scale == nullptr || P.D % 128 != 0)) return GDN_ERR_UNSUPPORTED;
  const int64_t rows = (int64_t)P.n_outer * P.n_inner;
  if (rows == 0) return GDN_OK;
  if (P.x == nullptr || P.w == nullptr || P.y == nullptr || (P.res != nullptr && P.r_out == nullptr))
    return GDN_ERR_NULL_POINTER;
  if (P.res == nullptr && P.r_dtype != P.x_dtype) return GDN_ERR_BAD_DTYPE;
  Args a = {};
  a.x = P.x;
  a.res = P.res;
  a.w = P.w;
  a.y = P.y;
  a.r_out = P.r_out;
  a.scale = P.scale;
  copy2(a.xs, P.x_stride);
  copy2(a.ress, P.res_stride);
  copy2(a.ys, P.y_stride);
  copy2(a.ros, P.r_out_stride);
  a.rows = (uint32_t)rows;
  a.n_inner = (uint32_t)P.n_inner;
  a.D = P.D;
  a.group = P.group;
  a.eps = P.eps;
  a.w_f32 = P.w_dtype == GDN_DTYPE_F32;
  const int eb = dtype_bytes(P.x_dtype), rb = dtype_bytes(P.r_dtype), wb = dtype_bytes(P.w_dtype);
  const int64_t dense[2] = {0, 0};
  const bool wide = P.D % 8 == 0 && rows_ok(P.x, P.x_stride, eb) && rows_ok(P.res, P.res_stride, rb) &&
                    rows_ok(P.res != nullptr ? P.r_out : nullptr, P.r_out_stride, rb) && rows_ok(P.w, dense, wb) &&
                    rows_ok(P.y, P.y_stride, P.scale != nullptr ? 1 : eb);
  return by_type(P.x_dtype, P.r_dtype, Fwd{a, wide, static_cast<hipStream_t>(stream)});
}

int64_t gdn_norm_bwd_workspace_size(const GdnNormParams* prm) {
  if (prm == nullptr || check_bwd(*prm) != GDN_OK) return -1;
  const int64_t rows = (int64_t)prm->n_outer * prm->n_inner;
  // partial rows of dw, and a float a row for rows that do not fit registers
  const int parts = std::max(parts_of(rows, prm->D, true), parts_of(rows, prm->D, false));
  return up256((int64_t)parts * prm->D * 4) + up256(rows * 4);
}

int gdn_norm_bwd_launch(const GdnNormParams* prm, void* stream) {
  if (prm == nullptr) return GDN_ERR_NULL_POINTER;
  const GdnNormParams& P = *prm;
  const int st = check_bwd(P);
  if (st != GDN_OK) return st;
  const int64_t rows = (int64_t)P.n_outer * P.n_inner;
  if (P.dw == nullptr || P.w == nullptr || (rows > 0 && (P.r == nullptr || P.dy == nullptr || P.dr == nullptr)))
    return GDN_ERR_NULL_POINTER;
  if (P.workspace == nullptr || P.workspace_bytes < gdn_norm_bwd_workspace_size(prm) ||
      reinterpret_cast<uintptr_t>(P.workspace) % 256 != 0)
    return GDN_ERR_WORKSPACE;
  Args a = {};
  a.w = P.w;
  a.r = P.r;
  a.dy = P.dy;
  a.dr_in = P.dr_in;
  a.dr = P.dr;
  a.dx = P.dx;
  a.dw = P.dw;
  copy2(a.rs, P.r_stride);
  copy2(a.dys, P.dy_stride);
  copy2(a.dris, P.dr_in_stride);
  copy2(a.drs, P.dr_stride);
  copy2(a.dxs, P.dx_stride);
  a.rows = (uint32_t)rows;
  a.n_inner = (uint32_t)std::max(1, P.n_inner);
  a.D = P.D;
  a.eps = P.eps;
  a.w_f32 = P.w_dtype == GDN_DTYPE_F32;
  const int eb = dtype_bytes(P.x_dtype), rb = dtype_bytes(P.r_dtype), wb = dtype_bytes(P.w_dtype);
  const int64_t dense[2] = {0, 0};
  const bool wide = P.D % 8 == 0 && rows_ok(P.r, P.r_stride, rb) && rows_ok(P.dy, P.dy_stride, eb) &&
                    rows_ok(P.dr_in, P.dr_in_stride, rb) && rows_ok(P.dr, P.dr_stride, rb) &&
                    rows_ok(P.dx, P.dx_stride, eb) && rows_ok(P.w, dense, wb);
  a.parts = parts_of(rows, P.D, wide);
  const int64_t most = std::max(parts_of(rows, P.D, true), parts_of(rows, P.D, false));
  a.part = static_cast<float*>(P.workspace);
  a.rstd = reinterpret_cast<float*>(static_cast<char*>(P.workspace) + up256(most * P.D * 4));
  return by_type(P.x_dtype, P.r_dtype, Bwd{a, wide, static_cast<hipStream_t>(stream)});
}

}  // extern "C"
