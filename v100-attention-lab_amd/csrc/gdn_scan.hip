// Elementwise gated linear recurrence and its gradient:
//     h_t = e^{g_t} h_{t-1} + x_t,  y_t = h_t
//     D_t = e^{g_t} dh_t,  dh_t = dy_t + D_{t+1},  dx_t = dh_t,
//     dg_t = dh_t e^{g_t} h_{t-1},  dh0 = D_1   (D_{T+1} = dfinal)
//
// Rows s..t together are h_t = e^G h_{s-1} + H with G the sum of their g, so a
// chunk of rows is one pair (G, H) per channel.  A gate near 1 enters as
// e^g - 1 (Decay below): its rounding does not add up over the rows that a
// state lives through.  A call of more than one chunk runs
//   agg    the pair of every chunk (forward from x, backward from dy),
//   carry  the state before every chunk, from the pairs of those before it,
//   main   every chunk from its state: rows in order, so that a row's value
//          comes from its own sequence of products and sums.
// A workgroup is kWaves waves on one chunk and 64 V channels; wave w holds R
// consecutive rows in registers and the waves exchange their pairs in LDS.
// Every sum has a fixed order.
//
// Bound by memory: x, g read and y written once, and the pairs' pass reads x
// and g once more, from the 256 MB cache where they fit.

#include <algorithm>

#include "gdn_row_io.h"

namespace gdn {
namespace scan {

using namespace rowio;

constexpr int kWaves = 16;
constexpr int kRows = 8;                   // rows a wave
constexpr int kChunk = kWaves * kRows;     // rows a workgroup
constexpr int kThreads = 64 * kWaves;

struct Args {
  const void* x;
  const void* g;
  const void* dy;
  void* y;
  void* dx;
  void* dg;
  const float* h0;
  const float* dfinal;
  float* fs;
  float* dh0;
  float* states;    // state before each chunk
  float* rstates;   // backward: D after each chunk
  float2* agg;      // pairs of the chunks
  const int64_t* cu;
  int64_t xs[2], gs[2], ys[2], dys[2], dxs[2], dgs[2];
  int64_t h0s, dfs;
  int T, D, N, nch, nblk;   // nch: chunks of a dense sequence; nblk: channel blocks
  uint32_t slots;
};

struct Job {
  int seq, chunk, len;   // rows of the sequence; chunk < 0: nothing to do
  int64_t row;           // first row of the sequence along t
  int b;                 // batch index
  int first;             // slot of the sequence's chunk 0
};

__device__ __forceinline__ int64_t clamp64(int64_t v, int64_t lo, int64_t hi) {
  return v < lo ? lo : (v > hi ? hi : v);
}

// Slot of chunk 0 of sequence i: floor(start / C) + i, which leaves every
// sequence room for ceil(len / C) chunks and at least one slot.
__device__ __forceinline__ int seq_slot(const Args& p, int i) {
  return (int)(clamp64(p.cu[i], 0, p.T) / kChunk) + i;
}

__device__ __forceinline__ Job seq_job(const Args& p, int seq) {
  Job j;
  j.seq = seq;
  j.chunk = 0;
  if (p.cu == nullptr) {
    j.b = seq;
    j.row = 0;
    j.len = p.T;
    j.first = seq * p.nch;
  } else {
    const int64_t s = clamp64(p.cu[seq], 0, p.T), e = clamp64(p.cu[seq + 1], s, p.T);
    j.b = 0;
    j.row = s;
    j.len = (int)(e - s);
    j.first = (int)(s / kChunk) + seq;
  }
  return j;
}

__device__ __forceinline__ Job slot_job(const Args& p, int slot) {
  int seq;
  if (p.cu == nullptr) {
    seq = slot / p.nch;
  } else {
    int lo = 0, hi = p.N;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (seq_slot(p, mid) <= slot) lo = mid; else hi = mid;
    }
    seq = lo;
  }
  Job j = seq_job(p, seq);
  j.chunk = slot - j.first;
  if (j.chunk * kChunk >= j.len && !(j.chunk == 0 && j.len == 0)) j.chunk = -1;
  return j;
}

// e^g in one float: for -1/8 < g <= 0 it is e^g - 1 (sign bit set, by its
// series, truncated below 2^-30), else e^g (sign bit clear).  e^g h is then
// h + (e^g - 1) h, exact to the rounding of the sum, where e^g itself would
// carry an error of 2^-25 a row.
__device__ __forceinline__ float decay(float g) {
  const float n = -g;
  float s = -1.f / 720.f;
  s = __builtin_fmaf(s, n, 1.f / 120.f);
  s = __builtin_fmaf(s, n, -1.f / 24.f);
  s = __builtin_fmaf(s, n, 1.f / 6.f);
  s = __builtin_fmaf(s, n, -0.5f);
  s = __builtin_fmaf(s, n, 1.f);
  return n >= 0.f && n < 0.125f ? -fabsf(n * s) : expf(g);
}

// e^g h + x from t = decay(g); an infinite sum stays what it is.
__device__ __forceinline__ float step(float t, float h, float x) {
  const bool near1 = __float_as_int(t) < 0;
  const float base = near1 ? h + x : x;
  const float r = __builtin_fmaf(t, h, base);
  return near1 && fabsf(base) == __builtin_inff() ? base : r;
}

// Exchange of the waves' pairs: decay(G) and H.
template <int V>
struct Exchange {
  float t[kWaves][64 * V], h[kWaves][64 * V];
};

template <typename TX, typename TG, int V>
__device__ __forceinline__ void load_rows(const TX* x, const TG* g, int64_t xs, int64_t gs, int n, bool ok,
                                          Pack<TX, V> (&xr)[kRows], Pack<TG, V> (&gr)[kRows]) {
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    xr[i].zero();
    gr[i].zero();
    if (i < n && ok) {
      xr[i].load(x + i * xs);
      gr[i].load(g + i * gs);
    }
  }
}

// The pair of every chunk.  REV: rows from the last to the first, D <- e^g (v + D).
template <typename TX, typename TG, int V, bool REV>
__global__ __launch_bounds__(kThreads) void agg_kernel(const Args p) {
  const uint32_t slot = blockIdx.x / p.nblk, blk = blockIdx.x % p.nblk;
  const Job j = slot_job(p, (int)slot);
  if (j.chunk < 0 || j.len == 0) return;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = (int)blk * 64 * V + lane * V;
  const bool ok = c < p.D;
  const int r0 = j.chunk * kChunk + w * kRows;
  const int n = min(max(j.len - r0, 0), kRows);
  const int64_t* vs = REV ? p.dys : p.xs;
  const TX* v = static_cast<const TX*>(REV ? p.dy : p.x) + j.b * vs[0] + (j.row + r0) * vs[1] + c;
  const TG* g = static_cast<const TG*>(p.g) + j.b * p.gs[0] + (j.row + r0) * p.gs[1] + c;
  Pack<TX, V> vr[kRows];
  Pack<TG, V> gr[kRows];
  load_rows<TX, TG, V>(v, g, vs[1], p.gs[1], n, ok, vr, gr);
  float G[V], H[V];
#pragma unroll
  for (int e = 0; e < V; ++e) G[e] = H[e] = 0.f;
#pragma unroll
  for (int s = 0; s < kRows; ++s) {
    const int i = REV ? kRows - 1 - s : s;
    if (i < n) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float gv = gr[i].get(e), t = decay(gv);
        H[e] = REV ? step(t, vr[i].get(e) + H[e], 0.f) : step(t, H[e], vr[i].get(e));
        G[e] += gv;
      }
    }
  }
  __shared__ float sh_g[kWaves][64 * V], sh_h[kWaves][64 * V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    sh_g[w][lane * V + e] = G[e];
    sh_h[w][lane * V + e] = H[e];
  }
  __syncthreads();
  const int ch = threadIdx.x;
  if (ch < 64 * V && (int)blk * 64 * V + ch < p.D) {
    float gs = 0.f, h = 0.f;
#pragma unroll
    for (int s = 0; s < kWaves; ++s) {
      const int i = REV ? kWaves - 1 - s : s;
      h = step(decay(sh_g[i][ch]), h, sh_h[i][ch]);
      gs += sh_g[i][ch];
    }
    p.agg[(int64_t)slot * p.D + (int)blk * 64 * V + ch] = make_float2(gs, h);
  }
}

// The state before every chunk of a sequence (REV: D after every chunk): wave
// w folds the pairs of its share of the chunks, the shares are joined in LDS,
// then every wave walks its share again.
template <bool REV>
__global__ __launch_bounds__(kThreads) void carry_kernel(const Args p) {
  const int nb = (p.D + 63) / 64;
  const int seq = blockIdx.x / nb, blk = blockIdx.x % nb;
  const Job j = seq_job(p, seq);
  const int n = (j.len + kChunk - 1) / kChunk;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = blk * 64 + lane;
  const bool ok = c < p.D;
  const int share = (n + kWaves - 1) / kWaves;
  const int k0 = min(w * share, n), k1 = min(k0 + share, n);
  // chunk of step k, in the order of the walk
  auto at = [&](int k) -> int64_t { return (int64_t)(j.first + (REV ? n - 1 - k : k)) * p.D + c; };
  float G = 0.f, H = 0.f;
  if (ok) {
#pragma unroll 8
    for (int k = k0; k < k1; ++k) {
      const float2 t = p.agg[at(k)];
      H = step(decay(t.x), H, t.y);
      G += t.x;
    }
  }
  __shared__ Exchange<1> sh;
  sh.t[w][lane] = decay(G);
  sh.h[w][lane] = H;
  __syncthreads();
  if (!ok) return;
  const float* init = REV ? p.dfinal : p.h0;
  const int64_t is = REV ? p.dfs : p.h0s;
  float h = init != nullptr ? init[seq * is + c] : 0.f;
  for (int i = 0; i < w; ++i) h = step(sh.t[i][lane], h, sh.h[i][lane]);
  float* out = REV ? p.rstates : p.states;
#pragma unroll 8
  for (int k = k0; k < k1; ++k) {
    const float2 t = p.agg[at(k)];
    out[at(k)] = h;
    h = step(decay(t.x), h, t.y);
  }
}

// y and the final state of every chunk; the state before it from `states`,
// or h0 where every sequence is one chunk (single).
template <typename TX, typename TG, int V>
__global__ __launch_bounds__(kThreads) void main_kernel(const Args p, bool single) {
  const uint32_t slot = blockIdx.x / p.nblk, blk = blockIdx.x % p.nblk;
  const Job j = slot_job(p, (int)slot);
  if (j.chunk < 0) return;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = (int)blk * 64 * V + lane * V;
  const bool ok = c < p.D;
  const int r0 = j.chunk * kChunk + w * kRows;
  const int n = min(max(j.len - r0, 0), kRows);
  const TX* x = static_cast<const TX*>(p.x) + j.b * p.xs[0] + (j.row + r0) * p.xs[1] + c;
  const TG* g = static_cast<const TG*>(p.g) + j.b * p.gs[0] + (j.row + r0) * p.gs[1] + c;
  TX* y = static_cast<TX*>(p.y) + j.b * p.ys[0] + (j.row + r0) * p.ys[1] + c;
  Pack<TX, V> xr[kRows];
  Pack<TG, V> gr[kRows];
  load_rows<TX, TG, V>(x, g, p.xs[1], p.gs[1], n, ok, xr, gr);
  float h[V];
#pragma unroll
  for (int e = 0; e < V; ++e) h[e] = 0.f;
  if (ok) {
    if (!single && j.len > 0) {
#pragma unroll
      for (int e = 0; e < V; ++e) h[e] = p.states[(int64_t)slot * p.D + c + e];
    } else if (p.h0 != nullptr) {
#pragma unroll
      for (int e = 0; e < V; ++e) h[e] = p.h0[j.seq * p.h0s + c + e];
    }
    if (single && p.states != nullptr && w == 0) {
#pragma unroll
      for (int e = 0; e < V; ++e) p.states[(int64_t)slot * p.D + c + e] = h[e];
    }
  }
  float a[kRows][V], G[V], H[V];
#pragma unroll
  for (int e = 0; e < V; ++e) G[e] = H[e] = 0.f;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      // rows past the end: g = 0 and x = 0 keep the state
      a[i][e] = decay(gr[i].get(e));
      H[e] = step(a[i][e], H[e], xr[i].get(e));
      G[e] += gr[i].get(e);
    }
  }
  __shared__ Exchange<V> sh;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    sh.t[w][lane * V + e] = decay(G[e]);
    sh.h[w][lane * V + e] = H[e];
  }
  __syncthreads();
  if (!ok) return;
  for (int i = 0; i < w; ++i) {
#pragma unroll
    for (int e = 0; e < V; ++e) h[e] = step(sh.t[i][lane * V + e], h[e], sh.h[i][lane * V + e]);
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    if (i < n) {
#pragma unroll
      for (int e = 0; e < V; ++e) h[e] = step(a[i][e], h[e], xr[i].get(e));
      Pack<TX, V> o;
      o.set(h);
      o.store(y + i * p.ys[1]);
    }
  }
  // the wave of the sequence's last row (of an empty sequence: the first wave)
  if ((n > 0 && r0 + n == j.len) || (j.len == 0 && w == 0)) {
#pragma unroll
    for (int e = 0; e < V; ++e) p.fs[(int64_t)j.seq * p.D + c + e] = h[e];
  }
}

// dx, dg of every chunk and dh0; the state before it from `states`, D after
// it from `rstates`, or h0 and dfinal where every sequence is one chunk.
template <typename TX, typename TG, int V>
__global__ __launch_bounds__(kThreads) void bwd_kernel(const Args p, bool single) {
  const uint32_t slot = blockIdx.x / p.nblk, blk = blockIdx.x % p.nblk;
  const Job j = slot_job(p, (int)slot);
  if (j.chunk < 0) return;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = (int)blk * 64 * V + lane * V;
  const bool ok = c < p.D;
  const int r0 = j.chunk * kChunk + w * kRows;
  const int n = min(max(j.len - r0, 0), kRows);
  const int64_t row = j.row + r0;
  const TX* x = static_cast<const TX*>(p.x) + j.b * p.xs[0] + row * p.xs[1] + c;
  const TG* g = static_cast<const TG*>(p.g) + j.b * p.gs[0] + row * p.gs[1] + c;
  const TX* dy = static_cast<const TX*>(p.dy) + j.b * p.dys[0] + row * p.dys[1] + c;
  TX* dx = static_cast<TX*>(p.dx) + j.b * p.dxs[0] + row * p.dxs[1] + c;
  TG* dg = static_cast<TG*>(p.dg) + j.b * p.dgs[0] + row * p.dgs[1] + c;
  Pack<TX, V> xr[kRows], dr[kRows];
  Pack<TG, V> gr[kRows];
  load_rows<TX, TG, V>(x, g, p.xs[1], p.gs[1], n, ok, xr, gr);
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    dr[i].zero();
    if (i < n && ok) dr[i].load(dy + i * p.dys[1]);
  }
  float h[V], d[V];
#pragma unroll
  for (int e = 0; e < V; ++e) h[e] = d[e] = 0.f;
  if (ok) {
    const bool many = !single && j.len > 0;
    if (many) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        h[e] = p.states[(int64_t)slot * p.D + c + e];
        d[e] = p.rstates[(int64_t)slot * p.D + c + e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (p.h0 != nullptr) h[e] = p.h0[j.seq * p.h0s + c + e];
        if (p.dfinal != nullptr) d[e] = p.dfinal[j.seq * p.dfs + c + e];
      }
    }
  }
  float a[kRows][V], G[V], H[V], R[V];
#pragma unroll
  for (int e = 0; e < V; ++e) G[e] = H[e] = R[e] = 0.f;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      // rows past the end: g = 0 and x = 0 keep the state
      a[i][e] = decay(gr[i].get(e));
      H[e] = step(a[i][e], H[e], xr[i].get(e));
      G[e] += gr[i].get(e);
    }
  }
#pragma unroll
  for (int i = kRows - 1; i >= 0; --i) {
#pragma unroll
    for (int e = 0; e < V; ++e) R[e] = step(a[i][e], dr[i].get(e) + R[e], 0.f);
  }
  __shared__ Exchange<V> sh;
  __shared__ float sh_r[kWaves][64 * V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    sh.t[w][lane * V + e] = decay(G[e]);
    sh.h[w][lane * V + e] = H[e];
    sh_r[w][lane * V + e] = R[e];
  }
  __syncthreads();
  if (!ok) return;
  for (int i = 0; i < w; ++i) {
#pragma unroll
    for (int e = 0; e < V; ++e) h[e] = step(sh.t[i][lane * V + e], h[e], sh.h[i][lane * V + e]);
  }
  for (int i = kWaves - 1; i > w; --i) {
#pragma unroll
    for (int e = 0; e < V; ++e) d[e] = step(sh.t[i][lane * V + e], d[e], sh_r[i][lane * V + e]);
  }
  float ah[kRows][V];   // e^{g_t} h_{t-1}
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      ah[i][e] = step(a[i][e], h[e], 0.f);
      h[e] = step(a[i][e], h[e], xr[i].get(e));
    }
  }
#pragma unroll
  for (int i = kRows - 1; i >= 0; --i) {
    if (i < n) {
      float dh[V], dgv[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        dh[e] = dr[i].get(e) + d[e];
        dgv[e] = dh[e] * ah[i][e];
        d[e] = step(a[i][e], dh[e], 0.f);
      }
      Pack<TX, V> ox;
      Pack<TG, V> og;
      ox.set(dh);
      og.set(dgv);
      ox.store(dx + i * p.dxs[1]);
      og.store(dg + i * p.dgs[1]);
    }
  }
  if (r0 == 0 && p.dh0 != nullptr) {
#pragma unroll
    for (int e = 0; e < V; ++e) p.dh0[(int64_t)j.seq * p.D + c + e] = d[e];
  }
}

// Sequences of at most kShort rows, dense: a thread walks its channels' rows
// in order, no exchange.
constexpr int kShort = 8;
template <typename TX, typename TG, int V>
__global__ __launch_bounds__(64) void short_kernel(const Args p) {
  const int b = blockIdx.x / p.nblk, blk = blockIdx.x % p.nblk;
  const int c = blk * 64 * V + threadIdx.x * V;
  if (c >= p.D) return;
  const TX* x = static_cast<const TX*>(p.x) + b * p.xs[0] + c;
  const TG* g = static_cast<const TG*>(p.g) + b * p.gs[0] + c;
  TX* y = static_cast<TX*>(p.y) + b * p.ys[0] + c;
  Pack<TX, V> xr[kShort];
  Pack<TG, V> gr[kShort];
  float h[V];
#pragma unroll
  for (int e = 0; e < V; ++e) h[e] = p.h0 != nullptr ? p.h0[b * p.h0s + c + e] : 0.f;
#pragma unroll
  for (int i = 0; i < kShort; ++i) {
    if (i < p.T) {
      xr[i].load(x + i * p.xs[1]);
      gr[i].load(g + i * p.gs[1]);
    }
  }
  if (p.states != nullptr) {
#pragma unroll
    for (int e = 0; e < V; ++e) p.states[(int64_t)b * p.D + c + e] = h[e];
  }
#pragma unroll
  for (int i = 0; i < kShort; ++i) {
    if (i < p.T) {
#pragma unroll
      for (int e = 0; e < V; ++e) h[e] = step(decay(gr[i].get(e)), h[e], xr[i].get(e));
      Pack<TX, V> o;
      o.set(h);
      o.store(y + i * p.ys[1]);
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) p.fs[(int64_t)b * p.D + c + e] = h[e];
}

int64_t slots_of(int64_t B, int64_t T, int64_t N, bool packed) {
  if (packed) return T / kChunk + N;
  return B * std::max<int64_t>(1, (T + kChunk - 1) / kChunk);
}

// Whether two channels at a time fit these rows.
bool pairs_ok(const void* p, const int64_t* s, int eb) {
  return reinterpret_cast<uintptr_t>(p) % (2 * eb) == 0 && s[0] % 2 == 0 && s[1] % 2 == 0;
}

template <typename TX, typename TG, int V>
int run_fwd(Args& a, bool single, hipStream_t s) {
  a.nblk = (a.D + 64 * V - 1) / (64 * V);
  if (a.cu == nullptr && a.T <= kShort) {
    hipLaunchKernelGGL((short_kernel<TX, TG, V>), dim3((uint32_t)a.N * a.nblk), dim3(64), 0, s, a);
    return (int)hipGetLastError();
  }
  const uint32_t grid = a.slots * a.nblk;
  if (!single) {
    hipLaunchKernelGGL((agg_kernel<TX, TG, V, false>), dim3(grid), dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL((carry_kernel<false>), dim3((uint32_t)a.N * ((a.D + 63) / 64)), dim3(kThreads), 0, s, a);
  }
  hipLaunchKernelGGL((main_kernel<TX, TG, V>), dim3(grid), dim3(kThreads), 0, s, a, single);
  return (int)hipGetLastError();
}

template <typename TX, typename TG, int V>
int run_bwd(Args& a, bool single, bool have_states, hipStream_t s) {
  a.nblk = (a.D + 64 * V - 1) / (64 * V);
  const uint32_t grid = a.slots * a.nblk;
  if (!single) {
    const dim3 cg((uint32_t)a.N * ((a.D + 63) / 64));
    if (!have_states) {
      hipLaunchKernelGGL((agg_kernel<TX, TG, V, false>), dim3(grid), dim3(kThreads), 0, s, a);
      hipLaunchKernelGGL((carry_kernel<false>), cg, dim3(kThreads), 0, s, a);
    }
    hipLaunchKernelGGL((agg_kernel<TX, TG, V, true>), dim3(grid), dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL((carry_kernel<true>), cg, dim3(kThreads), 0, s, a);
  }
  hipLaunchKernelGGL((bwd_kernel<TX, TG, V>), dim3(grid), dim3(kThreads), 0, s, a, single);
  return (int)hipGetLastError();
}

int check(const GdnScanParams& P) {
  if (P.B <= 0 || P.T < 0 || P.D <= 0 || P.N <= 0) return GDN_ERR_BAD_SHAPE;
  if (P.cu_seqlens == nullptr ? P.N != P.B : P.B != 1) return GDN_ERR_BAD_SHAPE;
  if (!scan_dtype_ok(P.x_dtype) || !(P.g_dtype == P.x_dtype || P.g_dtype == GDN_DTYPE_F32)) return GDN_ERR_BAD_DTYPE;
  // one workgroup a slot and 64 channels, and one a sequence and 64 channels
  const int64_t blocks = ((int64_t)P.D + 63) / 64;
  const int64_t slots = slots_of(P.B, P.T, P.N, P.cu_seqlens != nullptr);
  if (slots * blocks > 0x7fffffffLL) return GDN_ERR_BAD_SHAPE;
  return GDN_OK;
}

void common_args(const GdnScanParams& P, Args& a) {
  a.x = P.x;
  a.g = P.g;
  a.h0 = P.h0;
  a.cu = P.cu_seqlens;
  for (int d = 0; d < 2; ++d) {
    a.xs[d] = P.x_stride[d];
    a.gs[d] = P.g_stride[d];
  }
  a.h0s = P.h0_stride;
  a.T = P.T;
  a.D = P.D;
  a.N = P.N;
  a.nch = std::max(1, (P.T + kChunk - 1) / kChunk);
  a.slots = (uint32_t)slots_of(P.B, P.T, P.N, P.cu_seqlens != nullptr);
}

// Every sequence is one chunk for certain (packed offsets are not known here).
bool is_single(const GdnScanParams& P) { return P.T <= kChunk; }

template <int V, typename F>
int by_type(int xt, int gt, F f) {
  if (xt == GDN_DTYPE_F32) return f.template operator()<float, float, V>();
  if (xt == GDN_DTYPE_F16)
    return gt == GDN_DTYPE_F32 ? f.template operator()<f16, float, V>() : f.template operator()<f16, f16, V>();
  return gt == GDN_DTYPE_F32 ? f.template operator()<bf16_t, float, V>() : f.template operator()<bf16_t, bf16_t, V>();
}

struct Fwd {
  Args& a;
  bool single;
  hipStream_t s;
  template <typename TX, typename TG, int V>
  int operator()() {
    return run_fwd<TX, TG, V>(a, single, s);
  }
};
struct Bwd {
  Args& a;
  bool single, have;
  hipStream_t s;
  template <typename TX, typename TG, int V>
  int operator()() {
    return run_bwd<TX, TG, V>(a, single, have, s);
  }
};

int64_t up256(int64_t n) { return (n + 255) & ~(int64_t)255; }

}  // namespace scan
}  // namespace gdn

using namespace gdn;
using namespace gdn::scan;

extern "C" {

int gdn_scan_chunk(void) { return kChunk; }

int64_t gdn_scan_slots(int B, int T, int N, int packed) {
  if (B <= 0 || T < 0 || N <= 0) return -1;
  return slots_of(B, T, N, packed != 0);
}

int64_t gdn_scan_workspace_size(const GdnScanParams* prm) {
  if (prm == nullptr || check(*prm) != GDN_OK) return -1;
  if (is_single(*prm)) return 0;
  const int64_t n = slots_of(prm->B, prm->T, prm->N, prm->cu_seqlens != nullptr) * prm->D;
  return up256(8 * n) + (prm->states == nullptr ? up256(4 * n) : 0);
}

int64_t gdn_scan_bwd_workspace_size(const GdnScanParams* prm) {
  if (prm == nullptr || check(*prm) != GDN_OK) return -1;
  if (is_single(*prm)) return 0;
  const int64_t n = slots_of(prm->B, prm->T, prm->N, prm->cu_seqlens != nullptr) * prm->D;
  return up256(8 * n) + up256(4 * n) + (prm->states == nullptr ? up256(4 * n) : 0);
}

int gdn_scan_launch(const GdnScanParams* prm, void* stream) {
  if (prm == nullptr) return GDN_ERR_NULL_POINTER;
  const GdnScanParams& P = *prm;
  const int st = check(P);
  if (st != GDN_OK) return st;
  if (P.final_state == nullptr || (P.T > 0 && (P.x == nullptr || P.g == nullptr || P.y == nullptr)))
    return GDN_ERR_NULL_POINTER;
  const int64_t need = gdn_scan_workspace_size(prm);
  if (need > 0 && (P.workspace == nullptr || P.workspace_bytes < need ||
                   reinterpret_cast<uintptr_t>(P.workspace) % 256 != 0))
    return GDN_ERR_WORKSPACE;
  Args a = {};
  common_args(P, a);
  a.y = P.y;
  a.fs = P.final_state;
  a.states = P.states;
  for (int d = 0; d < 2; ++d) a.ys[d] = P.y_stride[d];
  if (need > 0) {
    a.agg = static_cast<float2*>(P.workspace);
    if (P.states == nullptr)
      a.states = reinterpret_cast<float*>(static_cast<char*>(P.workspace) + up256(8 * (int64_t)a.slots * a.D));
  }
  const int eb = dtype_bytes(P.x_dtype), gb = dtype_bytes(P.g_dtype);
  const bool two = P.D % 2 == 0 && pairs_ok(P.x, P.x_stride, eb) && pairs_ok(P.g, P.g_stride, gb) &&
                   pairs_ok(P.y, P.y_stride, eb);
  Fwd f{a, is_single(P), static_cast<hipStream_t>(stream)};
  return two ? by_type<2>(P.x_dtype, P.g_dtype, f) : by_type<1>(P.x_dtype, P.g_dtype, f);
}

int gdn_scan_bwd_launch(const GdnScanParams* prm, void* stream) {
  if (prm == nullptr) return GDN_ERR_NULL_POINTER;
  const GdnScanParams& P = *prm;
  const int st = check(P);
  if (st != GDN_OK) return st;
  if (P.T > 0 && (P.x == nullptr || P.g == nullptr || P.dy == nullptr || P.dx == nullptr || P.dg == nullptr))
    return GDN_ERR_NULL_POINTER;
  const int64_t need = gdn_scan_bwd_workspace_size(prm);
  if (need > 0 && (P.workspace == nullptr || P.workspace_bytes < need ||
                   reinterpret_cast<uintptr_t>(P.workspace) % 256 != 0))
    return GDN_ERR_WORKSPACE;
  Args a = {};
  common_args(P, a);
  a.dy = P.dy;
  a.dx = P.dx;
  a.dg = P.dg;
  a.dfinal = P.dfinal;
  a.dfs = P.dfinal_stride;
  a.dh0 = P.dh0;
  a.states = P.states;
  for (int d = 0; d < 2; ++d) {
    a.dys[d] = P.dy_stride[d];
    a.dxs[d] = P.dx_stride[d];
    a.dgs[d] = P.dg_stride[d];
  }
  if (need > 0) {
    char* ws = static_cast<char*>(P.workspace);
    const int64_t n = (int64_t)a.slots * a.D;
    a.agg = reinterpret_cast<float2*>(ws);
    a.rstates = reinterpret_cast<float*>(ws + up256(8 * n));
    if (P.states == nullptr) a.states = reinterpret_cast<float*>(ws + up256(8 * n) + up256(4 * n));
  }
  const int eb = dtype_bytes(P.x_dtype), gb = dtype_bytes(P.g_dtype);
  const bool two = P.D % 2 == 0 && pairs_ok(P.x, P.x_stride, eb) && pairs_ok(P.g, P.g_stride, gb) &&
                   pairs_ok(P.dy, P.dy_stride, eb) && pairs_ok(P.dx, P.dx_stride, eb) &&
                   pairs_ok(P.dg, P.dg_stride, gb);
  Bwd f{a, is_single(P), P.states != nullptr, static_cast<hipStream_t>(stream)};
  return two ? by_type<2>(P.x_dtype, P.g_dtype, f) : by_type<1>(P.x_dtype, P.g_dtype, f);
}

}  // extern "C"
