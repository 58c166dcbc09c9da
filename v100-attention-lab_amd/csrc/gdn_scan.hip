// Elementwise gated linear recurrence and its gradient:
//     h_t = e^{g_t} h_{t-1} + x_t,  y_t = h_t
//     D_t = e^{g_t} dh_t,  dh_t = dy_t + D_{t+1},  dx_t = dh_t,
//     dg_t = dh_t e^{g_t} h_{t-1},  dh0 = D_1   (D_{T+1} = dfinal)
//
// Rows s..t together are h_t = e^G h_{s-1} + H with G the sum of their g, so a
// chunk of rows is one pair (G, H) per channel.  A gate near 1 enters as
// e^g - 1 (decay() below): its rounding does not add up over the rows that a
// state lives through.
//
// A workgroup is kWaves waves on one chunk and 64 V channels; wave w holds
// kRows consecutive rows in registers and the waves exchange their pairs in
// LDS.  Sequences of one chunk need no more.  Else every workgroup leaves its
// chunk's pair in the workspace, takes the pairs of the chunks before it (in
// the backward, after it) and walks its rows from the state that they give: x,
// g and y pass through memory once.  Every 16th workgroup also leaves the pair
// of its 16 chunks, so that a chunk reads at most 46 pairs (15 before the first
// set, 31 behind the last) and one for each 16 chunks between.  All sums have a
// fixed order.
//
// Waiting: a channel block's chunks are dealt by its counter in the order of
// the walk, so whatever a workgroup waits for is left by workgroups that already
// run; each leaves its own pair before it waits for any, and what it leaves
// later depends on earlier ones alone.  A place in the workspace holds ~0 until its pair is there (one
// 8-byte store, seen by 8-byte loads past the caches), so no other order of
// memory is needed.  Chunk places that no sequence uses get a pair as well:
// offsets that make no sense give no meaningful rows, but every wait ends.
//
// Bound by memory, and by the walk's phases (rows in, pairs out and back, rows
// out), which the workgroups of a CU pass through side by side.  B4 T4096 D2048,
// bf16 with fp32 gates: forward 80 us (268 MB, 3.4 TB/s), backward from the
// forward's states 107 us (470 MB, 4.4 TB/s), a large copy 4.9 TB/s.  Chunks of
// 128 rows by 8 waves; of 64 by 4 waves (more pairs) forward and backward took 19 %
// more, of 256 by 16 waves (one workgroup a CU) 14 %.

#include <algorithm>

#include "gdn_row_io.h"

namespace gdn {
namespace scan {

using namespace rowio;

constexpr int kWaves = 8;
constexpr int kRows = 16;                  // rows a wave
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
  uint64_t* agg;    // pairs of the chunks in the order of the walk
  uint64_t* agg16;  // pairs of 16 chunks
  uint32_t* ticket;
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
  if (j.chunk < 0 || (j.chunk * kChunk >= j.len && !(j.chunk == 0 && j.len == 0))) j.chunk = -1;
  return j;
}

// e^g in one float: for -1/16 < g <= -0 it is e^g - 1 (sign bit set; four terms
// of its series, the next below 2^-26 of 1), else e^g (sign bit clear).  e^g h is
// then h + (e^g - 1) h, exact to the rounding of the sum, where e^g itself would
// carry an error of 2^-25 a row.  Below -1/16 a state lives for a few rows, and
// the hardware's 2^x of the rounded exponent is enough (2^-24 |g| beside the
// result's own unit).
__device__ __forceinline__ float decay(float g) {
  const float n = -g;
  float s = __builtin_fmaf(n, -1.f / 24.f, 1.f / 6.f);
  s = __builtin_fmaf(s, n, -0.5f);
  s = __builtin_fmaf(s, n, 1.f);
  const float e = __builtin_amdgcn_exp2f(g * 1.4426950408889634f);
  return __float_as_uint(n) < __float_as_uint(0.0625f) ? g * s : e;
}

// e^g h + x from t = decay(g).  Near 1 an infinite state stays what it is:
// (e^g - 1) times the largest finite number does not reach it.
__device__ __forceinline__ float step(float t, float h, float x) {
  const bool near1 = __float_as_int(t) < 0;
  const float top = 3.402823466e38f;
  return __builtin_fmaf(t, near1 ? __builtin_amdgcn_fmed3f(h, -top, top) : h, near1 ? h + x : x);
}

// e^G h + H for rows together, G the sum of their g.
struct Plain {
  __device__ __forceinline__ float operator()(float G, float h, float H) const { return step(decay(G), h, H); }
};
// The same where e^G leaves the range of floats and the rows' own gates do not:
// of a state 0 it stays 0, and an infinite one stays infinite (but under a gate of
// -inf, where it becomes NaN as 0 inf does for a row).
struct Careful {
  __device__ __forceinline__ float operator()(float G, float h, float H) const {
    const bool inf = fabsf(h) == __builtin_inff() && G > -__builtin_inff();
    return step(h == 0.f || inf ? 1.f : decay(G), h, H);
  }
};
// walk(join, h): a chain of joins from h on.  0 inf shows as NaN at its end: only
// then the chain is taken again, carefully (taken so at once, B4 T4096 D2048 takes
// 200 us forward and backward instead of 188).
template <int V, typename Walk>
__device__ __forceinline__ void chain(float (&h)[V], Walk walk) {
  float first[V];
  bool odd = false;
#pragma unroll
  for (int e = 0; e < V; ++e) first[e] = h[e];
  walk(Plain{}, h);
#pragma unroll
  for (int e = 0; e < V; ++e) odd |= h[e] != h[e];
  if (__builtin_expect(__any(odd), 0)) {
#pragma unroll
    for (int e = 0; e < V; ++e) h[e] = first[e];
    walk(Careful{}, h);
  }
}

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

// ---------------------------------------------------------------------------
// pairs in the workspace
// ---------------------------------------------------------------------------

constexpr uint64_t kAbsent = ~(uint64_t)0;
constexpr int kSet = 16;                   // chunks whose pairs are joined to one
constexpr int kLine = 32;                  // floats between two counters

__device__ __forceinline__ void leave_pair(uint64_t* at, float g, float h) {
  uint64_t v = ((uint64_t)__float_as_uint(h) << 32) | __float_as_uint(g);
  if (v == kAbsent) v = 0x7fc000007fc00000ull;   // a NaN of other bits
  __hip_atomic_store(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t look(const uint64_t* at) {
  return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float pair_g(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float pair_h(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }

// Every place of n pairs absent, and the counters at zero.
__global__ __launch_bounds__(256) void clear_kernel(uint64_t* agg, int64_t n, uint32_t* ticket, int nblk) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  for (int64_t k = i; k < nblk; k += (int64_t)gridDim.x * 256) ticket[k * kLine] = 0;
  for (int64_t k = i; k < n / 2; k += (int64_t)gridDim.x * 256)
    reinterpret_cast<ulonglong2*>(agg)[k] = make_ulonglong2(kAbsent, kAbsent);
}

// Channel block of a workgroup and its chunk's place in the order of the walk.
__device__ __forceinline__ uint32_t next_place(const Args& p, bool single, uint32_t& blk) {
  blk = blockIdx.x % p.nblk;
  if (single) return blockIdx.x / p.nblk;
  __shared__ uint32_t sh;
  if (threadIdx.x == 0) sh = atomicAdd(p.ticket + (int64_t)blk * kLine, 1u);
  __syncthreads();
  return sh;
}

// Scratch of the joins below.
template <int V>
struct Join {
  float g[kWaves][64 * V], h[kWaves][64 * V];
};

// Leaves the chunk's pair (from the waves' pairs in sh, in the order of the
// walk) and, at the end of a set, the set's.  u: the chunk's place.
template <int V, bool REV>
__device__ __forceinline__ void leave(const Args& p, const Join<V>& sh, uint32_t u, int c0) {
  const int ch = threadIdx.x, c = c0 + ch;
  if (ch >= 64 * V || c >= p.D) return;
  float g = 0.f, h[1] = {0.f};
#pragma unroll
  for (int i = 0; i < kWaves; ++i) g += sh.g[i][ch];
  chain<1>(h, [&](auto join, float (&h)[1]) {
#pragma unroll
    for (int s = 0; s < kWaves; ++s) {
      const int i = REV ? kWaves - 1 - s : s;
      h[0] = join(sh.g[i][ch], h[0], sh.h[i][ch]);
    }
  });
  leave_pair(p.agg + (int64_t)u * p.D + c, g, h[0]);
  if (u % kSet != kSet - 1) return;
  const uint64_t* first = p.agg + (int64_t)(u - (kSet - 1)) * p.D + c;
  constexpr int kBatch = 5;
  static_assert((kSet - 1) % kBatch == 0, "whole batches");
  float gs = 0.f, hs[1] = {0.f};
  chain<1>(hs, [&](auto join, float (&hs)[1]) {
    gs = 0.f;
#pragma unroll 1
    for (int k = 0; k < kSet - 1; k += kBatch) {
      uint64_t v[kBatch];
      bool all;
      do {
        all = true;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) v[i] = look(first + (int64_t)(k + i) * p.D);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) all &= v[i] != kAbsent;
      } while (!all);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        hs[0] = join(pair_g(v[i]), hs[0], pair_h(v[i]));
        gs += pair_g(v[i]);
      }
    }
    hs[0] = join(g, hs[0], h[0]);
  });
  leave_pair(p.agg16 + (int64_t)(u / kSet) * p.D + c, gs + g, hs[0]);
}

// The state h (of this lane's V channels) behind the places first .. u - 1, in
// order: single places up to a set's start, whole sets, single places again.
// Each wave takes a share of these pairs; the shares are joined in LDS.
template <int V, int BATCH>
__device__ __forceinline__ void carry(const Args& p, Join<V>& sh, uint32_t first, uint32_t u, int c, bool ok,
                                      float (&h)[V]) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int up = (int)(first + kSet - 1) / kSet * kSet;       // the first whole set's start
  const int head = min((int)u, up) - (int)first;
  // (the last 16 to 31 singly: by then a set before them has had its time)
  const int end = max(((int)u / kSet - 1) * kSet, up);
  const int sets = max((end - up) / kSet, 0);
  const int tail = max((int)u - end, 0);
  const int n = max(head, 0) + sets + tail;
  const int share = (n + kWaves - 1) / kWaves, k0 = min(w * share, n), k1 = min(k0 + share, n);
  auto at = [&](int k) -> const uint64_t* {
    if (k < head) return p.agg + ((int64_t)first + k) * p.D + c;
    if (k < head + sets) return p.agg16 + ((int64_t)(up / kSet) + (k - head)) * p.D + c;
    return p.agg + ((int64_t)(u - tail) + (k - head - sets)) * p.D + c;
  };
  float G[V], H[V];
#pragma unroll
  for (int e = 0; e < V; ++e) G[e] = H[e] = 0.f;
  if (ok) {
#pragma unroll 1
    for (int k = k0; k < k1; k += BATCH) {
      uint64_t v[BATCH][V];
      bool all;
      do {
        all = true;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          const uint64_t* a = at(min(k + i, k1 - 1));
#pragma unroll
          for (int e = 0; e < V; ++e) v[i][e] = look(a + e);
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
#pragma unroll
          for (int e = 0; e < V; ++e) all &= v[i][e] != kAbsent;
      } while (!all);
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        if (k + i < k1) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            H[e] = Plain{}(pair_g(v[i][e]), H[e], pair_h(v[i][e]));
            G[e] += pair_g(v[i][e]);
          }
        }
      }
    }
    // (see chain; here a loop of its own over pairs that are all there: as a chain
    // the loop above made the fp32 backward of 50001 rows of 640 143 us, not 135)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (__builtin_expect(H[e] != H[e], 0)) {
        H[e] = 0.f;
#pragma unroll 1
        for (int k = k0; k < k1; ++k) {
          const uint64_t v = look(at(k) + e);
          H[e] = Careful{}(pair_g(v), H[e], pair_h(v));
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    sh.g[w][lane * V + e] = G[e];
    sh.h[w][lane * V + e] = H[e];
  }
  __syncthreads();
  chain<V>(h, [&](auto join, float (&h)[V]) {
    for (int i = 0; i < kWaves && i * share < n; ++i) {
#pragma unroll
      for (int e = 0; e < V; ++e) h[e] = join(sh.g[i][lane * V + e], h[e], sh.h[i][lane * V + e]);
    }
  });
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------

// 16-bit gates: e^g is formed again in the second walk instead of held, which
// leaves room for 6 waves a SIMD (B4 T4096 D2048 bf16: 69 us, held with 4 waves 9 %
// more).  32-bit gates hold it: 6 waves would spill (19 % more than the 80 us).
template <typename TX, typename TG>
constexpr bool kMore = sizeof(TX) == 2 && sizeof(TG) == 2;

// y, the final states and (not nullptr) the states at the chunks' starts.
// ONLY_STATES: those alone.  single: every sequence is one chunk.
template <typename TX, typename TG, int V, bool ONLY_STATES>
__global__ __launch_bounds__(kThreads, (kMore<TX, TG> ? 6 : 4)) void fwd_kernel(const Args p, bool single) {
  uint32_t blk;
  const uint32_t slot = next_place(p, single, blk);
  const Job j = slot_job(p, (int)slot);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = (int)blk * 64 * V + lane * V;
  const bool ok = c < p.D;
  const int r0 = max(j.chunk, 0) * kChunk + w * kRows;
  const int n = j.chunk < 0 ? 0 : min(max(j.len - r0, 0), kRows);
  const TX* x = static_cast<const TX*>(p.x) + j.b * p.xs[0] + (j.row + r0) * p.xs[1] + c;
  const TG* g = static_cast<const TG*>(p.g) + j.b * p.gs[0] + (j.row + r0) * p.gs[1] + c;
  Pack<TX, V> xr[kRows];
  Pack<TG, V> gr[kRows];
  load_rows<TX, TG, V>(x, g, p.xs[1], p.gs[1], n, ok, xr, gr);
  float h[V];
#pragma unroll
  for (int e = 0; e < V; ++e) h[e] = ok && p.h0 != nullptr ? p.h0[j.seq * p.h0s + c + e] : 0.f;
  constexpr bool kHold = sizeof(TG) == 4;
  float a[kHold ? kRows : 1][V], G[V], H[V];
#pragma unroll
  for (int e = 0; e < V; ++e) G[e] = H[e] = 0.f;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      // rows past the end: g = 0 and x = 0 keep the state
      const float t = decay(gr[i].get(e));
      if constexpr (kHold) a[i][e] = t;
      H[e] = step(t, H[e], xr[i].get(e));
      G[e] += gr[i].get(e);
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    xr[i].repack();
    if constexpr (!kHold) gr[i].repack();
  }
  __shared__ Join<V> waves, shares;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    waves.g[w][lane * V + e] = G[e];
    waves.h[w][lane * V + e] = H[e];
  }
  __syncthreads();
  if (!single) {
    leave<V, false>(p, waves, slot, (int)blk * 64 * V);
    if (j.chunk < 0) return;
    carry<V, kMore<TX, TG> ? 2 : 4>(p, shares, (uint32_t)j.first, slot, c, ok, h);
  }
  if (j.chunk < 0 || !ok) return;
  if (p.states != nullptr && w == 0) {
#pragma unroll
    for (int e = 0; e < V; ++e) p.states[(int64_t)slot * p.D + c + e] = h[e];
  }
  if constexpr (ONLY_STATES) return;
  TX* y = static_cast<TX*>(p.y) + j.b * p.ys[0] + (j.row + r0) * p.ys[1] + c;
  chain<V>(h, [&](auto join, float (&h)[V]) {
    for (int i = 0; i < w; ++i) {
#pragma unroll
      for (int e = 0; e < V; ++e) h[e] = join(waves.g[i][lane * V + e], h[e], waves.h[i][lane * V + e]);
    }
  });
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    if (i < n) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float t;
        if constexpr (kHold) t = a[i][e];
        else t = decay(gr[i].get(e));
        h[e] = step(t, h[e], xr[i].get(e));
      }
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

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------

// dx, dg and dh0, the states at the chunks' starts from `states` (single: h0).
template <typename TX, typename TG, int V>
__global__ __launch_bounds__(kThreads, 4) void bwd_kernel(const Args p, bool single) {
  uint32_t blk;
  const uint32_t u = next_place(p, single, blk), slot = p.slots - 1 - u;
  const Job j = slot_job(p, (int)slot);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = (int)blk * 64 * V + lane * V;
  const bool ok = c < p.D;
  const int r0 = max(j.chunk, 0) * kChunk + w * kRows;
  const int n = j.chunk < 0 ? 0 : min(max(j.len - r0, 0), kRows);
  const int64_t row = j.row + r0;
  const TX* x = static_cast<const TX*>(p.x) + j.b * p.xs[0] + row * p.xs[1] + c;
  const TG* g = static_cast<const TG*>(p.g) + j.b * p.gs[0] + row * p.gs[1] + c;
  const TX* dy = static_cast<const TX*>(p.dy) + j.b * p.dys[0] + row * p.dys[1] + c;
  Pack<TX, V> xr[kRows], dr[kRows];
  Pack<TG, V> gr[kRows];
  load_rows<TX, TG, V>(x, g, p.xs[1], p.gs[1], n, ok, xr, gr);
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    dr[i].zero();
    if (i < n && ok) dr[i].load(dy + i * p.dys[1]);
  }
  float h[V], d[V];
  auto start = [&](int e) {
    if (!ok || j.chunk < 0) return 0.f;
    if (!single && j.len > 0) return p.states[(int64_t)slot * p.D + c + e];
    return p.h0 != nullptr ? p.h0[j.seq * p.h0s + c + e] : 0.f;
  };
#pragma unroll
  for (int e = 0; e < V; ++e) {
    h[e] = start(e);
    d[e] = ok && p.dfinal != nullptr ? p.dfinal[j.seq * p.dfs + c + e] : 0.f;
  }
  float a[kRows][V], G[V], H[V], R[V];
#pragma unroll
  for (int e = 0; e < V; ++e) G[e] = H[e] = R[e] = 0.f;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
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
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    xr[i].repack();
    dr[i].repack();
  }
  __shared__ Join<V> waves, shares;          // waves: G and the pairs of the backward walk
  __shared__ float sh_h[kWaves][64 * V];     // H of the forward walk
#pragma unroll
  for (int e = 0; e < V; ++e) {
    waves.g[w][lane * V + e] = G[e];
    waves.h[w][lane * V + e] = R[e];
    sh_h[w][lane * V + e] = H[e];
  }
  __syncthreads();
  if (!single) {
    leave<V, true>(p, waves, u, (int)blk * 64 * V);
    if (j.chunk < 0) return;
    const uint32_t last = j.first + (uint32_t)max((j.len + kChunk - 1) / kChunk, 1) - 1;
    carry<V, 4>(p, shares, p.slots - 1 - last, u, c, ok, d);
  }
  if (j.chunk < 0 || !ok) return;
  TX* dx = static_cast<TX*>(p.dx) + j.b * p.dxs[0] + row * p.dxs[1] + c;
  TG* dg = static_cast<TG*>(p.dg) + j.b * p.dgs[0] + row * p.dgs[1] + c;
  chain<V>(h, [&](auto join, float (&h)[V]) {
    for (int i = 0; i < w; ++i) {
#pragma unroll
      for (int e = 0; e < V; ++e) h[e] = join(waves.g[i][lane * V + e], h[e], sh_h[i][lane * V + e]);
    }
  });
  chain<V>(d, [&](auto join, float (&d)[V]) {
    for (int i = kWaves - 1; i > w; --i) {
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = join(waves.g[i][lane * V + e], d[e], waves.h[i][lane * V + e]);
    }
  });
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
// in order, no exchange.  16 single rows of 2048 channels: 2.8 us, of which most
// is the launch.
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

// The pairs' places before a walk.
void clear(const Args& a, hipStream_t s) {
  // agg, then agg16 (an even number of pairs in all, see pair_bytes)
  const int64_t n = ((int64_t)a.slots * a.D + 1) / 2 * 2 + (((int64_t)a.slots / kSet) * a.D + 1) / 2 * 2;
  const uint32_t grid = (uint32_t)std::min<int64_t>((n / 2 + 255) / 256, 2048);
  hipLaunchKernelGGL(clear_kernel, dim3(grid), dim3(256), 0, s, a.agg, n, a.ticket, a.nblk);
}

template <typename TX, typename TG, int V>
int run_fwd(Args& a, bool single, hipStream_t s) {
  a.nblk = (a.D + 64 * V - 1) / (64 * V);
  if (a.cu == nullptr && a.T <= kShort) {
    if (!grid_fits((int64_t)a.N * a.nblk, 64)) return GDN_ERR_BAD_SHAPE;
    hipLaunchKernelGGL((short_kernel<TX, TG, V>), dim3((uint32_t)a.N * a.nblk), dim3(64), 0, s, a);
    return (int)hipGetLastError();
  }
  if (!grid_fits((int64_t)a.slots * a.nblk, kThreads)) return GDN_ERR_BAD_SHAPE;
  if (!single) clear(a, s);
  hipLaunchKernelGGL((fwd_kernel<TX, TG, V, false>), dim3(a.slots * a.nblk), dim3(kThreads), 0, s, a, single);
  return (int)hipGetLastError();
}

template <typename TX, typename TG, int V>
int run_bwd(Args& a, bool single, bool have_states, hipStream_t s) {
  a.nblk = (a.D + 64 * V - 1) / (64 * V);
  if (!grid_fits((int64_t)a.slots * a.nblk, kThreads)) return GDN_ERR_BAD_SHAPE;
  const dim3 grid(a.slots * a.nblk);
  if (!single) {
    clear(a, s);
    if (!have_states) {
      hipLaunchKernelGGL((fwd_kernel<TX, TG, V, true>), grid, dim3(kThreads), 0, s, a, single);
      clear(a, s);
    }
  }
  hipLaunchKernelGGL((bwd_kernel<TX, TG, V>), grid, dim3(kThreads), 0, s, a, single);
  return (int)hipGetLastError();
}

int check(const GdnScanParams& P) {
  // (rows and channels are counted in 32 bits, a workgroup's past the last)
  if (P.B <= 0 || P.T < 0 || P.D <= 0 || P.N <= 0 || P.T > 0x7fffffff - 1024 || P.D > 0x7fffffff - 1024)
    return GDN_ERR_BAD_SHAPE;
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
    return run_bwd<TX, TG, std::is_same<TX, float>::value ? 1 : V>(a, single, have, s);
  }
};

int64_t up256(int64_t n) { return (n + 255) & ~(int64_t)255; }

// Workspace of a walk: the pairs (of chunks, then of sets, each an even number
// of places), the counters (of channel blocks of 64 or 128).
int64_t pair_bytes(int64_t slots, int64_t D) {
  return ((slots * D + 1) / 2 * 2 + (slots / kSet * D + 1) / 2 * 2) * 8;
}
int64_t walk_bytes(int64_t slots, int64_t D) { return up256(pair_bytes(slots, D) + (D + 63) / 64 * kLine * 4); }
void walk_space(Args& a, void* ws) {
  a.agg = static_cast<uint64_t*>(ws);
  a.agg16 = a.agg + ((int64_t)a.slots * a.D + 1) / 2 * 2;
  a.ticket = reinterpret_cast<uint32_t*>(static_cast<char*>(ws) + pair_bytes(a.slots, a.D));
}

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
  return walk_bytes(slots_of(prm->B, prm->T, prm->N, prm->cu_seqlens != nullptr), prm->D);
}

int64_t gdn_scan_bwd_workspace_size(const GdnScanParams* prm) {
  if (prm == nullptr || check(*prm) != GDN_OK) return -1;
  if (is_single(*prm)) return 0;
  const int64_t slots = slots_of(prm->B, prm->T, prm->N, prm->cu_seqlens != nullptr);
  return walk_bytes(slots, prm->D) + (prm->states == nullptr ? up256(4 * slots * prm->D) : 0);
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
  if (need > 0) walk_space(a, P.workspace);
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
    walk_space(a, P.workspace);
    if (P.states == nullptr)
      a.states = reinterpret_cast<float*>(static_cast<char*>(P.workspace) + walk_bytes(a.slots, a.D));
  }
  const int eb = dtype_bytes(P.x_dtype), gb = dtype_bytes(P.g_dtype);
  const bool two = P.D % 2 == 0 && pairs_ok(P.x, P.x_stride, eb) && pairs_ok(P.g, P.g_stride, gb) &&
                   pairs_ok(P.dy, P.dy_stride, eb) && pairs_ok(P.dx, P.dx_stride, eb) &&
                   pairs_ok(P.dg, P.dg_stride, gb);
  Bwd f{a, is_single(P), P.states != nullptr, static_cast<hipStream_t>(stream)};
  // fp32 rows of x, g and dy two channels wide do not fit the registers
  return two && P.x_dtype != GDN_DTYPE_F32 ? by_type<2>(P.x_dtype, P.g_dtype, f) : by_type<1>(P.x_dtype, P.g_dtype, f);
}

}  // extern "C"
