// Windowed attention of the newest tokens of each sequence over a cache.
//
// The G T query rows that share a key head (T tokens, G query heads) are the
// columns of the products, 32 at a time.  The visible key tiles of a sequence
// are dealt to `splits` workgroups and in each to its 4 waves; a wave brings
// its own tiles of 32 keys by LDS-DMA into two buffers and needs no barrier.
// The waves are joined in LDS; with more than one split the workgroups leave
// (m, l, O) in the workspace and a second kernel joins them, in order.
//
// Bound by reading the cache rows once (32 sequences, 4 key heads of 128, 4100
// visible keys, bf16: 51 us with the call, 5.3 TB/s), and for few sequences by the
// chain of one workgroup and the join (one sequence of the same: 6 to 8 us and
// 4 us for 8.4 MB).

#include <algorithm>

#include "gdn_attn.h"

namespace gdn {
namespace attn {

constexpr int kDN = 32;          // keys a tile
constexpr int kDWaves = 4;
constexpr int kMaxT = 16;
constexpr int kMaxSplits = 64;

struct DArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  const int32_t* lens;
  float* part;      // [units][splits][32][D + 2]
  int64_t qs[3], ks[3], vs[3], os[3];
  int B, T, S, Hk, G, tiles_r, splits, window, sinks;
  float scale_log2;
  uint32_t flip;
};

// Row (of 32) of a unit: query token, head, and whether it exists.
struct QRow {
  int t, h;
  bool ok;
  __device__ __forceinline__ QRow(const DArgs& a, int hk, int rt, int c) {
    const int r = rt * 32 + c;
    ok = r < a.G * a.T;
    const int rr = ok ? r : 0;
    t = rr / a.G;
    h = hk * a.G + rr % a.G;
  }
};

// Joins (m, l, O) pairs: factors of the two parts under the common maximum.
__device__ __forceinline__ float weight(float m, float top) {
  return m == -__builtin_inff() ? 0.f : exp2_fast(m - top);
}

template <typename T, int D>
__global__ __launch_bounds__(64 * kDWaves) void decode_kernel(const DArgs a) {
  using O = Ops<T>;
  using Vec = typename O::Vec;
  using TL = Tile<D>;
  constexpr uint32_t kTile = TL::bytes(kDN), kWave = 4 * kTile;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kDWaves * kWave];
  const int split = blockIdx.x % a.splits, unit = blockIdx.x / a.splits;
  const int rt = unit % a.tiles_r, bh = unit / a.tiles_r, hk = bh % a.Hk, b = bh / a.Hk;
  const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = __builtin_amdgcn_readfirstlane(max(0, min(a.lens[b], a.S)));
  const QRow qr(a, hk, rt, l32);
  const int p = n - a.T + qr.t;
  const int r0 = rt * 32, r1 = min(r0 + 32, a.G * a.T) - 1;
  const int p0 = n - a.T + r0 / a.G, p1 = n - a.T + r1 / a.G;

  Vec qf[D / 16];
  {
    const uint16_t* q = a.q + b * a.qs[0] + qr.t * a.qs[1] + qr.h * a.qs[2];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) qf[i] = signed_vec<T>(*reinterpret_cast<const uint4*>(q + 16 * i + 8 * half), a.flip);
  }
  // the tiles of any row; rows before the first key see none
  const KeyRange kr(max(p0, 0), p1, n, a.window, a.sinks, kDN);
  const int per = (kr.n + a.splits - 1) / a.splits;
  const int t0 = min(split * per, kr.n), t1 = min(t0 + per, kr.n);

  // a tile of 32 rows, 64 lanes a pass
  const uint16_t* kb = a.k + b * a.ks[0] + hk * a.ks[2];
  const uint16_t* vb = a.v + b * a.vs[0] + hk * a.vs[2];
  const uint32_t base = lds_addr(lds) + wv * kWave;
  auto fetch = [&](uint32_t at, const uint16_t* src, int64_t ld, int row0) {
    constexpr int kPasses = kDN * TL::kPieces / 64;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int e = i * 64 + lane, row = e / TL::kPieces, c = (e % TL::kPieces) ^ TL::swz(row);
      dma16(src + (int64_t)min(row0 + row, n - 1) * ld + 8 * c, at + i * TL::kGroupBytes);
    }
  };
  const TL tl(lane);
  Rows<T, D, 1> rows;
  if (t0 + wv < t1) {
    const int j = kr.tile(t0 + wv) * kDN;
    fetch(base, kb, a.ks[1], j);
    fetch(base + kTile, vb, a.vs[1], j);
  }
  for (int t = t0 + wv, k = 0; t < t1; t += kDWaves, ++k) {
    dma_wait();
    if (t + kDWaves < t1) {
      const uint32_t other = base + ((k + 1) & 1) * 2 * kTile;
      const int j = kr.tile(t + kDWaves) * kDN;
      fetch(other, kb, a.ks[1], j);
      fetch(other + kTile, vb, a.vs[1], j);
    }
    const uint32_t kt = base + (k & 1) * 2 * kTile;
    const Mask seen(p, kr.tile(t) * kDN, kDN, half, n, p0, p1, a.window, a.sinks);
    rows.template scores<1>(qf, tl, kt, seen, a.scale_log2);
    const uint32_t vt = kt + kTile;
    if (seen.any() && not_finite<T, kDN / TL::kGroup>(vt, lane)) {
      rows.template add_not_finite<1>(seen, tl, vt);
      make_finite<T, kDN / TL::kGroup>(vt, lane);
    }
    rows.template values<1>(tl, vt);
  }
  rows.l += swap_halves(rows.l);

  // the waves' parts, joined by all of them: wave w takes D / 4 columns of O
  __syncthreads();
  float* sm = reinterpret_cast<float*>(lds);                  // [4][32] m, [4][32] l, [4][D][32] O
  float* sl = sm + kDWaves * 32;
  float* so = sl + kDWaves * 32;
  static_assert((kDWaves * 32 * (D + 2)) * 4 <= (int)(kDWaves * kWave), "the parts fit the tiles' space");
  if (half == 0) {
    sm[wv * 32 + l32] = rows.m;
    sl[wv * 32 + l32] = rows.l;
  }
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) so[(wv * D + 32 * dt + acc_row(r, half)) * 32 + l32] = rows.acc[dt][r];
  __syncthreads();
  // thread: row c = tid / 8, D / 8 columns from 8 neighbouring threads
  const int c = threadIdx.x >> 3, d0 = (threadIdx.x & 7) * (D / 8);
  const QRow row(a, hk, rt, c);
  if (!row.ok) return;
  float top = sm[c];
#pragma unroll
  for (int w = 1; w < kDWaves; ++w) top = fmaxf(top, sm[w * 32 + c]);
  float l = 0.f, f[kDWaves];
#pragma unroll
  for (int w = 0; w < kDWaves; ++w) {
    f[w] = weight(sm[w * 32 + c], top);
    l += f[w] * sl[w * 32 + c];
  }
  float out[D / 8];
#pragma unroll
  for (int e = 0; e < D / 8; ++e) {
    out[e] = 0.f;
#pragma unroll
    for (int w = 0; w < kDWaves; ++w) out[e] += f[w] * so[(w * D + d0 + e) * 32 + c];
  }
  if (a.splits > 1) {
    float* part = a.part + ((int64_t)unit * a.splits + split) * 32 * (D + 2);
    if (d0 == 0) {
      part[c] = top;
      part[32 + c] = l;
    }
#pragma unroll
    for (int e = 0; e < D / 8; e += 4)
      *reinterpret_cast<float4*>(part + 64 + c * D + d0 + e) = make_float4(out[e], out[e + 1], out[e + 2], out[e + 3]);
    return;
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  uint16_t* o = a.o + b * a.os[0] + row.t * a.os[1] + row.h * a.os[2] + d0;
#pragma unroll
  for (int e = 0; e < D / 8; e += 2) *reinterpret_cast<uint32_t*>(o + e) = O::pack(out[e] * inv, out[e + 1] * inv);
}

// One workgroup a query row: every wave weighs the splits (one a lane), then
// groups of D / 4 threads add the splits g, g + groups, .. and the groups' sums
// are added in order.
constexpr int kJT = 256;
template <typename T, int D>
__global__ __launch_bounds__(kJT) void join_kernel(const DArgs a) {
  constexpr int L = D / 4, kGroups = kJT / L;
  const int rows = a.G * a.T, r = blockIdx.x % rows, bh = blockIdx.x / rows, hk = bh % a.Hk, b = bh / a.Hk;
  const int c = r % 32, unit = bh * a.tiles_r + r / 32;
  const float* part = a.part + (int64_t)unit * a.splits * 32 * (D + 2);
  const int64_t step = 32 * (D + 2);
  const int lane = threadIdx.x & 63, g = threadIdx.x / L, d = threadIdx.x % L;
  static_assert(kMaxSplits <= 64, "a split a lane");
  const float m = lane < a.splits ? part[lane * step + c] : -__builtin_inff();
  const float ls = lane < a.splits ? part[lane * step + 32 + c] : 0.f;
  float top = m;
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) top = fmaxf(top, __shfl_xor(top, s, 64));
  const float f = weight(m, top);
  float l = f * ls;
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) l += __shfl_xor(l, s, 64);
  // a split that saw no key (-1) is not read; one that saw only NaN has no maximum
  // either, but its sum is NaN, and what is not finite stays so at a weight of 0
  const float use = ls == 0.f ? -1.f : f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int k = 0; k < kMaxSplits / kGroups; ++k) {
    const int s = k * kGroups + g;
    const float fs = __shfl(use, s < a.splits ? s : 0, 64);
    if (s < a.splits && !(fs < 0.f)) {
      const float4 x = *reinterpret_cast<const float4*>(part + s * step + 64 + c * D + 4 * d);
      o.x += fs * x.x;
      o.y += fs * x.y;
      o.z += fs * x.z;
      o.w += fs * x.w;
    }
  }
  __shared__ float4 sums[kGroups][L];
  sums[g][d] = o;
  __syncthreads();
  if (g != 0) return;
#pragma unroll
  for (int k = 1; k < kGroups; ++k) {
    const float4 x = sums[k][d];
    o.x += x.x;
    o.y += x.y;
    o.z += x.z;
    o.w += x.w;
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  const QRow w(a, hk, r / 32, c);
  *reinterpret_cast<uint2*>(a.o + b * a.os[0] + w.t * a.os[1] + w.h * a.os[2] + 4 * d) =
      make_uint2(Ops<T>::pack(o.x * inv, o.y * inv), Ops<T>::pack(o.z * inv, o.w * inv));
}

int check(const GdnAttnDecodeParams& P) {
  if (P.B <= 0 || P.T < 1 || P.T > kMaxT || P.S <= 0 || P.Hq <= 0 || P.Hk <= 0 || P.Hq % P.Hk != 0) return GDN_ERR_BAD_SHAPE;
  if (P.window < 1 || P.sinks < 0 || P.S > 0x3fffffff) return GDN_ERR_BAD_SHAPE;
  if ((int64_t)P.B * P.Hq > 0x7fffffff / (2 * kMaxT)) return GDN_ERR_BAD_SHAPE;   // rows are 32-bit
  if (P.D != 64 && P.D != 128) return GDN_ERR_UNSUPPORTED;
  if (P.dtype != GDN_DTYPE_F16 && P.dtype != GDN_DTYPE_BF16) return GDN_ERR_BAD_DTYPE;
  return GDN_OK;
}

int row_tiles(const GdnAttnDecodeParams& P) { return (P.Hq / P.Hk * P.T + 31) / 32; }

// Workgroups a sequence and key head: one a CU (their tiles fill its LDS; 32
// sequences of 4 key heads with 4100 keys: 55 us with 256 workgroups, 60 with
// 512, 66 with 1024), over the tiles that the longest sequence can have.  Up to
// 4 tiles a wave stay in one workgroup: the join costs as much (a sequence of 4
// key heads, head size 128, one workgroup / joined: 128 keys 7.5 / 10.0 us, 512
// keys 10.6 / 10.8, 1024 keys 15.0 / 11.0, 4096 keys 40.0 / 11.9).
int splits_of(const GdnAttnDecodeParams& P) {
  const int64_t keys = std::min<int64_t>(P.S, (int64_t)P.window + P.T - 1 + P.sinks);
  const int64_t tiles = keys / kDN + 2;
  if (tiles <= 4 * kDWaves + 2) return 1;
  const int64_t units = (int64_t)P.B * P.Hk * row_tiles(P);
  const int64_t want = (256 + units - 1) / units;
  return (int)std::max<int64_t>(1, std::min({want, (tiles + kDWaves - 1) / kDWaves, (int64_t)kMaxSplits}));
}

template <typename T, int D>
int launch(const DArgs& a, hipStream_t s) {
  const uint32_t units = (uint32_t)a.B * a.Hk * a.tiles_r;
  hipLaunchKernelGGL((decode_kernel<T, D>), dim3(units * a.splits), dim3(64 * kDWaves), 0, s, a);
  if (a.splits > 1) hipLaunchKernelGGL((join_kernel<T, D>), dim3((uint32_t)(a.B * a.Hk * a.G * a.T)), dim3(kJT), 0, s, a);
  return (int)hipGetLastError();
}

}  // namespace attn
}  // namespace gdn

using namespace gdn;
using namespace gdn::attn;

extern "C" {

int64_t gdn_attn_decode_workspace_size(const GdnAttnDecodeParams* prm) {
  if (prm == nullptr || check(*prm) != GDN_OK) return -1;
  const int splits = splits_of(*prm);
  return splits == 1 ? 0 : (int64_t)prm->B * prm->Hk * row_tiles(*prm) * splits * 32 * (prm->D + 2) * 4;
}

int gdn_attn_decode_launch(const GdnAttnDecodeParams* prm, void* stream) {
  if (prm == nullptr) return GDN_ERR_NULL_POINTER;
  const GdnAttnDecodeParams& P = *prm;
  const int st = check(P);
  if (st != GDN_OK) return st;
  if (P.q == nullptr || P.k == nullptr || P.v == nullptr || P.o == nullptr || P.cache_seqlens == nullptr)
    return GDN_ERR_NULL_POINTER;
  if (!rows16(P.q, P.q_stride, P.B, P.T, P.Hq) || !rows16(P.o, P.o_stride, P.B, P.T, P.Hq) ||
      !rows16(P.k, P.k_stride, P.B, P.S, P.Hk) || !rows16(P.v, P.v_stride, P.B, P.S, P.Hk))
    return GDN_ERR_MISALIGNED;
  if (!grid_fits((int64_t)P.B * P.Hk * row_tiles(P) * splits_of(P), 64 * kDWaves) ||
      (splits_of(P) > 1 && !grid_fits((int64_t)P.B * P.Hq * P.T, kJT)))
    return GDN_ERR_BAD_SHAPE;
  const int64_t need = gdn_attn_decode_workspace_size(prm);
  if (need > 0 && (P.workspace == nullptr || P.workspace_bytes < need ||
                   reinterpret_cast<uintptr_t>(P.workspace) % 256 != 0))
    return GDN_ERR_WORKSPACE;
  DArgs a = {};
  a.q = static_cast<const uint16_t*>(P.q);
  a.k = static_cast<const uint16_t*>(P.k);
  a.v = static_cast<const uint16_t*>(P.v);
  a.o = static_cast<uint16_t*>(P.o);
  a.lens = P.cache_seqlens;
  a.part = static_cast<float*>(P.workspace);
  for (int d = 0; d < 3; ++d) {
    a.qs[d] = P.q_stride[d];
    a.ks[d] = P.k_stride[d];
    a.vs[d] = P.v_stride[d];
    a.os[d] = P.o_stride[d];
  }
  a.B = P.B;
  a.T = P.T;
  a.S = P.S;
  a.Hk = P.Hk;
  a.G = P.Hq / P.Hk;
  a.tiles_r = row_tiles(P);
  a.splits = splits_of(P);
  a.window = P.window;
  a.sinks = P.sinks;
  split_scale(P.scale, a.scale_log2, a.flip);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (P.dtype == GDN_DTYPE_F16) return P.D == 128 ? launch<f16, 128>(a, s) : launch<f16, 64>(a, s);
  return P.D == 128 ? launch<bf16_t, 128>(a, s) : launch<bf16_t, 64>(a, s);
}

}  // extern "C"
