// Windowed attention, forward: o = softmax(scale q k^T) v over the keys that
// each query row sees, one pass over the keys with the running maximum and sum.
//
// A workgroup is 4 waves on 128 query rows of one head, 32 rows a wave.  Key
// and value tiles of 64 rows come by LDS-DMA into two buffers, one ahead of
// the products.  A wave forms S^T = K Q^T (a lane then holds one query row's
// scores, so the softmax needs one exchange, between the lane's two halves)
// and O^T += V^T P^T with P^T straight from the accumulators.  Only tiles on
// the edges of the visible range are masked.  Few blocks of rows over many keys
// are cut along the keys, and a second kernel joins the parts.
//
// Bound by the matrix cores and, beside them, the exponentials: of 64 keys a
// wave's products take 1024 cycles of a SIMD at head size 128 and its softmax
// about as many (32 exponentials a lane at a quarter of the rate, a maximum, a
// sum, a scaling and a conversion), which overlap only between the two waves
// that share the SIMD.  At head size 64 the products are half of that.
// B2 Hq16 Hk4 D128 bf16: T16384 window 4096 950 us (1010 TFLOP/s of visible
// pairs; a large product reaches 1288), T4096 window 1024 97 us (615: every
// block's first and last tiles are masked, and 1024 blocks are two rounds of the
// card).  Tiles of 64 keys in two buffers leave room for two workgroups a CU.
// The half of an edge tile that no row sees is computed all the same: a form
// with 32-key steps there took 1214 us (registers).

#include <algorithm>

#include "gdn_attn.h"

namespace gdn {
namespace attn {

constexpr int kBM = 128;       // query rows a workgroup
constexpr int kBN = 64;        // keys a tile
constexpr int kNT = 256;
constexpr int kPlaces = 512;   // workgroups that the card holds at once

struct FArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  float* lse;
  SeqArgs seq;
  int64_t qs[3], ks[3], vs[3], os[3];
  int Hq, G, units, slots, splits, window, sinks;
  float* stat;      // [splits][B Tq Hq][2]: maximum (in powers of 2) and sum of a split
  float* part;      // [splits][B Tq Hq][D]: its O
  float scale_log2;
  uint32_t flip;
};

template <typename T, int D>
__global__ __launch_bounds__(kNT, 2) void fwd_kernel(const FArgs a) {
  using O = Ops<T>;
  using Vec = typename O::Vec;
  using TL = Tile<D>;
  constexpr uint32_t kTile = TL::bytes(kBN);     // K0 V0 K1 V1
  __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * kTile];
  // unit = (batch, head); neighbouring units share key heads, and workgroups
  // blockIdx.x % 8 run on one XCD: give each XCD a run of units.  Later blocks
  // see more keys and start first.
  const int unit_ix = blockIdx.x % a.units, rest = blockIdx.x / a.units;
  const int slot = a.slots - 1 - rest % a.slots, split = rest / a.slots;
  const int unit = a.units % 8 == 0 ? (unit_ix % 8) * (a.units / 8) + unit_ix / 8 : unit_ix;
  int block, si, head;
  if (a.seq.cu == nullptr) {
    si = unit / a.Hq;
    head = unit % a.Hq;
    block = slot;
  } else {
    head = unit;
    si = find_block(a.seq, slot, kBM, 0, block);
  }
  const Seq sq = get_seq(a.seq, si);
  const int m0 = block * kBM;
  if (block < 0 || m0 >= sq.nq) return;
  const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int shift = sq.nk - sq.nq;            // position of query row 0
  const int row = m0 + wv * 32 + l32;         // this lane's query row
  const int p = row + shift;
  const int hk = head / a.G;
  const uint16_t* kb = a.k + sq.b * a.ks[0] + sq.k0 * a.ks[1] + hk * a.ks[2];
  const uint16_t* vb = a.v + sq.b * a.vs[0] + sq.k0 * a.vs[1] + hk * a.vs[2];

  const int p0 = m0 + shift, p1 = min(m0 + kBM, sq.nq) - 1 + shift;
  const KeyRange kr(p0, p1, sq.nk, a.window, a.sinks, kBN);
  const int per = (kr.n + a.splits - 1) / a.splits;
  const int it0 = min(split * per, kr.n), n = min(per, kr.n - it0);
  const int wp0 = m0 + wv * 32 + shift, wp1 = min(wp0 + 31, sq.nq - 1 + shift);

  Vec qf[D / 16];
  {
    const uint16_t* qr = a.q + sq.b * a.qs[0] + (sq.q0 + min(row, sq.nq - 1)) * a.qs[1] + head * a.qs[2];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) qf[i] = signed_vec<T>(*reinterpret_cast<const uint4*>(qr + 16 * i + 8 * half), a.flip);
  }
  Rows<T, D, kBN / 32> rows;
  const Copier<D, kBN, kNT> ck(kb, a.ks[1], sq.nk), cv(vb, a.vs[1], sq.nk);
  const uint32_t base = lds_addr(lds);
  const TL tl(lane);
  // An infinity or NaN in a hidden place shows in the sums (0 times it is NaN):
  // only then the pass over the tiles is taken again, carefully.  Tiles on an
  // edge of any wave's range are then made finite where they are not, after
  // what they hold has reached the rows that see it.
  for (bool careful = false;; careful = true) {
    if (n > 0) {
      ck(base, kr.tile(it0) * kBN);
      cv(base + kTile, kr.tile(it0) * kBN);
    }
    for (int it = 0; it < n; ++it) {
      const int j0 = kr.tile(it0 + it) * kBN;
      const uint32_t kt = base + (it & 1) * 2 * kTile, vt = kt + kTile;
      dma_wait();
      __syncthreads();                        // tile `it` is here; every wave is done with the other buffer
      if (it + 1 < n) {
        const int jn = kr.tile(it0 + it + 1) * kBN;
        const uint32_t other = base + ((it + 1) & 1) * 2 * kTile;
        ck(other, jn);
        cv(other + kTile, jn);
      }
      const int j1 = min(j0 + kBN, sq.nk) - 1;
      const bool active = !none_visible(j0, j1, wp0, wp1, a.window, a.sinks);
      const Mask seen(p, j0, kBN, half, sq.nk, wp0, wp1, a.window, a.sinks);
      constexpr int kShare = kBN / TL::kGroup / 4;
      const uint32_t share = vt + wv * kShare * TL::kGroupBytes;
      if (active) rows.template scores<2>(qf, tl, kt, seen, a.scale_log2);
      if (careful && !(j0 + kBN <= sq.nk && all_visible(j0, j1, p0, p1, a.window, a.sinks)) &&
          __syncthreads_or(not_finite<T, kShare>(share, lane))) {
        if (active) rows.template add_not_finite<2>(seen, tl, vt);
        __syncthreads();
        make_finite<T, kShare>(share, lane);
        __syncthreads();
      }
      if (active) rows.template values<2>(tl, vt);
    }
    bool odd = !(fabsf(rows.l) < __builtin_inff());
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) odd |= !(fabsf(rows.acc[dt][r]) < __builtin_inff());
    if (careful || !__syncthreads_or(odd)) break;
    rows.clear();
  }

  const float l = rows.l + swap_halves(rows.l);
  if (row >= sq.nq) return;
  const int64_t at = ((int64_t)sq.b * a.seq.Tq + sq.q0 + row) * a.Hq + head;
  if (a.splits > 1) {
    const int64_t to = (int64_t)split * a.units * a.seq.Tq + at;
    if (half == 0) *reinterpret_cast<float2*>(a.stat + 2 * to) = make_float2(rows.m, l);
    float* pr = a.part + to * D + 4 * half;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        *reinterpret_cast<float4*>(pr + 32 * dt + 8 * c) =
            make_float4(rows.acc[dt][4 * c], rows.acc[dt][4 * c + 1], rows.acc[dt][4 * c + 2], rows.acc[dt][4 * c + 3]);
    return;
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  uint16_t* orow = a.o + sq.b * a.os[0] + (sq.q0 + row) * a.os[1] + head * a.os[2];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint2 w = make_uint2(O::pack(rows.acc[dt][4 * c] * inv, rows.acc[dt][4 * c + 1] * inv),
                                 O::pack(rows.acc[dt][4 * c + 2] * inv, rows.acc[dt][4 * c + 3] * inv));
      *reinterpret_cast<uint2*>(orow + 32 * dt + 8 * c + 4 * half) = w;
    }
  if (a.lse != nullptr && half == 0)
    a.lse[at] = l > 0.f || l != l ? (rows.m - O::kShift) * kLn2 + logf(l) : -__builtin_inff();
}

// The splits of a row joined, in order: D / 4 threads a row (of a dense batch).
template <typename T, int D>
__global__ __launch_bounds__(kNT) void join_rows_kernel(const FArgs a) {
  constexpr int L = D / 4;
  const int64_t rows = (int64_t)a.units * a.seq.Tq, at = (int64_t)blockIdx.x * (kNT / L) + threadIdx.x / L;
  if (at >= rows) return;
  const int d = 4 * (threadIdx.x % L);
  float top = -__builtin_inff();
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.stat[2 * (s * rows + at)]);
  float l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const float2 ml = *reinterpret_cast<const float2*>(a.stat + 2 * (s * rows + at));
    const float4 x = *reinterpret_cast<const float4*>(a.part + (s * rows + at) * D + d);
    // a split that saw no key adds nothing; one that saw only NaN has no maximum
    // either, but its sum is NaN
    if (ml.y == 0.f) continue;
    const float f = ml.x == -__builtin_inff() ? 0.f : exp2_fast(ml.x - top);
    l += f * ml.y;
    o.x += f * x.x;
    o.y += f * x.y;
    o.z += f * x.z;
    o.w += f * x.w;
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  const int head = (int)(at % a.Hq);
  const int64_t bt = at / a.Hq, b = bt / a.seq.Tq, t = bt % a.seq.Tq;
  *reinterpret_cast<uint2*>(a.o + b * a.os[0] + t * a.os[1] + head * a.os[2] + d) =
      make_uint2(Ops<T>::pack(o.x * inv, o.y * inv), Ops<T>::pack(o.z * inv, o.w * inv));
  if (a.lse != nullptr && d == 0)
    a.lse[at] = l > 0.f || l != l ? (top - Ops<T>::kShift) * kLn2 + logf(l) : -__builtin_inff();
}

int check_attn(const GdnAttnParams& P) {
  if (P.B <= 0 || P.Tq < 0 || P.Tk < 0 || P.N <= 0 || P.N > (1 << 22) || P.Hq <= 0 || P.Hk <= 0 || P.Hq % P.Hk != 0) return GDN_ERR_BAD_SHAPE;
  if (P.cu_seqlens == nullptr ? P.N != P.B : (P.B != 1 || P.Tq != P.Tk)) return GDN_ERR_BAD_SHAPE;
  if (P.window < 1 || P.sinks < 0) return GDN_ERR_BAD_SHAPE;
  if (P.D != 64 && P.D != 128) return GDN_ERR_UNSUPPORTED;
  if (P.dtype != GDN_DTYPE_F16 && P.dtype != GDN_DTYPE_BF16) return GDN_ERR_BAD_DTYPE;
  // positions and (batch, head) are 32-bit
  if ((int64_t)P.B * P.Hq > 0x7fffffffLL || (int64_t)P.Tq + P.Tk > 0x3fffffffLL) return GDN_ERR_BAD_SHAPE;
  return GDN_OK;
}

// Workgroups that share a block's keys: where a dense batch leaves most places
// on the card (two a CU) empty and has 1024 keys or more, as many as fill them,
// of at least 4 tiles each.  (Packed lengths are not known on the host.)  One
// workgroup a block / shared, bf16: 32 rows on 32768 keys, 16 heads of 128,
// 639 / 65 us; 512 on 4096 88 / 45; 1024 causal rows, 8 heads, 28 / 25; 2048 causal
// rows of 12 heads (192 blocks) 49 / 44, of 16 (256 blocks) 51 / 57; 512 causal
// rows of 16 heads 18 / 20.
int splits_of(const GdnAttnParams& P) {
  const int64_t blocks = (int64_t)P.B * P.Hq * ((P.Tq + kBM - 1) / kBM);
  const int64_t keys = std::min<int64_t>(P.Tk, (int64_t)P.window + kBM + P.sinks);
  if (P.cu_seqlens != nullptr || blocks == 0 || blocks >= kPlaces / 2 || keys < 1024) return 1;
  return (int)std::min<int64_t>(kPlaces / blocks, keys / kBN / 4);
}
int64_t stat_bytes(const GdnAttnParams& P, int splits) {
  return ((int64_t)splits * P.B * P.Tq * P.Hq * 8 + 255) & ~(int64_t)255;
}

template <typename T, int D>
int launch_td(const FArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((fwd_kernel<T, D>), dim3((uint32_t)a.units * a.slots * a.splits), dim3(kNT), 0, s, a);
  if (a.splits > 1) {
    constexpr int kRowsWg = kNT / (D / 4);
    const int64_t rows = (int64_t)a.units * a.seq.Tq;
    hipLaunchKernelGGL((join_rows_kernel<T, D>), dim3((uint32_t)((rows + kRowsWg - 1) / kRowsWg)), dim3(kNT), 0, s, a);
  }
  return (int)hipGetLastError();
}
template <typename T>
int launch_t(const FArgs& a, int D, hipStream_t s) {
  return D == 128 ? launch_td<T, 128>(a, s) : launch_td<T, 64>(a, s);
}

}  // namespace attn
}  // namespace gdn

using namespace gdn;
using namespace gdn::attn;

extern "C" {

int64_t gdn_attn_workspace_size(const GdnAttnParams* prm) {
  if (prm == nullptr || check_attn(*prm) != GDN_OK) return -1;
  const int splits = splits_of(*prm);
  return splits == 1 ? 0 : stat_bytes(*prm, splits) + (int64_t)splits * prm->B * prm->Tq * prm->Hq * prm->D * 4;
}

int gdn_attn_launch(const GdnAttnParams* prm, void* stream) {
  if (prm == nullptr) return GDN_ERR_NULL_POINTER;
  const GdnAttnParams& P = *prm;
  const int st = check_attn(P);
  if (st != GDN_OK) return st;
  if (P.Tq == 0) return GDN_OK;
  if (P.q == nullptr || P.o == nullptr || (P.Tk > 0 && (P.k == nullptr || P.v == nullptr))) return GDN_ERR_NULL_POINTER;
  if (!rows16(P.q, P.q_stride, P.B, P.Tq, P.Hq) || !rows16(P.o, P.o_stride, P.B, P.Tq, P.Hq) ||
      !rows16(P.k, P.k_stride, P.B, P.Tk, P.Hk) || !rows16(P.v, P.v_stride, P.B, P.Tk, P.Hk))
    return GDN_ERR_MISALIGNED;
  FArgs a = {};
  a.q = static_cast<const uint16_t*>(P.q);
  a.k = static_cast<const uint16_t*>(P.k);
  a.v = static_cast<const uint16_t*>(P.v);
  a.o = static_cast<uint16_t*>(P.o);
  a.lse = P.lse;
  a.seq = SeqArgs{P.cu_seqlens, P.Tq, P.Tk, P.N};
  for (int d = 0; d < 3; ++d) {
    a.qs[d] = P.q_stride[d];
    a.ks[d] = P.k_stride[d];
    a.vs[d] = P.v_stride[d];
    a.os[d] = P.o_stride[d];
  }
  a.Hq = P.Hq;
  a.G = P.Hq / P.Hk;
  a.window = P.window;
  a.sinks = P.sinks;
  split_scale(P.scale, a.scale_log2, a.flip);
  int64_t units = P.Hq, slots = 0;
  if (P.cu_seqlens == nullptr) {
    units *= P.B;
    slots = (P.Tq + kBM - 1) / kBM;
  } else {
    slots = P.Tq / kBM + P.N;
  }
  if (!grid_fits(units * slots * splits_of(P), kNT)) return GDN_ERR_BAD_SHAPE;
  a.units = (int)units;
  a.slots = (int)slots;
  a.splits = splits_of(P);
  if (a.splits > 1) {
    if (P.workspace == nullptr || P.workspace_bytes < gdn_attn_workspace_size(prm) ||
        reinterpret_cast<uintptr_t>(P.workspace) % 256 != 0)
      return GDN_ERR_WORKSPACE;
    a.stat = static_cast<float*>(P.workspace);
    a.part = reinterpret_cast<float*>(static_cast<char*>(P.workspace) + stat_bytes(P, a.splits));
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  return P.dtype == GDN_DTYPE_F16 ? launch_t<f16>(a, P.D, s) : launch_t<bf16_t>(a, P.D, s);
}

}  // extern "C"
