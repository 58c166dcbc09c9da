// Windowed attention, backward:
//     P = e^{scale q k^T - lse},  dP = dO v^T,  dS = P (dP - D),  D = dO . o
//     dv = P^T dO,  dk = scale dS^T q,  dq = scale dS k
// in two steps, each sum in one workgroup and in a fixed order:
//   q     128 query rows a workgroup, 32 a wave, key tiles of 64 as in the
//         forward: S^T, dP^T, dQ^T += K^T dS^T; it also leaves, per query row,
//         lse in powers of 2, D and (fp16) the largest |dO|;
//   kv    128 key rows a workgroup of 4 or 8 waves: query rows of all heads that
//         share the key head pass in tiles of 32 or 64, a wave taking 32 keys
//         and 32 of the rows (S and dP with a lane on one key; P and dS enter dV^T +=
//         dO^T P and dK^T += Q^T dS straight from their accumulators);
// Blocks of the first keys (the sinks) are seen by every later query row: the
// rows beyond the block's window are cut into segments with workgroups of
// their own, whose fp32 sums a last kernel adds in order.
//
// fp16 keeps P times 2^14 and dS in a unit of its own, 2^-7 of the product of
// the largest |dO| (of the row, or of the tiles so far) and the largest |v| of
// the sequence's head: |dS| <= 2 D of that product, so none overflows and small
// gradients keep their precision.  Neither looks beyond the sequence.
//
// Bound by the matrix cores and the operands' way through LDS: a wave's 32 keys
// by 32 rows at head size 128 are 32 products (1024 cycles of a SIMD) and 40 KB
// of LDS reads (320 cycles of the CU's 128 bytes a cycle, for each of 8 waves),
// and the accumulators of dk and dv with the keys take all registers of two
// waves a SIMD.  B2 Hq16 Hk4 T4096 D128 window 1024 bf16: kv 183 us (656
// TFLOP/s of visible pairs), q 126 us (716), parts 6 us; a matrix instruction runs
// in 30 and 34 % of the SIMD-cycles.  At head size 64 a tile's chain of reads,
// products and exponentials is short and its steps wait for one another (8192
// packed rows of 16 heads, window 512, fp16: kv 86 us, q 57, parts 9, the largest
// |v| 6; matrix instructions 15 to 18 %, all vector instructions 29 to 33 %, waves
// waiting 36 to 46 % of their time).  One kernel for dq, dk and dv would save two of
// seven products, but its dq needs atomics, whose order changes results.

#include <algorithm>

#include "gdn_attn.h"

namespace gdn {
namespace attn {

constexpr int kKB = 128;       // key rows a workgroup (kv)
constexpr int kSegRows = 64;   // rows of segments come in multiples of it
constexpr int kQB = 128;       // query rows a workgroup (q)
constexpr int kKT = 64;        // keys a tile (q)
constexpr int kFewTiles = 4;   // up to so many key tiles a block of rows sums D itself (q)
constexpr int kVParts = 128;   // partial maxima of |v| a head of a sequence, at most (two a lane)

struct BArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* o;
  const uint16_t* dO;
  const float* lse;
  uint16_t* dq;
  uint16_t* dk;
  uint16_t* dv;
  float* stat;      // [Hq][rows][2]: lse in powers of 2, D
  float* rmax;      // [Hq][rows] largest |dO| (fp16)
  float* vmax;      // [units_k][v_slots] (fp16)
  float* part;      // [units_k][sink blocks][slots_s][2][kKB][D], then own_part's
  SeqArgs seq;
  int64_t qs[3], ks[3], vs[3], os[3], dos[3], dqs[3], dks[3], dvs[3];
  int64_t rows;     // B Tq
  int Hq, Hk, G;
  int units_q, units_k;         // (batch and) heads of the q and kv grids
  int slots_q, slots_k;         // blocks of each
  int v_shift, v_slots;         // rows of a partial maximum of |v| (2^v_shift), slots of a unit's
  int kv_halves;                // waves of a workgroup / 4 (kv)
  int splits;                   // workgroups a key block
  int sink_blocks, seg, slots_s;  // blocks of the first keys, rows a segment, segment slots
  int longs, long_rows;           // places of long sequences (packed), rows of the shortest
  int window, sinks;
  float scale, scale_log2;
};

template <typename T>
constexpr bool kScaled = std::is_same<T, f16>::value;
// P is kept times 2^kPUp in the products of the backward.
template <typename T>
constexpr float kPUp = kScaled<T> ? 14.f : 0.f;

// The power of 2 above x (of fp16 magnitudes; above 2^-24 for zero), and the
// inverse of a power of 2: from the exponent's bits.
__device__ __forceinline__ float pow2_above(float x) {
  return __uint_as_float((__float_as_uint(fmaxf(x, 0x1p-24f)) & 0x7f800000u) + 0x00800000u);
}
__device__ __forceinline__ float pow2_inverse(float u) { return __uint_as_float(0x7f000000u - __float_as_uint(u)); }

// The largest x of each 32 lanes, in all of them (16 by rotations of a row).
__device__ __forceinline__ float max32(float x) {
#define ROTATED(c) __uint_as_float(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), c, 0xf, 0xf, false))
  x = fmaxf(x, ROTATED(0x128));
  x = fmaxf(x, ROTATED(0x124));
  x = fmaxf(x, ROTATED(0x122));
  x = fmaxf(x, ROTATED(0x121));
#undef ROTATED
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// ---------------------------------------------------------------------------
// v
// ---------------------------------------------------------------------------

__device__ __forceinline__ float finite_abs(float x) {
  const float y = fabsf(x);
  return y < __builtin_inff() ? y : 0.f;
}

// 2^v_shift keys of one head of a sequence: the largest |v|.
template <int D>
__global__ __launch_bounds__(256) void v_max_kernel(const BArgs a) {
  constexpr int L = D / 8, RPB = 256 / L;      // lanes a row, rows a workgroup
  const int slot = blockIdx.x % a.v_slots, unit = blockIdx.x / a.v_slots;
  int hk = unit, part;
  const int si = find_block(a.seq, slot, 1 << a.v_shift, a.v_slots, part);
  Seq sq = get_seq(a.seq, si);
  if (a.seq.cu == nullptr) {
    sq.b = unit / a.Hk;
    hk = unit % a.Hk;
  }
  if (part < 0) return;
  const int64_t t0 = (int64_t)part << a.v_shift;
  const int t1 = (int)min(t0 + (1 << a.v_shift), (int64_t)sq.nk);
  float m = 0.f;
  for (int64_t t = t0 + threadIdx.x / L; t < t1; t += RPB) {
    rowio::Pack<f16, 8> pv;
    pv.load(reinterpret_cast<const f16*>(a.v) + sq.b * a.vs[0] + (sq.k0 + t) * a.vs[1] + hk * a.vs[2] + 8 * (threadIdx.x % L));
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_abs(pv.get(i)));
  }
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) m = fmaxf(m, __shfl_xor(m, s, 64));
  __shared__ float sm[4];
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) a.vmax[(int64_t)unit * a.v_slots + slot] = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
}

// The largest |v| of a head of a sequence, as a power of 2.
__device__ __forceinline__ float v_unit(const BArgs& a, const Seq& sq, int si, int hk, int lane) {
  const int n = (int)((uint32_t)(sq.nk + (1 << a.v_shift) - 1) >> a.v_shift);    // kVParts at most
  const int64_t first = a.seq.cu == nullptr ? ((int64_t)sq.b * a.Hk + hk) * a.v_slots
                                            : (int64_t)hk * a.v_slots + (sq.k0 >> a.v_shift) + si;
  float m = 0.f;
  if (lane < n) m = a.vmax[first + lane];
  if (lane + 64 < n) m = fmaxf(m, a.vmax[first + lane + 64]);
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) m = fmaxf(m, __shfl_xor(m, s, 64));
  return pow2_above(m);
}

// Output rows from transposed accumulators: lane l holds row l % 32.
template <typename T, int D>
__device__ __forceinline__ void store_rows(uint16_t* row, const f32x16 (&acc)[D / 32], float f, int half) {
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      *reinterpret_cast<uint2*>(row + 32 * dt + 8 * c + 4 * half) =
          make_uint2(Ops<T>::pack(acc[dt][4 * c] * f, acc[dt][4 * c + 1] * f),
                     Ops<T>::pack(acc[dt][4 * c + 2] * f, acc[dt][4 * c + 3] * f));
}

// ---------------------------------------------------------------------------
// kv
// ---------------------------------------------------------------------------

// Query rows that a key block takes itself: those in reach of its window; the
// rest of a block of first keys goes to segments.  Rows of the sequence.
struct QRange {
  int r0, r1;        // [r0, r1)
};
__device__ __forceinline__ QRange own_rows(const BArgs& a, const Seq& s, int k0) {
  const int shift = s.nk - s.nq;
  QRange q;
  q.r0 = max(k0 - shift, 0);
  q.r1 = (int)min((int64_t)s.nq, max((int64_t)k0 + kKB - 1 + a.window - shift, (int64_t)0));
  return q;
}
__device__ __forceinline__ QRange seg_rows(const BArgs& a, const Seq& s, int k0, int seg) {
  const QRange own = own_rows(a, s, k0);
  QRange q;
  q.r0 = max(max(own.r0, own.r1), seg * a.seg);
  q.r1 = (int)min((int64_t)s.nq, (int64_t)(seg + 1) * a.seg);
  return q;
}

// Whether rows beyond a block of first keys' own see it: only then its sums are
// parts.  Packed sequences that have such rows are at least window + kKB long,
// so start / (window + kKB) numbers them without a place for the others; few
// sequences are numbered as they are.
__device__ __forceinline__ bool has_beyond(const BArgs& a, const Seq& s, int k0) { return own_rows(a, s, k0).r1 < s.nq; }
__device__ __forceinline__ int long_place(const BArgs& a, int64_t start, int i) {
  return a.longs == a.seq.N ? i : (int)((uint32_t)start / (uint32_t)a.long_rows);
}
// Slot of segment 0 of a packed long sequence (room for ceil(rows / seg)).
__device__ __forceinline__ int first_seg(const BArgs& a, int64_t start, int i) {
  return (int)((uint32_t)start / (uint32_t)a.seg) + long_place(a, start, i);
}

// Place of the part of a key block's own rows: with splits one for each slot
// and split, else one for each block of first keys of each long sequence.
__device__ __forceinline__ int64_t own_part(const BArgs& a, int unit, const Seq& sq, int si, int block, int slot,
                                            int split) {
  const int64_t first = (int64_t)a.units_k * a.sink_blocks * a.slots_s;
  if (a.splits > 1) return first + ((int64_t)unit * a.slots_k + slot) * a.splits + split;
  const int64_t seq = a.seq.cu == nullptr ? unit : (int64_t)unit * a.longs + long_place(a, sq.q0, si);
  return first + seq * a.sink_blocks + block;
}

// 4 bytes per lane from global memory to LDS at `at` + 4 * lane.
__device__ __forceinline__ void dma4(const void* src, uint32_t at) {
  at = __builtin_amdgcn_readfirstlane(at);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(at) : "memory", "m0");
}

template <typename T, int D, int QH>
__global__ __launch_bounds__(256 * QH, D == 64 && QH == 1 ? 3 : 2) void kv_kernel(const BArgs a) {
  constexpr int kQT = 32 * QH, kKVT = 256 * QH;     // query rows a tile, threads
  using O = Ops<T>;
  using Vec = typename O::Vec;
  using TL = Tile<D>;
  constexpr uint32_t kTile = TL::bytes(kQT), kBuf = 2 * kTile + 1024;    // Q, dO, lse, D, max
  constexpr uint32_t kV = 2 * kBuf;                                           // the block's v rows
  // the keys in registers, or (3 waves a SIMD) in LDS as well
  constexpr bool kKeysInLds = D == 64 && QH == 1;
  constexpr uint32_t kK = kV + TL::bytes(kKB);
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kK + (kKeysInLds ? TL::bytes(kKB) : 0)];
  const int unit_ix = blockIdx.x % a.units_k;
  const int unit = a.units_k % 8 == 0 ? (unit_ix % 8) * (a.units_k / 8) + unit_ix / 8 : unit_ix;
  // the segments last: they are short and fill the places of the blocks at the
  // sequences' ends
  const int at_item = blockIdx.x / a.units_k, own_items = a.slots_k * a.splits;
  const bool extra = at_item >= own_items;
  const int item = extra ? at_item - own_items : at_item / a.splits, split = extra ? 0 : at_item % a.splits;
  int si, hk, block, seg = 0;
  if (a.seq.cu == nullptr) {
    si = unit / a.Hk;
    hk = unit % a.Hk;
    block = extra ? item % a.sink_blocks : item;
    seg = extra ? item / a.sink_blocks : 0;
  } else {
    hk = unit;
    if (extra) {
      block = item % a.sink_blocks;
      const int slot = item / a.sink_blocks;
      si = last_seq(a.seq, slot, [&](int64_t start, int i) { return first_seg(a, start, i); });
      seg = slot - first_seg(a, clamp_row(a.seq.cu[si], 0, a.seq.Tq), si);
    } else {
      si = find_block(a.seq, item, kKB, 0, block);
    }
  }
  const Seq sq = get_seq(a.seq, si);
  const int k0 = block * kKB;
  if (block < 0 || k0 >= sq.nk || seg < 0 || (int64_t)seg * a.seg > sq.nq) return;
  const int shift = sq.nk - sq.nq;
  const QRange rg = extra ? seg_rows(a, sq, k0, seg) : own_rows(a, sq, k0);
  if (extra && rg.r1 <= rg.r0) return;
  const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kg = wv & 3, qh = wv >> 2;
  const int key = k0 + kg * 32 + l32;          // this lane's key row
  const int j0 = k0 + kg * 32, j1 = min(j0 + 32, sq.nk) - 1;
  const uint32_t base = lds_addr(lds);

  // the tiles of all heads in a row, of which this workgroup takes its share
  const int nt = (max(rg.r1 - rg.r0, 0) + kQT - 1) / kQT, all = nt * a.G;
  const int n0 = extra ? 0 : (int)((int64_t)all * split / a.splits);
  const int n = extra ? all : (int)((int64_t)all * (split + 1) / a.splits) - n0;
  Vec kf[D / 16];
  {
    if constexpr (kKeysInLds) {
      const Copier<D, kKB, kKVT> ck(a.k + sq.b * a.ks[0] + sq.k0 * a.ks[1] + hk * a.ks[2], a.ks[1], sq.nk);
      ck(base + kK, k0);
    } else {
      const uint16_t* kr = a.k + sq.b * a.ks[0] + (sq.k0 + min(key, sq.nk - 1)) * a.ks[1] + hk * a.ks[2];
#pragma unroll
      for (int i = 0; i < D / 16; ++i) kf[i] = as_vec<T>(*reinterpret_cast<const uint4*>(kr + 16 * i + 8 * half));
    }
    const Copier<D, kKB, kKVT> cv(a.v + sq.b * a.vs[0] + sq.k0 * a.vs[1] + hk * a.vs[2], a.vs[1], sq.nk);
    cv(base + kV, k0);
  }
  float vu = 1.f;
  if constexpr (kScaled<T>)
    if (n > 0) vu = v_unit(a, sq, si, hk, lane);
  float unit_do = 0x1p-24f;                     // unit of dO so far (fp16)
  f32x16 dk[D / 32] = {}, dv[D / 32] = {};

  const TL tl(lane);
  const uint32_t vt = base + kV + TL::bytes(32) * kg;
  const int fr_first = rg.r0 + (n > 0 ? n0 % nt : 0) * kQT;
  const int fh = hk * a.G + (n > 0 ? n0 / nt : 0);
  const uint16_t* const q_first = uniform_ptr(a.q + sq.b * a.qs[0] + sq.q0 * a.qs[1] + fh * a.qs[2]);
  const uint16_t* const d_first = uniform_ptr(a.dO + sq.b * a.dos[0] + sq.q0 * a.dos[1] + fh * a.dos[2]);
  const int64_t row_first = (int64_t)fh * a.rows + (int64_t)sq.b * a.seq.Tq + sq.q0;
  // the tile that is brought next: its rows and head
  int fr0;
  int64_t frow;
  Copier<D, kQT, kKVT> cq(q_first, a.qs[1], sq.nq), cd(d_first, a.dos[1], sq.nq);
  auto fetch = [&](uint32_t at) {
    cq(at, fr0);
    cd(at + kTile, fr0);
    const int64_t row = frow + min(fr0 + lane, sq.nq - 1);
    // (rows past the tile's are not read)
    if (wv < 2) dma4(a.stat + row * 2 + wv, at + 2 * kTile + 256 * wv);
    if constexpr (kScaled<T>)
      if (wv == 2) dma4(a.rmax + row, at + 2 * kTile + 512);
    fr0 += kQT;
    if (fr0 >= rg.r1) {
      fr0 = rg.r0;
      cq.src += a.qs[2];
      cd.src += a.dos[2];
      frow += a.rows;
    }
  };
  // two waves share a SIMD: with one of them ahead, its exponentials run beside
  // the other's products
  if (qh == 1) __builtin_amdgcn_s_setprio(1);
  // One pass over the tiles.  careful: tiles on an edge of any wave's range are
  // made finite where they are not, after S and dP.
  // An infinity or NaN in a hidden place shows in the sums (0 times it is NaN):
  // only then the careful pass is taken.
  for (bool careful = false;; careful = true) {
  fr0 = fr_first;
  cq.src = q_first;
  cd.src = d_first;
  frow = row_first;
  int t0 = fr0;                                   // the tile's first row
  if (n > 0) fetch(base);
  for (int it = 0; it < n; ++it) {
    dma_wait();
    __syncthreads();
    if (it + 1 < n) fetch(base + ((it + 1) & 1) * kBuf);
    const uint32_t buf = base + (it & 1) * kBuf;
    const uint32_t qt = buf + TL::bytes(32) * qh, dt_ = qt + kTile, st = buf + 2 * kTile + 128 * qh;
    const int r0 = t0 + 32 * qh, nr = min(32, rg.r1 - r0), p0 = r0 + shift, p1 = p0 + nr - 1;
    const bool active = nr > 0 && !none_visible(j0, j1, p0, p1, a.window, a.sinks);
    const bool masked = !(nr == 32 && j0 + 32 <= sq.nk && all_visible(j0, j1, p0, p1, a.window, a.sinks));
    // a tile on an edge of any wave's range: are all its rows finite?
    constexpr int kShare = 2 * kQT / TL::kGroup / (4 * QH);
    bool bad = false;
    if (careful && !(t0 + kQT <= rg.r1 && k0 + kKB <= sq.nk &&
          all_visible(k0, k0 + kKB - 1, t0 + shift, t0 + kQT - 1 + shift, a.window, a.sinks)))
      bad = __syncthreads_or(not_finite<T, kShare>(buf + wv * kShare * TL::kGroupBytes, lane));
    Vec pf[2], df[2];
    if (active) {
      float sc = 1.f;
      if constexpr (kScaled<T>) {
        // the unit of the wave's rows
        typedef __attribute__((address_space(3))) const float lds_float;
        const float u = pow2_above(max32(*(lds_float*)(st + 512 + 4 * l32)));
        if (__any(u > unit_do)) {
          const float f = unit_do * pow2_inverse(u);
#pragma unroll
          for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) dk[i][r] *= f;
          unit_do = u;
        }
        sc = 0x1p-7f * pow2_inverse(unit_do * vu);   // 2^7 / unit, and P's 2^14 taken out
      }
      f32x16 s = {}, dp = {};
      fed_products<D / 16, 2>(
          [&](int i) {
            Quad x{tl.row8(qt, i), tl.row8(dt_, i), tl.row8(vt, i), {}};
            if constexpr (kKeysInLds) x.d = tl.row8(vt + (kK - kV), i);
            return x;
          },
          [&](int i, const Quad& x) {
            if constexpr (kKeysInLds) s = O::mfma(as_vec<T>(x.a), as_vec<T>(x.d), s);
            else s = O::mfma(as_vec<T>(x.a), kf[i], s);
            dp = O::mfma(as_vec<T>(x.b), as_vec<T>(x.c), dp);
          });
      typedef float f32x4v __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) const f32x4v lds_f32x4;
      if (bad) {
        // a row of dO that is not finite reaches the keys that see it: its S is NaN
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const f32x4v de = *(lds_f32x4*)(st + 256 + 32 * c + 16 * half);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[4 * c + e] += fabsf(de[e]) < __builtin_inff() ? 0.f : __builtin_nanf("");
        }
      }
      // row c + 4 half of the tile sees the lane's key where lo <= c < top
      const int rel = p0 + 4 * half - key;
      const int64_t reach = key < a.sinks ? (int64_t)1 << 32 : (int64_t)a.window - rel;
      const int lo = -rel, top = key < sq.nk ? (int)min((int64_t)(nr - 4 * half), reach) : -1;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const f32x4v ls = *(lds_f32x4*)(st + 32 * c + 16 * half), de = *(lds_f32x4*)(st + 256 + 32 * c + 16 * half);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * c + e;
          const float x = exp2_fast(__builtin_fmaf(s[r], a.scale_log2, kPUp<T> - ls[e]));
          dp[r] = x * __builtin_fmaf(dp[r], sc, -de[e] * sc);
          s[r] = x;
        }
        if (masked) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 4 * c + e, at = 8 * c + e;
            const bool ok = (at >= lo) & (at < top);
            s[r] = ok ? s[r] : 0.f;
            dp[r] = ok ? dp[r] : 0.f;
          }
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        pf[t] = acc_operand<T>(s, t);
        df[t] = acc_operand<T>(dp, t);
      }
    }
    if (bad) {
      __syncthreads();
      make_finite<T, kShare>(buf + wv * kShare * TL::kGroupBytes, lane);
      __syncthreads();
    }
    if (active) {
      constexpr int N = D / 32;
      fed_products<4 * N, D == 128 ? 4 : 2>(
          [&](int i) { return tl.col8(i & 1 ? qt : dt_, i / 2 % N, 16 * (i / (2 * N))); },
          [&](int i, const uint4& x) {
            const int t = i / (2 * N), d = i / 2 % N;
            if (i & 1) dk[d] = O::mfma(as_vec<T>(x), df[t], dk[d]);
            else dv[d] = O::mfma(as_vec<T>(x), pf[t], dv[d]);
          });
    }
    t0 = t0 + kQT < rg.r1 ? t0 + kQT : rg.r0;
  }
  bool odd = false;
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) odd |= !(fabsf(dk[i][r]) < __builtin_inff()) | !(fabsf(dv[i][r]) < __builtin_inff());
  if (careful || !__syncthreads_or(odd)) break;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) dk[i] = dv[i] = f32x16{};
  unit_do = 0x1p-24f;
  }
  const float fv = exp2f(-kPUp<T>);
  const float fk = kScaled<T> ? a.scale * unit_do * vu * 0x1p-7f : a.scale;
  // the two halves of the query rows: the second's sums pass through LDS
  typedef float f32x4v __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) f32x4v lds_f32x4;
  static_assert(QH == 1 || 4 * 32 * D * 4 <= sizeof(lds), "a half's sums fit");
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      dk[i][r] *= fk;
      dv[i][r] *= fv;
    }
  const uint32_t mine = base + (kg * 64 + lane) * 16;
#pragma unroll
  for (int w = 0; w < 2 * (QH - 1); ++w) {
    f32x16(&x)[D / 32] = w == 0 ? dk : dv;
    dma_wait();
    __syncthreads();
    if (qh == 1) {
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          *(lds_f32x4*)(mine + (4 * i + c) * 4096) =
              f32x4v{x[i][4 * c], x[i][4 * c + 1], x[i][4 * c + 2], x[i][4 * c + 3]};
    }
    __syncthreads();
    if (qh == 0) {
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const f32x4v y = *(lds_f32x4*)(mine + (4 * i + c) * 4096);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[i][4 * c + e] += y[e];
        }
    }
  }
  if (qh == 1) return;
  if (extra || a.splits > 1 || (block < a.sink_blocks && has_beyond(a, sq, k0))) {
    // fp32 parts: of segments and, behind them, of the blocks' own rows
    if (extra && j0 >= a.sinks) return;
    const int64_t at = extra ? ((int64_t)unit * a.sink_blocks + block) * a.slots_s + item / a.sink_blocks
                             : own_part(a, unit, sq, si, block, item, split);
    float* pk = a.part + at * (2 * kKB * D) + (kg * 32 + l32) * D;
    float* pv = pk + kKB * D;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int d = 32 * i + 8 * c + 4 * half;
        *reinterpret_cast<float4*>(pk + d) = make_float4(dk[i][4 * c], dk[i][4 * c + 1], dk[i][4 * c + 2], dk[i][4 * c + 3]);
        *reinterpret_cast<float4*>(pv + d) = make_float4(dv[i][4 * c], dv[i][4 * c + 1], dv[i][4 * c + 2], dv[i][4 * c + 3]);
      }
    return;
  }
  if (key >= sq.nk) return;
  store_rows<T, D>(a.dk + sq.b * a.dks[0] + (sq.k0 + key) * a.dks[1] + hk * a.dks[2], dk, 1.f, half);
  store_rows<T, D>(a.dv + sq.b * a.dvs[0] + (sq.k0 + key) * a.dvs[1] + hk * a.dvs[2], dv, 1.f, half);
}

// Sums of the parts of a key block, in order: a workgroup a block and 8 rows.
template <typename T, int D>
__global__ __launch_bounds__(256) void part_sum_kernel(const BArgs a, int blocks) {
  constexpr int kRowsWg = 8;
  const int rg = blockIdx.x % (kKB / kRowsWg), rest = blockIdx.x / (kKB / kRowsWg);
  const int e = rest % blocks, unit = rest / blocks;
  int si, hk, block, slot = 0;
  if (a.seq.cu == nullptr) {
    si = unit / a.Hk;
    hk = unit % a.Hk;
    block = slot = e;
  } else {
    hk = unit;
    if (a.splits > 1) {
      slot = e;
      si = find_block(a.seq, slot, kKB, 0, block);
    } else {
      // the last sequence that starts at this place, if it is a long one
      const int place = e / a.sink_blocks;
      si = last_seq(a.seq, place, [&](int64_t start, int i) { return long_place(a, start, i); });
      if (long_place(a, clamp_row(a.seq.cu[si], 0, a.seq.Tq), si) != place) return;
      block = e % a.sink_blocks;
    }
  }
  const Seq sq = get_seq(a.seq, si);
  const int k0 = block * kKB;
  if (block < 0 || k0 >= sq.nk || (a.splits == 1 && !has_beyond(a, sq, k0))) return;
  const int64_t one = 2 * kKB * D;
  const float* own = a.part + own_part(a, unit, sq, si, block, slot, 0) * one;
  const int first = a.seq.cu == nullptr || a.seg == 0 ? 0 : first_seg(a, sq.q0, si);
  const int nseg = block < a.sink_blocks ? (sq.nq + a.seg - 1) / a.seg : 0;
  // segments that end before the rows beyond the block's own have no part
  const QRange mine = own_rows(a, sq, k0);
  const int end = max(mine.r0, mine.r1), seg0 = nseg == 0 ? 0 : (end < sq.nq ? end / a.seg : nseg);
  const float* segs = a.part + (((int64_t)unit * a.sink_blocks + block) * a.slots_s + first) * one;
  for (int e = threadIdx.x; e < kRowsWg * D / 4; e += 256) {
    const int r = rg * kRowsWg + e / (D / 4), d = 4 * (e % (D / 4)), key = k0 + r;
    if (key >= sq.nk) continue;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int64_t at = (w * kKB + r) * D + d;
      float4 s = *reinterpret_cast<const float4*>(own + at);
      auto add = [&](const float* p) {
        const float4 x = *reinterpret_cast<const float4*>(p + at);
        s.x += x.x;
        s.y += x.y;
        s.z += x.z;
        s.w += x.w;
      };
#pragma unroll 4
      for (int g = 1; g < a.splits; ++g) add(own + g * one);
      if (key < a.sinks) {
#pragma unroll 8
        for (int g = seg0; g < nseg; ++g) add(segs + g * one);
      }
      uint16_t* out = w == 0 ? a.dk + sq.b * a.dks[0] + (sq.k0 + key) * a.dks[1] + hk * a.dks[2]
                             : a.dv + sq.b * a.dvs[0] + (sq.k0 + key) * a.dvs[1] + hk * a.dvs[2];
      *reinterpret_cast<uint2*>(out + d) = make_uint2(Ops<T>::pack(s.x, s.y), Ops<T>::pack(s.z, s.w));
    }
  }
}

// ---------------------------------------------------------------------------
// q
// ---------------------------------------------------------------------------

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void q_kernel(const BArgs a) {
  using O = Ops<T>;
  using Vec = typename O::Vec;
  using TL = Tile<D>;
  constexpr uint32_t kTile = TL::bytes(kKT);
  __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * kTile];
  const int unit_ix = blockIdx.x % a.units_q, slot = a.slots_q - 1 - blockIdx.x / a.units_q;
  const int unit = a.units_q % 8 == 0 ? (unit_ix % 8) * (a.units_q / 8) + unit_ix / 8 : unit_ix;
  int block, si, head;
  if (a.seq.cu == nullptr) {
    si = unit / a.Hq;
    head = unit % a.Hq;
    block = slot;
  } else {
    head = unit;
    si = find_block(a.seq, slot, kQB, 0, block);
  }
  const Seq sq = get_seq(a.seq, si);
  const int m0 = block * kQB;
  if (block < 0 || m0 >= sq.nq) return;
  const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int shift = sq.nk - sq.nq;
  const int row = m0 + wv * 32 + l32, p = row + shift;
  const int hk = head / a.G;
  const int p0 = m0 + shift, p1 = min(m0 + kQB, sq.nq) - 1 + shift;
  const KeyRange kr(p0, p1, sq.nk, a.window, a.sinks, kKT);
  const int wp0 = m0 + wv * 32 + shift, wp1 = min(wp0 + 31, sq.nq - 1 + shift);

  Vec qf[D / 16], df[D / 16];
  const int64_t at = sq.q0 + min(row, sq.nq - 1);
  {
    const uint16_t* qr = a.q + sq.b * a.qs[0] + at * a.qs[1] + head * a.qs[2];
    const uint16_t* dr = a.dO + sq.b * a.dos[0] + at * a.dos[1] + head * a.dos[2];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      qf[i] = as_vec<T>(*reinterpret_cast<const uint4*>(qr + 16 * i + 8 * half));
      df[i] = as_vec<T>(*reinterpret_cast<const uint4*>(dr + 16 * i + 8 * half));
    }
  }
  // the largest |dO| of the row, left for the kv step
  float dmax = 0.f;
  if constexpr (kScaled<T>) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) dmax = fmaxf(dmax, finite_abs((float)df[i][e]));
    dmax = max_halves(dmax);
  }
  const float l = a.lse[((int64_t)sq.b * a.seq.Tq + at) * a.Hq + head];
  const float lse2 = l == -__builtin_inff() ? __builtin_inff() : l * kLog2e;
  const Copier<D, kKT, 256> ck(a.k + sq.b * a.ks[0] + sq.k0 * a.ks[1] + hk * a.ks[2], a.ks[1], sq.nk);
  const Copier<D, kKT, 256> cv(a.v + sq.b * a.vs[0] + sq.k0 * a.vs[1] + hk * a.vs[2], a.vs[1], sq.nk);
  const uint32_t base = lds_addr(lds);
  const TL tl(lane);
  // One walk over the key tiles: f(tile's K and V, its first key) for each half
  // of a tile that any of the wave's rows sees.
  auto walk = [&](auto f) {
    if (kr.n > 0) {
      ck(base, kr.tile(0) * kKT);
      cv(base + kTile, kr.tile(0) * kKT);
    }
    for (int it = 0; it < kr.n; ++it) {
      const uint32_t kt = base + (it & 1) * 2 * kTile, vt = kt + kTile;
      dma_wait();
      __syncthreads();
      if (it + 1 < kr.n) {
        const uint32_t other = base + ((it + 1) & 1) * 2 * kTile;
        ck(other, kr.tile(it + 1) * kKT);
        cv(other + kTile, kr.tile(it + 1) * kKT);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j0 = kr.tile(it) * kKT + 32 * h, j1 = min(j0 + 32, sq.nk) - 1;
        if (j0 >= sq.nk || none_visible(j0, j1, wp0, wp1, a.window, a.sinks)) continue;
        f(kt + TL::bytes(32) * h, vt + TL::bytes(32) * h, j0);
      }
    }
  };
  auto products = [&](uint32_t kh, uint32_t vh, f32x16& s, f32x16& dp) {
    fed_products<D / 8, 4>([&](int i) { return tl.row8(i & 1 ? vh : kh, i / 2); },
                           [&](int i, const uint4& x) {
                             if (i & 1) dp = O::mfma(as_vec<T>(x), df[i / 2], dp);
                             else s = O::mfma(as_vec<T>(x), qf[i / 2], s);
                           });
  };
  // D = dO . o.  Over few keys the rounding of o shows in dP - D (a row with one
  // key has dP = D): there D is the sum of P dP instead, from a walk of its own
  // (documents of 2 to 181 rows, bf16: gradients 0.0024 of their norm off, from o
  // 0.0028, rounding P, dS and the result alone 0.0024).  Of long sequences only
  // the first two blocks take it.
  float dsum = 0.f;
  if (kr.n <= kFewTiles) {
    walk([&](uint32_t kh, uint32_t vh, int j0) {
      const Mask seen(p, j0, 32, half, sq.nk, wp0, wp1, a.window, a.sinks);
      f32x16 s = {}, x[1] = {};
      products(kh, vh, s, x[0]);
#pragma unroll
      for (int r = 0; r < 16; ++r) x[0][r] *= exp2_fast(__builtin_fmaf(s[r], a.scale_log2, -lse2));
      seen.apply<1>(x, 0.f);
#pragma unroll
      for (int r = 0; r < 16; ++r) dsum += x[0][r];
    });
    __syncthreads();      // the next walk begins with the first buffer
  } else {
    const uint16_t* orow = a.o + sq.b * a.os[0] + at * a.os[1] + head * a.os[2];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      rowio::Pack<T, 8> po, pd;
      po.load(reinterpret_cast<const T*>(orow + 16 * i + 8 * half));
      pd.raw = __builtin_bit_cast(uint4, df[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) dsum = __builtin_fmaf(pd.get(e), po.get(e), dsum);
    }
  }
  dsum += swap_halves(dsum);
  if (half == 0 && row < sq.nq) {
    const int64_t sat = (int64_t)head * a.rows + (int64_t)sq.b * a.seq.Tq + at;
    *reinterpret_cast<float2*>(a.stat + sat * 2) = make_float2(lse2, dsum);
    if constexpr (kScaled<T>) a.rmax[sat] = dmax;
  }
  float u = 1.f, sc = 1.f;
  if constexpr (kScaled<T>) {
    u = pow2_above(dmax) * v_unit(a, sq, si, hk, lane);
    sc = 0x1p-7f * pow2_inverse(u);
  }
  const float lb = kPUp<T> - lse2, de = -dsum * sc;
  f32x16 dq[D / 32] = {};

  auto pass = [&](bool careful) {
    walk([&](uint32_t kh, uint32_t vh, int j0) {
      const Mask seen(p, j0, 32, half, sq.nk, wp0, wp1, a.window, a.sinks);
      f32x16 s = {}, dps[1] = {};
      f32x16& dp = dps[0];
      products(kh, vh, s, dp);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float x = exp2_fast(__builtin_fmaf(s[r], a.scale_log2, lb));
        dp[r] = x * __builtin_fmaf(dp[r], sc, de);
      }
      seen.apply<1>(dps, 0.f);
      const bool bad = careful && seen.any() && not_finite<T, 32 / TL::kGroup>(kh, lane);
      Vec sf[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) sf[t] = acc_operand<T>(dp, t);
      if (bad) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < D / 32; ++i)
            dq[i] = O::mfma(as_vec<T>(only_finite<T>(tl.col8(kh, i, 16 * t))), sf[t], dq[i]);
      } else {
        constexpr int N = D / 32;
        fed_products<2 * N, 4>([&](int i) { return tl.col8(kh, i % N, 16 * (i / N)); },
                               [&](int i, const uint4& x) { dq[i % N] = O::mfma(as_vec<T>(x), sf[i / N], dq[i % N]); });
      }
    });
  };
  // (see kv_kernel)
  pass(false);
  bool odd = false;
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) odd |= !(fabsf(dq[i][r]) < __builtin_inff());
  if (__syncthreads_or(odd)) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) dq[i] = f32x16{};
    pass(true);
  }
  if (row >= sq.nq) return;
  const float f = kScaled<T> ? a.scale * u * 0x1p-7f : a.scale;
  store_rows<T, D>(a.dq + sq.b * a.dqs[0] + (sq.q0 + row) * a.dqs[1] + head * a.dqs[2], dq, f, half);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

int64_t up256(int64_t n) { return (n + 255) & ~(int64_t)255; }

// Packed sequences of window + kKB rows or more, at most.
int64_t long_rows(const GdnAttnParams& P) { return (int64_t)P.window + kKB; }
int long_seqs(const GdnAttnParams& P) { return (int)std::min<int64_t>(P.N, P.Tq / long_rows(P)); }

// Blocks of first keys, rows a segment and segment slots of a call (none where
// no row lies beyond the first block's window: its last key kKB - 1 is in reach
// of positions up to kKB - 2 + window, and the last position is Tk - 1).
void sink_plan(const GdnAttnParams& P, int& blocks, int& seg, int& slots) {
  blocks = seg = slots = 0;
  const int64_t sinks = std::min<int64_t>(P.sinks, P.Tk);
  if (sinks == 0 || P.Tq == 0 || (int64_t)P.window + kKB > P.Tk) return;
  blocks = (int)((sinks + kKB - 1) / kKB);
  // half of a block's own tiles a segment, 16 at most (of all heads together),
  // and no more parts than rows of D floats for every query row, twice
  const int64_t group = P.Hq / P.Hk, own = ((int64_t)P.window + kKB) / kSegRows;
  const int64_t tiles = std::max<int64_t>(1, std::min<int64_t>(16 / group, own / 2));
  seg = (int)std::max<int64_t>(tiles * kSegRows, (int64_t)blocks * kKB);
  slots = P.cu_seqlens == nullptr ? (P.Tq + seg - 1) / seg : P.Tq / seg + long_seqs(P);
}

// Key blocks (slots) of a call, and the workgroups that share one: where the
// blocks leave CUs empty, each is cut into as many as fill them, of at least 4
// tiles of 64 rows.
int64_t key_slots(const GdnAttnParams& P) { return P.cu_seqlens == nullptr ? (P.Tk + kKB - 1) / kKB : P.Tk / kKB + P.N; }
int64_t key_units(const GdnAttnParams& P) { return P.cu_seqlens == nullptr ? (int64_t)P.B * P.Hk : P.Hk; }
int key_splits(const GdnAttnParams& P) {
  const int64_t blocks = std::max<int64_t>(1, key_units(P) * key_slots(P));
  const int64_t rows = std::min<int64_t>((int64_t)P.window + kKB, P.Tq);
  const int64_t tiles = (rows + 63) / 64 * (P.Hq / P.Hk);
  return (int)std::max<int64_t>(1, std::min<int64_t>(256 / blocks, tiles / 4));
}

// Partial maxima of |v|: rows of each (kVParts cover every sequence), slots a unit.
int v_shift(const GdnAttnParams& P) {
  int shift = 5;
  while (((int64_t)kVParts << shift) < P.Tk) ++shift;
  return shift;
}
int64_t v_slots(const GdnAttnParams& P) {
  const int shift = v_shift(P);
  return P.cu_seqlens == nullptr ? ((int64_t)P.Tk + (1 << shift) - 1) >> shift : (P.Tk >> shift) + (int64_t)P.N;
}

struct Space {
  int64_t stat, rmax, vmax, part, total;
};
Space space(const GdnAttnParams& P) {
  Space s;
  const int64_t rows = (int64_t)P.B * P.Tq;
  int blocks, seg, slots;
  sink_plan(P, blocks, seg, slots);
  s.stat = 0;
  s.rmax = s.stat + up256(rows * P.Hq * 8);
  s.vmax = s.rmax + (P.dtype == GDN_DTYPE_F16 ? up256(rows * P.Hq * 4) : 0);
  s.part = s.vmax + (P.dtype == GDN_DTYPE_F16 ? up256(key_units(P) * v_slots(P) * 4) : 0);
  const int64_t units = key_units(P), splits = key_splits(P);
  const int64_t own = splits > 1 ? key_slots(P) * splits : (int64_t)blocks * (P.cu_seqlens == nullptr ? 1 : long_seqs(P));
  s.total = s.part + up256(units * ((int64_t)blocks * slots + own) * 2 * kKB * P.D * 4);
  return s;
}

template <typename T, int D>
int launch(const BArgs& a, hipStream_t s) {
  const int64_t vb = kScaled<T> && a.rows > 0 ? (int64_t)a.units_k * a.v_slots : 0;
  const int64_t kvb = (int64_t)a.units_k * ((int64_t)a.slots_k * a.splits + (int64_t)a.sink_blocks * a.slots_s);
  const int64_t qb = (int64_t)a.units_q * a.slots_q;
  const int64_t blocks = a.splits > 1 ? a.slots_k : (int64_t)a.sink_blocks * (a.seq.cu == nullptr ? 1 : a.longs);
  const int64_t pb = a.sink_blocks > 0 || a.splits > 1 ? a.units_k * blocks * (kKB / 8) : 0;
  if (!grid_fits(vb, 256) || !grid_fits(kvb, 256 * a.kv_halves) || !grid_fits(qb, 256) || !grid_fits(pb, 256))
    return GDN_ERR_BAD_SHAPE;
  if (vb > 0) hipLaunchKernelGGL((v_max_kernel<D>), dim3((uint32_t)vb), dim3(256), 0, s, a);
  if (qb > 0) hipLaunchKernelGGL((q_kernel<T, D>), dim3((uint32_t)qb), dim3(256), 0, s, a);
  if (kvb > 0) {
    if (a.kv_halves == 1) hipLaunchKernelGGL((kv_kernel<T, D, 1>), dim3((uint32_t)kvb), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((kv_kernel<T, D, 2>), dim3((uint32_t)kvb), dim3(512), 0, s, a);
  }
  if (pb > 0) hipLaunchKernelGGL((part_sum_kernel<T, D>), dim3((uint32_t)pb), dim3(256), 0, s, a, (int)blocks);
  return (int)hipGetLastError();
}

}  // namespace attn
}  // namespace gdn

using namespace gdn;
using namespace gdn::attn;

extern "C" {

int64_t gdn_attn_bwd_workspace_size(const GdnAttnParams* prm) {
  if (prm == nullptr || check_attn(*prm) != GDN_OK) return -1;
  return space(*prm).total;
}

int gdn_attn_bwd_launch(const GdnAttnParams* prm, void* stream) {
  if (prm == nullptr) return GDN_ERR_NULL_POINTER;
  const GdnAttnParams& P = *prm;
  const int st = check_attn(P);
  if (st != GDN_OK) return st;
  if (P.Tq > 0 && (P.q == nullptr || P.o == nullptr || P.lse == nullptr || P.d_o == nullptr || P.dq == nullptr))
    return GDN_ERR_NULL_POINTER;
  if (P.Tk > 0 && (P.k == nullptr || P.v == nullptr || P.dk == nullptr || P.dv == nullptr)) return GDN_ERR_NULL_POINTER;
  if (!rows16(P.q, P.q_stride, P.B, P.Tq, P.Hq) || !rows16(P.o, P.o_stride, P.B, P.Tq, P.Hq) ||
      !rows16(P.d_o, P.do_stride, P.B, P.Tq, P.Hq) || !rows16(P.dq, P.dq_stride, P.B, P.Tq, P.Hq) ||
      !rows16(P.k, P.k_stride, P.B, P.Tk, P.Hk) || !rows16(P.v, P.v_stride, P.B, P.Tk, P.Hk) ||
      !rows16(P.dk, P.dk_stride, P.B, P.Tk, P.Hk) || !rows16(P.dv, P.dv_stride, P.B, P.Tk, P.Hk))
    return GDN_ERR_MISALIGNED;
  const Space sp = space(P);
  if (sp.total > 0 && (P.workspace == nullptr || P.workspace_bytes < sp.total ||
                       reinterpret_cast<uintptr_t>(P.workspace) % 256 != 0))
    return GDN_ERR_WORKSPACE;
  BArgs a = {};
  a.q = static_cast<const uint16_t*>(P.q);
  a.k = static_cast<const uint16_t*>(P.k);
  a.v = static_cast<const uint16_t*>(P.v);
  a.o = static_cast<const uint16_t*>(P.o);
  a.dO = static_cast<const uint16_t*>(P.d_o);
  a.lse = P.lse;
  a.dq = static_cast<uint16_t*>(P.dq);
  a.dk = static_cast<uint16_t*>(P.dk);
  a.dv = static_cast<uint16_t*>(P.dv);
  char* ws = static_cast<char*>(P.workspace);
  a.stat = reinterpret_cast<float*>(ws + sp.stat);
  a.rmax = reinterpret_cast<float*>(ws + sp.rmax);
  a.vmax = reinterpret_cast<float*>(ws + sp.vmax);
  a.part = reinterpret_cast<float*>(ws + sp.part);
  a.seq = SeqArgs{P.cu_seqlens, P.Tq, P.Tk, P.N};
  for (int d = 0; d < 3; ++d) {
    a.qs[d] = P.q_stride[d];
    a.ks[d] = P.k_stride[d];
    a.vs[d] = P.v_stride[d];
    a.os[d] = P.o_stride[d];
    a.dos[d] = P.do_stride[d];
    a.dqs[d] = P.dq_stride[d];
    a.dks[d] = P.dk_stride[d];
    a.dvs[d] = P.dv_stride[d];
  }
  a.rows = (int64_t)P.B * P.Tq;
  a.Hq = P.Hq;
  a.Hk = P.Hk;
  a.G = P.Hq / P.Hk;
  const bool packed = P.cu_seqlens != nullptr;
  a.units_q = packed ? P.Hq : P.B * P.Hq;
  a.units_k = (int)key_units(P);
  a.slots_q = packed ? P.Tq / kQB + P.N : (P.Tq + kQB - 1) / kQB;
  a.slots_k = (int)key_slots(P);
  a.splits = key_splits(P);
  // 4 waves a workgroup, several workgroups a CU, where there are that many;
  // else 8 waves, so that a SIMD still has two (B2 Hk4 T4096 window 1024 bf16,
  // 256 blocks: 348 us of backward with 8 waves, 390 with 4; B4, 512 blocks:
  // 602 and 581; 1040 blocks of D 64: 219 and 170)
  a.kv_halves = (int64_t)a.units_k * a.slots_k >= 512 ? 1 : 2;
  sink_plan(P, a.sink_blocks, a.seg, a.slots_s);
  a.v_shift = v_shift(P);
  a.v_slots = (int)v_slots(P);
  a.longs = long_seqs(P);
  a.long_rows = (int)std::min<int64_t>(long_rows(P), 0x7fffffff);
  a.window = P.window;
  a.sinks = P.sinks;
  a.scale = P.scale;
  a.scale_log2 = P.scale * kLog2e;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (P.dtype == GDN_DTYPE_F16) return P.D == 128 ? launch<f16, 128>(a, s) : launch<f16, 64>(a, s);
  return P.D == 128 ? launch<bf16_t, 128>(a, s) : launch<bf16_t, 64>(a, s);
}

}  // extern "C"
