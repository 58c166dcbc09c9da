// A key and value cache in e4m3 with a scale for each row and head: writing it,
// reading it back, and windowed attention of the newest tokens over it.
//     scale = max|x| / 448 over the D columns of a row, q = x / scale rounded,
//     o = softmax(q (k8 ks)^T) (v8 vs)  over the visible keys
//
// Decode: as over a 16-bit cache, the G T query rows that share a key head are the
// columns of 32-wide products, and the visible key tiles are dealt to `splits`
// workgroups and there to their 8 waves, each of which brings its own tiles of 32
// keys by LDS-DMA into two buffers.  The bytes go to the operands' type in
// registers (e4m3 is exact in both); keys meet their scales behind the product.
// Values meet theirs inside the exponential, 2^(s + log2 vs - M), M the running
// maximum of s + log2 vs: so P vs has the range of a probability whatever the
// scales are, and is rounded once to the operands' type as P is over a 16-bit
// cache.  The sum l of P without vs keeps a running maximum m of its own; the
// result is O 2^(M - m) / l.
//
// Bound by reading 2 D + 8 bytes of each visible key and head: 32 sequences of up to
// 16384 keys, 4 heads of 128 in a window of 4096, 27 us at 4.8 TB/s, the rate of a copy;
// one sequence of 65536 keys 17.3 to 18 us at 3.6 TB/s (4 tiles a wave, of which the first two
// wait for the length, the query and memory alone), its join 5 us.  Two tiles on
// the way before the first is used changed nothing.
// Writing 8 x 2048 rows of 4 heads from bf16: 12.5 us, 4 TB/s; reading 8 x 4096 back:
// 17.7 us, 5.7 TB/s (partly from the last-level cache).
#include <algorithm>

#include "gdn_attn.h"
#include "gdn_fp8.h"

namespace gdn {
namespace cache8 {

using namespace attn;
using fp8::kFp8Max;
using fp8::lanes_max;
using fp8::nan_max;
using fp8::Quant;
using fp8::pack_fp8;
using rowio::Pack;

struct Args {
  const void* k;        // new rows; read back: written
  const void* v;
  const uint16_t* q;
  uint16_t* o;
  uint8_t* kc;
  uint8_t* vc;
  float* ks;
  float* vs;
  const int32_t* lens;
  float* part;          // [units][splits][32][D + 3]
  int64_t kst[3], vst[3], qst[3], ost[3], kcst[3], vcst[3], ksst[3], vsst[3];
  int B, T, S, Hk, G, tiles_r, splits, window, sinks;
  uint32_t first;       // workgroup of a launch (write, read)
  float scale_log2;
  uint32_t flip;
};

__device__ __forceinline__ int64_t at3(const int64_t* st, int b, int t, int h) {
  return b * st[0] + t * st[1] + h * st[2];
}

// ---------------------------------------------------------------------------
// writing and reading back
// ---------------------------------------------------------------------------

constexpr int kRowNT = 256;

// D / 16 lanes a row; blockIdx.y: keys, values.
template <typename E, int D>
__global__ __launch_bounds__(kRowNT) void write_kernel(const Args a) {
  constexpr int L = D / 16;
  const uint32_t row = (a.first + blockIdx.x) * (kRowNT / L) + threadIdx.x / L, e0 = threadIdx.x % L * 16;
  const uint32_t per = a.T * a.Hk;
  if (row >= a.B * per) return;       // (the row's lanes leave together)
  const int b = row / per, r = row - b * per, t = r / a.Hk, h = r - t * a.Hk;
  const int s = max(0, min(a.lens[b], a.S)) - a.T + t;
  if (s < 0) return;
  const bool v = blockIdx.y;
  const E* from = (v ? static_cast<const E*>(a.v) + at3(a.vst, b, t, h) : static_cast<const E*>(a.k) + at3(a.kst, b, t, h)) + e0;
  Pack<E, 8> x[2];
  x[0].load(from);
  x[1].load(from + 8);
  float f[16], m = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    f[e] = x[e / 8].get(e % 8);
    m = nan_max(m, fabsf(f[e]));
  }
  m = lanes_max<L>(m) / kFp8Max;
  const Quant quant(m);
  uint32_t q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = pack_fp8(quant(f[4 * i]), quant(f[4 * i + 1]), quant(f[4 * i + 2]), quant(f[4 * i + 3]));
  *reinterpret_cast<uint4*>((v ? a.vc + at3(a.vcst, b, s, h) : a.kc + at3(a.kcst, b, s, h)) + e0) =
      make_uint4(q[0], q[1], q[2], q[3]);
  if (e0 == 0) {
    if (v) a.vs[at3(a.vsst, b, s, h)] = m;
    else a.ks[at3(a.ksst, b, s, h)] = m;
  }
}

// D / 16 lanes a row.
template <typename E, int D>
__global__ __launch_bounds__(kRowNT) void read_kernel(const Args a) {
  constexpr int L = D / 16;
  const uint32_t row = (a.first + blockIdx.x) * (kRowNT / L) + threadIdx.x / L, e0 = threadIdx.x % L * 16;
  const uint32_t per = a.S * a.Hk;
  if (row >= a.B * per) return;
  const int b = row / per, r = row - b * per, s = r / a.Hk, h = r - s * a.Hk;
  const bool v = blockIdx.y;
  const uint4 q = *reinterpret_cast<const uint4*>((v ? a.vc + at3(a.vcst, b, s, h) : a.kc + at3(a.kcst, b, s, h)) + e0);
  const float scale = v ? a.vs[at3(a.vsst, b, s, h)] : a.ks[at3(a.ksst, b, s, h)];
  E* out = (v ? (E*)a.v + at3(a.vst, b, s, h) : (E*)a.k + at3(a.kst, b, s, h)) + e0;
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  float f[16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[4 * i] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 0) * scale;
    f[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 1) * scale;
    f[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 2) * scale;
    f[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 3) * scale;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    Pack<E, 8> p;
    p.set(f + 8 * i);
    p.store(out + 8 * i);
  }
}

// ---------------------------------------------------------------------------
// decode
// ---------------------------------------------------------------------------

constexpr int kDN = 32;          // keys a tile
constexpr int kDWaves = 8;
constexpr int kNT = 64 * kDWaves;
constexpr int kMaxT = 16;
constexpr int kMaxSplits = 64;

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
typedef __attribute__((address_space(3))) f32x4 lds_f32x4;

// 4 bytes of e4m3 as two pairs of the operands' type.
template <typename T>
__device__ __forceinline__ uint2 widen4(int w);
template <>
__device__ __forceinline__ uint2 widen4<f16>(int w) {
  return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true)));
}
template <>
__device__ __forceinline__ uint2 widen4<bf16_t>(int w) {
  return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true)));
}
template <typename T>
__device__ __forceinline__ typename Ops<T>::Vec widen8(int lo, int hi) {
  const uint2 a = widen4<T>(lo), b = widen4<T>(hi);
  return as_vec<T>(make_uint4(a.x, a.y, b.x, b.y));
}

// 32 rows of D bytes in LDS, 16-byte piece c of row r at place c ^ swz(r): 16 rows
// at one piece (the keys' operand) and the 8 rows {0..3, 8..11} at 32 neighbouring
// bytes (the values', transposing) each cover all banks once.
template <int D>
struct Tile8 {
  static constexpr int kPieces = D / 16, kRowsDma = 64 / kPieces, kDmas = kDN / kRowsDma;
  static constexpr uint32_t kBytes = kDN * D;
  __device__ static __forceinline__ int swz(int r) {
    return D == 128 ? ((r >> 2) & 1) | (((r >> 1) & 1) << 1) | (((r >> 3) & 1) << 2) : (r >> 2) & 3;
  }
  uint32_t row, col;
  __device__ __forceinline__ explicit Tile8(int lane) {
    const int r = lane & 31, h = lane >> 5;
    row = r * D + 16 * (h ^ swz(r));
    const int j = (lane & 15) >> 1, key = 8 * (j >> 2) + 4 * h + (j & 3);
    col = key * D + 16 * (((lane >> 4) & 1) ^ swz(key)) + 8 * (lane & 1);
  }
  // 16 elements 32 u + 16 (l / 32) .. of row l % 32
  __device__ __forceinline__ u32x4 row16(uint32_t tile, int u) const {
    return *(const lds_u32x4*)(tile + (row ^ (32 * u)));
  }
  // element 32 dt + l % 32 of rows 16 s + 4 (l / 32) + {0..3, 8..11}
  // (ds_read_b64_tr_b8: lane i of 16 receives byte i % 8 of the 8 bytes addressed by
  // lanes 2 j + i / 8, j = 0..7)
  __device__ __forceinline__ i32x2 col8(uint32_t tile, int dt, int s) const {
    return __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(tile + (col ^ (32 * dt)) + 16 * D * s));
  }
};

// Row (of 32) of a unit: query token, head, and whether it exists.
struct QRow {
  int t, h;
  bool ok;
  __device__ __forceinline__ QRow(const Args& a, int hk, int rt, int c) {
    const int r = rt * 32 + c;
    ok = r < a.G * a.T;
    const int rr = ok ? r : 0;
    t = rr / a.G;
    h = hk * a.G + rr % a.G;
  }
};

// The factor of a part with maximum m under the common one.
__device__ __forceinline__ float weight(float m, float top) { return m == -__builtin_inff() ? 0.f : exp2_fast(m - top); }

// log2 of a value's scale, of the smallest ones too (the instruction takes those below
// 2^-126 for 0).
__device__ __forceinline__ float log2_scale(float x) {
  return x < 0x1p-126f ? __builtin_amdgcn_logf(x * 0x1p32f) - 32.f : __builtin_amdgcn_logf(x);
}

// What O becomes the result by: 2^(M - m) / l (0 where no key was seen, NaN where l is),
// in two factors where the power is no normal number.
template <typename T>
struct Result {
  float f, down;
  __device__ __forceinline__ Result(float m, float l, float M) {
    const float e = M - m - Ops<T>::kShift;
    const bool small = e < -64.f;
    down = small ? 0x1p-64f : 1.f;
    f = l == 0.f ? 0.f : M == -__builtin_inff() ? (l != l ? l : 0.f) : exp2_fast(small ? e + 64.f : e) / l;
  }
  __device__ __forceinline__ float operator()(float o) const { return o * f * down; }
};

constexpr uint32_t kNan = 0x7f7f7f7fu;       // e4m3: all ones but the sign
// Bits 0x80 of the bytes that are NaN.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & kNan) + 0x01010101u) & 0x80808080u; }

template <typename T, int D>
__global__ __launch_bounds__(kNT) void decode_kernel(const Args a) {
  using O = Ops<T>;
  using Vec = typename O::Vec;
  using TL = Tile8<D>;
  constexpr uint32_t kTile = TL::kBytes, kBuf = 2 * kTile + 256, kWave = 2 * kBuf;
  constexpr int kRow = D + 3, kPitch = D + 4;
  constexpr uint32_t kJoin = kDWaves * 32 * (kPitch + 3) * 4, kTiles = kDWaves * kWave;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kJoin > kTiles ? kJoin : kTiles];
  const int split = blockIdx.x % a.splits, unit = blockIdx.x / a.splits;
  const int rt = unit % a.tiles_r, bh = unit / a.tiles_r, hk = bh % a.Hk, b = bh / a.Hk;
  const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int len = a.lens[b];
  const QRow qr(a, hk, rt, l32);
  Vec qf[D / 16];      // elements 32 u + 16 half + 8 w of product 2 u + w
  {
    const uint16_t* q = a.q + at3(a.qst, b, qr.t, qr.h);
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
      qf[i] = signed_vec<T>(*reinterpret_cast<const uint4*>(q + 32 * (i >> 1) + 16 * half + 8 * (i & 1)), a.flip);
  }
  const int n = __builtin_amdgcn_readfirstlane(max(0, min(len, a.S)));
  const int p = n - a.T + qr.t;
  const int r0 = rt * 32, rows = min(32, a.G * a.T - r0);
  const int p0 = n - a.T + r0 / a.G, p1 = n - a.T + (r0 + rows - 1) / a.G;

  // the tiles of any row; rows before the first key see none
  const KeyRange kr(max(p0, 0), p1, n, a.window, a.sinks, kDN);
  const int per = (kr.n + a.splits - 1) / a.splits;
  const int t0 = min(split * per, kr.n), t1 = min(t0 + per, kr.n);

  const uint8_t* kb = a.kc + b * a.kcst[0] + hk * a.kcst[2];
  const uint8_t* vb = a.vc + b * a.vcst[0] + hk * a.vcst[2];
  // lanes 0..31 bring the keys' scales of a tile, the others the values'
  const float* sb = half == 0 ? a.ks + b * a.ksst[0] + hk * a.ksst[2] : a.vs + b * a.vsst[0] + hk * a.vsst[2];
  const int64_t sld = half == 0 ? a.ksst[1] : a.vsst[1];
  const uint32_t base = lds_addr(lds) + wv * kWave;
  auto fetch = [&](uint32_t at, int row0) {
    dma4(sb + (int64_t)min(row0 + l32, n - 1) * sld, at + 2 * kTile);
#pragma unroll
    for (int i = 0; i < TL::kDmas; ++i) {
      const int row = i * TL::kRowsDma + lane / TL::kPieces, c = (lane % TL::kPieces) ^ TL::swz(row);
      const int64_t r = min(row0 + row, n - 1);
      dma16(kb + r * a.kcst[1] + 16 * c, at + i * 1024);
      dma16(vb + r * a.vcst[1] + 16 * c, at + kTile + i * 1024);
    }
  };
  const TL tl(lane);
  f32x16 acc[D / 32] = {};
  float m = -__builtin_inff(), l = 0.f, M = -__builtin_inff();
  if (t0 + wv < t1) fetch(base, kr.tile(t0 + wv) * kDN);
  for (int t = t0 + wv, k = 0; t < t1; t += kDWaves, ++k) {
    dma_wait();
    const uint32_t kt = base + (k & 1) * kBuf, vt = kt + kTile, st = vt + kTile;
    if (t + kDWaves < t1) fetch(base + ((k + 1) & 1) * kBuf, kr.tile(t + kDWaves) * kDN);
    // the scales as the scores need them: times log2 e and the scale, and log2
    {
      lds_f32* at = (lds_f32*)(st + 4 * lane);
      const float x = *at;
      *at = half == 0 ? x * a.scale_log2 : log2_scale(x);
    }
    const Mask seen(p, kr.tile(t) * kDN, kDN, half, n, p0, p1, a.window, a.sinks);
    f32x16 s[1] = {};
#pragma unroll
    for (int u = 0; u < D / 32; ++u) {
      const u32x4 x = tl.row16(kt, u);
      s[0] = O::mfma(widen8<T>((int)x[0], (int)x[1]), qf[2 * u], s[0]);
      s[0] = O::mfma(widen8<T>((int)x[2], (int)x[3]), qf[2 * u + 1], s[0]);
    }
    f32x16 w;      // s + log2 of the value's scale
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 x = *(const lds_f32x4*)(st + 32 * g + 16 * half), y = *(const lds_f32x4*)(st + 128 + 32 * g + 16 * half);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[0][4 * g + e] *= x[e];
        w[4 * g + e] = y[e];
      }
    }
    seen.apply<1>(s, -__builtin_inff());
#pragma unroll
    for (int r = 0; r < 16; ++r) w[r] += s[0][r];
    if (seen.any()) {      // what is hidden stays so, whatever its scale
#pragma unroll
      for (int r = 0; r < 16; ++r) w[r] = s[0][r] == -__builtin_inff() ? -__builtin_inff() : w[r];
    }
    float ms = s[0][0], mw = w[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) {
      ms = fmaxf(ms, s[0][r]);
      mw = fmaxf(mw, w[r]);
    }
    ms = max_halves(ms);
    mw = max_halves(mw);
    if (__any(ms > m + kLazy || mw > M + kLazy)) {
      // each row by its own scores, so that no row's bits depend on another's
      if (ms > m + kLazy) {
        l *= exp2_fast(m - ms);
        m = ms;
      }
      const float f = mw > M + kLazy ? exp2_fast(M - mw) : 1.f;
      M = mw > M + kLazy ? mw : M;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] *= f;
    }
    const float mb = m == -__builtin_inff() ? 0.f : -m, Mb = M == -__builtin_inff() ? 0.f : O::kShift - M;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      l += exp2_fast(s[0][r] + mb);
      w[r] = exp2_fast(w[r] + Mb);
    }
    const Vec pf[2] = {acc_operand<T>(w, 0), acc_operand<T>(w, 1)};
    if (seen.any()) {
      // a NaN in a hidden place would enter as 0 NaN: the sums that see one become
      // NaN by a product of 0/1 matrices, and the tile is made finite
      uint32_t bad = 0;
#pragma unroll
      for (int i = 0; i < TL::kDmas; ++i) {
        const u32x4 x = *(const lds_u32x4*)(vt + i * 1024 + 16 * lane);
        bad |= nan_bytes(x[0]) | nan_bytes(x[1]) | nan_bytes(x[2]) | nan_bytes(x[3]);
      }
      if (__any(bad != 0)) {
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) {
          f32x16 hit = {};
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const i32x2 x = tl.col8(vt, dt, i);
            // e4m3's 1 is 0x38
            const int nan[2] = {(int)((nan_bytes(x[0]) >> 7) * 0x38u), (int)((nan_bytes(x[1]) >> 7) * 0x38u)};
            uint32_t one[2] = {0, 0};
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (seen(0, 8 * i + e)) one[e >> 2] |= 0x38u << (8 * (e & 3));
            hit = O::mfma(widen8<T>(nan[0], nan[1]), widen8<T>((int)one[0], (int)one[1]), hit);
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[dt][r] += hit[r] > 0.f ? __builtin_nanf("") : 0.f;
        }
#pragma unroll
        for (int i = 0; i < TL::kDmas; ++i) {
          lds_u32x4* at = (lds_u32x4*)(vt + i * 1024 + 16 * lane);
          u32x4 x = *at;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] &= ~((nan_bytes(x[e]) >> 7) * 0xffu);
          *at = x;
        }
      }
    }
    // O^T += V^T P^T
    fed_products<2 * (D / 32), 4>([&](int i) { return tl.col8(vt, i % (D / 32), i / (D / 32)); },
                                  [&](int i, const i32x2& x) {
                                    acc[i % (D / 32)] = O::mfma(widen8<T>(x[0], x[1]), pf[i / (D / 32)], acc[i % (D / 32)]);
                                  });
  }
  l += swap_halves(l);

  // the waves' parts, joined by all of them
  __syncthreads();
  float* sm = reinterpret_cast<float*>(lds);        // [8][32] m, l, M, then [8][32][D + 4] O
  float* sl = sm + kDWaves * 32;
  float* sM = sl + kDWaves * 32;
  float* so = sM + kDWaves * 32;
  if (l32 < rows) {
    if (half == 0) {
      sm[wv * 32 + l32] = m;
      sl[wv * 32 + l32] = l;
      sM[wv * 32 + l32] = M;
    }
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(so + (wv * 32 + l32) * kPitch + 32 * dt + 8 * g + 4 * half) =
            make_float4(acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]);
  }
  __syncthreads();
  // two columns of a row a thread
  for (int e = threadIdx.x; e < rows * (D / 2); e += kNT) {
    const int c = e / (D / 2), d = e % (D / 2) * 2;
    float top = sm[c], topM = sM[c];
#pragma unroll
    for (int w = 1; w < kDWaves; ++w) {
      top = fmaxf(top, sm[w * 32 + c]);
      topM = fmaxf(topM, sM[w * 32 + c]);
    }
    // (a wave without a key holds zeros; one that saw NaN alone has no maximum and keeps
    // it: 0 NaN is NaN, in the sum too)
    float sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < kDWaves; ++w) {
      sum += weight(sm[w * 32 + c], top) * sl[w * 32 + c];
      const float f = weight(sM[w * 32 + c], topM);
      const float2 o = *reinterpret_cast<const float2*>(so + (w * 32 + c) * kPitch + d);
      x += f * o.x;
      y += f * o.y;
    }
    if (a.splits > 1) {
      float* part = a.part + ((int64_t)unit * a.splits + split) * 32 * kRow;
      if (d == 0) {
        part[c] = top;
        part[32 + c] = sum;
        part[64 + c] = topM;
      }
      *reinterpret_cast<float2*>(part + 96 + c * D + d) = make_float2(x, y);
    } else {
      const Result<T> result(top, sum, topM);
      const QRow row(a, hk, rt, c);
      *reinterpret_cast<uint32_t*>(a.o + at3(a.ost, b, row.t, row.h) + d) = O::pack(result(x), result(y));
    }
  }
}

// One workgroup a query row: every wave weighs the splits (one a lane), then
// groups of D / 4 threads add the splits g, g + groups, .. and the groups' sums
// are added in order.
constexpr int kJT = 256;
template <typename T, int D>
__global__ __launch_bounds__(kJT) void join_kernel(const Args a) {
  constexpr int L = D / 4, kGroups = kJT / L, kRow = D + 3;
  const int rows = a.G * a.T, r = blockIdx.x % rows, bh = blockIdx.x / rows, hk = bh % a.Hk, b = bh / a.Hk;
  const int c = r % 32, unit = bh * a.tiles_r + r / 32;
  const float* part = a.part + (int64_t)unit * a.splits * 32 * kRow;
  const int64_t step = 32 * kRow;
  const int lane = threadIdx.x & 63, g = threadIdx.x / L, d = threadIdx.x % L;
  static_assert(kMaxSplits <= 64, "a split a lane");
  const bool mine = lane < a.splits;
  const float m = mine ? part[lane * step + c] : -__builtin_inff(), ls = mine ? part[lane * step + 32 + c] : 0.f;
  const float M = mine ? part[lane * step + 64 + c] : -__builtin_inff();
  float top = m, topM = M;
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) {
    top = fmaxf(top, __shfl_xor(top, s, 64));
    topM = fmaxf(topM, __shfl_xor(topM, s, 64));
  }
  float l = weight(m, top) * ls;
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) l += __shfl_xor(l, s, 64);
  const float f = weight(M, topM);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int k = 0; k < kMaxSplits / kGroups; ++k) {
    const int s = k * kGroups + g;
    const float fs = __shfl(f, s < a.splits ? s : 0, 64);
    if (s < a.splits) {
      const float4 x = *reinterpret_cast<const float4*>(part + s * step + 96 + c * D + 4 * d);
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
  const Result<T> result(top, l, topM);
  const QRow w(a, hk, r / 32, c);
  *reinterpret_cast<uint2*>(a.o + at3(a.ost, b, w.t, w.h) + 4 * d) =
      make_uint2(Ops<T>::pack(result(o.x), result(o.y)), Ops<T>::pack(result(o.z), result(o.w)));
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

int check(const GdnCache8Params& P) {
  if (P.B <= 0 || P.S <= 0 || P.S > 0x3fffffff || P.Hk <= 0) return GDN_ERR_BAD_SHAPE;
  if (P.D != 64 && P.D != 128) return GDN_ERR_UNSUPPORTED;
  return GDN_OK;
}
int check_decode(const GdnCache8Params& P) {
  if (const int st = check(P)) return st;
  if (P.T < 1 || P.T > kMaxT || P.Hq <= 0 || P.Hq % P.Hk != 0 || P.window < 1 || P.sinks < 0) return GDN_ERR_BAD_SHAPE;
  if ((int64_t)P.B * P.Hq > 0x7fffffff / (2 * kMaxT)) return GDN_ERR_BAD_SHAPE;   // rows are 32-bit
  if (P.dtype != GDN_DTYPE_F16 && P.dtype != GDN_DTYPE_BF16) return GDN_ERR_BAD_DTYPE;
  return GDN_OK;
}

// Rows of n elements of es bytes, 16 bytes at a time; a stride that no index uses
// may be anything.
bool rows_ok(const void* p, const int64_t* s, int64_t b, int64_t t, int64_t h, int es) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (b <= 1 || s[0] * es % 16 == 0) && (t <= 1 || s[1] * es % 16 == 0) &&
         (h <= 1 || s[2] * es % 16 == 0);
}
bool cache_ok(const GdnCache8Params& P) {
  return rows_ok(P.k_cache, P.kc_stride, P.B, P.S, P.Hk, 1) && rows_ok(P.v_cache, P.vc_stride, P.B, P.S, P.Hk, 1);
}

int row_tiles(const GdnCache8Params& P) { return (P.Hq / P.Hk * P.T + 31) / 32; }

// Workgroups a sequence and key head: one a CU over the tiles that the longest
// sequence can have, at least a tile a wave; up to 2 tiles a wave stay in one
// workgroup, without a second kernel (one sequence in us, one workgroup and joined: 512
// keys 9.8 and 11.1, 1024 keys 13.6 and 11.3, 2048 keys 20.3 and 11.6).
int splits_of(const GdnCache8Params& P) {
  const int64_t keys = std::min<int64_t>(P.S, (int64_t)P.window + P.T - 1 + P.sinks);
  const int64_t tiles = keys / kDN + 2;
  if (tiles <= 2 * kDWaves + 2) return 1;
  const int64_t units = (int64_t)P.B * P.Hk * row_tiles(P);
  const int64_t want = (256 + units - 1) / units;
  return (int)std::max<int64_t>(1, std::min({want, (tiles + kDWaves - 1) / kDWaves, (int64_t)kMaxSplits}));
}

Args args_of(const GdnCache8Params& P) {
  Args a = {};
  a.k = P.k;
  a.v = P.v;
  a.q = static_cast<const uint16_t*>(P.q);
  a.o = static_cast<uint16_t*>(P.o);
  a.kc = static_cast<uint8_t*>(P.k_cache);
  a.vc = static_cast<uint8_t*>(P.v_cache);
  a.ks = P.k_scale;
  a.vs = P.v_scale;
  a.lens = P.cache_seqlens;
  for (int d = 0; d < 3; ++d) {
    a.kst[d] = P.k_stride[d];
    a.vst[d] = P.v_stride[d];
    a.qst[d] = P.q_stride[d];
    a.ost[d] = P.o_stride[d];
    a.kcst[d] = P.kc_stride[d];
    a.vcst[d] = P.vc_stride[d];
    a.ksst[d] = P.ks_stride[d];
    a.vsst[d] = P.vs_stride[d];
  }
  a.B = P.B;
  a.T = P.T;
  a.S = P.S;
  a.Hk = P.Hk;
  return a;
}

// launch(args, grid) for keys and values of all rows, as many launches as they take
// (see grid_fits).
template <typename F>
int by_rows(Args a, int64_t rows, int D, F launch) {
  constexpr uint32_t kMost = 1 << 22;
  static_assert(2 * kMost <= 0xffffffffu / kRowNT, "one launch holds them");
  const int64_t per = kRowNT / (D / 16);
  const uint32_t all = (uint32_t)((rows + per - 1) / per);
  for (; a.first < all; a.first += kMost) {
    launch(a, dim3(std::min(kMost, all - a.first), 2));
    if (const int st = (int)hipGetLastError()) return st;
  }
  return GDN_OK;
}
template <typename E>
int launch_write(const Args& a, int D, hipStream_t s) {
  return by_rows(a, (int64_t)a.B * a.T * a.Hk, D, [&](const Args& b, dim3 grid) {
    if (D == 128) hipLaunchKernelGGL((write_kernel<E, 128>), grid, dim3(kRowNT), 0, s, b);
    else hipLaunchKernelGGL((write_kernel<E, 64>), grid, dim3(kRowNT), 0, s, b);
  });
}
template <typename E>
int launch_read(const Args& a, int D, hipStream_t s) {
  return by_rows(a, (int64_t)a.B * a.S * a.Hk, D, [&](const Args& b, dim3 grid) {
    if (D == 128) hipLaunchKernelGGL((read_kernel<E, 128>), grid, dim3(kRowNT), 0, s, b);
    else hipLaunchKernelGGL((read_kernel<E, 64>), grid, dim3(kRowNT), 0, s, b);
  });
}
template <typename T, int D>
void launch_decode(const Args& a, hipStream_t s) {
  const uint32_t units = (uint32_t)a.B * a.Hk * a.tiles_r;
  hipLaunchKernelGGL((decode_kernel<T, D>), dim3(units * a.splits), dim3(kNT), 0, s, a);
  if (a.splits > 1) hipLaunchKernelGGL((join_kernel<T, D>), dim3((uint32_t)(a.B * a.Hk * a.G * a.T)), dim3(kJT), 0, s, a);
}

}  // namespace cache8
}  // namespace gdn

using namespace gdn;
using namespace gdn::cache8;

extern "C" {

int gdn_cache8_write_launch(const GdnCache8Params* prm, void* stream) {
  if (prm == nullptr) return GDN_ERR_NULL_POINTER;
  const GdnCache8Params& P = *prm;
  if (const int st = check(P)) return st;
  if (P.T < 0) return GDN_ERR_BAD_SHAPE;
  if (!scan_dtype_ok(P.dtype)) return GDN_ERR_BAD_DTYPE;
  if (P.T == 0) return GDN_OK;
  if (P.k == nullptr || P.v == nullptr || P.k_cache == nullptr || P.v_cache == nullptr || P.k_scale == nullptr ||
      P.v_scale == nullptr || P.cache_seqlens == nullptr)
    return GDN_ERR_NULL_POINTER;
  const int es = dtype_bytes(P.dtype);
  if (!rows_ok(P.k, P.k_stride, P.B, P.T, P.Hk, es) || !rows_ok(P.v, P.v_stride, P.B, P.T, P.Hk, es) || !cache_ok(P))
    return GDN_ERR_MISALIGNED;
  if ((int64_t)P.T * P.Hk > 0x7fffffff / P.B) return GDN_ERR_BAD_SHAPE;      // rows are 32-bit
  const Args a = args_of(P);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (P.dtype == GDN_DTYPE_F16) return launch_write<f16>(a, P.D, s);
  if (P.dtype == GDN_DTYPE_BF16) return launch_write<bf16_t>(a, P.D, s);
  return launch_write<float>(a, P.D, s);
}

int gdn_cache8_read_launch(const GdnCache8Params* prm, void* stream) {
  if (prm == nullptr) return GDN_ERR_NULL_POINTER;
  const GdnCache8Params& P = *prm;
  if (const int st = check(P)) return st;
  if (!scan_dtype_ok(P.dtype)) return GDN_ERR_BAD_DTYPE;
  if (P.k == nullptr || P.v == nullptr || P.k_cache == nullptr || P.v_cache == nullptr || P.k_scale == nullptr ||
      P.v_scale == nullptr)
    return GDN_ERR_NULL_POINTER;
  const int es = dtype_bytes(P.dtype);
  if (!rows_ok(P.k, P.k_stride, P.B, P.S, P.Hk, es) || !rows_ok(P.v, P.v_stride, P.B, P.S, P.Hk, es) || !cache_ok(P))
    return GDN_ERR_MISALIGNED;
  if ((int64_t)P.S * P.Hk > 0x7fffffff / P.B) return GDN_ERR_BAD_SHAPE;      // rows are 32-bit
  const Args a = args_of(P);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (P.dtype == GDN_DTYPE_F16) return launch_read<f16>(a, P.D, s);
  if (P.dtype == GDN_DTYPE_BF16) return launch_read<bf16_t>(a, P.D, s);
  return launch_read<float>(a, P.D, s);
}

int64_t gdn_cache8_decode_workspace_size(const GdnCache8Params* prm) {
  if (prm == nullptr || check_decode(*prm) != GDN_OK) return -1;
  const int splits = splits_of(*prm);
  return splits == 1 ? 0 : (int64_t)prm->B * prm->Hk * row_tiles(*prm) * splits * 32 * (prm->D + 3) * 4;
}

int gdn_cache8_decode_launch(const GdnCache8Params* prm, void* stream) {
  if (prm == nullptr) return GDN_ERR_NULL_POINTER;
  const GdnCache8Params& P = *prm;
  if (const int st = check_decode(P)) return st;
  if (P.q == nullptr || P.o == nullptr || P.k_cache == nullptr || P.v_cache == nullptr || P.k_scale == nullptr ||
      P.v_scale == nullptr || P.cache_seqlens == nullptr)
    return GDN_ERR_NULL_POINTER;
  if (!rows16(P.q, P.q_stride, P.B, P.T, P.Hq) || !rows16(P.o, P.o_stride, P.B, P.T, P.Hq) || !cache_ok(P))
    return GDN_ERR_MISALIGNED;
  const int splits = splits_of(P);
  if (!grid_fits((int64_t)P.B * P.Hk * row_tiles(P) * splits, kNT) ||
      (splits > 1 && !grid_fits((int64_t)P.B * P.Hq * P.T, kJT)))
    return GDN_ERR_BAD_SHAPE;
  const int64_t need = gdn_cache8_decode_workspace_size(prm);
  if (need > 0 && (P.workspace == nullptr || P.workspace_bytes < need ||
                   reinterpret_cast<uintptr_t>(P.workspace) % 256 != 0))
    return GDN_ERR_WORKSPACE;
  Args a = args_of(P);
  a.part = static_cast<float*>(P.workspace);
  a.G = P.Hq / P.Hk;
  a.tiles_r = row_tiles(P);
  a.splits = splits;
  a.window = P.window;
  a.sinks = P.sinks;
  split_scale(P.scale, a.scale_log2, a.flip);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (P.dtype == GDN_DTYPE_F16) P.D == 128 ? launch_decode<f16, 128>(a, s) : launch_decode<f16, 64>(a, s);
  else P.D == 128 ? launch_decode<bf16_t, 128>(a, s) : launch_decode<bf16_t, 64>(a, s);
  return (int)hipGetLastError();
}

}  // extern "C"
