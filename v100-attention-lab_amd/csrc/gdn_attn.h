// Shared parts of the windowed attention kernels: operand types, the LDS tile
// of key or query rows, the visible range of keys, and the map from workgroups
// to sequences.
//
// Matrix products are v_mfma_f32_32x32x16: lane l supplies row (A) or column
// (B) l % 32 and 8 contraction slots of half l / 32; accumulator register r
// holds column l % 32, row 8 (r / 4) + 4 (l / 32) + r % 4.  Contraction order
// is free, so a product P whose rows are the contraction of the next product
// enters it straight from its accumulators: registers 8 s .. 8 s + 7 are the
// slots of step s, contraction index 16 s + 8 (i / 4) + 4 (l / 32) + i % 4,
// and the other operand is read in that order by two transposing LDS reads.
#pragma once

#include "gdn_row_io.h"

namespace gdn {
namespace attn {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_void;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// fp16 probabilities are kept times 2^7: with the running maximum at most 2^8
// behind (kLazy) none overflows, and 2^-21 of the largest is still normal.
template <typename T>
struct Ops;
template <>
struct Ops<f16> {
  typedef f16x8 Vec;
  static constexpr float kShift = 7.f;
  static constexpr uint32_t kExp = 0x7c00u;
  static constexpr uint32_t kOne = 0x3c00u;
  __device__ static __forceinline__ f32x16 mfma(Vec a, Vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  __device__ static __forceinline__ uint32_t pack(float a, float b) {
    typedef f16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, f16x2{(f16)a, (f16)b});
  }
};
template <>
struct Ops<bf16_t> {
  typedef bf16x8 Vec;
  static constexpr float kShift = 0.f;
  static constexpr uint32_t kExp = 0x7f80u;
  static constexpr uint32_t kOne = 0x3f80u;
  __device__ static __forceinline__ f32x16 mfma(Vec a, Vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  __device__ static __forceinline__ uint32_t pack(float a, float b) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
  }
};
// How far (in powers of 2) the row maximum may rise before the accumulators
// are rescaled.
constexpr float kLazy = 8.f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// The value of the lane in the other half (l ^ 32), without a way through LDS.
__device__ __forceinline__ float swap_halves(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}
// The larger of the two halves' values, in both.
__device__ __forceinline__ float max_halves(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Registers 8 s .. 8 s + 7 of a product as the operand of the next one.
template <typename T>
__device__ __forceinline__ typename Ops<T>::Vec acc_operand(const f32x16& p, int s) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = Ops<T>::pack(p[8 * s + 2 * i], p[8 * s + 2 * i + 1]);
  typename Ops<T>::Vec v;
  __builtin_memcpy(&v, w, 16);
  return v;
}

// N products, each with its LDS operand read AHEAD products before it: left
// alone the compiler puts each read right before its product, and the wave
// waits for it there.
template <int N, int AHEAD, typename Load, typename Use>
__device__ __forceinline__ void fed_products(Load load, Use use) {
  decltype(load(0)) f[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) f[i] = load(i);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    use(i, f[i % AHEAD]);
    if (i + AHEAD < N) f[i % AHEAD] = load(i + AHEAD);
    __builtin_amdgcn_sched_barrier(0);
  }
}
struct Quad {
  uint4 a, b, c, d;
};

// Accumulator row of register r.
__device__ __forceinline__ int acc_row(int r, int half) { return 8 * (r >> 2) + 4 * half + (r & 3); }

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) float lds_f32;

// LDS byte address of a shared array.
__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)(lds_void*)p; }

// 16 bytes per lane from global memory to LDS at `at` + 16 * lane (at
// uniform).  Written out, so that the compiler does not take every LDS read
// that follows for a reader of these bytes and wait for them there: a buffer
// is read only after dma_wait() in every wave that filled it and a barrier.
// The instruction has no result registers, and a count of outstanding loads
// that the compiler waits for is only met later for it, never earlier.
__device__ __forceinline__ void dma16(const void* src, uint32_t at) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(at) : "memory", "m0");
}
// the same from a uniform base and a byte offset per lane
__device__ __forceinline__ void dma16(const void* base, uint32_t ofs, uint32_t at) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(ofs), "s"(base), "s"(at)
               : "memory", "m0");
}
// 4 bytes per lane from global memory to LDS at `at` + 4 * lane (dma16's rules).
__device__ __forceinline__ void dma4(const void* src, uint32_t at) {
  at = __builtin_amdgcn_readfirstlane(at);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(at) : "memory", "m0");
}
// Every load of this wave so far, from memory and from LDS, is done.
__device__ __forceinline__ void dma_wait() {
  __builtin_amdgcn_s_waitcnt(7 << 4);   // vmcnt(0) lgkmcnt(0)
  asm volatile("" ::: "memory");
}
// A value that is the same in every lane, in scalar registers.
__device__ __forceinline__ int64_t uniform64(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ const uint16_t* uniform_ptr(const uint16_t* p) {
  return (const uint16_t*)(uintptr_t)uniform64((int64_t)(uintptr_t)p);
}

// Rows of D 16-bit elements in LDS: groups of 1 KB (kGroup rows, one LDS-DMA of
// a wave) 1040 bytes apart, in 16-byte pieces; piece c of row r lies at place
// c ^ swz(r) of the row.  16 rows at one piece (a product's operand) and 4 rows
// at 64 neighbouring bytes (a transposing read) then each cover all banks once,
// and a lane's addresses differ by constants but for four of them.
template <int D>
struct Tile {
  static constexpr int kPieces = D / 8, kRowBytes = 2 * D, kGroup = 1024 / kRowBytes;
  static constexpr uint32_t kGroupBytes = 1040;
  static constexpr uint32_t bytes(int rows) { return rows / kGroup * kGroupBytes; }   // rows: a multiple of kGroup
  __device__ static __forceinline__ int swz(int row) {
    return D == 128 ? (row & 3) << 2 : (((row >> 1) & 1) << 2) | (((row >> 2) & 1) << 1);
  }
  __device__ static __forceinline__ uint32_t place(int row, int piece) {
    return row / kGroup * kGroupBytes + row % kGroup * kRowBytes + 16 * (piece ^ swz(row));
  }
  // A lane's byte offsets in a tile.
  uint32_t row[4], col[D / 32];
  __device__ __forceinline__ explicit Tile(int lane) {
    const int h = lane >> 5, a = lane & 15;
#pragma unroll
    for (int j = 0; j < 4; ++j) row[j] = place(lane & 31, h + (D == 128 ? 4 : 2) * j);
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
      col[dt] = place(4 * h + (a >> 2), 4 * dt + 2 * ((lane >> 4) & 1) + ((a & 3) >> 1)) + 8 * (a & 1);
  }
  // Operand of step i: row r0 + l % 32, elements 16 i + 8 (l / 32) .. (r0 a
  // multiple of kGroup).
  __device__ __forceinline__ uint4 row8(uint32_t tile, int i, int r0 = 0) const {
    const u32x4 v = *(const lds_u32x4*)(tile + row[D == 128 ? i >> 1 : i] + (D == 128 ? 32 * (i & 1) : 0) + bytes(r0));
    return make_uint4(v[0], v[1], v[2], v[3]);
  }
  // Transposed operand: lane l receives element 32 dt + l % 32 of rows k0 + 4 h
  // + {0..3} and k0 + 8 + 4 h + {0..3}, h = l / 32 (k0 a multiple of 16).
  // ds_read_b64_tr_b16: lane i of 16 receives halfword i % 4 of the 8 bytes
  // addressed by lanes 4 j + i / 4, j = 0..3.
  __device__ __forceinline__ uint4 col8(uint32_t tile, int dt, int k0) const {
    union {
      s16x4 h[2];
      uint4 v;
    } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + col[dt] + bytes(k0)));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + col[dt] + bytes(k0 + 8)));
    return u.v;
  }
};

// Copies rows row0 .. row0 + ROWS - 1 of a [rows, D] matrix (row stride ld
// elements) into a tile by LDS-DMA, NT threads; rows past the last one are
// copies of it.  A pass moves NT / kPieces rows (a multiple of kGroup, so a
// lane's piece is the same in every pass).
template <int D, int ROWS, int NT>
struct Copier {
  using TL = Tile<D>;
  static constexpr int kPass = NT / TL::kPieces, kPasses = ROWS / kPass;
  static_assert(kPass % TL::kGroup == 0 && ROWS % kPass == 0, "whole passes");
  const uint16_t* src;
  int64_t ld;
  int rows;          // of the matrix
  int row, piece;    // of this lane in the first pass
  uint32_t ofs;      // its byte offset where that fits 31 bits
  bool small;
  __device__ __forceinline__ Copier(const uint16_t* s, int64_t ld_, int rows_)
      : src(uniform_ptr(s)), ld(ld_), rows(__builtin_amdgcn_readfirstlane(rows_)) {
    const int tid = threadIdx.x % NT;
    row = tid / TL::kPieces;
    piece = (tid % TL::kPieces) ^ TL::swz(row);
    small = ld >= 0 && ld < (1 << 24);
    ofs = (uint32_t)(row * (uint32_t)ld * 2u) + 16u * piece;
  }
  __device__ __forceinline__ void operator()(uint32_t tile, int row0) const {
    constexpr uint32_t kStep = NT / 64 * TL::kGroupBytes;
    const uint32_t at = tile + TL::kGroupBytes * __builtin_amdgcn_readfirstlane(threadIdx.x % NT / 64);
    if (small && row0 + ROWS <= rows) {
#pragma unroll
      for (int i = 0; i < kPasses; ++i)
        dma16(src + (int64_t)(row0 + i * kPass) * ld, ofs, at + i * kStep);
    } else {
      int r = row0 + row;
      asm volatile("" : "+v"(r));     // (not kept in registers from tile to tile)
#pragma unroll
      for (int i = 0; i < kPasses; ++i)
        dma16(src + (int64_t)min(r + i * kPass, rows - 1) * ld + 8 * piece, at + i * kStep);
    }
  }
};

template <typename T>
__device__ __forceinline__ typename Ops<T>::Vec as_vec(const uint4& u) {
  return __builtin_bit_cast(typename Ops<T>::Vec, u);
}

// ---------------------------------------------------------------------------
// sequences
// ---------------------------------------------------------------------------

struct Seq {
  int b;             // batch index
  int64_t q0, k0;    // first query and key row along t
  int nq, nk;        // rows
};

struct SeqArgs {
  const int64_t* cu;
  int Tq, Tk, N;
};

__device__ __forceinline__ int64_t clamp_row(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }

__device__ __forceinline__ Seq get_seq(const SeqArgs& a, int i) {
  Seq s;
  if (a.cu == nullptr) {
    s.b = i;
    s.q0 = s.k0 = 0;
    s.nq = a.Tq;
    s.nk = a.Tk;
  } else {
    const int64_t b = clamp_row(a.cu[i], 0, a.Tq), e = clamp_row(a.cu[i + 1], b, a.Tq);
    s.b = 0;
    s.q0 = s.k0 = uniform64(b);
    s.nq = s.nk = __builtin_amdgcn_readfirstlane((int)(e - b));
  }
  return s;
}

// The last of N packed sequences whose first(start row, sequence) is at most
// `at` (it rises along the sequences).
template <typename First>
__device__ __forceinline__ int last_seq(const SeqArgs& a, int at, First first) {
  int lo = 0, hi = a.N;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first(clamp_row(a.cu[mid], 0, a.Tq), mid) <= at) lo = mid; else hi = mid;
  }
  return lo;
}

// Blocks of `rows` rows: a dense sequence has ceil(T / rows); packed sequence
// i has its first at slot start / rows + i, which leaves each room for
// ceil(len / rows) blocks.  Returns the sequence and the block in it (which
// may lie past its end: nothing to do).
__device__ __forceinline__ int find_block(const SeqArgs& a, int slot, int rows, int nblk, int& block) {
  if (a.cu == nullptr) {
    block = slot % nblk;
    return slot / nblk;
  }
  auto first = [&](int64_t start, int i) { return (int)((uint32_t)start / (uint32_t)rows) + i; };
  const int i = last_seq(a, slot, first);
  block = slot - first(clamp_row(a.cu[i], 0, a.Tq), i);
  return i;
}

// Key tiles of TK keys that query positions [p0, p1] see: tiles [0, ns) of the
// first keys, then [w0, w1).
struct KeyRange {
  int ns, w0, n;
  __device__ __forceinline__ KeyRange(int p0, int p1, int nk, int window, int sinks, int tk) {
    const int lo = (int)max((int64_t)p0 - window + 1, (int64_t)0);
    const int hi = min(p1, nk - 1);
    w0 = lo / tk;
    const int w1 = hi < lo ? w0 : hi / tk + 1;
    const int s = min(sinks, max(hi + 1, 0));
    ns = min((s + tk - 1) / tk, w0);
    n = ns + (w1 - w0);
  }
  __device__ __forceinline__ int tile(int i) const { return i < ns ? i : w0 + (i - ns); }
};

// Visibility of the accumulator rows of a lane whose column is query position
// p: row c = 32 t + 8 (r / 4) + r % 4 of a key tile from j0 (the half's 4 rows
// folded in) is seen where c <= hi and (c > lo or c < first).  `ends` and
// `starts` say (for the wave) whether any row's visible keys end, or start,
// inside the tile, `firsts` whether the first keys reach into it.
struct Mask {
  int hi, lo, first;
  bool ends, starts, firsts;
  // The tile's keys [j0, j0 + n), the wave's positions [p0, p1].
  __device__ __forceinline__ Mask(int p, int j0, int n, int half, int nk, int p0, int p1, int window, int sinks) {
    const int j = j0 + 4 * half;
    hi = min(p, nk - 1) - j;
    lo = (int)max((int64_t)p - window, (int64_t)-1) - j;
    first = sinks - j;
    ends = j0 + n - 1 > p0 || j0 + n > nk;
    starts = p1 - j0 >= window && j0 + n > sinks;
    firsts = j0 < sinks;
  }
  __device__ __forceinline__ bool any() const { return ends || starts; }
  __device__ __forceinline__ static int at(int t, int r) { return 32 * t + 8 * (r >> 2) + (r & 3); }
  __device__ __forceinline__ bool operator()(int t, int r) const {
    const int c = at(t, r);
    return (c <= hi) & ((c > lo) | (c < first));
  }
  // x where it is seen, else `hidden`
  template <int KS>
  __device__ __forceinline__ void apply(f32x16 (&x)[KS], float hidden) const {
    if (ends) {
#pragma unroll
      for (int t = 0; t < KS; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[t][r] = at(t, r) <= hi ? x[t][r] : hidden;
    }
    if (starts) {
      if (firsts) {
#pragma unroll
        for (int t = 0; t < KS; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) x[t][r] = (at(t, r) > lo) | (at(t, r) < first) ? x[t][r] : hidden;
      } else {
#pragma unroll
        for (int t = 0; t < KS; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) x[t][r] = at(t, r) > lo ? x[t][r] : hidden;
      }
    }
  }
};

// An operand with its infinities and NaN replaced by zero.
template <typename T>
__device__ __forceinline__ uint4 only_finite(const uint4& x) {
  constexpr uint32_t E = Ops<T>::kExp;
  uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((w[i] & E) == E) w[i] &= 0xffff0000u;
    if ((w[i] & (E << 16)) == (E << 16)) w[i] &= 0x0000ffffu;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// A product over rows of which some are hidden from some columns adds 0 times
// what the hidden places hold.  Where that is an infinity or NaN, the tile is
// made finite before the product: these look at and change N groups of a tile,
// one wave, a group a step.
template <typename T, int N>
__device__ __forceinline__ bool not_finite(uint32_t at, int lane) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  u16x2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const u32x4 x = *(const lds_u32x4*)(at + i * 1040 + 16 * lane);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t w = x[e] & 0x7fff7fffu;
      m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w));
    }
  }
  return __any(m[0] >= Ops<T>::kExp || m[1] >= Ops<T>::kExp);
}
template <typename T, int N>
__device__ __forceinline__ void make_finite(uint32_t at, int lane) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    lds_u32x4* p = (lds_u32x4*)(at + i * 1040 + 16 * lane);
    const u32x4 x = *p;
    const uint4 y = only_finite<T>(make_uint4(x[0], x[1], x[2], x[3]));
    *p = u32x4{y.x, y.y, y.z, y.w};
  }
}

// An operand with its sign turned where flip = 0x80008000 (else 0).
template <typename T>
__device__ __forceinline__ typename Ops<T>::Vec signed_vec(const uint4& x, uint32_t flip) {
  return as_vec<T>(make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip));
}

// 32 query rows of a wave (lane l: row l % 32) against key tiles of 32 KS rows
// (KS up to MAX): the running maximum m (in powers of 2, as the scores are),
// this lane's share l of the sum, and O^T.
template <typename T, int D, int MAX>
struct Rows {
  using O = Ops<T>;
  using Vec = typename O::Vec;
  using TL = Tile<D>;
  f32x16 acc[D / 32] = {};
  float m = -__builtin_inff(), l = 0.f;

  Vec pf[2 * MAX];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = f32x16{};
    m = -__builtin_inff();
    l = 0.f;
  }

  // Scores and probabilities of one tile.
  template <int KS>
  __device__ __forceinline__ void scores(const Vec (&qf)[D / 16], const TL& tl, uint32_t kt, const Mask& seen,
                                         float scale_log2) {
    f32x16 s[KS] = {};
    fed_products<KS * D / 16, 4>([&](int i) { return tl.row8(kt, i / KS, 32 * (i % KS)); },
                                 [&](int i, const uint4& x) { s[i % KS] = O::mfma(as_vec<T>(x), qf[i / KS], s[i % KS]); });
    seen.apply<KS>(s, -__builtin_inff());
    float mx = s[0][0];
#pragma unroll
    for (int t = 0; t < KS; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[t][r]);
    mx = max_halves(mx) * scale_log2;
    if (__any(mx > m + kLazy)) {
      // each row by its own scores, so that no row's bits depend on another's
      const float mn = mx > m + kLazy ? mx : m;
      const float f = mn == m ? 1.f : exp2_fast(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] *= f;
    }
    const float mb = m == -__builtin_inff() ? 0.f : O::kShift - m;
#pragma unroll
    for (int t = 0; t < KS; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[t][r] = exp2_fast(__builtin_fmaf(s[t][r], scale_log2, mb));
        l += s[t][r];
      }
#pragma unroll
    for (int t = 0; t < 2 * KS; ++t) pf[t] = acc_operand<T>(s[t >> 1], t & 1);
  }

  // What the infinities and NaN of a value tile add to the rows that see them:
  // two products of 0/1 matrices say which sums meet a +inf or NaN, and which a
  // -inf or NaN.
  template <int KS>
  __device__ __forceinline__ void add_not_finite(const Mask& seen, const TL& tl, uint32_t vt) {
    constexpr uint32_t E = O::kExp, ONE = O::kOne;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
      f32x16 up = {}, dn = {};
#pragma unroll
      for (int s = 0; s < 2 * KS; ++s) {
        const uint4 raw = tl.col8(vt, dt, 16 * s);
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        uint32_t u[4], d[4], one[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          u[i] = d[i] = one[i] = 0;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t x = (w[i] >> (16 * h)) & 0xffffu, mag = x & 0x7fffu;
            if (mag > E || x == E) u[i] |= ONE << (16 * h);
            if (mag > E || x == (E | 0x8000u)) d[i] |= ONE << (16 * h);
            if (seen(s >> 1, 8 * (s & 1) + 2 * i + h)) one[i] |= ONE << (16 * h);
          }
        }
        const Vec sv = as_vec<T>(make_uint4(one[0], one[1], one[2], one[3]));
        up = O::mfma(as_vec<T>(make_uint4(u[0], u[1], u[2], u[3])), sv, up);
        dn = O::mfma(as_vec<T>(make_uint4(d[0], d[1], d[2], d[3])), sv, dn);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        acc[dt][r] += up[r] > 0.f ? __builtin_inff() : 0.f;
        acc[dt][r] -= dn[r] > 0.f ? __builtin_inff() : 0.f;
      }
    }
  }

  // O^T += V^T P^T
  template <int KS>
  __device__ __forceinline__ void values(const TL& tl, uint32_t vt) {
    constexpr int N = D / 32;
    fed_products<2 * KS * N, 4>([&](int i) { return tl.col8(vt, i % N, 16 * (i / N)); },
                                [&](int i, const uint4& x) { acc[i % N] = O::mfma(as_vec<T>(x), pf[i / N], acc[i % N]); });
  }
};

// Whether every key of [j0, j1] is visible to every position of [p0, p1].
__device__ __forceinline__ bool all_visible(int j0, int j1, int p0, int p1, int window, int sinks) {
  return j1 <= p0 && (p1 - j0 < window || j1 < sinks);
}
// Whether none is.
__device__ __forceinline__ bool none_visible(int j0, int j1, int p0, int p1, int window, int sinks) {
  return j0 > p1 || (p0 - j1 >= window && j0 >= sinks);
}

// Rows of D 16-bit elements are read 16 bytes at a time; a stride that no
// index uses may be anything.
inline bool rows16(const void* p, const int64_t* s, int64_t b, int64_t t, int64_t h) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (b <= 1 || s[0] % 8 == 0) && (t <= 1 || s[1] % 8 == 0) &&
         (h <= 1 || s[2] % 8 == 0);
}

// The scale in powers of 2 and the sign that goes into q: the running maximum
// is taken of the products, so the factor after it is positive (of a scale of
// zero, so small that every visible score is zero and hidden ones stay -inf).
inline void split_scale(float scale, float& log2, uint32_t& flip) {
  flip = scale < 0.f ? 0x80008000u : 0u;
  log2 = scale == 0.f ? 1e-30f : (scale < 0.f ? -scale : scale) * kLog2e;
}

int check_attn(const GdnAttnParams& P);

}  // namespace attn
}  // namespace gdn
