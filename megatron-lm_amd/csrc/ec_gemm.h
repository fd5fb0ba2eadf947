// ec_gemm.h — matrix products on the matrix cores for ec_ff.hip and ec_ortho.hip.
//
// C[m][n] = sum over k of A(m, k) * B(n, k).  A workgroup computes a BM x BN tile, a wave a
// WM x WN part of it, in fp32 accumulators.  A step of the loop over k covers 128 bytes of a
// row: 64 16-bit values, 32 fp32 ones, or 32 pairs (below).  Its BM + BN rows go from memory
// straight to LDS (buffer_load ... lds, 16 bytes a lane), one step ahead of the products, and
// from LDS to fragments of 16 rows by 16 bytes a lane.
//
// An operand lies in memory in one of two ways: along k ([rows][k], the tile in LDS is
// [rows][128 bytes]), or across it ([k][rows], the tile is [k][rows], and the 16-bit fragments are
// transposed on the way out of LDS, by ds_read_b64_tr_b16: of 16 lanes that give the
// addresses of four times 16 values, lane i gets the four i-th ones).  So no operand is
// ever transposed in memory.  16-byte chunks are exchanged within their row of the tile by an
// exclusive or with a function of the row, so that neither form of reading meets bank conflicts.
//
// Ends: the buffer's size bounds the reads, which give zeros past it; chunks past the end of a row are
// pointed there.  So operands are 16-byte aligned, rows a multiple of 16 bytes apart, and the
// dimension along a row a multiple of 16 bytes (or padded to one, with zeros if it is k).
//
// Pairs: a value as the sum of two fp16 ones, 22 bits of significand: eight high parts, then the
// eight low parts, in 32 bytes.  A product of two pairs takes three of the matrix cores' products
// (the low parts' is below the fp32 accumulator's rounding), at three tenths of the time of fp32 products.  The matrix
// cores truncate where they add to an accumulator, so the two small products have accumulators of their own, which
// are added at the end: five Newton-Schulz steps on 1001 x 777 are 3.5e-6 off with one accumulator, 2.0e-6 with two, and
// those of fp32 products 2.3e-6.
#pragma once

#include <algorithm>

#include "ec_types.h"
#include "routes.h"

namespace ec {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f8 __attribute__((ext_vector_type(8)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));

template <typename T>
using local = __attribute__((address_space(3))) T;

struct pair_t {   // 4 bytes of a matrix of pairs
  uint32_t bits;
};

constexpr int kRowBytes = 128;   // of a step along k
constexpr uint32_t kNowhere = 0x80000000u;   // an offset past any buffer below

template <typename T>
struct Kind {   // bf16, fp16
  static constexpr int kBytes = 2, kSubs = 2, kParts = 1;
};
template <>
struct Kind<float> {
  static constexpr int kBytes = 4, kSubs = 2, kParts = 1;
};
template <>
struct Kind<pair_t> {
  static constexpr int kBytes = 4, kSubs = 1, kParts = 2;
};

template <typename T>
struct Frag {
  s8 part[Kind<T>::kParts];
};

// acc[m = lane % 16][n = 4 (lane / 16) + i] += A B: the second operand's rows go along the accumulators
// of a lane, so that a lane stores four neighbours of a row of C.
template <typename T>
__device__ __forceinline__ void mma(f4& acc, const Frag<T>& a, const Frag<T>& b) {
  typedef bf16_t __attribute__((ext_vector_type(8))) b8;
  typedef fp16_t __attribute__((ext_vector_type(8))) h8;
  if constexpr (__is_same(T, bf16_t)) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, b.part[0]),
                                                  __builtin_bit_cast(b8, a.part[0]), acc, 0, 0, 0);
  } else if constexpr (__is_same(T, fp16_t)) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, b.part[0]),
                                                 __builtin_bit_cast(h8, a.part[0]), acc, 0, 0, 0);
  } else if constexpr (__is_same(T, float)) {
    const f4 x = __builtin_bit_cast(f4, a.part[0]), y = __builtin_bit_cast(f4, b.part[0]);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(y[e], x[e], acc, 0, 0, 0);
  }
}

// The same of pairs: what the high parts give, and the rest.
__device__ __forceinline__ void mma_pairs(f4& acc, f4& rest, const Frag<pair_t>& a, const Frag<pair_t>& b) {
  typedef fp16_t __attribute__((ext_vector_type(8))) h8;
  const h8 ah = __builtin_bit_cast(h8, a.part[0]), al = __builtin_bit_cast(h8, a.part[1]);
  const h8 bh = __builtin_bit_cast(h8, b.part[0]), bl = __builtin_bit_cast(h8, b.part[1]);
  rest = __builtin_amdgcn_mfma_f32_16x16x32_f16(bl, ah, rest, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(bh, ah, acc, 0, 0, 0);
  rest = __builtin_amdgcn_mfma_f32_16x16x32_f16(bh, al, rest, 0, 0, 0);
}

// Which of a wave's 32 rows fragment h (0, 1) of a pair of fragments holds in lane i of 16:
// 8 (i / 4) + 4 h + i % 4, so that both accumulators of a lane together are eight neighbours of a row of C,
// 64 bytes of four lanes.

// The exclusive or on the 16-byte chunks of row r of a tile along k: i % 8 for the row above.
__device__ __forceinline__ uint32_t along_swizzle(uint32_t r) { return (r & 3) | (r >> 1 & 4); }

// That of row k of a tile across k: the rows that are read together, four neighbours, or for fp32 four that are
// four apart, are exchanged into different banks.
template <typename T>
__device__ __forceinline__ uint32_t across_swizzle(uint32_t k, uint32_t chunks) {
  const uint32_t f = __is_same(T, float) ? k >> 2 & 3 : along_swizzle(k);
  return (Kind<T>::kBytes == 4 ? (f >> 1) * 8 | (f & 1) : f * 4) & (chunks - 1);
}

// Fragment `block` (of 16 rows of the operand) of sub-step `sub` of a tile of ROWS rows.
template <typename T, int ROWS, bool ACROSS>
__device__ __forceinline__ Frag<T> read_frag(const local<char>* tile, int block, int sub) {
  constexpr int P = Kind<T>::kParts;
  const uint32_t l = threadIdx.x % 64, i = l % 16, q = l / 16, pair = block / 2 * 32, h = block % 2;
  Frag<T> f;
  if constexpr (!ACROSS) {
    const local<char>* row = tile + (pair + i / 4 * 8 + h * 4 + i % 4) * kRowBytes;
#pragma unroll
    for (int p = 0; p < P; ++p)
      f.part[p] = *(const local<s8>*)(row + (((sub * 4 + q) * P + p) ^ (i & 7)) * 16);
  } else if constexpr (__is_same(T, float)) {
    f4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t k = sub * 16 + 4 * q + e;
      const uint32_t chunk = (pair / 4 + i / 4 * 2 + h) ^ across_swizzle<T>(k, ROWS / 4);
      v[e] = *(const local<float>*)(tile + k * (ROWS * 4) + chunk * 16 + i % 4 * 4);
    }
    f.part[0] = __builtin_bit_cast(s8, v);
  } else {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      s4 half[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t k = sub * 32 + 8 * q + 4 * e + i / 4;
        const uint32_t chunk = ((pair / 8 + i % 4) * P + p) ^
                               across_swizzle<T>(k, ROWS * Kind<T>::kBytes / 16);
        half[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (local<s4>*)(tile + k * (ROWS * Kind<T>::kBytes) + chunk * 16 + h * 8));
      }
      f.part[p] = __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  return f;
}

// A value that is the same in every lane, for the scalar unit: buffers are described by scalars.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }

// An operand: `rows` of it and K values along k; consecutive rows of memory are ld bytes apart.
struct Operand {
  const char* p;
  uint64_t ld;
  uint32_t rows;
};

// 16 bytes a lane from the buffer at byte `offset` to LDS at `lds` + 16 * lane.  The nop stands
// between the write of m0 and its use.  (m0 is reserved: the compiler keeps nothing in it.)
__device__ __forceinline__ void to_lds(uint32_t lds, uint32_t offset, const i4& buffer) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds), "v"(offset), "s"(buffer)
               : "memory");
}

__device__ __forceinline__ uint32_t lds_address(const local<char>* p) { return (uint32_t)(uintptr_t)p; }

// Brings the ROWS rows of an operand's tile to LDS step by step.  DUAL: 32 rows of a first operand,
// 32 of a second one, and so on; both with the same number of rows, equally far apart.
template <typename T, int ROWS, int WAVES, bool ACROSS, bool DUAL>
struct Loader {
  static_assert(!(ACROSS && DUAL), "only operands along k are taken in turns");
  static constexpr int kLoads = ROWS * kRowBytes / (WAVES * 1024);
  static constexpr int kStep = kRowBytes / Kind<T>::kBytes;
  uint32_t offset[kLoads];
  uint64_t base, other;
  uint64_t ld;
  // bytes along k not yet brought, or rows across it; signed, as a saturating difference would
  // leave the scalar unit
  int32_t left;
  uint32_t last_row;   // byte offset of the tile's last row of memory, where it bounds the buffer
  uint32_t row_bytes;  // ACROSS: bytes of the tile's part of a row
  uint32_t wave;

  // up to the end of the last 16 bytes, or eight pairs
  static __device__ __forceinline__ uint32_t whole(uint32_t bytes) {
    constexpr uint32_t unit = 16 * Kind<T>::kParts;
    return (bytes + unit - 1) & ~(unit - 1);
  }

  // Along k, the chunk of its rows that a lane brings: they are a multiple of 16 rows apart.
  __device__ __forceinline__ uint32_t chunk() const {
    static_assert(WAVES % 2 == 0, "rows of one swizzle");
    return (threadIdx.x % 8) ^ along_swizzle(wave * 8 + threadIdx.x % 64 / 8);
  }

  __device__ __forceinline__ void init(const Operand& a, const Operand& b, uint32_t row0, uint32_t k,
                                       uint32_t w) {
    const uint32_t l = threadIdx.x % 64;
    wave = w;
    ld = a.ld;
    if constexpr (!ACROSS) {
      const uint32_t first = DUAL ? row0 / 2 : row0, most = DUAL ? ROWS / 2 : ROWS;
      base = (uint64_t)(uintptr_t)a.p + first * a.ld;
      other = DUAL ? (uint64_t)(uintptr_t)b.p + first * b.ld : 0;
      left = (int32_t)whole(k * Kind<T>::kBytes);
      last_row = (min(most, a.rows - first) - 1) * (uint32_t)ld;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const uint32_t r = (i * WAVES + wave) * 8 + l / 8;
        const uint32_t from = DUAL ? r / 64 * 32 + r % 32 : r;
        offset[i] = from * (uint32_t)ld + chunk() * 16;
      }
    } else {
      base = (uint64_t)(uintptr_t)a.p + (uint64_t)row0 * Kind<T>::kBytes;
      left = (int32_t)k;
      row_bytes = whole(min((uint32_t)ROWS, a.rows - row0) * Kind<T>::kBytes);
      constexpr uint32_t chunks = ROWS * Kind<T>::kBytes / 16;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const uint32_t slot = (i * WAVES + wave) * 64 + l, r = slot / chunks;
        const uint32_t c = slot % chunks ^ across_swizzle<T>(r, chunks);
        offset[i] = c * 16 < row_bytes ? r * (uint32_t)ld + c * 16 : kNowhere;
      }
    }
  }

  static __device__ __forceinline__ i4 buffer(uint64_t at, uint32_t bytes) {
    return i4{(int)(uint32_t)at, (int)((uint32_t)(at >> 32) & 0xffffu), (int)bytes, 0x00020000};
  }

  i4 one, two;         // what begin() describes: the next step's tile
  uint32_t to;         // and where it goes in LDS
  bool in;             // whether the lane's chunk of its rows is before their end

  // The next step's tile, to LDS at `lds`: begin(), then every bring(i).  At most kStages steps past the last.
  __device__ __forceinline__ void begin(uint32_t lds) {
    uint32_t bytes;   // 0 past the last step
    if constexpr (!ACROSS) {
      in = chunk() * 16 < (uint32_t)max(left, 0);
      bytes = left > 0 ? last_row + (uint32_t)left : 0;
      left -= kRowBytes;
    } else {
      bytes = left > 0 ? (uint32_t)(min(left, kStep) - 1) * (uint32_t)ld + row_bytes : 0;
      left -= kStep;
    }
    one = buffer(base, bytes);
    if (DUAL) two = buffer(other, bytes);
    to = lds + wave * 1024;
    const uint64_t step = ACROSS ? kStep * ld : kRowBytes;
    base += step;
    if (DUAL) other += step;
  }

  __device__ __forceinline__ void bring(int i) {
    const bool second = DUAL && ((i * WAVES + wave) / 4 & 1);
    to_lds(to + i * WAVES * 1024, ACROSS || in ? offset[i] : kNowhere, second ? two : one);
  }

  __device__ __forceinline__ void issue(uint32_t lds) {
    begin(lds);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) bring(i);
  }
};

// A tile's geometry: BM x BN by waves of WM x WN, STAGES steps of it in LDS.  The smaller a tile, the sooner a step is
// multiplied, so small ones are brought from further ahead.
template <int BM_, int BN_, int WM_, int WN_, int STAGES_>
struct Shape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, kStages = STAGES_;
  static constexpr int kWavesN = BN / WN, kWaves = (BM / WM) * kWavesN, kLanes = kWaves * 64;
  static constexpr int MI = WM / 16, NI = WN / 16;
  static constexpr int kPerSimd = 2;   // waves, at least
  static constexpr int kStage = (BM + BN) * kRowBytes, kLds = kStages * kStage;
};

typedef Shape<256, 256, 128, 64, 2> Large;    // 8 waves, a workgroup per CU
typedef Shape<128, 128, 64, 64, 2> Middle;    // 4 waves, two workgroups per CU
typedef Shape<64, 128, 32, 64, 3> Flat;       // 4 waves, two workgroups per CU
typedef Shape<64, 64, 32, 32, 3> Small;       // 4 waves, three workgroups per CU

template <class S>
struct Acc {
  f4 v[S::MI][S::NI];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < S::MI; ++i)
#pragma unroll
      for (int j = 0; j < S::NI; ++j) v[i][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  __device__ __forceinline__ void add(const Acc& x) {
#pragma unroll
    for (int i = 0; i < S::MI; ++i)
#pragma unroll
      for (int j = 0; j < S::NI; ++j) v[i][j] += x.v[i][j];
  }

  // f(m, n, values): row m and columns n ... n + 7 of the tile.
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    const uint32_t l = threadIdx.x % 64, w = threadIdx.x / 64, i = l % 16;
    const uint32_t m0 = w / S::kWavesN * S::WM + i / 4 * 8 + i % 4;
    const uint32_t n0 = w % S::kWavesN * S::WN + l / 16 * 8;
#pragma unroll
    for (int r = 0; r < S::MI; ++r)
#pragma unroll
      for (int j = 0; j < S::NI; j += 2) f(m0 + r / 2 * 32 + r % 2 * 4, n0 + j * 16, pair(r, j));
  }

  // The values become f(m, n).
  template <typename F>
  __device__ __forceinline__ void start(F f) {
    const uint32_t l = threadIdx.x % 64, w = threadIdx.x / 64, i = l % 16;
    const uint32_t m0 = w / S::kWavesN * S::WM + i / 4 * 8 + i % 4;
    const uint32_t n0 = w % S::kWavesN * S::WN + l / 16 * 8;
#pragma unroll
    for (int r = 0; r < S::MI; ++r) {
#pragma unroll
      for (int j = 0; j < S::NI; j += 2) {
        const f8 x = f(m0 + r / 2 * 32 + r % 2 * 4, n0 + j * 16);
        v[r][j] = __builtin_shufflevector(x, x, 0, 1, 2, 3);
        v[r][j + 1] = __builtin_shufflevector(x, x, 4, 5, 6, 7);
      }
      if (r % 4 == 3) __builtin_amdgcn_sched_barrier(0);   // all at once would take too many registers
    }
  }

  // g(m, n, values, f(m, n)), where f loads and g stores: the loads are two rows ahead, as the compiler would not
  // let them overtake a store.
  template <typename F, typename G>
  __device__ __forceinline__ void each_with(F f, G g) const {
    const uint32_t l = threadIdx.x % 64, w = threadIdx.x / 64, i = l % 16;
    const uint32_t m0 = w / S::kWavesN * S::WM + i / 4 * 8 + i % 4;
    const uint32_t n0 = w % S::kWavesN * S::WN + l / 16 * 8;
    constexpr int kAhead = 2;
    const auto m = [&](int r) { return m0 + r / 2 * 32 + r % 2 * 4; };
    f8 x[kAhead][S::NI / 2];
#pragma unroll
    for (int r = -kAhead; r < S::MI; ++r) {
      f8 now[S::NI / 2];
#pragma unroll
      for (int j = 0; j < S::NI; j += 2) {
        const int at = (r + kAhead) % kAhead;
        now[j / 2] = x[at][j / 2];
        if (r + kAhead < S::MI) x[at][j / 2] = f(m(r + kAhead), n0 + j * 16);
      }
#pragma unroll
      for (int j = 0; j < S::NI; j += 2)
        if (r >= 0) g(m(r), n0 + j * 16, pair(r, j), now[j / 2]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  __device__ __forceinline__ f8 pair(int r, int j) const {
    return __builtin_shufflevector(v[r][j], v[r][j + 1], 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// All of this wave's loads to LDS but the last LATER ones have landed and its reads of LDS are done, and the same
// holds for the other waves.
template <int LATER = 0>
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LATER) : "memory");
}

// The compiler would put the reads of a group right before their use, to save registers.
__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(0); }

__device__ __forceinline__ void loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// A wave's way through a step: kSubs sub-steps of kParts groups of its rows each.  Two groups' fragments are in
// registers: that which is multiplied and the next one, which is read meanwhile.
template <class S, typename T, bool ACROSS_A, bool ACROSS_B>
struct Groups {
  static constexpr int kParts = S::MI >= 4 ? 2 * Kind<T>::kParts : 2;
  static constexpr int kRows = S::MI / kParts, kGroups = Kind<T>::kSubs * kParts;
  static_assert(kGroups % 2 == 0, "the groups' fragments take turns");
  Frag<T> a[2][kRows], b[2][S::NI];
  int blockA, blockB;

  // Group g of a tile; the second operand's fragments go to b[turn].
  __device__ __forceinline__ void read(const local<char>* tile, int g, int turn) {
    const int sub = g / kParts, at = g % kParts;
    if (at == 0) {
#pragma unroll
      for (int j = 0; j < S::NI; ++j)
        b[turn][j] = read_frag<T, S::BN, ACROSS_B>(tile + S::BM * kRowBytes, blockB + j, sub);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      a[g & 1][i] = read_frag<T, S::BM, ACROSS_A>(tile, blockA + at * kRows + i, sub);
  }

  // acc += A B for group g (of pairs acc + rest), with between(i) behind each row of products.
  template <typename F>
  __device__ __forceinline__ void multiply(Acc<S>& acc, Acc<S>& rest, int g, int turn, F between) const {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int r = g % kParts * kRows + i;
#pragma unroll
      for (int j = 0; j < S::NI; ++j) {
        if constexpr (Kind<T>::kParts == 2)
          mma_pairs(acc.v[r][j], rest.v[r][j], a[g & 1][i], b[turn][j]);
        else
          mma<T>(acc.v[r][j], a[g & 1][i], b[turn][j]);
      }
      between(i);
    }
  }
};

// acc += A B over K values along k, for the tile at (m0, n0); b2 is the second operand of a DUAL product.
//
// A step's tile is read group by group, each while the one before is multiplied.  Before the last group is
// multiplied comes the step's barrier, behind which the tile's place in LDS is free and the next tile has
// landed: the next tile's first group is read, and the loads of the tile after that go out one by one between
// the products (all at once they fill the queue, and the waves stand).  So products cover both latencies.
// The steps past the last one bring zeros, which nobody multiplies.
template <class S, typename T, bool ACROSS_A, bool ACROSS_B, bool DUAL>
__device__ __forceinline__ void product(Acc<S>& acc, local<char>* lds, const Operand& a,
                                        const Operand& b, const Operand& b2, uint32_t m0, uint32_t n0,
                                        uint32_t K) {
  typedef Loader<T, S::BM, S::kWaves, ACROSS_A, false> LoadA;
  typedef Loader<T, S::BN, S::kWaves, ACROSS_B, DUAL> LoadB;
  typedef Groups<S, T, ACROSS_A, ACROSS_B> G;
  LoadA la;
  LoadB lb;
  const uint32_t wave = uniform(threadIdx.x / 64);
  la.init(a, a, m0, K, wave);
  lb.init(b, b2, n0, K, wave);
  constexpr uint32_t step = kRowBytes / Kind<T>::kBytes;
  const uint32_t steps = (K + step - 1) / step;
  const uint32_t at = lds_address(lds);
  G g;
  g.blockA = wave / S::kWavesN * S::MI, g.blockB = wave % S::kWavesN * S::NI;
  Acc<S> rest;   // of pairs
  if (Kind<T>::kParts == 2) rest.clear();
  // loads of the stages behind the one that is waited for
  constexpr int kLater = (S::kStages - 2) * (LoadA::kLoads + LoadB::kLoads);
  uint32_t here = 0;   // the step's place in LDS
  const auto one_step = [&](int parity) {
    const uint32_t ahead = here + S::kStage < (uint32_t)S::kLds ? here + S::kStage : 0;
    // which of b's halves a sub-step's fragments are in
    const auto turn = [&](int group) { return Kind<T>::kSubs == 1 ? parity : group / G::kParts; };
#pragma unroll
    for (int i = 0; i < G::kGroups; ++i) {
      if (i + 1 < G::kGroups) {
        g.read(lds + here, i + 1, turn(i + 1));
        keep_order();
        g.multiply(acc, rest, i, turn(i), [](int) {});
        keep_order();
      } else {
        stage_barrier<kLater>();
        g.read(lds + ahead, 0, Kind<T>::kSubs == 1 ? parity ^ 1 : 0);
        keep_order();
        la.begin(at + here);
        lb.begin(at + here + S::BM * kRowBytes);
        constexpr int kAll = LoadA::kLoads + LoadB::kLoads, kEach = (kAll + G::kRows - 1) / G::kRows;
        g.multiply(acc, rest, i, turn(i), [&](int row) {
#pragma unroll
          for (int l = row * kEach; l < (row + 1) * kEach && l < kAll; ++l) {
            if (l < LoadA::kLoads)
              la.bring(l);
            else
              lb.bring(l - LoadA::kLoads);
          }
          keep_order();
        });
      }
    }
    here = ahead;
  };
  stage_barrier();   // what was in LDS before is read
#pragma unroll
  for (int s = 0; s < S::kStages; ++s) {
    la.issue(at + s * S::kStage);
    lb.issue(at + s * S::kStage + S::BM * kRowBytes);
  }
  stage_barrier<(S::kStages - 1) * (LoadA::kLoads + LoadB::kLoads)>();
  g.read(lds, 0, 0);
  for (uint32_t s = 0; s < steps; ++s) {
    one_step(0);
    if constexpr (Kind<T>::kSubs == 1) {
      if (++s < steps) one_step(1);
    }
  }
  if (Kind<T>::kParts == 2) acc.add(rest);
  loads_done();   // none to LDS is under way when the workgroup gives it back
}

// Which tile a workgroup computes.  Workgroups go to the 8 XCDs in turns, each with an L2 of
// its own: each XCD gets a run of tiles, in strips of kStrip tiles of rows, so that those at work
// together share rows of both operands.
constexpr uint32_t kXcds = 8, kStrip = 8;

__device__ __forceinline__ uint32_t xcd_order(uint32_t b, uint32_t n) {
  const uint32_t x = b % kXcds, whole = n / kXcds, more = n % kXcds;
  return x * whole + min(x, more) + b / kXcds;
}

__device__ __forceinline__ void tile_at(uint32_t t, uint32_t tiles_m, uint32_t tiles_n, uint32_t& m,
                                        uint32_t& n) {
  const uint32_t strip = t / (kStrip * tiles_n), in = t % (kStrip * tiles_n);
  const uint32_t high = min(kStrip, tiles_m - strip * kStrip);
  m = uniform(strip * kStrip + in % high);
  n = uniform(in / high);
}

// Few tiles with a long way along k are split: each split's sums go to memory as they lie in the accumulators, in
// fp32, and a second launch adds them in order and goes on as a product of one split would.
struct Splits {
  uint32_t n, steps;   // steps along k of each but the last; n 1: not split
  float* parts;
};

template <class S>
__device__ __forceinline__ float* part_at(float* parts, uint64_t tile) {
  return parts + tile * (S::BM * S::BN) + threadIdx.x * 4;
}

template <class S>
__device__ __forceinline__ void store_part(const Acc<S>& acc, float* parts, uint64_t tile) {
  float* to = part_at<S>(parts, tile);
#pragma unroll
  for (int r = 0; r < S::MI; ++r)
#pragma unroll
    for (int j = 0; j < S::NI; ++j) *(global<f4>*)(uintptr_t)(to + (r * S::NI + j) * S::kLanes * 4) = acc.v[r][j];
}

// acc += the parts of `tile` of each split, `tiles` apart.
template <class S>
__device__ __forceinline__ void add_parts(Acc<S>& acc, float* parts, uint64_t tile, uint64_t tiles,
                                          uint32_t splits) {
  for (uint32_t s = 0; s < splits; ++s) {
    const float* from = part_at<S>(parts, tile + s * tiles);
#pragma unroll
    for (int r = 0; r < S::MI; ++r) {
#pragma unroll
      for (int j = 0; j < S::NI; ++j)
        acc.v[r][j] += *(const global<f4>*)(uintptr_t)(from + (r * S::NI + j) * S::kLanes * 4);
      if (r % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// The part of an operand along or across k from step s0 on.
template <typename T, bool ACROSS>
__device__ __forceinline__ Operand from_step(Operand a, uint32_t s0) {
  a.p += ACROSS ? (uint64_t)s0 * (kRowBytes / Kind<T>::kBytes) * a.ld : (uint64_t)s0 * kRowBytes;
  return a;
}

// Values along k of a split, of K.
template <typename T>
__device__ __forceinline__ uint32_t split_length(const Splits& s, uint32_t split, uint32_t K) {
  constexpr uint32_t step = kRowBytes / Kind<T>::kBytes;
  const uint32_t from = split * s.steps * step;
  return min(K - from, s.steps * step);
}

constexpr uint64_t kCus = 256;

inline uint64_t tiles_of(uint64_t m, uint64_t n, uint64_t bm, uint64_t bn) {
  return (m + bm - 1) / bm * ((n + bn - 1) / bn);
}

// What a step takes a CU full of such workgroups for each of them, and what a tile takes beside its steps, in ns as
// measured. 16-bit products of small tiles are bound by what comes from L2 (64 bytes a clock and CU), others by the matrix
// cores. A workgroup of four waves that has a CU for itself takes a quarter longer (2048 x 2048 pairs over 2048: 136
// middle tiles 63 us, 528 small ones 49).
template <class S, typename T>
constexpr uint64_t step_ns() {
  constexpr int at = __is_same(S, Large) ? 0 : __is_same(S, Middle) ? 1 : __is_same(S, Flat) ? 2 : 3;
  constexpr uint64_t narrow[] = {1470, 610, 400, 260}, pairs[] = {0, 720, 400, 250}, wide[] = {6800, 1720, 880, 450};
  return __is_same(T, float) ? wide[at] : __is_same(T, pair_t) ? pairs[at] : narrow[at];
}
// Tiles of few steps are bound by what they write, in bursts that only other workgroups of the CU fill the pauses of (gradients of
// 4096 rows 64 -> 1000 bf16 52 us with large tiles, 39 with middle ones).
template <class S>
constexpr uint64_t tile_ns(bool few_steps) {
  if (few_steps) return __is_same(S, Large) ? 13000 : __is_same(S, Middle) ? 3500 : S::BN > 64 ? 2500 : 1500;
  return __is_same(S, Large) ? 8000 : __is_same(S, Middle) ? 5000 : 3500;
}
constexpr uint64_t kFewSteps = 4;

struct Choice {
  int shape;           // 0: Large, 1: Middle, 2: the least
  Splits splits;
  uint64_t bytes;      // of the parts
  uint64_t ns;
};

constexpr uint64_t kMostPartBytes = 256u << 20;   // bytes of parts

// The best shape and number of splits for `tiles(S())` tiles of `steps` steps: the CUs take the workgroups in
// turns; parts are written and read at 5.5 KB a ns in all, and read at 35 bytes a ns by a workgroup, in a launch of 4 us.
// (2048 -> 8192 bf16, dx of 256 rows: 8 large tiles in 32 splits 301 us, most of them in the join.)
template <typename T, class Least, typename F>
Choice choose(F tiles, uint64_t steps, bool may_split = true) {
  Choice best = {};
  best.ns = ~0ull;
  steps = steps ? steps : 1;
  const auto consider = [&](auto s, int shape) {
    typedef decltype(s) S;
    const uint64_t n = tiles(s);
    for (uint64_t splits = 1; splits <= (may_split ? 32 : 1); splits += splits < 4 ? 1 : splits / 2) {
      const uint64_t each = (steps + splits - 1) / splits;
      if (splits > 1 && (!n || each < 4 || n >= 2 * kCus)) break;   // (no tiles, no rows: nothing to split)
      const uint64_t real = (steps + each - 1) / each, bytes = real > 1 ? n * real * S::BM * S::BN * 4 : 0;
      if (bytes > kMostPartBytes) break;
      const uint64_t turns = (n * real + kCus - 1) / kCus;
      const uint64_t join = real == 1 ? 0 : 4000 + std::max(bytes * 2 / 5500, (n + kCus - 1) / kCus * (bytes / n) / 35);
      const uint64_t step = step_ns<S, T>() * (turns == 1 && S::kWaves == 4 ? 5 : 4) / 4;
      const uint64_t ns = turns * (each * step + tile_ns<S>(steps <= kFewSteps)) + join;
      if (ns < best.ns) best = {shape, {(uint32_t)real, (uint32_t)each, nullptr}, bytes, ns};
    }
  };
  if constexpr (!__is_same(T, pair_t)) consider(Large(), 0);   // pairs' accumulators would not fit
  consider(Middle(), 1);
  consider(Least(), 2);
  return best;
}

template <typename T, class Least, typename G>
void with_shape(const Choice& c, G f) {
  if constexpr (!__is_same(T, pair_t)) {
    if (c.shape == 0) return f(Large());
  }
  if (c.shape == 1) return f(Middle());
  return f(Least());
}

template <typename T>
uint64_t steps_of(uint64_t K) {
  constexpr uint64_t step = kRowBytes / Kind<T>::kBytes;
  return (K + step - 1) / step;
}

template <typename T>
__device__ __forceinline__ f8 load8(const T* p) {
  typedef T __attribute__((ext_vector_type(8), aligned(sizeof(T)))) any8;
  return __builtin_convertvector(*(const global<any8>*)(uintptr_t)p, f8);
}

// Eight neighbours of a row, at column n of `cols`.
template <typename T>
__device__ __forceinline__ void store8(T* row, uint32_t n, uint32_t cols, const f8& v) {
  typedef T __attribute__((ext_vector_type(8))) t8;
  typedef T __attribute__((ext_vector_type(8), aligned(sizeof(T)))) any8;
  if (n + 8 <= cols) {
    *(global<any8>*)(uintptr_t)(row + n) = __builtin_convertvector(v, t8);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (n + e < cols) gp(row)[n + e] = (T)v[e];
  }
}

template <typename T>
__device__ __forceinline__ f8 load8(const T* row, uint32_t n, uint32_t cols) {
  f8 v = {};
  if (n + 8 <= cols) {
    v = load8(row + n);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (n + e < cols) v[e] = (float)gp(row)[n + e];
  }
  return v;
}

}  // namespace
}  // namespace ec
