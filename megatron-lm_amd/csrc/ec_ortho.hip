// ec_ortho.hip — ec_orthogonalize: Newton-Schulz steps on a batch of matrices.
//
// X = x / (|x| + eps), then `steps` times A = X X', B = a I + b A + c A A, X = B X (from the
// other side, X' X and X B, where the matrix is tall, so that A is as small as can be), which
// takes every singular value through a s + b s^3 + c s^5.  A and B are symmetric: only the tiles on
// and above the diagonal are computed, and written twice.
//
// Small singular values grow by `a` a step, and so do the rounding errors of what is
// stored in between: with X, A and B in 16 bits 0.2 % (fp16) or 2 % (bf16) of the result after five
// steps.  There are two kinds of steps:
// - exact ones: all matrices are pairs of fp16 values (22 bits, ec_gemm.h).  The result is as good as that of fp32 products
//   (five steps, off by 1.2e-6 at 128 x 128, 2.0e-6 at 1001 x 777 and 2.7e-6 at 2048 x 2048, where those are by 1.4e-6, 2.3e-6
//   and 2.9e-6; at 16 x 256 9.5e-7 against 7.4e-7), at a third of the fp16 rate instead of a tenth.
// - fast ones: the products are of fp16 values, but all but the last two steps take X = a X + (b A + c A A) X, and
//   the X that a stands before has a second fp16 part.  What small singular values consist of is that first
//   term; the products' errors are small where they are.  Five steps leave 0.7e-3 to 0.8e-3 of the result
//   (with second parts in the last two steps too 0.8e-3 to 1.1e-3, without any 1.9e-3 to 2.5e-3), against 1.7e-3 by the
//   rounding to bf16; an update of a single nonzero row, whose roundings do not average out, has 1.5e-3 to 2.7e-3.
// A bf16 result takes fast steps, from kFastSide rows and columns on (smaller matrices are bound by the launches, and
// their roundings average out less); an fp16 or fp32 one exact steps.
//
// What is stored is 2^12 times the value, as ordinary entries are of 1 / sqrt(columns) and less: X has none above its largest
// singular value, A none above that squared.  Those are 1 at first, for the norm, and with coefficients that orthogonalise about
// 1.2 later.  Where the coefficients let them grow or shrink, the host follows them (exponents_of) and scales so that fp16 holds them.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "ec_gemm.h"
#include "ec_pack.h"

namespace ec {
namespace {

constexpr int kLanes = 256;
constexpr int kAhead = 4;
constexpr uint32_t kMostParts = 1024;     // of a matrix's sum of squares
constexpr uint32_t kPiece = 8192;         // elements of a contiguous matrix that are summed at a time
constexpr int kStored = 12;               // matrices are stored times 2^12,
constexpr int kMostStored = 42;           // or up to this where values shrink
constexpr uint32_t kMostSide = 1u << 16;
constexpr uint32_t kMostBatch = 65535;

constexpr uint32_t kFastSide = 64;
constexpr int kPlainSteps = 2;   // the last fast steps, whose X has no second part

struct Matrices {
  const char* p;
  uint64_t stride, matrix;   // elements from row to row, from matrix to matrix
};

template <int LANES>
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double shared[LANES / 64];
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  if (threadIdx.x % 64 == 0) shared[threadIdx.x / 64] = v;
  __syncthreads();
  v = shared[0];
  for (int w = 1; w < LANES / 64; ++w) v += shared[w];
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kLanes) square_kernel(const T* x, uint64_t stride, uint64_t matrix,
                                                        uint64_t pieces, uint64_t total, uint32_t width,
                                                        double* parts) {
  typedef Group<T> G;
  const T* base = x + blockIdx.y * matrix;
  double sum = 0.0;
  for (uint64_t i = blockIdx.x; i < pieces; i += gridDim.x) {
    const T* p = base + i * stride;
    const uint32_t n = (uint32_t)min((uint64_t)width, total - i * width);
    const uint32_t groups = n / G::kN;
    for (uint32_t g = threadIdx.x; g < groups; g += kLanes * kAhead) {
      typename G::vec v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)   // without conditions, so that all are in flight together
        v[u] = load_group<T, false>(p + (uint64_t)min(g + u * kLanes, groups - 1) * G::kN);
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (g + u * kLanes < groups) {
          const typename G::wide w = widen<T>(v[u]);
#pragma unroll
          for (int e = 0; e < G::kN; ++e) sum = __builtin_fma((double)w[e], (double)w[e], sum);
        }
    }
    const uint32_t rest = groups * G::kN + threadIdx.x;
    if (rest < n) {
      const double v = (double)(float)gp(p)[rest];
      sum = __builtin_fma(v, v, sum);
    }
  }
  sum = block_sum<kLanes>(sum);
  if (threadIdx.x == 0) gp(parts)[blockIdx.y * gridDim.x + blockIdx.x] = sum;
}

// The exponents that a step's X, A, B and the next X (of a result 0) are stored with.
struct Exponents {
  int8_t x, gram, poly, next;
};

struct Coefficients {
  float a, b, c, b_by_c;   // b / c where it is finite
};

// A step's factors between stored values.
struct Factors {
  float gram;       // of the product of X with itself: A
  float poly;       // c, of ratio * A + A A, beside the diagonal: B
  float ratio;      // b / c
  float own;        // a, of the diagonal, or of an X that is added to B X
  float next;       // of B X
};

__host__ __device__ __forceinline__ Factors factors_of(const Exponents& at, const Coefficients& k) {
  Factors f;
  f.gram = __builtin_ldexpf(1.0f, at.gram - 2 * at.x);
  // where there is no A A, or next to none, so little of it that it is rounded off (as stored it is below 2^30) and b / c
  // is finite
  f.poly = k.c * __builtin_ldexpf(1.0f, at.poly - 2 * at.gram);
  const bool none = __builtin_fabsf(f.poly) < 0x1p-72f;
  f.ratio = none ? __builtin_ldexpf(k.b, at.poly - at.gram + 72) : __builtin_ldexpf(k.b_by_c, at.gram);
  f.poly = none ? 0x1p-72f : f.poly;
  f.own = k.a * __builtin_ldexpf(1.0f, at.poly);
  f.next = __builtin_ldexpf(1.0f, at.next - at.poly - at.x);
  return f;
}

typedef fp16_t __attribute__((ext_vector_type(8))) h8;

// Two fp16 values whose sum is v to 22 bits.  `high` is made a value of its own: where v is a product, the compiler would
// round the unrounded product to the `high` that the difference takes and the rounded one to the `high` that is
// stored, which are a step of 11 bits apart in one of 2^14 elements (and left one matrix in 20 with 1e-5 of its result).
__device__ __forceinline__ void split(const f8& v, h8& high, h8& low) {
  high = __builtin_convertvector(v, h8);
  asm("" : "+v"(high));
  low = __builtin_convertvector(v - __builtin_convertvector(high, f8), h8);
}

// Columns n ... n + 7 (n a multiple of 8) of a row of pairs; or of one of fp16 values, of a matrix whose second parts
// are `low_at` bytes behind (0: it has none).
template <typename K>
__device__ __forceinline__ void put8(char* row, uint32_t n, const f8& v, uint64_t low_at) {
  h8 high, low;
  split(v, high, low);
  global<char>* to = gp(row) + n * Kind<K>::kBytes;
  *(global<h8>*)to = high;
  if (Kind<K>::kParts == 2)
    *(global<h8>*)(to + 16) = low;
  else if (low_at)
    *(global<h8>*)(to + low_at) = low;
}

template <typename K>
__device__ __forceinline__ f8 get8(const char* row, uint32_t n, uint64_t low_at) {
  const global<char>* from = gp(row) + n * Kind<K>::kBytes;
  f8 v = __builtin_convertvector(*(const global<h8>*)from, f8);
  if (Kind<K>::kParts == 2 || low_at)
    v += __builtin_convertvector(*(const global<h8>*)(from + (Kind<K>::kParts == 2 ? 16 : low_at)), f8);
  return v;
}

// x / (|x| + eps) as a matrix of K, 8 elements a lane, with zeros behind a row's end.  |x| comes from the partial
// sums in order, in every workgroup.
template <typename T, typename K>
__global__ void __launch_bounds__(kLanes) scale_kernel(const T* x, uint64_t stride, uint64_t matrix,
                                                       uint32_t rows, uint32_t cols, const double* parts,
                                                       uint32_t n_parts, double eps, char* out, uint64_t low_at) {
  double sum = 0.0;
  for (uint32_t i = threadIdx.x; i < n_parts; i += kLanes) sum += gp(parts)[blockIdx.y * n_parts + i];
  sum = block_sum<kLanes>(sum);
  const double by = (double)(1 << kStored) / (__builtin_sqrt(sum) + eps);
  const T* from = x + blockIdx.y * matrix;
  const uint32_t groups = (cols + 7) / 8, all = rows * groups;
  constexpr uint32_t kGroup = 8 * Kind<K>::kBytes;
  char* to = out + (uint64_t)blockIdx.y * all * kGroup;
  for (uint32_t g = blockIdx.x * kLanes + threadIdx.x; g < all; g += gridDim.x * kLanes) {
    const uint32_t row = g / groups, at = g % groups * 8;
    f8 v = load8<T>(from + row * stride, at, cols);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)((double)v[e] * by);
    put8<K>(to + (uint64_t)g * kGroup, 0, v, low_at);
  }
}

struct NsArgs {
  Operand a, b;
  uint64_t a_matrix, b_matrix;   // bytes from matrix to matrix
  uint32_t K, M, N;
  uint32_t tiles_m, tiles_n;     // tiles_m 0: those on and above the diagonal of tiles_n x tiles_n
  uint32_t tiles;                // of a matrix
  char* out;
  uint64_t out_ld, out_matrix;   // bytes
  float by;                      // the result: by * product
  uint64_t out_low;              // from a value to its second part, in bytes
  const char* add;               // a matrix like the result: by * (linear * add + product), or none
  uint64_t add_ld, add_matrix, add_low;
  float linear, diagonal;        // POLY: + diagonal * I
  Matrices base;                 // LAST: + keep * base, or none
  float keep;
  Splits splits;                 // GRAM
};

// A wave's LDS to turn a block of 32 x 32 round: rows of 36 meet no bank conflicts either way.
constexpr uint32_t kTurnRow = 36, kTurn = 32 * kTurnRow;

// What becomes of a product: A, B, the next X, or the result.
enum { kGram, kPoly, kNext, kLast };

// The t-th tile on and above the diagonal, column by column.
__device__ __forceinline__ void upper_tile_at(uint32_t t, uint32_t& tm, uint32_t& tn) {
  t = uniform(t);
  for (tn = 0; (tn + 1) * (tn + 2) / 2 <= t;) ++tn;
  tm = t - tn * (tn + 1) / 2;
}

// A split of A's product.
template <class S, typename In, bool ACROSS>
__global__ void __launch_bounds__(S::kLanes, S::kPerSimd) gram_part_kernel(NsArgs p) {
  __shared__ __attribute__((aligned(1024))) char lds[S::kLds];
  const uint32_t t = xcd_order(blockIdx.x, gridDim.x), all = gridDim.x / p.splits.n, split = uniform(t / all);
  const uint32_t matrix = uniform(t % all / p.tiles);
  uint32_t tm, tn;
  upper_tile_at(t % all % p.tiles, tm, tn);
  Operand a = from_step<In, ACROSS>(p.a, split * p.splits.steps), b = from_step<In, ACROSS>(p.b, split * p.splits.steps);
  a.p += matrix * p.a_matrix;
  b.p += matrix * p.b_matrix;
  Acc<S> acc;
  acc.clear();
  product<S, In, ACROSS, ACROSS, false>(acc, (local<char>*)lds, a, b, b, tm * S::BM, tn * S::BN,
                                        split_length<In>(p.splits, split, p.K));
  store_part(acc, p.splits.parts, t);
}

template <class S, typename In, bool ACROSS_A, bool ACROSS_B, int WHAT, typename Out, bool JOIN>
__global__ void __launch_bounds__(S::kLanes, S::kPerSimd) ns_kernel(NsArgs p) {
  __shared__ __attribute__((aligned(1024))) char lds[JOIN ? S::kWaves * kTurn * 4 : S::kLds];
  const uint32_t t = xcd_order(blockIdx.x, gridDim.x), matrix = uniform(t / p.tiles);
  uint32_t tm, tn;
  constexpr bool kSymmetric = WHAT == kGram || WHAT == kPoly;
  if (kSymmetric)
    upper_tile_at(t % p.tiles, tm, tn);
  else
    tile_at(t % p.tiles, p.tiles_m, p.tiles_n, tm, tn);
  Operand a = p.a, b = p.b;
  a.p += matrix * p.a_matrix;
  b.p += matrix * p.b_matrix;
  const uint32_t m0 = tm * S::BM, n0 = tn * S::BN, padded = (p.N + 7) & ~7u;
  // zeros below the last row, which the mirrored tile has as columns of padding; past the columns some other value,
  // which is not stored
  const auto added = [&](uint32_t m, uint32_t n) {
    return (m0 + m < p.M ? p.linear : 0.0f) *
           get8<In>(p.add + matrix * p.add_matrix + min(m0 + m, p.M - 1) * p.add_ld, min(n0 + n, padded - 8),
                    p.add_low);
  };
  constexpr bool kStarts = WHAT == kPoly || (WHAT != kGram && Kind<In>::kParts == 1);
  Acc<S> acc;
  if (kStarts && p.add)
    acc.start(added);
  else
    acc.clear();
  if constexpr (JOIN)
    add_parts(acc, p.splits.parts, t, gridDim.x, p.splits.n);
  else
    product<S, In, ACROSS_A, ACROSS_B, false>(acc, (local<char>*)lds, a, b, b, m0, n0, p.K);
  char* out = p.out + matrix * p.out_matrix;
  const auto value = [&](uint32_t m, uint32_t n, f8 v) {
    v *= p.by;
    if constexpr (WHAT == kPoly) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (m == n + e) v[e] += p.diagonal;
    }
    return v;
  };
  if constexpr (WHAT == kLast) {
    const auto put = [&](uint32_t m, uint32_t n, const f8& v) {
      m += m0;
      n += n0;
      if (m < p.M && n < p.N) store8<Out>((Out*)(out + m * p.out_ld), n, p.N, v);
    };
    if (p.base.p) {
      const Out* base = (const Out*)p.base.p + matrix * p.base.matrix;
      acc.each_with(
          [&](uint32_t m, uint32_t n) {
            return load8(base + min(m0 + m, p.M - 1) * p.base.stride, n0 + n, p.N);
          },
          [&](uint32_t m, uint32_t n, const f8& v, const f8& x) { put(m, n, p.by * v + p.keep * x); });
    } else {
      acc.each([&](uint32_t m, uint32_t n, const f8& v) { put(m, n, p.by * v); });
    }
  } else if (!kSymmetric || tm == tn) {
    acc.each([&](uint32_t m, uint32_t n, f8 v) {
      m += m0;
      n += n0;
      if (m < p.M && n < padded) put8<Out>(out + m * p.out_ld, n, value(m, n, v), p.out_low);
    });
  } else {
    // and the mirrored tile, 32 x 32 at a time turned round in the wave's part of LDS
    stage_barrier();
    local<float>* turn = (local<float>*)(local<char>*)lds + threadIdx.x / 64 * kTurn;
    static_assert(S::kWaves * kTurn * 4 <= S::kLds, "a part for each wave");
    const uint32_t l = threadIdx.x % 64, w = threadIdx.x / 64, i = l % 16;
    const uint32_t mw = m0 + w / S::kWavesN * S::WM, nw = n0 + w % S::kWavesN * S::WN;
    const auto in_step = [] {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    };
#pragma unroll
    for (int r = 0; r < S::MI; r += 2) {
#pragma unroll
      for (int j = 0; j < S::NI; j += 2) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t mr = i / 4 * 8 + h * 4 + i % 4, nr = l / 16 * 8;
          const uint32_t m = mw + r * 16 + mr, n = nw + j * 16 + nr;
          const f8 v = value(m, n, acc.pair(r + h, j));
          if (m < p.M && n < padded) put8<Out>(out + m * p.out_ld, n, v, p.out_low);
          *(local<f4>*)(turn + mr * kTurnRow + nr) = __builtin_shufflevector(v, v, 0, 1, 2, 3);
          *(local<f4>*)(turn + mr * kTurnRow + nr + 4) = __builtin_shufflevector(v, v, 4, 5, 6, 7);
        }
        in_step();
        const uint32_t row = nw + j * 16 + l / 2, col = mw + r * 16 + l % 2 * 16;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          f8 v;
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = turn[(l % 2 * 16 + h * 8 + e) * kTurnRow + l / 2];
          if (row < p.N && col + h * 8 < padded) put8<Out>(out + row * p.out_ld, col + h * 8, v, p.out_low);
        }
        in_step();
      }
    }
  }
}

// The tiles of M x N results, or (symmetric) those on and above the diagonal.
template <class S>
uint64_t ns_tiles(uint64_t m, uint64_t n, bool symmetric) {
  const uint64_t wide = (n + S::BN - 1) / S::BN;
  return symmetric ? wide * (wide + 1) / 2 : tiles_of(m, n, S::BM, S::BN);
}

template <typename In>
Choice choose_ns(uint32_t m, uint32_t n, uint32_t K, uint32_t batch, int what) {
  const bool symmetric = what == kGram || what == kPoly;
  return choose<In, Small>([&](auto s) { return batch * ns_tiles<decltype(s)>(m, n, symmetric); }, steps_of<In>(K),
                           what == kGram);   // only A's products are split
}

template <typename In, bool ACROSS_A, bool ACROSS_B, int WHAT, typename Out>
int run_ns(NsArgs& p, uint32_t batch, char* parts, hipStream_t st) {
  constexpr bool kSymmetric = WHAT == kGram || WHAT == kPoly;
  int status = EC_OK;
  const Choice c = choose_ns<In>(p.M, p.N, p.K, batch, WHAT);
  p.splits = c.splits;
  p.splits.parts = (float*)parts;
  with_shape<In, Small>(c, [&](auto s) {
    typedef decltype(s) S;
    p.tiles_m = (p.M + S::BM - 1) / S::BM;
    p.tiles_n = (p.N + S::BN - 1) / S::BN;
    p.tiles = (uint32_t)ns_tiles<S>(p.M, p.N, kSymmetric);
    const uint64_t all = (uint64_t)p.tiles * batch;
    if (all >= (1ull << 32) / S::kLanes) {
      status = EC_ERANGE;
      return;
    }
    if constexpr (WHAT == kGram) {
      if (c.splits.n > 1) {
        gram_part_kernel<S, In, ACROSS_A><<<(uint32_t)all * c.splits.n, S::kLanes, 0, st>>>(p);
        ns_kernel<S, In, ACROSS_A, ACROSS_B, WHAT, Out, true><<<(uint32_t)all, S::kLanes, 0, st>>>(p);
        return;
      }
    }
    ns_kernel<S, In, ACROSS_A, ACROSS_B, WHAT, Out, false><<<(uint32_t)all, S::kLanes, 0, st>>>(p);
  });
  return status;
}

// A matrix of at most D x D: one workgroup takes all steps, with everything in LDS, one launch instead of seventeen.  A tall
// matrix is taken transposed.  A matrix lies there as D-row tiles along k, one behind another; B takes A's place and
// the next X that of X, when all waves have read them.
// The arguments of up to five steps are in 128 bytes.
struct SmallArgs {
  Matrices x, base;
  char* out;
  uint64_t out_stride, out_matrix;   // elements
  uint16_t rows, cols;
  uint32_t steps;
  Coefficients k;
  float scale, keep, eps;
  Exponents at[EC_MAX_STEPS];
};

constexpr int kSmallSide = 128;

template <typename K, int D>
struct Resident {
  static constexpr int kBlock = D * kRowBytes, kBlocks = D * Kind<K>::kBytes / kRowBytes, kSize = kBlock * kBlocks;

  // 16-byte chunk c of row r
  __device__ __forceinline__ static uint32_t chunk_at(uint32_t r, uint32_t c) {
    return c / 8 * kBlock + r * kRowBytes + ((c % 8) ^ along_swizzle(r)) * 16;
  }
  __device__ __forceinline__ static void put(local<char>* m, local<char>* low, uint32_t row, uint32_t n, const f8& v) {
    h8 h, l;
    split(v, h, l);
    if constexpr (Kind<K>::kParts == 2) {
      *(local<h8>*)(m + chunk_at(row, n / 4)) = h;
      *(local<h8>*)(m + chunk_at(row, n / 4 + 1)) = l;
    } else {
      *(local<h8>*)(m + chunk_at(row, n / 8)) = h;
      if (low) *(local<h8>*)(low + chunk_at(row, n / 8)) = l;
    }
  }
  __device__ __forceinline__ static f8 get(const local<char>* m, const local<char>* low, uint32_t row, uint32_t n) {
    if constexpr (Kind<K>::kParts == 2)
      return __builtin_convertvector(*(const local<h8>*)(m + chunk_at(row, n / 4)), f8) +
             __builtin_convertvector(*(const local<h8>*)(m + chunk_at(row, n / 4 + 1)), f8);
    f8 v = __builtin_convertvector(*(const local<h8>*)(m + chunk_at(row, n / 8)), f8);
    if (low) v += __builtin_convertvector(*(const local<h8>*)(low + chunk_at(row, n / 8)), f8);
    return v;
  }
  // The fragment whose rows are the matrix's columns and whose k its rows, of step k0 / 32: read_frag's across k.
  __device__ __forceinline__ static Frag<K> turned(const local<char>* m, int block, uint32_t k0) {
    constexpr int P = Kind<K>::kParts;
    const uint32_t l = threadIdx.x % 64, i = l % 16, q = l / 16;
    Frag<K> f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      s4 half[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t k = k0 + 8 * q + 4 * e + i / 4;
        half[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (local<s4>*)(m + chunk_at(k, (block / 2 * 4 + i % 4) * P + p) + block % 2 * 8));
      }
      f.part[p] = __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
    }
    return f;
  }
};

// Waves: four for 64 x 64, eight for 128 x 128, so that one's products cover another's reads.
template <int D>
using SmallShape = Shape<D, D, D / 2, D == 128 ? D / 4 : D / 2, 2>;

template <typename T, typename Out, typename K, int D>
__global__ void __launch_bounds__(SmallShape<D>::kLanes) small_kernel(SmallArgs p) {
  typedef Resident<K, D> R;
  typedef SmallShape<D> S;
  constexpr bool kFast = Kind<K>::kParts == 1;
  __shared__ __attribute__((aligned(1024))) char lds[R::kSize * (kFast ? 3 : 2)];
  local<char>* x = (local<char>*)lds;
  local<char>* a = x + R::kSize;
  local<char>* low = kFast ? a + R::kSize : nullptr;
  const uint32_t matrix = blockIdx.x, wave = threadIdx.x / 64;
  const int blockA = wave / S::kWavesN * S::MI, blockB = wave % S::kWavesN * S::NI;
  const bool tall = p.rows > p.cols;
  {   // X = x / (|x| + eps), groups of 8 along x's rows
    const T* from = (const T*)p.x.p + matrix * p.x.matrix;
    constexpr int kGroups = D * D / 8 / S::kLanes;
    f8 v[kGroups];
    double sum = 0.0;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const uint32_t at = g * S::kLanes + threadIdx.x, row = at / (D / 8), col = at % (D / 8) * 8;
      v[g] = f8{};
      if (row < p.rows) v[g] = load8(from + row * p.x.stride, col, p.cols);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = __builtin_fma((double)v[g][e], (double)v[g][e], sum);
    }
    const double by = (double)(1 << kStored) / (__builtin_sqrt(block_sum<S::kLanes>(sum)) + (double)p.eps);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const uint32_t at = g * S::kLanes + threadIdx.x, row = at / (D / 8), col = at % (D / 8) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[g][e] = (float)((double)v[g][e] * by);
      if (!tall) {
        R::put(x, low, row, col, v[g]);
      } else {
        h8 h, l;
        split(v[g], h, l);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t c = row / 8 * Kind<K>::kParts, in = row % 8 * 2;
          *(local<fp16_t>*)(x + R::chunk_at(col + e, c) + in) = h[e];
          *(local<fp16_t>*)((kFast ? low : x) + R::chunk_at(col + e, kFast ? c : c + 1) + in) = l[e];
        }
      }
    }
  }
  // acc += the product with the second matrix's rows, or (TURNED) its columns, of what is `first` along k
  Acc<S> acc;
  const auto multiply = [&](const local<char>* first, const local<char>* second, auto turned) {
    constexpr bool kTurned = decltype(turned)::value;
    Acc<S> rest;   // of pairs
    if (!kFast) rest.clear();
#pragma unroll
    for (int t = 0; t < R::kBlocks; ++t) {
#pragma unroll
      for (int sub = 0; sub < Kind<K>::kSubs; ++sub) {
        Frag<K> fa[S::MI], fb[S::NI];
#pragma unroll
        for (int j = 0; j < S::NI; ++j) {
          if constexpr (kTurned)
            fb[j] = R::turned(second, blockB + j, (t * Kind<K>::kSubs + sub) * 32);
          else
            fb[j] = read_frag<K, D, false>(second + t * R::kBlock, blockB + j, sub);
        }
#pragma unroll
        for (int i = 0; i < S::MI; ++i) fa[i] = read_frag<K, D, false>(first + t * R::kBlock, blockA + i, sub);
#pragma unroll
        for (int i = 0; i < S::MI; ++i)
#pragma unroll
          for (int j = 0; j < S::NI; ++j) {
            if constexpr (kFast)
              mma<K>(acc.v[i][j], fa[i], fb[j]);
            else
              mma_pairs(acc.v[i][j], rest.v[i][j], fa[i], fb[j]);
          }
      }
    }
    if (!kFast) acc.add(rest);
  };
  for (uint32_t s = 0; s < p.steps; ++s) {
    const bool adds = kFast && s + kPlainSteps < p.steps;
    __syncthreads();
    const Factors f = factors_of(p.at[s], p.k);   // behind the barrier: 64 x 64 9.3 us, before it 9.5
    const float diagonal = adds ? 0.0f : f.own;
    acc.clear();
    multiply(x, x, std::false_type());
    acc.each([&](uint32_t m, uint32_t n, f8 v) { R::put(a, nullptr, m, n, f.gram * v); });
    __syncthreads();
    acc.start([&](uint32_t m, uint32_t n) { return f.ratio * R::get(a, nullptr, m, n); });
    multiply(a, a, std::false_type());
    __syncthreads();
    acc.each([&](uint32_t m, uint32_t n, f8 v) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = m == n + e ? __builtin_fmaf(v[e], f.poly, diagonal) : v[e] * f.poly;
      R::put(a, nullptr, m, n, v);
    });
    __syncthreads();
    if (adds)
      acc.start([&](uint32_t m, uint32_t n) { return f.own * R::get(x, low, m, n); });
    else
      acc.clear();
    multiply(a, x, std::true_type());
    if (s + 1 < p.steps) {
      __syncthreads();
      acc.each([&](uint32_t m, uint32_t n, f8 v) { R::put(x, low, m, n, f.next * v); });
      continue;
    }
    const float scale = p.scale * f.next;
    Out* out = (Out*)p.out + matrix * p.out_matrix;
    const Out* base = (const Out*)p.base.p + matrix * p.base.matrix;
    acc.each([&](uint32_t m, uint32_t n, f8 v) {
      v *= scale;
      if (!tall) {
        if (m >= p.rows || n >= p.cols) return;
        if (p.base.p) v += p.keep * load8(base + m * p.base.stride, n, p.cols);
        store8<Out>(out + m * p.out_stride, n, p.cols, v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (n + e >= p.rows || m >= p.cols) continue;
          float w = v[e];
          if (p.base.p) w += p.keep * (float)gp(base)[(n + e) * p.base.stride + m];
          gp(out)[(n + e) * p.out_stride + m] = (Out)w;
        }
      }
    });
  }
}

struct Plan {
  uint32_t batch, rows, cols, side, other;   // side: of the symmetric matrices
  uint32_t sums;                             // parts of a matrix's sum of squares
  uint64_t parts, x[2], gram, poly, splits, total;
};

Plan plan_of(uint32_t batch, uint32_t rows, uint32_t cols) {
  Plan p = {};
  p.batch = batch, p.rows = rows, p.cols = cols;
  p.side = std::min(rows, cols), p.other = std::max(rows, cols);
  // enough workgroups in all to keep the memory busy
  p.sums = std::min(kMostParts, std::max(1u, 2 * kMostParts / batch));
  const auto take = [&](uint64_t bytes) {
    const uint64_t at = p.total;
    p.total += part(bytes);
    return at;
  };
  const uint64_t x = (uint64_t)batch * rows * up_to(cols, 8) * 4;
  const uint64_t square = (uint64_t)batch * p.side * up_to(p.side, 8) * 4;
  p.parts = take((uint64_t)batch * p.sums * sizeof(double));
  p.x[0] = take(x), p.x[1] = take(x);
  p.gram = take(square), p.poly = take(square);
  p.splits = take(std::max(choose_ns<pair_t>(p.side, p.side, p.other, batch, kGram).bytes,
                           choose_ns<fp16_t>(p.side, p.side, p.other, batch, kGram).bytes));
  return p;
}

int check_sizes(uint64_t batch, uint64_t rows, uint64_t cols) {
  if (!rows || !cols) return EC_EINVAL;
  if (rows > kMostSide || cols > kMostSide || batch > kMostBatch) return EC_ERANGE;
  return EC_OK;
}

struct Call {
  Matrices x, base;
  char* out;
  uint64_t out_stride, out_matrix;
  int type, out_type, steps;
  Coefficients k;
  float eps, scale, keep;
  Exponents at[EC_MAX_STEPS];
};

bool fast(const Plan& p, int out_type) { return out_type == EC_BF16 && p.side >= kFastSide; }

bool small(uint64_t rows, uint64_t cols) { return std::max(rows, cols) <= kSmallSide; }

// A matrix of K in the workspace, the bytes of one of the batch, and those to its second parts.
struct Stored {
  Operand m;
  uint64_t matrix, low;
};

template <typename K>
Stored stored(char* at, uint32_t batch, uint32_t rows, uint32_t cols, bool low) {
  Stored s;
  s.m = {at, up_to(cols, 8) * Kind<K>::kBytes, rows};
  s.matrix = s.m.ld * rows;
  s.low = Kind<K>::kParts == 1 && low ? s.matrix * batch : 0;
  return s;
}

// The exponent that values up to `most` are stored with: at most half of what fp16 holds, as roundings may pass the bounds, and
// so much that ordinary entries, a fraction of the largest, keep their second parts' bits.
int stored_at(double most) {
  int e;
  const bool exact = std::frexp(most, &e) == 0.5;   // most is in [2^(e - 1), 2^e)
  const int high = 15 - e + exact, low = 10 - e;    // most 2^high is at most 2^15, most 2^low at least 2^9
  return std::max(std::min(kStored, high), std::min(kMostStored, most > 0.0 ? low : kMostStored));
}

// The largest singular value after a step from values in [0, most]: s (a + b s^2 + c s^4) at the end, or where
// a + 3 b t + 5 c t^2 = 0, t = s^2.
double largest_next(double a, double b, double c, double most) {
  const auto at = [&](double s) { return std::fabs(s * (a + s * s * (b + c * s * s))); };
  double next = at(most);
  const auto turn = [&](double t) {
    if (t > 0.0 && t < most * most) next = std::max(next, at(std::sqrt(t)));
  };
  const double root = std::sqrt(std::max(0.0, 9.0 * b * b - 20.0 * a * c));
  const double q = -0.5 * (3.0 * b + std::copysign(root, b));   // both roots without cancellation
  if (c != 0.0) turn(q / (5.0 * c));
  if (q != 0.0) turn(a / q);
  return next;
}

// Bounds of singular values are followed up to here: the factors stay within fp32's exponents.
constexpr double kMostSingular = 1u << 20;

// The exponents of all steps; `fast`: all but the last kPlainSteps add a X by themselves.
void exponents_of(const Coefficients& k, int steps, bool fast, Exponents* to) {
  const double a = k.a, b = k.b, c = k.c;
  double most = 1.0;   // singular values of X
  int x = kStored;
  for (int s = 0; s < steps; ++s) {
    const bool adds = fast && s + kPlainSteps < steps;
    const double a_most = most * most, in_poly = std::max(2.0, a_most);
    const int gram = stored_at(a_most);
    const int poly = stored_at((adds ? 0.0 : std::fabs(a)) + in_poly * (std::fabs(b) + in_poly * std::fabs(c)));
    most = std::min(largest_next(a, b, c, most), kMostSingular);
    const int next = s + 1 < steps ? stored_at(most) : 0;
    to[s] = {(int8_t)x, (int8_t)gram, (int8_t)poly, (int8_t)next};
    x = next;
  }
}

// Step s: the next step's X, or the result.
template <bool TALL, typename In>
int run_step(const Plan& p, const Call& c, char* work, int s, hipStream_t st) {
  constexpr bool kFast = Kind<In>::kParts == 1;
  // X has a second part, and a step adds a X by itself, up to the last steps
  const bool adds = kFast && s + kPlainSteps < c.steps, next_adds = kFast && s + 1 + kPlainSteps < c.steps;
  const Stored x = stored<In>(work + p.x[s & 1], p.batch, p.rows, p.cols, true);
  const Stored gram = stored<In>(work + p.gram, p.batch, p.side, p.side, false);
  const Stored poly = stored<In>(work + p.poly, p.batch, p.side, p.side, false);
  const Factors f = factors_of(c.at[s], c.k);

  NsArgs n = {};
  n.a = n.b = x.m;
  n.a.rows = n.b.rows = p.side;
  n.a_matrix = n.b_matrix = x.matrix;
  n.K = p.other, n.M = n.N = p.side;
  n.out = work + p.gram, n.out_ld = gram.m.ld, n.out_matrix = gram.matrix;
  n.by = f.gram;
  if (const int e = run_ns<In, TALL, TALL, kGram, In>(n, p.batch, work + p.splits, st)) return e;

  n.a = n.b = gram.m;
  n.a_matrix = n.b_matrix = gram.matrix;
  n.K = p.side;
  n.out = work + p.poly;
  n.add = work + p.gram, n.add_ld = gram.m.ld, n.add_matrix = gram.matrix;
  n.by = f.poly, n.linear = f.ratio, n.diagonal = adds ? 0.0f : f.own;
  if (const int e = run_ns<In, false, false, kPoly, In>(n, p.batch, work + p.splits, st)) return e;

  // B X, X across; or X B, X along
  n.a = TALL ? x.m : poly.m, n.b = TALL ? poly.m : x.m;
  n.a.rows = p.rows, n.b.rows = p.cols;
  n.a_matrix = TALL ? x.matrix : poly.matrix, n.b_matrix = TALL ? poly.matrix : x.matrix;
  n.M = p.rows, n.N = p.cols;
  n.add = adds ? x.m.p : nullptr, n.add_ld = x.m.ld, n.add_matrix = x.matrix, n.add_low = x.low;
  n.linear = f.own;
  if (s + 1 < c.steps) {
    n.out = work + p.x[(s + 1) & 1], n.out_ld = x.m.ld, n.out_matrix = x.matrix;
    n.out_low = next_adds ? x.low : 0;
    n.by = f.next;
    return run_ns<In, false, !TALL, kNext, In>(n, p.batch, work + p.splits, st);
  }
  const uint32_t w = type_bytes(c.out_type);
  n.out = c.out, n.out_ld = c.out_stride * w, n.out_matrix = c.out_matrix * w;
  n.by = c.scale * f.next;
  n.base = c.base, n.keep = c.keep;
  if constexpr (kFast)
    return run_ns<In, false, !TALL, kLast, bf16_t>(n, p.batch, work + p.splits, st);
  else
    return with_type(c.out_type, [&](auto o) {
      return run_ns<In, false, !TALL, kLast, decltype(o)>(n, p.batch, work + p.splits, st);
    });
}

template <bool TALL>
int run_steps(const Plan& p, const Call& c, char* work, hipStream_t st) {
  for (int s = 0; s < c.steps; ++s) {
    const int e = fast(p, c.out_type) ? run_step<TALL, fp16_t>(p, c, work, s, st)
                                      : run_step<TALL, pair_t>(p, c, work, s, st);
    if (e) return e;
  }
  return EC_OK;
}

template <typename T, typename Out, typename K>
void run_small(const Plan& p, const Call& c, hipStream_t st) {
  SmallArgs a = {};
  a.x = c.x, a.base = c.base;
  a.out = c.out, a.out_stride = c.out_stride, a.out_matrix = c.out_matrix;
  a.rows = (uint16_t)p.rows, a.cols = (uint16_t)p.cols, a.steps = (uint32_t)c.steps;
  a.scale = c.scale, a.keep = c.keep, a.eps = c.eps;
  a.k = c.k;
  std::copy(c.at, c.at + c.steps, a.at);
  if (p.other <= kSmallSide / 2)
    small_kernel<T, Out, K, kSmallSide / 2><<<p.batch, SmallShape<kSmallSide / 2>::kLanes, 0, st>>>(a);
  else
    small_kernel<T, Out, K, kSmallSide><<<p.batch, SmallShape<kSmallSide>::kLanes, 0, st>>>(a);
}

}  // namespace
}  // namespace ec

using namespace ec;

extern "C" {

uint64_t ec_orthogonalize_workspace(uint64_t batch, uint64_t rows, uint64_t cols) {
  if (!batch || check_sizes(batch, rows, cols) != EC_OK || small(rows, cols)) return 0;
  return plan_of((uint32_t)batch, (uint32_t)rows, (uint32_t)cols).total;
}

int ec_orthogonalize(const void* d_x, int type, uint64_t batch, uint64_t rows, uint64_t cols,
                     uint64_t x_stride, uint64_t x_matrix, int steps, const float* coefficients,
                     float eps, float scale, const void* d_base, uint64_t base_stride,
                     uint64_t base_matrix, float keep, void* d_out, int out_type, uint64_t out_stride,
                     uint64_t out_matrix, void* d_work, uint64_t work_bytes, ec_stream_t stream) {
  if (!known_type(type) || !known_type(out_type) || !coefficients) return EC_EINVAL;
  if (const int st = check_sizes(batch, rows, cols)) return st;
  if (steps < 1 || steps > EC_MAX_STEPS) return EC_ERANGE;
  for (int i = 0; i < 3; ++i)
    if (!std::isfinite(coefficients[i]) || std::fabs(coefficients[i]) > 1024.0f) return EC_EINVAL;
  if (!(eps > 0.0f) || !std::isfinite(eps) || !std::isfinite(scale) || !std::isfinite(keep)) return EC_EINVAL;
  if (x_stride < cols || out_stride < cols || (d_base && base_stride < cols)) return EC_EINVAL;
  if (!batch) return EC_OK;
  if (!d_x || !d_out) return EC_EINVAL;
  const Plan p = plan_of((uint32_t)batch, (uint32_t)rows, (uint32_t)cols);
  if (!small(rows, cols) && (!d_work || work_bytes < p.total)) return EC_EINVAL;
  if ((uintptr_t)d_work & 15u) return EC_EALIGN;
  char* work = (char*)d_work;
  const auto st = (hipStream_t)stream;
  Call c = {};
  c.x = {(const char*)d_x, x_stride, x_matrix};
  c.base = {(const char*)d_base, base_stride, base_matrix};
  c.out = (char*)d_out, c.out_stride = out_stride, c.out_matrix = out_matrix;
  c.out_type = out_type, c.steps = steps;
  c.eps = eps, c.scale = scale, c.keep = keep;
  c.k = {coefficients[0], coefficients[1], coefficients[2], 0.0f};
  if (std::isfinite(c.k.b / c.k.c)) c.k.b_by_c = c.k.b / c.k.c;
  exponents_of(c.k, steps, fast(p, out_type), c.at);
  if (small(rows, cols)) {
    with_type(type, [&](auto t) {
      return with_type(out_type, [&](auto o) {
        typedef decltype(t) T;
        typedef decltype(o) Out;
        if constexpr (__is_same(Out, bf16_t)) {
          if (fast(p, out_type)) {
            run_small<T, Out, fp16_t>(p, c, st);
            return EC_OK;
          }
        }
        run_small<T, Out, pair_t>(p, c, st);
        return EC_OK;
      });
    });
    return launched();
  }
  // rows without gaps are summed as one
  const bool dense = x_stride == cols;
  const uint64_t total = rows * cols;
  const uint64_t pieces = dense ? (total + kPiece - 1) / kPiece : rows;
  const uint32_t parts = (uint32_t)std::min<uint64_t>(p.sums, pieces);
  double* sums = (double*)(work + p.parts);
  const uint64_t blocks = (rows * ((cols + 7) / 8) + kLanes - 1) / kLanes;
  const uint32_t grid = (uint32_t)std::min<uint64_t>(blocks, std::max<uint64_t>(1, 8192 / batch));
  with_type(type, [&](auto t) {
    typedef decltype(t) T;
    square_kernel<T><<<dim3(parts, (uint32_t)batch), kLanes, 0, st>>>(
        (const T*)d_x, dense ? kPiece : x_stride, x_matrix, pieces, total, dense ? kPiece : (uint32_t)cols, sums);
    if (fast(p, out_type)) {
      const Stored x = stored<fp16_t>(work + p.x[0], p.batch, p.rows, p.cols, steps > kPlainSteps);
      scale_kernel<T, fp16_t><<<dim3(grid, (uint32_t)batch), kLanes, 0, st>>>(
          (const T*)d_x, x_stride, x_matrix, p.rows, p.cols, sums, parts, (double)eps, work + p.x[0], x.low);
    } else {
      scale_kernel<T, pair_t><<<dim3(grid, (uint32_t)batch), kLanes, 0, st>>>(
          (const T*)d_x, x_stride, x_matrix, p.rows, p.cols, sums, parts, (double)eps, work + p.x[0], 0);
    }
    return EC_OK;
  });
  const int e = rows > cols ? run_steps<true>(p, c, work, st) : run_steps<false>(p, c, work, st);
  return e ? e : launched();
}

}  // extern "C"
