// ec_ortho.hip — ec_orthogonalize: Newton-Schulz steps on a batch of matrices.
//
// X = x / (|x| + eps), then `steps` times A = X X', B = a I + b A + c A A, X = B X (from the
// other side, X' X and X B, where the matrix is tall, so that A is as small as can be), which
// takes every singular value through a s + b s^3 + c s^5.  A and B are symmetric: only the tiles on
// and above the diagonal are computed, and written twice.
//
// Small singular values grow by `a` a step, and so do the rounding errors of what is
// stored in between: with 16-bit matrices 0.2 % (fp16) or 2 % (bf16) of the result after five
// steps.  So the matrices in between are pairs of fp16 values (22 bits, ec_gemm.h), and the result is as
// good as that of fp32 products, at a third of the fp16 rate instead of the fp32 products' sixteenth.
// What is stored is 2^12 times the value: X and A have entries of at most about 1.5 (the norm
// bounds them), and ordinary ones of 1 / sqrt(columns) and less.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "ec_gemm.h"
#include "ec_pack.h"

namespace ec {
namespace {

constexpr int kLanes = 256;
constexpr uint32_t kMostParts = 64;       // of a matrix's sum of squares
constexpr uint32_t kPiece = 8192;         // elements of a contiguous matrix that are summed at a time
constexpr int kStored = 12;               // matrices are stored times 2^12
constexpr uint32_t kMostSide = 1u << 16;
constexpr uint32_t kMostBatch = 1u << 16;

struct Matrices {
  const char* p;
  uint64_t stride, matrix;   // elements from row to row, from matrix to matrix
};

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
    for (uint32_t g = threadIdx.x; g < groups; g += kLanes) {
      const typename G::wide v = widen<T>(load_group<T, false>(p + g * G::kN));
#pragma unroll
      for (int e = 0; e < G::kN; ++e) sum = __builtin_fma((double)v[e], (double)v[e], sum);
    }
    const uint32_t rest = groups * G::kN + threadIdx.x;
    if (rest < n) {
      const double v = (double)(float)gp(p)[rest];
      sum = __builtin_fma(v, v, sum);
    }
  }
  __shared__ double shared[kLanes / 64];
#pragma unroll
  for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
  if (threadIdx.x % 64 == 0) shared[threadIdx.x / 64] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kLanes / 64; ++w) sum += shared[w];
    gp(parts)[blockIdx.y * kMostParts + blockIdx.x] = sum;
  }
}

// Two fp16 values whose sum is v to 22 bits.
__device__ __forceinline__ void split(float v, fp16_t& high, fp16_t& low) {
  high = (fp16_t)v;
  low = (fp16_t)(v - (float)high);
}

typedef fp16_t __attribute__((ext_vector_type(4))) h4;
typedef fp16_t __attribute__((ext_vector_type(8))) h8;

// Columns n ... n + 3 (n a multiple of 4) of a row of pairs, or of fp16 values.
template <typename K>
__device__ __forceinline__ void put4(char* row, uint32_t n, const f4& v) {
  if constexpr (__is_same(K, pair_t)) {
    h4 high, low;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      fp16_t h, l;
      split(v[e], h, l);
      high[e] = h;
      low[e] = l;
    }
    global<char>* to = gp(row) + n / 8 * 32 + n % 8 * 2;
    *(global<h4>*)to = high;
    *(global<h4>*)(to + 16) = low;
  } else {
    *(global<h4>*)(gp(row) + n * 2) = __builtin_convertvector(v, h4);
  }
}

template <typename K>
__device__ __forceinline__ f4 get4(const char* row, uint32_t n) {
  if constexpr (__is_same(K, pair_t)) {
    const global<char>* from = gp(row) + n / 8 * 32 + n % 8 * 2;
    return __builtin_convertvector(*(const global<h4>*)from, f4) +
           __builtin_convertvector(*(const global<h4>*)(from + 16), f4);
  } else {
    return __builtin_convertvector(*(const global<h4>*)(gp(row) + n * 2), f4);
  }
}

// x / (|x| + eps) as pairs, 8 elements a lane, with zeros behind a row's end.  |x| comes from the partial sums
// in order, in every workgroup.
template <typename T>
__global__ void __launch_bounds__(kLanes) scale_kernel(const T* x, uint64_t stride, uint64_t matrix,
                                                       uint32_t rows, uint32_t cols, const double* parts,
                                                       uint32_t n_parts, double eps, char* out) {
  double sum = 0.0;
  for (uint32_t i = 0; i < n_parts; ++i) sum += gp(parts)[blockIdx.y * kMostParts + i];
  const double by = (double)(1 << kStored) / (__builtin_sqrt(sum) + eps);
  const T* from = x + blockIdx.y * matrix;
  const uint32_t groups = (cols + 7) / 8, all = rows * groups;
  char* to = out + (uint64_t)blockIdx.y * all * 32;
  for (uint32_t g = blockIdx.x * kLanes + threadIdx.x; g < all; g += gridDim.x * kLanes) {
    const uint32_t row = g / groups, at = g % groups * 8;
    const T* p = from + row * stride;
    const f4 a = load4<T>(p, at, cols);
    f4 b = {};
    if (at + 4 < cols) b = load4<T>(p, at + 4, cols);
    h8 high, low;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      fp16_t h, l;
      split((float)((double)(e < 4 ? a[e % 4] : b[e % 4]) * by), h, l);
      high[e] = h;
      low[e] = l;
    }
    global<char>* q = gp(to) + (uint64_t)g * 32;
    *(global<h8>*)q = high;
    *(global<h8>*)(q + 16) = low;
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
  const char* add;               // POLY: + linear * add + diagonal * I
  float linear, diagonal;
  Matrices base;                 // LAST: + keep * base, or none
  float keep;
};

// What becomes of a product: a symmetric matrix of K, one plus a polynomial's other terms, a matrix of
// K, or the result.
enum { kGram, kPoly, kNext, kLast };

template <class S, typename In, bool ACROSS_A, bool ACROSS_B, int WHAT, typename Out>
__global__ void __launch_bounds__(S::kLanes) ns_kernel(NsArgs p) {
  __shared__ __attribute__((aligned(1024))) char lds[S::kLds];
  const uint32_t t = xcd_order(blockIdx.x, gridDim.x), matrix = uniform(t / p.tiles);
  uint32_t tm, tn;
  constexpr bool kSymmetric = WHAT == kGram || WHAT == kPoly;
  if (kSymmetric) {   // the tiles above the diagonal, column by column
    const uint32_t i = uniform(t % p.tiles);
    for (tn = 0; (tn + 1) * (tn + 2) / 2 <= i;) ++tn;
    tm = i - tn * (tn + 1) / 2;
  } else {
    tile_at(t % p.tiles, p.tiles_m, p.tiles_n, tm, tn);
  }
  Operand a = p.a, b = p.b;
  a.p += matrix * p.a_matrix;
  b.p += matrix * p.b_matrix;
  Acc<S> acc;
  acc.clear();
  product<S, In, ACROSS_A, ACROSS_B, false>(acc, (local<char>*)lds, a, b, b, tm * S::BM, tn * S::BN, p.K);
  char* out = p.out + matrix * p.out_matrix;
  if constexpr (WHAT == kLast) {
    const uint64_t first = matrix * p.base.matrix;
    acc.each([&](uint32_t m, uint32_t n, f4 v) {
      m += tm * S::BM;
      n += tn * S::BN;
      if (m >= p.M || n >= p.N) return;
      v *= p.by;
      if (p.base.p) v += p.keep * load4<Out>((const Out*)p.base.p + first + m * p.base.stride, n, p.N);
      store4<Out>((Out*)(out + m * p.out_ld), n, p.N, v);
    });
  } else {
    const uint32_t padded = (p.N + 7) & ~7u;
    const auto value = [&](uint32_t m, uint32_t n, f4 v) {
      v *= p.by;
      if constexpr (WHAT == kPoly) {
        if (m < p.M && n < padded) {
          v += p.linear * get4<In>(p.add + matrix * p.out_matrix + m * p.out_ld, n);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (m == n + e) v[e] += p.diagonal;
        }
      }
      return v;
    };
    if (!kSymmetric || tm == tn) {
      acc.each([&](uint32_t m, uint32_t n, f4 v) {
        m += tm * S::BM;
        n += tn * S::BN;
        v = value(m, n, v);
        if (m < p.M && n < padded) put4<Out>(out + m * p.out_ld, n, v);
      });
    } else {
      // and the mirrored tile, 16 x 16 at a time turned round in the wave's part of LDS
      stage_barrier();
      constexpr uint32_t kRow = 20;
      local<float>* turn = (local<float>*)(local<char>*)lds + threadIdx.x / 64 * (16 * kRow);
      const uint32_t l = threadIdx.x % 64;
      acc.each([&](uint32_t m, uint32_t n, f4 v) {
        m += tm * S::BM;
        n += tn * S::BN;
        v = value(m, n, v);
        if (m < p.M && n < padded) put4<Out>(out + m * p.out_ld, n, v);
        *(local<f4>*)(turn + l % 16 * kRow + l / 16 * 4) = v;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        f4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = turn[(l / 16 * 4 + e) * kRow + l % 16];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        // the block's rows are at m - l % 16, its columns at n - 4 (l / 16)
        const uint32_t row = n - l / 16 * 4 + l % 16, col = m - l % 16 + l / 16 * 4;
        if (row < p.N && col < padded) put4<Out>(out + row * p.out_ld, col, w);
      });
    }
  }
}

template <typename In, bool ACROSS_A, bool ACROSS_B, int WHAT, typename Out>
int run_ns(NsArgs& p, uint32_t batch, hipStream_t st) {
  constexpr bool kSymmetric = WHAT == kGram || WHAT == kPoly;
  int status = EC_OK;
  const auto tiles = [&](uint64_t side) {
    const uint64_t n = (p.N + side - 1) / side;
    return kSymmetric ? n * (n + 1) / 2 * batch : tiles_of(p.M, p.N, side) * batch;
  };
  with_shape<true>(tiles, [&](auto s) {
    typedef decltype(s) S;
    p.tiles_m = (p.M + S::BM - 1) / S::BM;
    p.tiles_n = (p.N + S::BN - 1) / S::BN;
    p.tiles = (uint32_t)(tiles(S::BM) / batch);
    if ((uint64_t)p.tiles * batch >= (1ull << 32) / S::kLanes)
      status = EC_ERANGE;
    else
      ns_kernel<S, In, ACROSS_A, ACROSS_B, WHAT, Out><<<p.tiles * batch, S::kLanes, 0, st>>>(p);
  });
  return status;
}

struct Plan {
  uint32_t batch, rows, cols, side, other;   // side: of the symmetric matrices
  uint64_t parts, x[2], gram, poly, total;
};

Plan plan_of(uint32_t batch, uint32_t rows, uint32_t cols) {
  Plan p = {};
  p.batch = batch, p.rows = rows, p.cols = cols;
  p.side = std::min(rows, cols), p.other = std::max(rows, cols);
  const auto take = [&](uint64_t bytes) {
    const uint64_t at = p.total;
    p.total += part(bytes);
    return at;
  };
  const uint64_t x = (uint64_t)batch * rows * up_to(cols, 8) * 4;
  const uint64_t square = (uint64_t)batch * p.side * up_to(p.side, 8) * 4;
  p.parts = take((uint64_t)batch * kMostParts * sizeof(double));
  p.x[0] = take(x), p.x[1] = take(x);
  p.gram = take(square), p.poly = take(square);
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
  float a, b, c, eps, scale, keep;
};

template <bool TALL>
int run_steps(const Plan& p, const Call& c, char* work, hipStream_t st) {
  const auto matrix = [&](uint64_t at, uint32_t rows, uint32_t cols) {
    return Operand{work + at, up_to(cols, 8) * 4, rows};
  };
  // stored times 2^at so that a I + b A + c A A stays below fp16's largest value
  const float most = std::fabs(c.a) + 2.0f * std::fabs(c.b) + 4.0f * std::fabs(c.c);
  int at = kStored;
  while (at > 0 && std::ldexp(most, at) > 32768.0f) --at;
  for (int s = 0; s < c.steps; ++s) {
    const Operand x = matrix(p.x[s & 1], p.rows, p.cols);
    const uint64_t xm = x.ld * p.rows;
    Operand gram = matrix(p.gram, p.side, p.side), poly = matrix(p.poly, p.side, p.side);
    const uint64_t gm = gram.ld * p.side;
    NsArgs n = {};
    n.a = n.b = x;
    n.a.rows = n.b.rows = p.side;
    n.a_matrix = n.b_matrix = xm;
    n.K = p.other, n.M = n.N = p.side;
    n.out = work + p.gram, n.out_ld = gram.ld, n.out_matrix = gm;
    n.by = std::ldexp(1.0f, -kStored);
    if (const int e = run_ns<pair_t, TALL, TALL, kGram, pair_t>(n, p.batch, st)) return e;
    n.a = n.b = gram;
    n.a_matrix = n.b_matrix = gm;
    n.K = p.side;
    n.out = work + p.poly;
    n.add = work + p.gram;
    n.by = c.c * std::ldexp(1.0f, at - 2 * kStored);
    n.linear = c.b * std::ldexp(1.0f, at - kStored);
    n.diagonal = c.a * std::ldexp(1.0f, at);
    if (const int e = run_ns<pair_t, false, false, kPoly, pair_t>(n, p.batch, st)) return e;
    // X = B X, X across; or X B, X along
    n.a = TALL ? x : poly, n.b = TALL ? poly : x;
    n.a.rows = p.rows, n.b.rows = p.cols;
    n.a_matrix = TALL ? xm : gm, n.b_matrix = TALL ? gm : xm;
    n.M = p.rows, n.N = p.cols;
    if (s + 1 < c.steps) {
      n.out = work + p.x[(s + 1) & 1], n.out_ld = x.ld, n.out_matrix = xm;
      n.by = std::ldexp(1.0f, -at);
      if (const int e = run_ns<pair_t, false, !TALL, kNext, pair_t>(n, p.batch, st)) return e;
    } else {
      const uint32_t w = type_bytes(c.out_type);
      n.out = c.out, n.out_ld = c.out_stride * w, n.out_matrix = c.out_matrix * w;
      n.by = c.scale * std::ldexp(1.0f, -at - kStored);
      n.base = c.base, n.keep = c.keep;
      const int e = with_type(c.out_type, [&](auto o) {
        return run_ns<pair_t, false, !TALL, kLast, decltype(o)>(n, p.batch, st);
      });
      if (e) return e;
    }
  }
  return EC_OK;
}

}  // namespace
}  // namespace ec

using namespace ec;

extern "C" {

uint64_t ec_orthogonalize_workspace(uint64_t batch, uint64_t rows, uint64_t cols) {
  if (!batch || check_sizes(batch, rows, cols) != EC_OK) return 0;
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
  if (!d_work || work_bytes < p.total) return EC_EINVAL;
  if ((uintptr_t)d_work & 15u) return EC_EALIGN;
  char* work = (char*)d_work;
  const auto st = (hipStream_t)stream;
  // rows without gaps are summed as one
  const bool dense = x_stride == cols;
  const uint64_t total = rows * cols;
  const uint64_t pieces = dense ? (total + kPiece - 1) / kPiece : rows;
  const uint32_t parts = (uint32_t)std::min<uint64_t>(kMostParts, pieces);
  double* sums = (double*)(work + p.parts);
  const uint64_t blocks = (rows * ((cols + 7) / 8) + kLanes - 1) / kLanes;
  const uint32_t grid = (uint32_t)std::min<uint64_t>(blocks, std::max<uint64_t>(1, 8192 / batch));
  with_type(type, [&](auto t) {
    typedef decltype(t) T;
    square_kernel<T><<<dim3(parts, (uint32_t)batch), kLanes, 0, st>>>(
        (const T*)d_x, dense ? kPiece : x_stride, x_matrix, pieces, total, dense ? kPiece : (uint32_t)cols, sums);
    scale_kernel<T><<<dim3(grid, (uint32_t)batch), kLanes, 0, st>>>(
        (const T*)d_x, x_stride, x_matrix, (uint32_t)rows, (uint32_t)cols, sums, parts, (double)eps,
        work + p.x[0]);
    return EC_OK;
  });
  Call c = {};
  c.base = {(const char*)d_base, base_stride, base_matrix};
  c.out = (char*)d_out, c.out_stride = out_stride, c.out_matrix = out_matrix;
  c.out_type = out_type, c.steps = steps;
  c.a = coefficients[0], c.b = coefficients[1], c.c = coefficients[2];
  c.scale = scale, c.keep = keep;
  const int e = rows > cols ? run_steps<true>(p, c, work, st) : run_steps<false>(p, c, work, st);
  return e ? e : launched();
}

}  // extern "C"
