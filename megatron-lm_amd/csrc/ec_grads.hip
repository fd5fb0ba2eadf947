// ec_grads.hip — ec_grad_norm and ec_grad_clip: the norm of a list of gradient
// tensors and the list scaled to at most a given norm.
//
// The list comes as pieces of at most EC_GRAD_PIECE elements, so that one large
// matrix and a thousand biases spread over the workgroups alike.  Each of up to
// kParts workgroups adds the squares of every kParts-th piece in fp64 (a square of an
// fp32 value is exact there, cannot overflow, and the sum's error is far below the
// result's fp32 rounding) and leaves one partial; the next launch adds the partials in
// order.  Two launches, no atomics, and the norm does not depend on timing.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "ec_types.h"
#include "routes.h"

namespace ec {
namespace {

constexpr int kLanes = 64;
constexpr int kBlockLanes = 256;
constexpr int kWaves = kBlockLanes / kLanes;
constexpr uint32_t kParts = EC_GRAD_WORK / sizeof(double);
constexpr int kAhead = 4;
constexpr float kEps = 1e-6f;

// The largest magnitude as the bits of its absolute value: their order as
// integers is the values' order, with NaN above infinity.
struct Acc {
  double sum = 0.0;
  uint32_t most = 0;

  template <int NORM>
  __device__ __forceinline__ void add(float v) {
    if (NORM == EC_NORM_2)
      sum = __builtin_fma((double)v, (double)v, sum);
    else
      most = max(most, __float_as_uint(v) & 0x7fffffffu);
  }
};

// f with the element type of `type`.
template <typename F>
__device__ __forceinline__ void with_element(uint32_t type, F f) {
  if (type == EC_F32)
    f(float());
  else if (type == EC_BF16)
    f(bf16_t());
  else
    f(fp16_t());
}

template <int NORM>
__device__ __forceinline__ double block_reduce(const Acc& acc) {
  __shared__ double shared[kWaves];
  double v = NORM == EC_NORM_2 ? acc.sum : (double)__uint_as_float(acc.most);
  // a NaN stays one through the maxima: it compares false, so it is looked at first
  const auto join = [](double x, double y) {
    if (NORM == EC_NORM_2) return x + y;
    return x != x ? x : y != y ? y : x > y ? x : y;
  };
#pragma unroll
  for (int o = 32; o; o >>= 1) v = join(v, __shfl_xor(v, o));
  if (threadIdx.x % kLanes == 0) shared[threadIdx.x / kLanes] = v;
  __syncthreads();
  v = shared[0];
  for (int w = 1; w < kWaves; ++w) v = join(v, shared[w]);
  return v;
}

template <int NORM, bool STREAM, typename T>
__device__ __forceinline__ void add_piece(Acc& acc, const T* p, uint32_t n) {
  typedef Group<T> G;
  const uint32_t groups = n / G::kN;
  for (uint32_t g = threadIdx.x; g < groups; g += kBlockLanes * kAhead) {
    typename G::vec v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)   // without conditions, so that all are in flight together
      v[u] = load_group<T, STREAM>(p + (uint64_t)min(g + u * kBlockLanes, groups - 1) * G::kN);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (g + u * kBlockLanes < groups) {
        const typename G::wide x = widen<T>(v[u]);
#pragma unroll
        for (int e = 0; e < G::kN; ++e) acc.template add<NORM>(x[e]);
      }
  }
  const uint32_t rest = groups * G::kN + threadIdx.x;
  if (rest < n) acc.template add<NORM>((float)gp(p)[rest]);
}

template <int NORM, bool STREAM>
__global__ void __launch_bounds__(kBlockLanes) grad_parts_kernel(const ec_grad_item* items,
                                                                 uint32_t n_items, double* parts) {
  Acc acc;
  for (uint32_t i = blockIdx.x; i < n_items; i += gridDim.x) {
    const ec_grad_item it = items[i];
    with_element(it.src_type, [&](auto t) {
      typedef decltype(t) T;
      add_piece<NORM, STREAM, T>(acc, (const T*)it.src, it.n);
    });
  }
  const double v = block_reduce<NORM>(acc);
  if (threadIdx.x == 0) gp(parts)[blockIdx.x] = v;
}

// The norm from the partials, the same in every workgroup.
template <int NORM>
__device__ __forceinline__ float join_parts(const double* parts, uint32_t n, float scale) {
  Acc acc;
  for (uint32_t i = threadIdx.x; i < n; i += kBlockLanes) {
    const double v = gp(parts)[i];
    if (NORM == EC_NORM_2)
      acc.sum += v;
    else
      acc.template add<NORM>((float)v);
  }
  const double v = block_reduce<NORM>(acc);
  return (float)((NORM == EC_NORM_2 ? __builtin_sqrt(v) : v) * (double)__builtin_fabsf(scale));
}

template <int NORM>
__global__ void __launch_bounds__(kBlockLanes) grad_norm_kernel(const double* parts, uint32_t n,
                                                                float scale, float* norm) {
  const float v = join_parts<NORM>(parts, n, scale);
  if (threadIdx.x == 0) *gp(norm) = v;
}

// The factor of ec_grad_clip for a norm.
__device__ __forceinline__ float clip_factor(float norm, float scale, float max_norm) {
  return __builtin_isfinite(norm) ? scale * fminf(1.0f, max_norm / (norm + kEps)) : scale;
}

// Group g of 16 bytes of a piece, as its raw bits; nothing where it is not whole.
typedef uint32_t __attribute__((ext_vector_type(4))) raw_t;
template <bool STREAM>
__device__ __forceinline__ raw_t load_raw(const ec_grad_item& it, uint32_t g) {
  typedef uint32_t __attribute__((ext_vector_type(4), aligned(2))) any_t;
  const uint32_t groups = it.n / (it.src_type == EC_F32 ? 4 : 8);
  raw_t v = {};
  if (g < groups) {
    const auto* p = (const global<any_t>*)(uintptr_t)(it.src + (uint64_t)g * 16);
    v = STREAM ? __builtin_nontemporal_load(p) : *p;
  }
  return v;
}

// The elements of group g, scaled.  Where a lane's result is two groups (16-bit to
// fp32) the stores go through the caches, which join the halves of a line: 534 M
// elements, norm and clip, 730 us against 814 streamed.
template <typename T, typename O>
__device__ __forceinline__ void scale_group(const ec_grad_item& it, uint32_t g, const raw_t& raw,
                                            float by) {
  typedef Group<T> G;
  constexpr int N = G::kN;
  const T* src = (const T*)it.src;
  O* dst = (O*)it.dst;
  const uint32_t j = g * N;
  if (j + N <= it.n) {
    const typename G::wide w = widen<T>(__builtin_bit_cast(typename G::vec, raw)) * by;
    if constexpr (N > Group<O>::kN) {
      store_wide<O, false>(dst + j, __builtin_shufflevector(w, w, 0, 1, 2, 3));
      store_wide<O, false>(dst + j + 4, __builtin_shufflevector(w, w, 4, 5, 6, 7));
    } else {
      typedef O __attribute__((ext_vector_type(N), aligned(sizeof(O)))) some;
      __builtin_nontemporal_store((some)__builtin_convertvector(w, some),
                                  (global<some>*)(uintptr_t)(dst + j));
    }
  } else {
    for (uint32_t e = j; e < it.n; ++e) gp(dst)[e] = (O)((float)gp(src)[e] * by);
  }
}

// f(T(), O()) with the types of a piece.
template <typename F>
__device__ __forceinline__ void with_types(const ec_grad_item& it, F f) {
  with_element(it.src_type, [&](auto t) { with_element(it.dst_type, [&](auto o) { f(t, o); }); });
}

__device__ __forceinline__ bool unchanged(const ec_grad_item& it, float by) {
  return by == 1.0f && it.src == it.dst && it.src_type == it.dst_type;
}

// kSplit workgroups for a piece, which take neighbouring 4 KiB of it, one or two
// groups a lane, from the list's end (what the norm read last may still be in the
// Infinity Cache).  1.3 G fp32 elements: norm 740 us (7.1 TB/s; 850 with cached reads),
// clip 1630 us (6.4 TB/s) against 2050 with 2048 workgroups that walk whole pieces.
// JOIN: each workgroup joins the norm's partials by itself, a launch less.
constexpr uint32_t kSplit = 8;

template <int NORM, bool JOIN, bool STREAM>
__global__ void __launch_bounds__(kBlockLanes) grad_clip_kernel(
    const ec_grad_item* items, uint32_t n_items, const double* parts, uint32_t n_parts, float scale,
    float max_norm, const float* given, float* norm) {
  const uint32_t back = gridDim.x - 1 - blockIdx.x;
  ec_grad_item it = {};
  if (back / kSplit < n_items) it = items[back / kSplit];
  // a lane's groups are under way while the norm is found; of long lists the second (of
  // fp32) only behind the first one's store, which keeps to the memory's order (1.3 G
  // elements, norm and clip, 2385 us against 2415)
  constexpr uint32_t kStep = kSplit * kBlockLanes;
  const uint32_t g = back % kSplit * kBlockLanes + threadIdx.x;
  const raw_t first = load_raw<STREAM>(it, g);
  raw_t second = {};
  if (!STREAM) second = load_raw<STREAM>(it, g + kStep);
  const float v = JOIN ? join_parts<NORM>(parts, n_parts, scale) : *gp(given);
  if (norm != given && blockIdx.x == 0 && threadIdx.x == 0) *gp(norm) = v;
  const float by = clip_factor(v, scale, max_norm);
  if (unchanged(it, by)) return;
  with_types(it, [&](auto t, auto o) {
    typedef decltype(t) T;
    typedef decltype(o) O;
    static_assert(EC_GRAD_PIECE <= 2 * kStep * 4, "two groups a lane");
    scale_group<T, O>(it, g, first, by);
    if (STREAM) second = load_raw<STREAM>(it, g + kStep);
    scale_group<T, O>(it, g + kStep, second, by);
  });
}

constexpr uint32_t kMaxPieces = 1u << 28;   // of 16384 elements: more than any memory

int check_list(const ec_grad_item* items, uint32_t n, float scale, int norm, const void* work,
               const float* out) {
  if (!std::isfinite(scale) || (norm != EC_NORM_2 && norm != EC_NORM_INF)) return EC_EINVAL;
  if (!work || !out || (n && !items)) return EC_EINVAL;
  if (n > kMaxPieces) return EC_ERANGE;
  if ((uintptr_t)work & 7u) return EC_EALIGN;
  return EC_OK;
}

// Pieces above which reads are streamed (about 128 MiB of fp32, half the Infinity Cache),
// and up to which the clip joins the partials itself.
constexpr uint32_t kManyPieces = 2048;
constexpr uint32_t kFewPieces = 256;

template <int NORM>
uint32_t run_parts(const ec_grad_item* items, uint32_t n, double* parts, hipStream_t st) {
  const uint32_t blocks = std::min(n, kParts);
  if (n > kManyPieces)
    grad_parts_kernel<NORM, true><<<blocks, kBlockLanes, 0, st>>>(items, n, parts);
  else if (blocks)
    grad_parts_kernel<NORM, false><<<blocks, kBlockLanes, 0, st>>>(items, n, parts);
  return blocks;
}

template <int NORM>
int run_norm(const ec_grad_item* items, uint32_t n, float scale, double* parts, float* norm,
             hipStream_t st) {
  const uint32_t blocks = run_parts<NORM>(items, n, parts, st);
  grad_norm_kernel<NORM><<<1, kBlockLanes, 0, st>>>(parts, blocks, scale, norm);
  return launched();
}

template <int NORM>
int run_clip(const ec_grad_item* items, uint32_t n, float scale, float max_norm, const float* given,
             double* parts, float* norm, hipStream_t st) {
  if (n && n <= kFewPieces && !given) {
    const uint32_t n_parts = run_parts<NORM>(items, n, parts, st);
    grad_clip_kernel<NORM, true, false><<<n * kSplit, kBlockLanes, 0, st>>>(
        items, n, parts, n_parts, scale, max_norm, given, norm);
    return launched();
  }
  if (!given) {
    const int status = run_norm<NORM>(items, n, scale, parts, norm, st);
    if (status != EC_OK || !n) return status;
    given = norm;
  }
  const auto kernel = n > kManyPieces ? grad_clip_kernel<NORM, false, true>
                                      : grad_clip_kernel<NORM, false, false>;
  // what a launch takes at most, from the list's end; an empty list's norm is still written
  constexpr uint32_t kMost = (uint32_t)(max_grid(kBlockLanes) / kSplit);
  do {
    const uint32_t some = std::min(n, kMost);
    n -= some;
    kernel<<<std::max(1u, some) * kSplit, kBlockLanes, 0, st>>>(items + n, some, parts, 0, scale, max_norm,
                                                                given, norm);
  } while (n);
  return launched();
}

}  // namespace
}  // namespace ec

using namespace ec;

extern "C" {

int ec_grad_norm(const ec_grad_item* d_items, uint32_t n_items, float grad_scale, int norm,
                 void* d_work, float* d_norm, ec_stream_t stream) {
  if (const int st = check_list(d_items, n_items, grad_scale, norm, d_work, d_norm)) return st;
  const auto run = norm == EC_NORM_2 ? run_norm<EC_NORM_2> : run_norm<EC_NORM_INF>;
  return run(d_items, n_items, grad_scale, (double*)d_work, d_norm, (hipStream_t)stream);
}

int ec_grad_clip(const ec_grad_item* d_items, uint32_t n_items, float grad_scale, int norm,
                 float max_norm, const float* d_given, void* d_work, float* d_norm,
                 ec_stream_t stream) {
  if (const int st = check_list(d_items, n_items, grad_scale, norm, d_work, d_norm)) return st;
  if (!(max_norm > 0.0f)) return EC_EINVAL;
  const auto run = norm == EC_NORM_2 ? run_clip<EC_NORM_2> : run_clip<EC_NORM_INF>;
  return run(d_items, n_items, grad_scale, max_norm, d_given, (double*)d_work, d_norm,
             (hipStream_t)stream);
}

}  // extern "C"
