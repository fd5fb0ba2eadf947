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

// Every element of a piece through f (groups, and the elements behind the last).
template <typename T, typename F, typename S>
__device__ __forceinline__ void each_group(uint64_t src, uint32_t n, F group, S single) {
  typedef Group<T> G;
  const T* p = (const T*)src;
  const uint32_t groups = n / G::kN;
  for (uint32_t g = threadIdx.x; g < groups; g += kBlockLanes * kAhead) {
    typename G::vec v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (g + u * kBlockLanes < groups)
        v[u] = load_group<T, false>(p + (uint64_t)(g + u * kBlockLanes) * G::kN);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (g + u * kBlockLanes < groups) group(g + u * kBlockLanes, widen<T>(v[u]));
  }
  const uint32_t rest = groups * G::kN + threadIdx.x;
  if (rest < n) single(rest, (float)gp(p)[rest]);
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

template <int NORM>
__global__ void __launch_bounds__(kBlockLanes) grad_parts_kernel(const ec_grad_item* items,
                                                                 uint32_t n_items, double* parts) {
  Acc acc;
  for (uint32_t i = blockIdx.x; i < n_items; i += gridDim.x) {
    const ec_grad_item it = items[i];
    const auto piece = [&](auto t) {
      typedef decltype(t) T;
      each_group<T>(it.src, it.n,
                    [&](uint32_t, const typename Group<T>::wide& x) {
#pragma unroll
                      for (int e = 0; e < Group<T>::kN; ++e) acc.template add<NORM>(x[e]);
                    },
                    [&](uint32_t, float x) { acc.template add<NORM>(x); });
    };
    if (it.src_type == EC_F32)
      piece(float());
    else if (it.src_type == EC_BF16)
      piece(bf16_t());
    else
      piece(fp16_t());
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

template <int NORM>
__global__ void __launch_bounds__(kBlockLanes) grad_clip_kernel(
    const ec_grad_item* items, uint32_t n_items, const double* parts, uint32_t n_parts,
    float scale, float max_norm, const float* given, float* norm) {
  const float v = given ? *gp(given) : join_parts<NORM>(parts, n_parts, scale);
  if (blockIdx.x == 0 && threadIdx.x == 0) *gp(norm) = v;
  float by = scale;
  if (__builtin_isfinite(v)) by *= fminf(1.0f, max_norm / (v + kEps));
  // from the list's end: what the norm read last may still be in the Infinity Cache
  for (uint32_t k = blockIdx.x; k < n_items; k += gridDim.x) {
    const ec_grad_item it = items[n_items - 1 - k];
    if (by == 1.0f && it.src == it.dst && it.src_type == it.dst_type) continue;
    const auto piece = [&](auto t, auto o) {
      typedef decltype(t) T;
      typedef decltype(o) O;
      constexpr int N = Group<T>::kN, M = Group<O>::kN;
      O* out = (O*)it.dst;
      each_group<T>(it.src, it.n,
                    [&](uint32_t g, const typename Group<T>::wide& x) {
                      const typename Group<T>::wide w = x * by;
                      O* to = out + (uint64_t)g * N;
                      if constexpr (N == M) {
                        store_wide<O, true>(to, w);
                      } else if constexpr (N > M) {   // 16-bit to fp32: two groups
                        store_wide<O, true>(to, __builtin_shufflevector(w, w, 0, 1, 2, 3));
                        store_wide<O, true>(to + M, __builtin_shufflevector(w, w, 4, 5, 6, 7));
                      } else {                        // fp32 to 16-bit
#pragma unroll
                        for (int e = 0; e < N; ++e) gp(to)[e] = (O)w[e];
                      }
                    },
                    [&](uint32_t j, float x) { gp(out)[j] = (O)(x * by); });
    };
    const auto from = [&](auto t) {
      if (it.dst_type == EC_F32)
        piece(t, float());
      else if (it.dst_type == EC_BF16)
        piece(t, bf16_t());
      else
        piece(t, fp16_t());
    };
    if (it.src_type == EC_F32)
      from(float());
    else if (it.src_type == EC_BF16)
      from(bf16_t());
    else
      from(fp16_t());
  }
}

int check_list(const ec_grad_item* items, uint32_t n, float scale, int norm, const void* work,
               const float* out) {
  if (!std::isfinite(scale) || (norm != EC_NORM_2 && norm != EC_NORM_INF)) return EC_EINVAL;
  if (!work || !out || (n && !items)) return EC_EINVAL;
  if ((uintptr_t)work & 7u) return EC_EALIGN;
  return EC_OK;
}

template <int NORM>
uint32_t run_parts(const ec_grad_item* items, uint32_t n, double* parts, hipStream_t st) {
  const uint32_t blocks = std::min(n, kParts);
  if (blocks) grad_parts_kernel<NORM><<<blocks, kBlockLanes, 0, st>>>(items, n, parts);
  return blocks;
}

template <int NORM>
int run_norm(const ec_grad_item* items, uint32_t n, float scale, double* parts, float* norm,
             hipStream_t st) {
  const uint32_t blocks = run_parts<NORM>(items, n, parts, st);
  grad_norm_kernel<NORM><<<1, kBlockLanes, 0, st>>>(parts, blocks, scale, norm);
  return launched();
}

constexpr uint32_t kClipBlocks = 2048;

template <int NORM>
int run_clip(const ec_grad_item* items, uint32_t n, float scale, float max_norm, const float* given,
             double* parts, float* norm, hipStream_t st) {
  const uint32_t blocks = given ? 0 : run_parts<NORM>(items, n, parts, st);
  grad_clip_kernel<NORM><<<std::max(1u, std::min(n, kClipBlocks)), kBlockLanes, 0, st>>>(
      items, n, parts, blocks, scale, max_norm, given, norm);
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
