// ec_pack.h — rows brought to where ec_gemm.h can read them: 16-byte aligned, a multiple of 16
// bytes apart, zeros behind a row's end.  Memory-bound, one pass; taken for operands that are not so.
#pragma once

#include "ec_gemm.h"

namespace ec {
namespace {

inline uint64_t up_to(uint64_t n, uint64_t unit) { return (n + unit - 1) / unit * unit; }
inline uint64_t part(uint64_t bytes) { return up_to(bytes, 256); }   // of a workspace

// Whether ec_gemm.h can read rows of `width` elements of `bytes` as they are: also rows so far
// apart that a tile's would not lie within one buffer are copied.
inline bool readable(const void* p, uint64_t width, uint64_t stride, uint32_t bytes) {
  return (uintptr_t)p % 16 == 0 && width * bytes % 16 == 0 && stride * bytes % 16 == 0 &&
         stride * bytes <= (4u << 20);
}

constexpr int kPackLanes = 256;

// What is packed in one launch, blockIdx.y's each.
template <typename T>
struct PackArgs {
  const T* src[3];
  uint64_t stride[3], rows[3];
  T* dst[3];
  uint32_t width, groups;
};

// 16 bytes of the result a lane.
template <typename T>
__global__ void __launch_bounds__(kPackLanes) pack_kernel(PackArgs<T> p) {
  typedef Group<T> G;
  const T* src = p.src[blockIdx.y];
  const uint64_t stride = p.stride[blockIdx.y], n = p.rows[blockIdx.y] * p.groups;
  T* dst = p.dst[blockIdx.y];
  for (uint64_t g = (uint64_t)blockIdx.x * kPackLanes + threadIdx.x; g < n;
       g += (uint64_t)gridDim.x * kPackLanes) {
    const uint64_t row = g / p.groups;
    const uint32_t at = (uint32_t)(g % p.groups) * G::kN;
    const T* from = src + row * stride + at;
    typename G::vec v = {};
    if (at + G::kN <= p.width) {
      v = load_group<T, true>(from);
    } else {
#pragma unroll
      for (int e = 0; e < G::kN; ++e)
        if (at + e < p.width) v[e] = gp(from)[e];
    }
    store_group<T, false>(dst + g * G::kN, v);
  }
}

// Rows of one width, up to three times, in one launch.
template <typename T>
struct Packer {
  PackArgs<T> p = {};
  uint32_t n = 0;
  uint64_t most = 0;

  explicit Packer(uint32_t width) {
    p.width = width;
    p.groups = (uint32_t)(up_to(width, Group<T>::kN) / Group<T>::kN);
  }
  void add(const T* src, uint64_t stride, uint64_t rows, T* dst) {
    p.src[n] = src, p.stride[n] = stride, p.rows[n] = rows, p.dst[n] = dst;
    most = rows > most ? rows : most;
    ++n;
  }
  void run(hipStream_t st) const {
    const uint64_t blocks = (most * p.groups + kPackLanes - 1) / kPackLanes;
    if (n) pack_kernel<T><<<dim3((uint32_t)(blocks < 8192 ? blocks : 8192), n), kPackLanes, 0, st>>>(p);
  }
};

}  // namespace
}  // namespace ec
