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

// 16 bytes of the result a lane.
template <typename T>
__global__ void __launch_bounds__(kPackLanes) pack_kernel(const T* src, uint64_t stride, uint64_t rows,
                                                          uint32_t width, uint32_t groups, T* dst) {
  typedef Group<T> G;
  const uint64_t n = rows * groups;
  for (uint64_t g = (uint64_t)blockIdx.x * kPackLanes + threadIdx.x; g < n;
       g += (uint64_t)gridDim.x * kPackLanes) {
    const uint64_t row = g / groups;
    const uint32_t at = (uint32_t)(g % groups) * G::kN;
    const T* from = src + row * stride + at;
    typename G::vec v = {};
    if (at + G::kN <= width) {
      v = load_group<T, true>(from);
    } else {
#pragma unroll
      for (int e = 0; e < G::kN; ++e)
        if (at + e < width) v[e] = gp(from)[e];
    }
    store_group<T, false>(dst + g * G::kN, v);
  }
}

template <typename T>
void pack(const T* src, uint64_t stride, uint64_t rows, uint32_t width, T* dst, hipStream_t st) {
  const uint32_t groups = (uint32_t)(up_to(width, Group<T>::kN) / Group<T>::kN);
  const uint64_t blocks = (rows * groups + kPackLanes - 1) / kPackLanes;
  pack_kernel<T><<<(uint32_t)(blocks < 8192 ? blocks : 8192), kPackLanes, 0, st>>>(src, stride, rows, width,
                                                                                  groups, dst);
}

}  // namespace
}  // namespace ec
