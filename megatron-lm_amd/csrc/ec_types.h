// ec_types.h — element types and group accesses of the training-step kernels
// (ec_embed.hip, ec_logprobs.hip, ec_grads.hip) and the block's (ec_ff.hip, ec_norms.hip, ec_ortho.hip).
//
// A group is the 16 bytes one lane moves at once: 4 fp32 or 8 bf16 / fp16
// elements, at any address that is a multiple of the element's size (the vector
// types are declared with that alignment; gfx950 loads and stores them as one
// dwordx4 all the same).  All arithmetic is in fp32 and more; a result is
// rounded to the element's type once, to nearest even, where it is stored.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ec_mi355.h"

namespace ec {
namespace {

typedef __bf16 bf16_t;
typedef _Float16 fp16_t;

template <typename T>
struct Group {
  static constexpr int kN = 16 / (int)sizeof(T);
  typedef T __attribute__((ext_vector_type(16 / sizeof(T)))) vec;
  typedef T __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T)))) any;
  typedef float __attribute__((ext_vector_type(16 / sizeof(T)))) wide;
};

template <typename T>
using global = __attribute__((address_space(1))) T;

template <typename T>
__device__ __forceinline__ const global<T>* gp(const T* p) {
  return (const global<T>*)(uintptr_t)p;
}
template <typename T>
__device__ __forceinline__ global<T>* gp(T* p) {
  return (global<T>*)(uintptr_t)p;
}

// Raw groups (kept packed until they are used, half the registers of the
// converted ones for 16-bit types), streamed (STREAM: read or written once, not
// worth a place in the caches) or cached.
template <typename T, bool STREAM>
__device__ __forceinline__ typename Group<T>::vec load_group(const T* p) {
  typedef typename Group<T>::any any;
  const auto* q = (const global<any>*)(uintptr_t)p;
  if constexpr (STREAM) return __builtin_nontemporal_load(q);
  return *q;
}

template <typename T, bool STREAM>
__device__ __forceinline__ void store_group(T* p, const typename Group<T>::vec& v) {
  typedef typename Group<T>::any any;
  auto* q = (global<any>*)(uintptr_t)p;
  if constexpr (STREAM)
    __builtin_nontemporal_store((any)v, q);
  else
    *q = v;
}

template <typename T>
__device__ __forceinline__ typename Group<T>::wide widen(const typename Group<T>::vec& v) {
  return __builtin_convertvector(v, typename Group<T>::wide);
}

// `n` floats rounded to T, stored at p as one group (n = Group<T>::kN) at any
// element address.
template <typename T, bool STREAM, typename W>
__device__ __forceinline__ void store_wide(T* p, const W& w) {
  store_group<T, STREAM>(p, __builtin_convertvector(w, typename Group<T>::vec));
}

template <typename T>
__device__ __forceinline__ float to_float(T v) {
  return (float)v;
}

inline bool known_type(int type) { return type == EC_F32 || type == EC_BF16 || type == EC_F16; }
inline uint32_t type_bytes(int type) { return type == EC_F32 ? 4u : 2u; }

// f(T()) with the element type of the status-checked `type`.
template <typename F>
inline int with_type(int type, F f) {
  switch (type) {
    case EC_F32: return f(float());
    case EC_BF16: return f(bf16_t());
    default: return f(fp16_t());
  }
}

inline int launched() { return hipGetLastError() == hipSuccess ? EC_OK : EC_EHIP; }

}  // namespace
}  // namespace ec
