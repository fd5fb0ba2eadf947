// torch_checks.h — what the torch-tensor bindings of the operators (step_torch.cpp, block_torch.cpp)
// check of their tensors, and torch's current stream.
#pragma once

#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cstdint>
#include <optional>
#include <string>
#include <vector>

#include "ec_mi355.h"

namespace {

using at::Tensor;

inline int type_code(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return EC_F32;
    case at::kBFloat16: return EC_BF16;
    case at::kHalf: return EC_F16;
    default:
      throw py::value_error(std::string(what) + " must be float32, bfloat16 or float16, not " +
                            c10::toString(t.scalar_type()));
  }
}

inline at::ScalarType torch_type(int64_t code) {
  return code == EC_F32 ? at::kFloat : code == EC_BF16 ? at::kBFloat16 : at::kHalf;
}

inline void check_device(const Tensor& t, const char* what, const c10::Device* device) {
  // (the operators have no forward-mode derivatives, and a result without a tangent would pass for one whose is zero)
  if (t._fw_grad(/*level=*/0).defined())
    throw py::value_error(std::string(what) + " has a forward-mode tangent, which the operators do not pass on");
  if (!t.is_cuda()) throw py::value_error(std::string(what) + " must be a device (HIP) tensor");
  if (device && t.device() != *device)
    throw py::value_error(std::string(what) + " is on " + t.device().str() +
                          ", the other operands on " + device->str());
}

inline void check_dense(const Tensor& t, const char* what, const c10::Device* device) {
  check_device(t, what, device);
  if (!t.is_contiguous()) throw py::value_error(std::string(what) + " must be contiguous");
}

inline void check_type(const Tensor& t, const char* what, at::ScalarType want) {
  if (t.scalar_type() != want)
    throw py::value_error(std::string(what) + " must be " + c10::toString(want) + ", not " +
                          c10::toString(t.scalar_type()));
}

inline std::string shape_text(at::IntArrayRef s) {
  std::string r = "[";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + "]";
}

inline void check_shape(const Tensor& t, const char* what, at::IntArrayRef want) {
  if (t.sizes() != want)
    throw py::value_error(std::string(what) + " has shape " + shape_text(t.sizes()) +
                          ", expected " + shape_text(want));
}

// Rows of adjacent elements: [..., width] contiguous, or [rows, width] with any
// row stride of at least width.
struct Rows {
  uint64_t n, width, stride;
};

inline Rows rows_of(const Tensor& t, const char* what, const c10::Device* device) {
  check_device(t, what, device);
  if (t.dim() < 1) throw py::value_error(std::string(what) + " must have at least one dimension");
  const int64_t width = t.size(-1);
  int64_t n = 1;
  for (int64_t d = 0; d + 1 < t.dim(); ++d) n *= t.size(d);
  const int64_t least = std::max<int64_t>(width, 1);
  if (t.is_contiguous() || t.numel() == 0)
    return {(uint64_t)n, (uint64_t)width, (uint64_t)least};
  if (t.dim() == 2 && (width == 1 || t.stride(1) == 1) && (n == 1 || t.stride(0) >= width))
    return {(uint64_t)n, (uint64_t)width, (uint64_t)(n == 1 ? least : t.stride(0))};
  throw py::value_error(std::string(what) +
                        " must be contiguous, or two-dimensional with adjacent elements in "
                        "rows that do not overlap");
}

// torch's current stream of the operands' device, for a call under a DeviceGuard: the
// default stream's handle is null, which is that of whatever device is current.
inline ec_stream_t stream_of(const c10::Device& device) {
  return reinterpret_cast<ec_stream_t>(c10::hip::getCurrentHIPStream(device.index()).stream());
}

// Whether rows of a and rows of b, written and read by one call, share memory.
// Rows of one pitch that lie beside each other (columns of one buffer) do not.
inline bool share(const void* a, const Rows& ra, uint64_t wa, const void* b, const Rows& rb, uint64_t wb) {
  if (!ra.n || !ra.width || !rb.n || !rb.width) return false;
  const uint64_t a0 = reinterpret_cast<uint64_t>(a), b0 = reinterpret_cast<uint64_t>(b);
  const uint64_t a1 = a0 + ((ra.n - 1) * ra.stride + ra.width) * wa;
  const uint64_t b1 = b0 + ((rb.n - 1) * rb.stride + rb.width) * wb;
  if (a1 <= b0 || b1 <= a0) return false;
  const uint64_t pitch = ra.stride * wa;
  if (pitch != rb.stride * wb) return true;
  const uint64_t d = a0 <= b0 ? (b0 - a0) % pitch : (pitch - (a0 - b0) % pitch) % pitch;
  return !(d >= ra.width * wa && d + rb.width * wb <= pitch);
}

// A caller's tensor was written: as after torch's own in-place operations, a backward pass that
// saved it before raises.
inline void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

inline void check_apart(bool together, const char* a, const char* b) {
  if (together) throw py::value_error(std::string(a) + " shares memory with " + b);
}

inline std::vector<int64_t> with_last(at::IntArrayRef lead, int64_t last) {
  std::vector<int64_t> s(lead.begin(), lead.end());
  s.push_back(last);
  return s;
}

}  // namespace
