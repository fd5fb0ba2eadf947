// Torch-tensor binding of the training-step operators (ec_embed ... ec_grad_clip),
// part of the _ec_shards extension: the checks on the tensors, the outputs'
// allocation, torch's current stream and the C call in one crossing from Python.
// Each function returns the status of the C call first, for the caller to turn into
// its error type, then what it allocated.
#include <cstring>
#include <unordered_set>

#include "torch_checks.h"

namespace {

int token_bytes(const Tensor& t) {
  if (t.scalar_type() == at::kLong) return 8;
  if (t.scalar_type() == at::kInt) return 4;
  throw py::value_error(std::string("tokens must be int32 or int64, not ") +
                        c10::toString(t.scalar_type()));
}

py::tuple embed(const Tensor& tokens, const Tensor& table, double scale, int64_t start,
                std::optional<Tensor> out) {
  const int type = type_code(table, "table");
  if (table.dim() != 2)
    throw py::value_error("table must be [vocabulary, hidden], has shape " +
                          shape_text(table.sizes()));
  const Rows rows = rows_of(table, "table", nullptr);
  const c10::Device device = table.device();
  const c10::DeviceGuard guard(device);
  check_dense(tokens, "tokens", &device);
  const int bytes = token_bytes(tokens);
  const auto shape = with_last(tokens.sizes(), (int64_t)rows.width);
  Tensor result;
  if (out.has_value()) {
    result = *out;
    check_dense(result, "out", &device);
    check_type(result, "out", table.scalar_type());
    check_shape(result, "out", shape);
    const Rows o = {1, (uint64_t)result.numel(), (uint64_t)std::max<int64_t>(result.numel(), 1)};
    const uint64_t w = result.element_size();
    check_apart(share(result.data_ptr(), o, w, table.data_ptr(), rows, w), "out", "table");
  } else {
    result = at::empty(shape, table.options().requires_grad(false));
  }
  const uint64_t n = (uint64_t)tokens.numel();
  const ec_stream_t st = stream_of(device);
  const int status =
      rows.width > 0xffffffffull
          ? EC_ERANGE
          : ec_embed(tokens.data_ptr(), bytes, n, table.data_ptr(), type, rows.n,
                     (uint32_t)rows.width, rows.stride, start, (float)scale, result.data_ptr(), st);
  if (out.has_value()) written(result);
  return py::make_tuple(status, result);
}

py::tuple embed_grad(const Tensor& tokens, const Tensor& dout, int64_t vocab, double scale,
                     int64_t start, int64_t grad_type, std::optional<Tensor> out, bool accumulate) {
  const int type = type_code(dout, "dout");
  const Rows rows = rows_of(dout, "dout", nullptr);
  const c10::Device device = dout.device();
  const c10::DeviceGuard guard(device);
  check_dense(tokens, "tokens", &device);
  const int bytes = token_bytes(tokens);
  if (vocab < 0) throw py::value_error("vocab_size must not be negative");
  if (rows.n != (uint64_t)tokens.numel())
    throw py::value_error("dout has " + std::to_string(rows.n) + " rows, got " +
                          std::to_string(tokens.numel()) + " tokens");
  Tensor grad;
  Rows g = {(uint64_t)vocab, rows.width, std::max<uint64_t>(rows.width, 1)};
  if (out.has_value()) {
    grad = *out;
    check_shape(grad, "out", {vocab, (int64_t)rows.width});
    g = rows_of(grad, "out", &device);
    grad_type = type_code(grad, "out");
    check_apart(share(grad.data_ptr(), g, grad.element_size(), dout.data_ptr(), rows,
                      dout.element_size()), "out", "dout");
  } else {
    if (accumulate) throw py::value_error("accumulate needs out");
    grad = at::empty({vocab, (int64_t)rows.width},
                     at::TensorOptions().dtype(torch_type(grad_type)).device(device));
  }
  if (grad_type != EC_F32 && grad_type != type)
    throw py::value_error("the gradient's type must be float32 or dout's");
  const uint32_t hidden = (uint32_t)std::min<uint64_t>(rows.width, 0xffffffffull);
  const uint64_t need = ec_embed_grad_workspace(rows.n, (uint64_t)vocab, hidden);
  const Tensor work =
      at::empty({(int64_t)need}, at::TensorOptions().dtype(at::kByte).device(device));
  const int status = ec_embed_grad(tokens.data_ptr(), bytes, rows.n, dout.data_ptr(), type,
                                   rows.stride, (uint64_t)vocab, hidden, start, (float)scale,
                                   grad.data_ptr(), (int)grad_type, g.stride, accumulate,
                                   work.data_ptr(), need, stream_of(device));
  if (out.has_value()) written(grad);
  return py::make_tuple(status, grad, work);
}

py::tuple token_logprobs(const Tensor& logits, const Tensor& targets, double scale, bool entropy,
                         int64_t top) {
  const int type = type_code(logits, "logits");
  const Rows rows = rows_of(logits, "logits", nullptr);
  const c10::Device device = logits.device();
  const c10::DeviceGuard guard(device);
  check_dense(targets, "targets", &device);
  check_type(targets, "targets", at::kLong);
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  check_shape(targets, "targets", lead);
  if (top < 0 || top > EC_MAX_TOP || (uint64_t)top > rows.width)
    throw py::value_error("top must be between 0 and " +
                          std::to_string(std::min<uint64_t>(EC_MAX_TOP, rows.width)) + ", got " +
                          std::to_string(top));
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(device);
  const Tensor logprobs = at::empty(lead, f32), lse = at::empty(lead, f32);
  std::optional<Tensor> ent, top_logprobs, top_tokens;
  if (entropy) ent = at::empty(lead, f32);
  if (top) {
    const auto shape = with_last(lead, top);
    top_logprobs = at::empty(shape, f32);
    top_tokens = at::empty(shape, f32.dtype(at::kLong));
  }
  const int status = ec_token_logprobs(
      logits.data_ptr(), type, rows.n, rows.width, rows.stride, targets.data_ptr<int64_t>(),
      (float)scale, logprobs.data_ptr<float>(), lse.data_ptr<float>(),
      ent ? ent->data_ptr<float>() : nullptr, (int)top,
      top ? top_logprobs->data_ptr<float>() : nullptr,
      top ? top_tokens->data_ptr<int64_t>() : nullptr, stream_of(device));
  return py::make_tuple(status, logprobs, lse, ent, top_logprobs, top_tokens);
}

py::tuple token_logprobs_grad(const Tensor& logits, const Tensor& targets, const Tensor& lse,
                              const Tensor& dlogprobs, std::optional<Tensor> entropy,
                              std::optional<Tensor> dentropy, double scale,
                              std::optional<Tensor> out) {
  const int type = type_code(logits, "logits");
  const Rows rows = rows_of(logits, "logits", nullptr);
  const c10::Device device = logits.device();
  const c10::DeviceGuard guard(device);
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  check_dense(targets, "targets", &device);
  check_type(targets, "targets", at::kLong);
  check_shape(targets, "targets", lead);
  const auto per_row = [&](const Tensor& t, const char* what) {
    check_dense(t, what, &device);
    check_type(t, what, at::kFloat);
    check_shape(t, what, lead);
    return t.data_ptr<float>();
  };
  if (entropy.has_value() != dentropy.has_value())
    throw py::value_error("entropy and dentropy go together");
  const float* l = per_row(lse, "lse");
  const float* g = per_row(dlogprobs, "dlogprobs");
  const float* h = entropy ? per_row(*entropy, "entropy") : nullptr;
  const float* dh = dentropy ? per_row(*dentropy, "dentropy") : nullptr;
  Tensor result;
  Rows o = {rows.n, rows.width, std::max<uint64_t>(rows.width, 1)};
  if (out.has_value()) {
    result = *out;
    check_type(result, "out", logits.scalar_type());
    check_shape(result, "out", logits.sizes());
    o = rows_of(result, "out", &device);
    const uint64_t w = result.element_size();
    const bool same = result.data_ptr() == logits.data_ptr() && (o.stride == rows.stride || o.n < 2);
    check_apart(!same && share(result.data_ptr(), o, w, logits.data_ptr(), rows, w), "out",
                "logits");
  } else {
    result = at::empty(logits.sizes(), logits.options().requires_grad(false));
  }
  const int status = ec_token_logprobs_grad(
      logits.data_ptr(), type, rows.n, rows.width, rows.stride, targets.data_ptr<int64_t>(), l, g,
      h, dh, (float)scale, result.data_ptr(), o.stride, stream_of(device));
  if (out.has_value()) written(result);
  return py::make_tuple(status, result);
}

// The tensors that a clip of a list writes, of views of one buffer, which share its version,
// only the buffer: a call raises each version once (120 small tensors one by one: 0.7 us).
struct Written {
  std::vector<Tensor> tensors;

  explicit Written(const std::vector<Tensor>& list) {
    std::unordered_set<const void*> seen;
    for (const Tensor& t : list) {
      const Tensor root = t.is_view() ? Tensor(t._base()) : t;
      if (seen.insert(root.unsafeGetTensorImpl()).second) tensors.push_back(root);
    }
  }
};

// The pieces of a list of gradients, as the bytes of an ec_grad_item array (a CPU
// tensor), and the tensors that a clip writes; clips false: a list for norms only, whose tensors
// may overlap.
py::tuple grad_items(const std::vector<Tensor>& grads, const std::optional<std::vector<Tensor>>& out,
                     bool clips) {
  if (out && out->size() != grads.size())
    throw py::value_error("out: expected " + std::to_string(grads.size()) + " tensors, got " +
                          std::to_string(out->size()));
  std::vector<ec_grad_item> items;
  struct Span {
    uint64_t from, to;
    size_t i;
    bool operator<(const Span& o) const { return from < o.from; }
  };
  std::vector<Span> read, written;
  for (size_t i = 0; i < grads.size(); ++i) {
    const std::string name = "grads[" + std::to_string(i) + "]";
    const Tensor& src = grads[i];
    const c10::Device device = grads[0].device();
    check_dense(src, name.c_str(), &device);
    const int st = type_code(src, name.c_str());
    const Tensor& dst = out ? (*out)[i] : src;
    int dt = st;
    if (out) {
      const std::string to = "out[" + std::to_string(i) + "]";
      check_dense(dst, to.c_str(), &device);
      dt = type_code(dst, to.c_str());
      if (dst.numel() != src.numel())
        throw py::value_error(to + " has " + std::to_string(dst.numel()) + " elements, " + name +
                              " " + std::to_string(src.numel()));
    }
    const uint64_t n = (uint64_t)src.numel();
    const uint64_t from = reinterpret_cast<uint64_t>(src.data_ptr());
    const uint64_t to = reinterpret_cast<uint64_t>(dst.data_ptr());
    if (n && clips) {
      read.push_back({from, from + n * src.element_size(), i});
      written.push_back({to, to + n * dst.element_size(), i});
    }
    for (uint64_t at = 0; at < n; at += EC_GRAD_PIECE)
      items.push_back({from + at * (uint64_t)src.element_size(),
                       to + at * (uint64_t)dst.element_size(),
                       (uint32_t)std::min<uint64_t>(EC_GRAD_PIECE, n - at), (uint16_t)st,
                       (uint16_t)dt});
  }
  if (items.size() > 0xffffffffull) throw py::value_error("too many gradients");
  // no element is written twice, and none that another tensor is read from
  const std::string side = out ? "out" : "grads";
  const auto name = [](const std::string& list, size_t i) { return list + "[" + std::to_string(i) + "]"; };
  std::sort(written.begin(), written.end());
  for (size_t j = 1; j < written.size(); ++j)
    check_apart(written[j].from < written[j - 1].to, name(side, written[j].i).c_str(),
                name(side, written[j - 1].i).c_str());
  if (out) {
    std::sort(read.begin(), read.end());
    std::vector<uint64_t> reach(read.size());   // the furthest end of the reads up to here
    for (size_t j = 0; j < read.size(); ++j)
      reach[j] = std::max(read[j].to, j ? reach[j - 1] : 0);
    for (const Span& w : written) {
      size_t j = std::lower_bound(read.begin(), read.end(), Span{w.to, 0, 0}) - read.begin();
      for (; j > 0 && reach[j - 1] > w.from; --j) {
        const Span& r = read[j - 1];
        if (r.to > w.from && !(r.i == w.i && r.from == w.from && r.to == w.to))
          check_apart(true, name("out", w.i).c_str(), name("grads", r.i).c_str());
      }
    }
  }
  const Tensor bytes = at::empty({(int64_t)(items.size() * sizeof(ec_grad_item))}, at::kByte);
  if (!items.empty()) std::memcpy(bytes.data_ptr(), items.data(), items.size() * sizeof(ec_grad_item));
  return py::make_tuple(bytes, Written(!clips ? std::vector<Tensor>() : out ? *out : grads));
}

// ec_grad_norm (max_norm empty) or ec_grad_clip over an uploaded list.
py::tuple grad_call(const Tensor& items, const Written& list, double grad_scale, int64_t norm,
                    std::optional<double> max_norm, std::optional<Tensor> given) {
  const c10::Device device = items.device();
  const c10::DeviceGuard guard(device);
  const auto opts = at::TensorOptions().device(device);
  const Tensor work = at::empty({EC_GRAD_WORK}, opts.dtype(at::kByte));
  const Tensor result = at::empty({}, opts.dtype(at::kFloat));
  const auto* d = reinterpret_cast<const ec_grad_item*>(items.data_ptr());
  const uint32_t n = (uint32_t)(items.numel() / (int64_t)sizeof(ec_grad_item));
  const ec_stream_t st = stream_of(device);
  int status;
  if (max_norm.has_value()) {
    const float* g = nullptr;
    if (given.has_value()) {
      check_device(*given, "norm", &device);
      check_type(*given, "norm", at::kFloat);
      if (given->numel() != 1) throw py::value_error("norm must hold one value");
      g = given->data_ptr<float>();
    }
    status = ec_grad_clip(d, n, (float)grad_scale, (int)norm, (float)*max_norm, g, work.data_ptr(),
                          result.data_ptr<float>(), st);
    for (const Tensor& t : list.tensors) written(t);
  } else {
    status = ec_grad_norm(d, n, (float)grad_scale, (int)norm, work.data_ptr(),
                          result.data_ptr<float>(), st);
  }
  return py::make_tuple(status, result, work);
}

}  // namespace

void bind_step(py::module_& mod) {
  const auto none = py::none();
  mod.def("embed", &embed, py::arg("tokens"), py::arg("table"), py::arg("scale"), py::arg("start"),
          py::arg("out") = none);
  mod.def("embed_grad", &embed_grad, py::arg("tokens"), py::arg("dout"), py::arg("vocab"),
          py::arg("scale"), py::arg("start"), py::arg("grad_type"), py::arg("out") = none,
          py::arg("accumulate") = false);
  mod.def("token_logprobs", &token_logprobs, py::arg("logits"), py::arg("targets"),
          py::arg("scale"), py::arg("entropy"), py::arg("top"));
  mod.def("token_logprobs_grad", &token_logprobs_grad, py::arg("logits"), py::arg("targets"),
          py::arg("lse"), py::arg("dlogprobs"), py::arg("entropy"), py::arg("dentropy"),
          py::arg("scale"), py::arg("out") = none);
  py::class_<Written>(mod, "Written");
  mod.def("grad_items", &grad_items, py::arg("grads"), py::arg("out") = none,
          py::arg("clips") = true);
  mod.def("grad_call", &grad_call, py::arg("items"), py::arg("list"), py::arg("grad_scale"), py::arg("norm"),
          py::arg("max_norm") = none, py::arg("given") = none);
}
