// Torch-tensor binding of the block operators (ec_gated_ff ... ec_orthogonalize), part of the
// _ec_shards extension: as step_torch.cpp, the checks on the tensors, the outputs' and the
// workspace's allocation and the C call, whose status comes first in what is returned.
#include "torch_checks.h"

namespace {

at::TensorOptions like(const Tensor& t) { return t.options().requires_grad(false); }

Tensor bytes_on(const c10::Device& device, uint64_t n) {
  return at::empty({(int64_t)n}, at::TensorOptions().dtype(at::kByte).device(device));
}

// Nobody takes a result for a differentiable one that is not.
bool needs_grad(const Tensor& t) { return t.requires_grad(); }
bool needs_grad(const std::optional<Tensor>& t) { return t && t->requires_grad(); }
template <typename... T>
void no_graph(const char* name, const T&... operands) {
  if (at::GradMode::is_enabled() && (needs_grad(operands) || ...))
    throw py::value_error(std::string(name) +
                          " has no gradient: call it under torch.no_grad(), or with detached tensors");
}

uint32_t narrow(uint64_t v) { return (uint32_t)std::min<uint64_t>(v, 0xffffffffull); }

Rows weight_rows(const Tensor& t, const char* what, const Tensor& x, const Rows& rows) {
  const c10::Device device = x.device();
  check_device(t, what, &device);
  check_type(t, what, x.scalar_type());
  if (t.dim() != 2)
    throw py::value_error(std::string(what) + " must be [inner, width], has shape " +
                          shape_text(t.sizes()));
  if ((uint64_t)t.size(1) != rows.width)
    throw py::value_error(std::string(what) + " has width " + std::to_string(t.size(1)) +
                          ", x " + std::to_string(rows.width));
  return rows_of(t, what, &device);
}

// A caller's result of a shape and type, or a new one; its rows in `rows`.
Tensor result_of(const std::optional<Tensor>& out, const char* what, at::IntArrayRef shape,
                 const at::TensorOptions& options, Rows& rows) {
  if (!out.has_value()) {
    const Tensor t = at::empty(shape, options);
    rows = rows_of(t, what, nullptr);
    return t;
  }
  const c10::Device device = options.device();
  check_device(*out, what, &device);
  check_shape(*out, what, shape);
  check_type(*out, what, c10::typeMetaToScalarType(options.dtype()));
  rows = rows_of(*out, what, &device);
  return *out;
}

struct Named {
  const Tensor& t;
  Rows rows;
  const char* name;
};

void apart(const Named& a, const Named& b) {
  check_apart(share(a.t.data_ptr(), a.rows, a.t.element_size(), b.t.data_ptr(), b.rows,
                    b.t.element_size()),
              a.name, b.name);
}

struct Ff {
  Rows x, gate, up;
  int type;
};

Ff ff_of(const Tensor& x, const Tensor& gate, const Tensor& up) {
  Ff f;
  f.type = type_code(x, "x");
  f.x = rows_of(x, "x", nullptr);
  f.gate = weight_rows(gate, "w_gate", x, f.x);
  f.up = weight_rows(up, "w_up", x, f.x);
  if (f.gate.n != f.up.n)
    throw py::value_error("w_gate has " + std::to_string(f.gate.n) + " rows, w_up " +
                          std::to_string(f.up.n));
  if (!f.x.width || !f.gate.n) throw py::value_error("width and inner must be positive");
  return f;
}

Tensor ff_work(const Ff& f, const Tensor& x, const Tensor& gate, const Tensor& up, bool grad) {
  return bytes_on(x.device(), ec_gated_ff_workspace(x.data_ptr(), f.x.stride, gate.data_ptr(),
                                                    f.gate.stride, up.data_ptr(), f.up.stride,
                                                    f.type, f.x.n, narrow(f.x.width),
                                                    narrow(f.gate.n), grad));
}

py::tuple gated_ff(const Tensor& x, const Tensor& gate, const Tensor& up, int64_t activation,
                   std::optional<Tensor> out) {
  const Ff f = ff_of(x, gate, up);
  const c10::DeviceGuard guard(x.device());
  Rows o;
  const auto shape = with_last(x.sizes().slice(0, x.dim() - 1), (int64_t)f.gate.n);
  const Tensor h = result_of(out, "out", shape, like(x), o);
  if (out.has_value())
    for (const Named& in : {Named{x, f.x, "x"}, {gate, f.gate, "w_gate"}, {up, f.up, "w_up"}})
      apart({h, o, "out"}, in);
  const Tensor work = ff_work(f, x, gate, up, false);
  const int status = ec_gated_ff(x.data_ptr(), f.x.stride, gate.data_ptr(), f.gate.stride,
                                 up.data_ptr(), f.up.stride, f.type, f.x.n, narrow(f.x.width),
                                 narrow(f.gate.n), (int)activation, h.data_ptr(), o.stride,
                                 work.data_ptr(), (uint64_t)work.numel(), stream_of(x.device()));
  if (out.has_value()) written(h);
  return py::make_tuple(status, h, work);
}

py::tuple gated_ff_grad(const Tensor& dh, const Tensor& x, const Tensor& gate, const Tensor& up,
                        int64_t activation, bool with_dx, bool with_dw, int64_t grad_type,
                        std::optional<Tensor> dgate_out, std::optional<Tensor> dup_out,
                        bool accumulate) {
  no_graph("gated_ff_grad", dh, x, gate, up, dgate_out, dup_out);
  const Ff f = ff_of(x, gate, up);
  const c10::Device device = x.device();
  const c10::DeviceGuard guard(device);
  check_type(dh, "dh", x.scalar_type());
  check_shape(dh, "dh", with_last(x.sizes().slice(0, x.dim() - 1), (int64_t)f.gate.n));
  const Rows d = rows_of(dh, "dh", &device);
  if (dgate_out.has_value() != dup_out.has_value())
    throw py::value_error("the weights' gradients are given both or neither");
  if (dgate_out.has_value()) {
    if (!with_dw) throw py::value_error("the weights' gradients are given, but not asked for");
    grad_type = type_code(*dgate_out, "dw_gate");
  } else if (accumulate) {
    throw py::value_error("accumulate needs the gradients to add to");
  }
  if (grad_type != EC_F32 && grad_type != f.type)
    throw py::value_error("the weights' gradients' type must be float32 or x's");
  std::optional<Tensor> dx, dgate, dup;
  Rows rx = {}, rg = {}, ru = {};
  if (with_dx) dx = result_of(std::nullopt, "dx", x.sizes(), like(x), rx);
  if (with_dw) {
    const auto options = like(gate).dtype(torch_type(grad_type));
    dgate = result_of(dgate_out, "dw_gate", gate.sizes(), options, rg);
    dup = result_of(dup_out, "dw_up", up.sizes(), options, ru);
    if (dgate_out.has_value()) {
      const Named g = {*dgate, rg, "dw_gate"}, u = {*dup, ru, "dw_up"};
      for (const Named& in : {Named{x, f.x, "x"}, {gate, f.gate, "w_gate"}, {up, f.up, "w_up"},
                              {dh, d, "dh"}}) {
        apart(g, in);
        apart(u, in);
      }
      apart(g, u);
    }
  }
  const Tensor work = ff_work(f, x, gate, up, true);
  const int status = ec_gated_ff_grad(
      dh.data_ptr(), d.stride, x.data_ptr(), f.x.stride, gate.data_ptr(), f.gate.stride,
      up.data_ptr(), f.up.stride, f.type, f.x.n, narrow(f.x.width), narrow(f.gate.n),
      (int)activation, dx ? dx->data_ptr() : nullptr, rx.stride, dgate ? dgate->data_ptr() : nullptr,
      rg.stride, dup ? dup->data_ptr() : nullptr, ru.stride, (int)grad_type, accumulate,
      work.data_ptr(), (uint64_t)work.numel(), stream_of(device));
  if (dgate_out.has_value()) {
    written(*dgate);
    written(*dup);
  }
  return py::make_tuple(status, dx, dgate, dup, work);
}

// [..., rows, cols]: a batch of matrices, contiguous, or one two-dimensional with strided rows.
struct Matrix {
  uint64_t batch, rows, cols, stride;
};

Matrix matrix_of(const Tensor& t, const char* what, const c10::Device* device) {
  if (t.dim() < 2) throw py::value_error(std::string(what) + " must have at least two dimensions");
  const Rows r = rows_of(t, what, device);
  Matrix m = {1, (uint64_t)t.size(-2), (uint64_t)t.size(-1), r.stride};
  for (int64_t d = 0; d + 2 < t.dim(); ++d) m.batch *= (uint64_t)t.size(d);
  return m;
}

// Whether two tensors are the same elements: a result over its own operand.
bool same_place(const Tensor& a, const Tensor& b) {
  return a.data_ptr() == b.data_ptr() && a.strides() == b.strides() &&
         a.scalar_type() == b.scalar_type();
}

py::tuple orthogonalize(const Tensor& x, int64_t steps, double a, double b, double c, double eps,
                        double scale, std::optional<Tensor> base, double keep, int64_t out_type,
                        std::optional<Tensor> out) {
  no_graph("orthogonalize", x, base, out);
  const int type = type_code(x, "x");
  const Matrix m = matrix_of(x, "x", nullptr);
  const c10::Device device = x.device();
  const c10::DeviceGuard guard(device);
  if (!m.rows || !m.cols) throw py::value_error("a matrix has at least one row and one column");
  if (out.has_value()) out_type = type_code(*out, "out");
  if (out_type < 0) out_type = base ? type_code(*base, "base") : type;
  const auto options = like(x).dtype(torch_type(out_type));
  Rows o, br = {};
  const Tensor result = result_of(out, "out", x.sizes(), options, o);
  const Rows xr = rows_of(x, "x", nullptr);
  if (base) {
    check_type(*base, "base", torch_type(out_type));
    check_shape(*base, "base", x.sizes());
    br = rows_of(*base, "base", &device);
  }
  if (out.has_value()) {
    if (base && !same_place(result, *base)) apart({result, o, "out"}, {*base, br, "base"});
    if (!same_place(result, x)) apart({result, o, "out"}, {x, xr, "x"});
  }
  const Tensor work = bytes_on(device, ec_orthogonalize_workspace(m.batch, m.rows, m.cols));
  const float coefficients[3] = {(float)a, (float)b, (float)c};
  const int status = ec_orthogonalize(
      x.data_ptr(), type, m.batch, m.rows, m.cols, m.stride, m.rows * m.stride, (int)steps,
      coefficients, (float)eps, (float)scale, base ? base->data_ptr() : nullptr, br.stride,
      m.rows * br.stride, (float)keep, result.data_ptr(), (int)out_type, o.stride,
      m.rows * o.stride, work.data_ptr(), (uint64_t)work.numel(), stream_of(device));
  if (out.has_value()) written(result);
  return py::make_tuple(status, result, work);
}

Tensor vector_of(const Tensor& t, const char* what, const Tensor& x, uint64_t width) {
  const c10::Device device = x.device();
  check_dense(t, what, &device);
  check_type(t, what, x.scalar_type());
  check_shape(t, what, {(int64_t)width});
  return t;
}

// Rows of the gate: those of [..., width], which the rows of x share evenly, in order. Of more than two dimensions
// x's leading ones have to be the gate's (and ones after them), so that none is taken for another.
uint64_t gate_rows(const std::optional<Tensor>& gate, const Tensor& x, const Rows& rows) {
  if (!gate) return 1;
  const c10::Device device = x.device();
  check_dense(*gate, "gate", &device);
  check_type(*gate, "gate", x.scalar_type());
  if (gate->dim() < 1 || (uint64_t)gate->size(-1) != rows.width)
    throw py::value_error("gate must be [..., " + std::to_string(rows.width) + "], has shape " +
                          shape_text(gate->sizes()));
  uint64_t n = 1;
  for (int64_t d = 0; d + 1 < gate->dim(); ++d) n *= (uint64_t)gate->size(d);
  bool ones = false, fits = x.dim() <= 2 || gate->dim() <= x.dim();
  for (int64_t d = 0; x.dim() > 2 && fits && d + 1 < gate->dim(); ++d) {
    ones = ones || gate->size(d) != x.size(d);
    fits = !ones || gate->size(d) == 1;
  }
  if (!fits || (rows.n && (!n || rows.n % n)))
    throw py::value_error("gate of shape " + shape_text(gate->sizes()) + ": the rows of " +
                          shape_text(x.sizes()) + " do not share its rows evenly, in order");
  return std::max<uint64_t>(n, 1);
}

Rows rows_like(const Tensor& t, const char* what, const Tensor& x) {
  const c10::Device device = x.device();
  check_type(t, what, x.scalar_type());
  check_shape(t, what, x.sizes());
  return rows_of(t, what, &device);
}

void* place(const std::optional<Tensor>& t) { return t ? t->data_ptr() : nullptr; }
float* floats(const std::optional<Tensor>& t) { return t ? t->data_ptr<float>() : nullptr; }

py::tuple residual_norm(const Tensor& residual, std::optional<Tensor> branch,
                        std::optional<Tensor> gate, double scale,
                        std::optional<Tensor> branch_weight, std::optional<Tensor> weight, double eps,
                        std::optional<Tensor> out) {
  const int type = type_code(residual, "residual");
  const Rows rows = rows_of(residual, "residual", nullptr);
  const c10::Device device = residual.device();
  const c10::DeviceGuard guard(device);
  if (!rows.width) throw py::value_error("rows must not be empty");
  if (!branch && (gate || branch_weight || out))
    throw py::value_error("gate, branch_weight and out go with a branch");
  if (!branch && !weight) throw py::value_error("neither a branch to add nor a weight to norm with");
  const Rows b = branch ? rows_like(*branch, "branch", residual) : Rows{0, 0, 0};
  const uint64_t gates = gate_rows(gate, residual, rows);
  if (branch_weight) vector_of(*branch_weight, "branch_weight", residual, rows.width);
  if (weight) vector_of(*weight, "weight", residual, rows.width);
  const auto lead = residual.sizes().slice(0, residual.dim() - 1);
  std::optional<Tensor> sum, normed, rstd, branch_rstd;
  Rows s = {};
  if (branch) {
    sum = result_of(out, "out", residual.sizes(), like(residual), s);
    if (out.has_value()) {
      const Named o = {*sum, s, "out"};
      if (!same_place(*sum, residual)) apart(o, {residual, rows, "residual"});
      if (!same_place(*sum, *branch)) apart(o, {*branch, b, "branch"});
      const Rows one = {1, rows.width, rows.width};
      if (branch_weight) apart(o, {*branch_weight, one, "branch_weight"});
      if (weight) apart(o, {*weight, one, "weight"});
      if (gate) apart(o, {*gate, {gates, rows.width, rows.width}, "gate"});
    }
  }
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(device);
  if (weight) {
    normed = at::empty(residual.sizes(), like(residual));
    rstd = at::empty(lead, f32);
  }
  if (branch_weight) branch_rstd = at::empty(lead, f32);
  // (tensors without rows have no addresses to tell given ones by)
  const int status = !rows.n ? EC_OK : ec_residual_norm(
      residual.data_ptr(), rows.stride, place(branch), b.stride, type, rows.n, narrow(rows.width),
      place(gate), gates, (float)scale, place(branch_weight), place(weight), (float)eps, place(sum),
      s.stride, place(normed), floats(rstd), floats(branch_rstd), stream_of(device));
  if (out.has_value()) written(*sum);
  return py::make_tuple(status, sum, normed, rstd, branch_rstd);
}

py::tuple residual_norm_grad(std::optional<Tensor> dsum, std::optional<Tensor> dnormed,
                             const Tensor& sum, std::optional<Tensor> branch,
                             std::optional<Tensor> rstd, std::optional<Tensor> branch_rstd,
                             std::optional<Tensor> gate, double scale,
                             std::optional<Tensor> branch_weight, std::optional<Tensor> weight) {
  no_graph("residual_norm_grad", dsum, dnormed, sum, branch, rstd, branch_rstd, gate, branch_weight, weight);
  const int type = type_code(sum, "sum");
  const Rows rows = rows_of(sum, "sum", nullptr);
  const c10::Device device = sum.device();
  const c10::DeviceGuard guard(device);
  if (!rows.width) throw py::value_error("rows must not be empty");
  if (!dsum && !dnormed) throw py::value_error("neither of the two gradients is given");
  if (dnormed && (!weight || !rstd)) throw py::value_error("dnormed needs weight and rstd");
  if (!branch && (gate || branch_weight))
    throw py::value_error("gate and branch_weight go with a branch");
  if (branch_weight && !branch_rstd) throw py::value_error("branch_weight needs branch_rstd");
  if (!dnormed) weight.reset();   // nothing of the second norm is read, and its weight has no gradient
  const Rows ds = dsum ? rows_like(*dsum, "dresidual", sum) : Rows{0, 0, 0};
  const Rows dn = dnormed ? rows_like(*dnormed, "dnormed", sum) : Rows{0, 0, 0};
  const Rows b = branch ? rows_like(*branch, "branch", sum) : Rows{0, 0, 0};
  const uint64_t gates = gate_rows(gate, sum, rows);
  const auto lead = sum.sizes().slice(0, sum.dim() - 1);
  const auto per_row = [&](const Tensor& t, const char* what) {
    check_dense(t, what, &device);
    check_type(t, what, at::kFloat);
    check_shape(t, what, lead);
  };
  if (branch_weight) {
    vector_of(*branch_weight, "branch_weight", sum, rows.width);
    per_row(*branch_rstd, "branch_rstd");
  }
  if (weight) {
    vector_of(*weight, "weight", sum, rows.width);
    per_row(*rstd, "rstd");
  }
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(device);
  const Tensor dresidual = at::empty(sum.sizes(), like(sum));
  std::optional<Tensor> dbranch, dgate, dbranch_weight, dweight;
  if (branch) dbranch = at::empty(sum.sizes(), like(sum));
  if (gate) dgate = at::empty(gate->sizes(), f32);
  if (branch_weight) dbranch_weight = at::empty({(int64_t)rows.width}, f32);
  if (weight) dweight = at::empty({(int64_t)rows.width}, f32);
  const Tensor work =
      bytes_on(device, ec_residual_norm_grad_workspace(rows.n, narrow(rows.width), gates));
  if (!rows.n)
    for (std::optional<Tensor>* t : {&dgate, &dbranch_weight, &dweight})
      if (*t) (*t)->zero_();
  const int status = !rows.n ? EC_OK : ec_residual_norm_grad(
      place(dsum), ds.stride, weight ? place(dnormed) : nullptr, dn.stride,
      weight ? sum.data_ptr() : nullptr, rows.stride, place(branch), b.stride, type, rows.n,
      narrow(rows.width), weight ? floats(rstd) : nullptr,
      branch_weight ? floats(branch_rstd) : nullptr, place(gate), gates, (float)scale,
      place(branch_weight), place(weight), dresidual.data_ptr(), place(dbranch), floats(dgate),
      floats(dbranch_weight), floats(dweight), work.data_ptr(), (uint64_t)work.numel(),
      stream_of(device));
  return py::make_tuple(status, dresidual, dbranch, dgate, dbranch_weight, dweight, work);
}

}  // namespace

void bind_block(py::module_& mod) {
  const auto none = py::none();
  mod.def("gated_ff", &gated_ff, py::arg("x"), py::arg("w_gate"), py::arg("w_up"),
          py::arg("activation"), py::arg("out") = none);
  mod.def("gated_ff_grad", &gated_ff_grad, py::arg("dh"), py::arg("x"), py::arg("w_gate"),
          py::arg("w_up"), py::arg("activation"), py::arg("with_dx"), py::arg("with_dw"),
          py::arg("grad_type"), py::arg("dw_gate") = none, py::arg("dw_up") = none,
          py::arg("accumulate") = false);
  mod.def("orthogonalize", &orthogonalize, py::arg("x"), py::arg("steps"), py::arg("a"),
          py::arg("b"), py::arg("c"), py::arg("eps"), py::arg("scale"), py::arg("base") = none,
          py::arg("keep") = 1.0, py::arg("out_type") = -1, py::arg("out") = none);
  mod.def("residual_norm", &residual_norm, py::arg("residual"), py::arg("branch") = none,
          py::arg("gate") = none, py::arg("scale") = 1.0, py::arg("branch_weight") = none,
          py::arg("weight") = none, py::arg("eps") = 1e-6, py::arg("out") = none);
  mod.def("residual_norm_grad", &residual_norm_grad, py::arg("dresidual") = none,
          py::arg("dnormed") = none, py::arg("sum"), py::arg("branch") = none,
          py::arg("rstd") = none, py::arg("branch_rstd") = none, py::arg("gate") = none,
          py::arg("scale") = 1.0, py::arg("branch_weight") = none, py::arg("weight") = none);
}
