// Native host side of medvision_amd.ops: argument checks, allocation, workspace and autograd nodes around the C
// entry points of libmedvision_hip.
//
// Small calls of these operators last 5 - 20 us on the GPU, about what the same steps cost in Python (12 us for a
// resampling call, 70 - 150 us for a training step whose backward node has to take the interpreter's lock in the
// autograd thread).  Here a forward call costs ~4 us and backward nodes never enter the interpreter.
// Errors keep the types and texts of the Python layer.
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/numpy.h>

#include <optional>

#include "../../include/medvision_hip.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

[[noreturn]] void raise(PyObject *type, const std::string &text) {
  py::gil_scoped_acquire gil;
  PyErr_SetString(type, text.c_str());
  throw py::error_already_set();
}

// None of the operators has a forward-mode derivative: a dual tensor is refused instead of losing its tangent (it need
// not require a gradient, so the short ways around the autograd nodes would take it).
void no_forward_mode(const Tensor &t) {
  if (t.defined() && t._fw_grad(/*level=*/0).defined())
    raise(PyExc_NotImplementedError, "forward-mode AD is not implemented for this operator");
}

// (std::runtime_error becomes RuntimeError without the C++ backtrace that TORCH_CHECK appends)
#define MVB_CHECK(cond, ...) \
  do {                       \
    if (!(cond)) throw std::runtime_error(c10::str(__VA_ARGS__)); \
  } while (0)

void check(int status) {
  if (status != MV_OK) throw std::runtime_error(mv_last_error());
}

std::string dtype_name(const Tensor &t) {
  py::gil_scoped_acquire gil;
  return py::str(py::cast(t).attr("dtype")).cast<std::string>();
}

int dtype_code(const Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return MV_F32;
    case at::kHalf: return MV_F16;
    case at::kBFloat16: return MV_BF16;
    case at::kDouble: return MV_F64;
    default: throw std::runtime_error("unsupported dtype " + dtype_name(t));
  }
}

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void same_device(const Tensor &ref, const Tensor &t, const char *name) {
  MVB_CHECK(!t.defined() || t.device() == ref.device(), name, " is on ", t.device().str(), ", expected ", ref.device().str(),
            " like the input tensor");
}

Tensor bytes_on(const Tensor &like, size_t n) {
  return n ? at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte)) : Tensor();
}

// sampling_ratio, order, im2col_step: any number, as int() takes it
int64_t whole(double v) {
  MVB_CHECK(v > -9e18 && v < 9e18, "expected a whole number, got ", v);
  return static_cast<int64_t>(v);
}

void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

using Dims = std::array<int, 3>;

// "output_size": one integer or a tuple of ndim integers
Dims parse_size(const py::handle &size, int ndim) {
  Dims out{1, 1, 1};
  if (PyLong_Check(size.ptr())) {
    for (int a = 3 - ndim; a < 3; ++a) out[a] = static_cast<int>(PyLong_AsLong(size.ptr()));
  } else if (PyTuple_Check(size.ptr())) {
    if (PyTuple_GET_SIZE(size.ptr()) != ndim) raise(PyExc_AssertionError, "");
    for (int a = 0; a < ndim; ++a) {
      PyObject *v = PyTuple_GET_ITEM(size.ptr(), a);
      if (!PyLong_Check(v)) raise(PyExc_AssertionError, "");
      out[3 - ndim + a] = static_cast<int>(PyLong_AsLong(v));
    }
  } else {
    raise(PyExc_TypeError, "\"output_size\" must be an integer or tuple of integers");
  }
  if (PyErr_Occurred()) throw py::error_already_set();
  return out;
}

// stride / padding / dilation of a layer: one integer for all axes or one per axis
Dims per_axis(const py::handle &value, int ndim, int absent) {
  Dims out{absent, absent, absent};
  if (PySequence_Check(value.ptr())) {
    const py::sequence seq = py::reinterpret_borrow<py::sequence>(value);
    if (static_cast<int>(seq.size()) != ndim) raise(PyExc_TypeError, "one value per axis is needed");
    for (int a = 0; a < ndim; ++a) out[3 - ndim + a] = seq[a].cast<int>();
  } else {
    const int v = value.cast<int>();
    for (int a = 3 - ndim; a < 3; ++a) out[a] = v;
  }
  return out;
}

// ---- RoIAlign, RoIAlignRotated and the affine engines -----------------------------------------------------------
enum RoiKind { kPlain, kRotated, kAffine };

struct RoiCall {
  int kind, ndim, ratio, order;
  bool aligned;
  float scale;
  Dims out;
  const char *what() const { return kind == kPlain ? "RoIAlign" : kind == kRotated ? "RoIAlignRotated" : "affine"; }
  int columns() const { return kind == kPlain ? 1 + 2 * ndim : ndim == 2 ? 6 : 10; }
};

Tensor prepared_rois(const RoiCall &c, const Tensor &rois, const Tensor &features) {
  MVB_CHECK(rois.dim() == 2 && rois.size(1) == c.columns(), "wrong roi size! size_rois should be ", c.columns());
  const auto want = features.scalar_type() == at::kDouble ? at::kDouble : at::kFloat;
  if (rois.scalar_type() == want && rois.device() == features.device() && rois.is_contiguous()) return rois;
  return rois.to(features.options().dtype(want)).contiguous();
}

// [N, C, D, H, W] of a feature tensor or gradient (images: D = 1)
std::array<int, 5> five_dims(const at::IntArrayRef &s, int ndim) {
  if (ndim == 2) return {int(s[0]), int(s[1]), 1, int(s[2]), int(s[3])};
  return {int(s[0]), int(s[1]), int(s[2]), int(s[3]), int(s[4])};
}

Tensor roi_forward(const RoiCall &c, const Tensor &input, const Tensor &rois_in, const Tensor &prepared) {
  MVB_CHECK(input.is_cuda(), c.what(), " is not implemented on CPU");
  const Tensor features = input.contiguous();
  const Tensor rois = prepared_rois(c, rois_in, features);
  MVB_CHECK(features.dim() == c.ndim + 2, "expected a ", c.ndim + 2, "-d feature tensor, got ", features.dim(), "-d");
  const bool labels = features.scalar_type() == at::kInt && c.kind == kAffine;
  const int code = labels ? static_cast<int>(MV_I32) : dtype_code(features);
  const auto d = five_dims(features.sizes(), c.ndim);
  const int n = static_cast<int>(rois.size(0));
  const c10::DeviceGuard guard(features.device());
  const Tensor output = c.ndim == 2 ? at::empty({n, d[1], c.out[1], c.out[2]}, features.options())
                                    : at::empty({n, d[1], c.out[0], c.out[1], c.out[2]}, features.options());
  void *const stream = stream_of(features);
  if (prepared.defined()) {
    same_device(features, prepared, "prepared");
    MVB_CHECK(static_cast<size_t>(prepared.numel()) ==
                  mv_roi_align_prepared_bytes(code, c.ndim, d[0], d[1], d[2], d[3], d[4]),
              "prepared copy does not belong to features of this shape");
    // four bytes per roi for the order the rois are worked in; what heads the copy does not serve need
    const size_t bytes = std::max<size_t>(4 * static_cast<size_t>(n),
        mv_roi_align_forward_workspace_bytes(code, c.ndim, d[1], n, c.out[0], c.out[1], c.out[2], c.ratio));
    const Tensor ws = bytes_on(features, bytes);
    check(mv_roi_align_forward_prepared(ptr(features), ptr(prepared), ptr(rois), ptr(output), code, c.ndim, d[0], d[1],
                                        d[2], d[3], d[4], n, c.out[0], c.out[1], c.out[2], c.scale, c.ratio, c.order,
                                        ptr(ws), bytes, stream));
    return output;
  }
  const size_t bytes = mv_roi_align_forward_workspace_bytes_for_input(code, c.ndim, d[0], d[1], d[2], d[3], d[4], n,
                                                                      c.out[0], c.out[1], c.out[2], c.ratio);
  const Tensor ws = bytes_on(features, bytes);
  int status;
  if (c.kind == kPlain && c.ndim == 2)
    status = mv_roi_align_2d_forward(ptr(features), ptr(rois), ptr(output), code, d[0], d[1], d[3], d[4], n, c.out[1],
                                     c.out[2], c.scale, c.ratio, c.order, ptr(ws), bytes, stream);
  else if (c.kind == kPlain)
    status = mv_roi_align_3d_forward(ptr(features), ptr(rois), ptr(output), code, d[0], d[1], d[2], d[3], d[4], n,
                                     c.out[0], c.out[1], c.out[2], c.scale, c.ratio, c.order, ptr(ws), bytes, stream);
  else if (c.ndim == 2)
    status = (c.kind == kRotated ? mv_roi_align_rotated_2d_forward : mv_affine_2d)(
        ptr(features), ptr(rois), ptr(output), code, d[0], d[1], d[3], d[4], n, c.out[1], c.out[2], c.scale, c.ratio,
        c.aligned, c.order, ptr(ws), bytes, stream);
  else
    status = (c.kind == kRotated ? mv_roi_align_rotated_3d_forward : mv_affine_3d)(
        ptr(features), ptr(rois), ptr(output), code, d[0], d[1], d[2], d[3], d[4], n, c.out[0], c.out[1], c.out[2],
        c.scale, c.ratio, c.aligned, c.order, ptr(ws), bytes, stream);
  check(status);
  return output;
}

Tensor roi_backward(const RoiCall &c, const Tensor &grad_output, const Tensor &rois_in, at::IntArrayRef feature_size) {
  MVB_CHECK(grad_output.is_cuda(), c.what(), " is not implemented on CPU");
  const c10::DeviceGuard guard(grad_output.device());
  const Tensor g = grad_output.contiguous();
  const Tensor rois = prepared_rois(c, rois_in, g);
  const int code = dtype_code(g);
  const auto d = five_dims(feature_size, c.ndim);
  const int n = static_cast<int>(rois.size(0));
  const Tensor grad_input = at::empty(feature_size, g.options());
  const size_t bytes = mv_roi_align_backward_write_workspace_bytes(code, c.ndim, c.kind == kRotated, d[0], d[1], d[2], d[3], d[4], n,
                                                                   c.out[0], c.out[1], c.out[2], c.ratio, c.order);
  const Tensor ws = bytes_on(g, bytes);
  check(mv_roi_align_backward_replace(ptr(g), ptr(rois), ptr(grad_input), code, c.ndim, c.kind == kRotated, d[0], d[1], d[2],
                                      d[3], d[4], n, c.out[0], c.out[1], c.out[2], c.scale, c.ratio, c.aligned, c.order,
                                      ptr(ws), bytes, stream_of(g)));
  return grad_input;
}

struct RoiAlignFunction : torch::autograd::Function<RoiAlignFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &features, const Tensor &rois,
                        const std::optional<Tensor> &prepared, const RoiCall &call) {
    ctx->save_for_backward({rois});
    ctx->saved_data["size"] = features.sizes();
    ctx->saved_data["call"] = std::vector<int64_t>{call.kind, call.ndim, call.ratio, call.order, call.aligned};
    ctx->saved_data["scale"] = static_cast<double>(call.scale);
    return roi_forward(call, features, rois, prepared.value_or(Tensor()));
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    if (!ctx->needs_input_grad(0) || !grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const at::NoGradGuard no_grad;
    const auto call = ctx->saved_data["call"].toIntVector();
    RoiCall c{int(call[0]), int(call[1]), int(call[2]), int(call[3]), call[4] != 0,
              static_cast<float>(ctx->saved_data["scale"].toDouble()), {1, 1, 1}};
    for (int a = 0; a < c.ndim; ++a) c.out[3 - c.ndim + a] = static_cast<int>(grads[0].size(2 + a));
    return {roi_backward(c, grads[0], ctx->get_saved_variables()[0], ctx->saved_data["size"].toIntVector()), Tensor(),
            Tensor(), Tensor()};
  }
};

// features that need no gradient (or a call under no_grad) get no node
Tensor roi_align(int ndim, bool rotated, const Tensor &features, const Tensor &rois, const py::object &output_size,
                 double spatial_scale, double sampling_ratio, bool aligned, double order, const std::optional<Tensor> &prepared) {
  const RoiCall c{rotated ? kRotated : kPlain, ndim, static_cast<int>(whole(sampling_ratio)), static_cast<int>(whole(order)), aligned, static_cast<float>(spatial_scale),
                  parse_size(output_size, ndim)};
  no_forward_mode(features);
  no_forward_mode(rois);
  const py::gil_scoped_release no_gil;
  if (!(at::GradMode::is_enabled() && (features.requires_grad() || rois.requires_grad()))) {
    const at::NoGradGuard no_grad;
    return roi_forward(c, features, rois, prepared.value_or(Tensor()));
  }
  return RoiAlignFunction::apply(features, rois, prepared, c);
}

Tensor affine(int ndim, const Tensor &features, const Tensor &rois, const py::object &out_size, double spatial_scale,
              double sampling_ratio, bool aligned, double given_order) {
  const int order = static_cast<int>(whole(given_order));
  RoiCall c{kAffine, ndim, static_cast<int>(whole(sampling_ratio)), order, aligned, static_cast<float>(spatial_scale), parse_size(out_size, ndim)};
  const auto t = features.scalar_type();
  // (int32: label maps at order 0, sampled as they are -- the reference resamples a float copy of them)
  if (!(t == at::kFloat || t == at::kHalf || t == at::kBFloat16 || t == at::kDouble || (t == at::kInt && order == 0)))
    raise(PyExc_AssertionError, "input must be a floating tensor but got " + dtype_name(features));
  if ((order != 0 && order != 1 && order != 3) || order != given_order)
    raise(PyExc_AssertionError, c10::str("order ", given_order, " is not supported!"));
  if (order == 0) c.ratio = 1;   // never average nearest-neighbour samples (reference cuda_fun_tools.py:72-74)
  const py::gil_scoped_release no_gil;
  const at::NoGradGuard no_grad;
  return roi_forward(c, features, rois, Tensor());
}

// The same for a sample [C, *spatial] as for a batch of one
Tensor affine_sample(int ndim, const Tensor &sample, const Tensor &rois, const py::object &out_size, double sampling_ratio, double order) {
  return affine(ndim, sample.unsqueeze(0), rois, out_size, 1.0, sampling_ratio, true, order).squeeze(0);
}

// ---- deformable convolution -----------------------------------------------------------------------------------------
struct DcnCall {
  int nd, groups, dg;
  Dims stride, pad, dil;
};

struct DcnShape {
  int nd;
  mv_dcn3d_shape v;
  mv_dcn2d_shape i;
  std::vector<int64_t> out;   // [B, Cout, *spatial]
  int taps;
};

DcnShape dcn_shape(const DcnCall &c, const Tensor &input, const Tensor &weight) {
  MVB_CHECK(input.is_contiguous(), "input tensor has to be contiguous");
  MVB_CHECK(weight.is_contiguous(), "weight tensor has to be contiguous");
  MVB_CHECK(input.dim() == c.nd + 2 && weight.dim() == c.nd + 2, "expected ", c.nd + 2, "-d input and weight tensors");
  const auto x = five_dims(input.sizes(), c.nd), w = five_dims(weight.sizes(), c.nd);
  const int C = x[1], Cout = w[0], ck = w[1];
  MVB_CHECK(c.groups > 0 && c.dg > 0, "groups must be positive");   // (divided by below)
  MVB_CHECK(C == ck * c.groups, "Input shape and kernel channels wont match: (", C, " vs ", ck * c.groups, ").");
  MVB_CHECK(C % c.groups == 0 && Cout % c.groups == 0, "channels(", C, ") and channels_out(", Cout, ") must divide group(",
            c.groups, ")");
  MVB_CHECK(C % c.dg == 0, "channels(", C, ") must divide deformable_group(", c.dg, ")");
  DcnShape s{};
  s.nd = c.nd;
  s.v = {x[0], C, x[2], x[3], x[4], Cout, w[2], w[3], w[4], c.stride[0], c.stride[1], c.stride[2],
         c.pad[0], c.pad[1], c.pad[2], c.dil[0], c.dil[1], c.dil[2], c.groups, c.dg};
  s.i = {x[0], C, x[3], x[4], Cout, w[3], w[4], c.stride[1], c.stride[2], c.pad[1], c.pad[2], c.dil[1], c.dil[2],
         c.groups, c.dg};
  s.taps = w[2] * w[3] * w[4];
  int d = 1, h = 1, wd = 1;
  check(c.nd == 3 ? mv_dcn3d_output_dims(&s.v, &d, &h, &wd) : mv_dcn2d_output_dims(&s.i, &h, &wd));
  s.out = {x[0], Cout};
  if (c.nd == 3) s.out.push_back(d);
  s.out.push_back(h);
  s.out.push_back(wd);
  return s;
}

std::string shape_text(at::IntArrayRef s) {
  std::string t = "(";
  for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
  return t + ")";
}

void check_aux(const DcnShape &s, const Tensor &t, int channels, const char *name) {
  std::vector<int64_t> want = s.out;
  want[1] = channels;
  MVB_CHECK(t.sizes() == at::IntArrayRef(want), name, " has shape ", shape_text(t.sizes()), ", expected ", shape_text(want));
}

Tensor dcn_forward(const DcnCall &c, const Tensor &input, const Tensor &offset_in, const Tensor &mask_in,
                   const Tensor &weight, const Tensor &bias_in) {
  const DcnShape s = dcn_shape(c, input, weight);
  same_device(input, offset_in, "offset");
  same_device(input, mask_in, "mask");
  same_device(input, weight, "weight");
  same_device(input, bias_in, "bias");
  const Tensor bias = bias_in.defined() ? bias_in.contiguous() : bias_in;
  const Tensor offset = offset_in.to(input.scalar_type()).contiguous();
  const Tensor mask = mask_in.defined() ? mask_in.to(input.scalar_type()).contiguous() : mask_in;
  check_aux(s, offset, c.dg * c.nd * s.taps, "offset");
  if (mask.defined()) check_aux(s, mask, c.dg * s.taps, "mask");
  MVB_CHECK(weight.scalar_type() == input.scalar_type() && (!bias.defined() || bias.scalar_type() == input.scalar_type()),
            "input, weight and bias must share one dtype");
  const int code = dtype_code(input);
  const c10::DeviceGuard guard(input.device());
  const Tensor output = at::empty(s.out, input.options());
  const Tensor ws = bytes_on(input, c.nd == 3 ? mv_dcn3d_forward_workspace_bytes(&s.v, code)
                                              : mv_dcn2d_forward_workspace_bytes(&s.i, code));
  void *const stream = stream_of(input);
  check(c.nd == 3 ? mv_dcn3d_forward(ptr(input), ptr(offset), ptr(mask), ptr(weight), ptr(bias), ptr(output), &s.v, code,
                                     ptr(ws), stream)
                  : mv_dcn2d_forward(ptr(input), ptr(offset), ptr(mask), ptr(weight), ptr(bias), ptr(output), &s.i, code,
                                     ptr(ws), stream));
  return output;
}

struct DcnGrads {
  Tensor input, offset, mask, weight, bias;
};

DcnGrads dcn_backward(const DcnCall &c, const Tensor &input, const Tensor &offset_in, const Tensor &mask_in,
                      const Tensor &weight, const Tensor &bias, const Tensor &grad_in) {
  const c10::DeviceGuard guard(input.device());
  const DcnShape s = dcn_shape(c, input, weight);
  same_device(input, grad_in, "grad_output");
  const Tensor offset = offset_in.to(input.scalar_type()).contiguous();
  const Tensor mask = mask_in.defined() ? mask_in.to(input.scalar_type()).contiguous() : mask_in;
  const Tensor grad = grad_in.to(input.scalar_type()).contiguous();
  MVB_CHECK(grad.sizes() == at::IntArrayRef(s.out), "Input shape and grad_out shape wont match: (", shape_text(s.out), " vs ",
            shape_text(grad.sizes()), ").");
  DcnGrads g;
  g.input = at::empty_like(input);
  g.weight = at::empty_like(weight);
  if (bias.defined()) g.bias = at::empty_like(bias, at::MemoryFormat::Contiguous);
  g.offset = at::empty_like(offset);
  if (mask.defined()) g.mask = at::empty_like(mask);
  const int code = dtype_code(input);
  const Tensor ws = bytes_on(input, c.nd == 3 ? mv_dcn3d_backward_workspace_bytes(&s.v, code)
                                              : mv_dcn2d_backward_workspace_bytes(&s.i, code));
  void *const stream = stream_of(input);
  check(c.nd == 3 ? mv_dcn3d_backward_write(ptr(input), ptr(offset), ptr(mask), ptr(weight), ptr(grad), ptr(g.input), ptr(g.offset),
                                      ptr(g.mask), ptr(g.weight), ptr(g.bias), &s.v, code, ptr(ws), stream)
                  : mv_dcn2d_backward_write(ptr(input), ptr(offset), ptr(mask), ptr(weight), ptr(grad), ptr(g.input), ptr(g.offset),
                                      ptr(g.mask), ptr(g.weight), ptr(g.bias), &s.i, code, ptr(ws), stream));
  return g;
}

struct DeformConvFunction : torch::autograd::Function<DeformConvFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &input_in, const Tensor &offset,
                        const std::optional<Tensor> &mask_in, const Tensor &weight_in,
                        const std::optional<Tensor> &bias_in, const DcnCall &c) {
    Tensor input = input_in, weight = weight_in, bias = bias_in.value_or(Tensor());
    const Tensor mask = mask_in.value_or(Tensor());
    if (offset.scalar_type() == at::kHalf || offset.scalar_type() == at::kBFloat16) {   // autocast: follow the offset branch
      input = input.to(offset.scalar_type());
      weight = weight.to(offset.scalar_type());
      if (bias.defined()) bias = bias.to(offset.scalar_type());
    }
    const Tensor output = dcn_forward(c, input, offset, mask, weight, bias);
    ctx->save_for_backward({input, offset, mask, weight, bias});
    ctx->saved_data["call"] = std::vector<int64_t>{c.nd, c.groups, c.dg, c.stride[0], c.stride[1], c.stride[2], c.pad[0],
                                                   c.pad[1], c.pad[2], c.dil[0], c.dil[1], c.dil[2]};
    return output;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    if (!grads[0].defined()) return variable_list(6);
    variable_list out;
    {
      const at::NoGradGuard no_grad;
      MVB_CHECK(grads[0].is_cuda(), "Not implemented on the CPU");
      const auto v = ctx->saved_data["call"].toIntVector();
      const DcnCall c{int(v[0]), int(v[1]), int(v[2]), {int(v[3]), int(v[4]), int(v[5])}, {int(v[6]), int(v[7]), int(v[8])},
                      {int(v[9]), int(v[10]), int(v[11])}};
      const auto saved = ctx->get_saved_variables();
      const DcnGrads g = dcn_backward(c, saved[0], saved[1], saved[2], saved[3], saved[4], grads[0]);
      out = {g.input, g.offset, g.mask, g.weight, g.bias, Tensor()};
    }
    // the gradients cannot be differentiated again: say so when someone tries
    if (at::GradMode::is_enabled() && grads[0].requires_grad()) {
      for (Tensor &t : out) {
        if (!t.defined()) continue;
        auto once = std::make_shared<torch::autograd::DelayedError>(
            "trying to differentiate twice a function that was marked with @once_differentiable", 1);
        t.set_requires_grad(true);
        t = (*once)(variable_list{t})[0];
      }
    }
    return out;
  }
};

void im2col_step_check(int64_t batch, int64_t im2col_step) {
  const int64_t step = std::min(batch, im2col_step);
  MVB_CHECK(step != 0 && batch % step == 0, "batch(", batch, ") must divide im2col_step(", step, ")");
}

// DCNv2: scalar stride / padding / dilation, optional bias
Tensor modulated_deform_conv(int nd, const Tensor &input, const Tensor &offset, const Tensor &mask, const Tensor &weight,
                             const std::optional<Tensor> &bias, int stride, int padding, int dilation, int groups, int dg) {
  if (!input.is_cuda()) raise(PyExc_NotImplementedError, "");
  const int s0 = nd == 3 ? stride : 1, p0 = nd == 3 ? padding : 0, d0 = nd == 3 ? dilation : 1;
  const DcnCall c{nd, groups, dg, {s0, stride, stride}, {p0, padding, padding}, {d0, dilation, dilation}};
  for (const Tensor &t : {input, offset, mask, weight, bias.value_or(Tensor())}) no_forward_mode(t);
  const py::gil_scoped_release no_gil;
  return DeformConvFunction::apply(input, offset, mask, weight, bias, c);
}

// DCNv1: the bias is always added
Tensor deform_conv(int nd, const Tensor &input, const Tensor &offset, const Tensor &weight, const Tensor &bias,
                   const py::object &stride, const py::object &padding, const py::object &dilation, int groups, int dg,
                   double im2col_step) {
  const DcnCall c{nd, groups, dg, per_axis(stride, nd, 1), per_axis(padding, nd, 0), per_axis(dilation, nd, 1)};
  for (const Tensor &t : {input, offset, weight, bias}) no_forward_mode(t);
  const py::gil_scoped_release no_gil;
  MVB_CHECK(input.is_cuda(), "Not implemented on the CPU");
  im2col_step_check(input.size(0), whole(im2col_step));
  return DeformConvFunction::apply(input, offset, std::nullopt, weight, bias, c);
}

// ---- displacement-field warp ------------------------------------------------------------------------------------------
Tensor deform_warp(const Tensor &img_in, const Tensor &offset_in, double given_order) {
  const int order = given_order == 0.0 || given_order == 1.0 || given_order == 3.0 ? static_cast<int>(given_order) : -1;
  const py::gil_scoped_release no_gil;
  const at::NoGradGuard no_grad;
  MVB_CHECK(img_in.is_cuda(), "Not implemented on the CPU");
  const int ndim = static_cast<int>(img_in.dim()) - 2;
  MVB_CHECK(ndim == 2 || ndim == 3, "expected a 4-d or 5-d image, got ", img_in.dim(), "-d");
  const c10::DeviceGuard guard(img_in.device());
  const Tensor img = img_in.contiguous();
  const bool labels = img.scalar_type() == at::kInt;   // label maps: order 0 picks voxels, so they are warped as they are
  MVB_CHECK(!labels || order == 0, "int32 label maps are warped at order 0 only");
  const Tensor offset = offset_in.to(img.options().dtype(labels ? at::kFloat : img.scalar_type())).contiguous();
  std::vector<int64_t> want = img.sizes().vec();
  if (want.size() > 1) want[1] = ndim;
  MVB_CHECK(offset.sizes() == at::IntArrayRef(want), "offset must have shape [B, ", ndim, ", *spatial]");
  MVB_CHECK(order >= 0, "order ", given_order, " is not supported (0 nearest, 1 linear, 3 cubic)");
  const int code = labels ? static_cast<int>(MV_I32) : dtype_code(img);
  const Tensor out = at::empty_like(img);
  const auto d = five_dims(img.sizes(), ndim);
  void *const stream = stream_of(img);
  check(ndim == 2 ? mv_deform_warp_2d(ptr(img), ptr(offset), ptr(out), code, d[0], d[1], d[3], d[4], order, stream)
                  : mv_deform_warp_3d(ptr(img), ptr(offset), ptr(out), code, d[0], d[1], d[2], d[3], d[4], order, stream));
  return out;
}

// A volume [B,C,D,H,W], or a sample [C,D,H,W] as a batch of one, warped by the field that its control grids [B,3,z,y,x] give over the
// window [border, points - border]; nothing where that has to be done in two calls.
std::optional<Tensor> elastic_warp(const Tensor &given, const Tensor &grid, double border) {
  const py::gil_scoped_release no_gil;
  const at::NoGradGuard no_grad;
  const bool sample = given.dim() == 4;
  const Tensor img_in = sample ? given.unsqueeze(0) : given;
  if (!img_in.is_cuda() || img_in.dim() != 5 || grid.dim() != 5 || grid.device() != img_in.device() || grid.scalar_type() != at::kFloat ||
      grid.size(0) != img_in.size(0) || grid.size(1) != 3 || img_in.numel() == 0)
    return std::nullopt;
  const auto type = img_in.scalar_type();
  if (type != at::kInt && type != at::kFloat && type != at::kHalf && type != at::kBFloat16) return std::nullopt;
  for (const Tensor &t : {img_in, grid})
    for (int64_t n : t.sizes())
      if (n > std::numeric_limits<int>::max()) return std::nullopt;
  const int code = type == at::kInt ? static_cast<int>(MV_I32) : dtype_code(img_in);
  const auto d = five_dims(img_in.sizes(), 3);
  const auto g = five_dims(grid.sizes(), 3);
  const float edge = static_cast<float>(border);
  if (!mv_elastic_warp_3d_applies(code, d[0], d[2], d[3], d[4], g[2], g[3], g[4], edge)) return std::nullopt;
  const c10::DeviceGuard guard(img_in.device());
  const Tensor img = img_in.contiguous(), points = grid.contiguous();
  const Tensor out = at::empty_like(img);
  check(mv_elastic_warp_3d(ptr(img), ptr(points), ptr(out), code, d[0], d[1], d[2], d[3], d[4], g[2], g[3], g[4], edge, stream_of(img)));
  return sample ? out.squeeze(0) : out;
}

// ---- region decoders: cross attention, RMS norm with residual, 8-bit products -------------------------------------------
int float_code(const Tensor &t, const char *what) {
  const auto type = t.scalar_type();
  MVB_CHECK(type == at::kFloat || type == at::kHalf || type == at::kBFloat16, what, " takes float32, float16 or bfloat16, got ", dtype_name(t));
  return dtype_code(t);
}

int to_int(int64_t n, const char *what) {
  MVB_CHECK(n <= std::numeric_limits<int>::max(), what, " is too large: ", n);
  return static_cast<int>(n);
}

bool wants_gradient(std::initializer_list<Tensor> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor &t : tensors)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// Gradients that cannot be differentiated again: say so when someone tries
void differentiable_once(const variable_list &grads, variable_list &out) {
  bool again = false;
  for (const Tensor &g : grads) again |= g.defined() && g.requires_grad();
  if (!at::GradMode::is_enabled() || !again) return;
  for (Tensor &t : out) {
    if (!t.defined()) continue;
    auto once = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that was marked with @once_differentiable", 1);
    t.set_requires_grad(true);
    t = (*once)(variable_list{t})[0];
  }
}

std::optional<Tensor> maybe(const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// Neighbouring channels of a head; every other stride is the kernels' to follow
Tensor rows_of_heads(const Tensor &t) { return t.size(3) <= 1 || t.stride(3) == 1 ? t : t.contiguous(); }

struct AttentionCall {
  Tensor q, k, v, mask, lengths;
  mv_attention_shape shape;
  int code;
};

AttentionCall attention_call(const Tensor &query, const Tensor &key, const Tensor &value, const Tensor &key_mask, const Tensor &key_lengths) {
  MVB_CHECK(query.is_cuda(), "cross_attention is not implemented on CPU");
  MVB_CHECK(query.dim() == 4 && key.dim() == 4 && value.dim() == 4, "query, key and value have to be [batch, length, heads, channels]");
  AttentionCall c;
  c.code = float_code(query, "cross_attention");
  MVB_CHECK(key.scalar_type() == query.scalar_type() && value.scalar_type() == query.scalar_type(), "query, key and value must share one dtype");
  same_device(query, key, "key");
  same_device(query, value, "value");
  same_device(query, key_mask, "key_mask");
  same_device(query, key_lengths, "key_lengths");
  MVB_CHECK(key.sizes() == value.sizes(), "key has shape ", shape_text(key.sizes()), ", value ", shape_text(value.sizes()));
  MVB_CHECK(key.size(0) == query.size(0), "key has a batch of ", key.size(0), ", expected ", query.size(0), " like the query");
  MVB_CHECK(key.size(3) == query.size(3), "key has heads of ", key.size(3), " channels, expected ", query.size(3), " like the query");
  MVB_CHECK(key.size(2) > 0 && query.size(2) > 0 && query.size(2) % key.size(2) == 0, query.size(2), " heads cannot share ", key.size(2), " heads of keys");
  MVB_CHECK(query.size(3) >= 1 && query.size(3) <= 128, "heads of ", query.size(3), " channels: 1 to 128 are possible");
  mv_attention_shape &s = c.shape;
  s = {to_int(query.size(0), "the batch"), to_int(query.size(1), "the number of queries"), to_int(key.size(1), "the number of keys"),
       to_int(query.size(2), "the number of heads"), to_int(key.size(2), "the number of heads"), static_cast<int>(query.size(3)), {}, {}, {}, 0};
  c.q = rows_of_heads(query), c.k = rows_of_heads(key), c.v = rows_of_heads(value);
  for (int a = 0; a < 3; ++a) s.q_strides[a] = c.q.stride(a), s.k_strides[a] = c.k.stride(a), s.v_strides[a] = c.v.stride(a);
  if (key_mask.defined()) {
    MVB_CHECK(key_mask.scalar_type() == at::kBool, "key_mask has to be bool, got ", dtype_name(key_mask));
    MVB_CHECK(key_mask.dim() == 2 && key_mask.size(0) == s.batch && key_mask.size(1) == s.keys, "key_mask has shape ", shape_text(key_mask.sizes()),
              ", expected (", s.batch, ", ", s.keys, ")");
    c.mask = s.keys <= 1 || key_mask.stride(1) == 1 ? key_mask : key_mask.contiguous();
    s.mask_stride = c.mask.stride(0);
  }
  if (key_lengths.defined()) {
    MVB_CHECK(at::isIntegralType(key_lengths.scalar_type(), false), "key_lengths have to be whole numbers, got ", dtype_name(key_lengths));
    MVB_CHECK(key_lengths.dim() == 1 && key_lengths.size(0) == s.batch, "key_lengths has shape ", shape_text(key_lengths.sizes()), ", expected (", s.batch, ")");
    // (the kernels clamp; types that 32 bits do not hold are clamped first, and none in a type that may not hold the keys' number)
    const auto type = key_lengths.scalar_type();
    MVB_CHECK(type != at::kUInt64, "key_lengths have to fit into int64, got ", dtype_name(key_lengths));
    c.lengths = type == at::kLong || type == at::kUInt32 ? key_lengths.to(at::kLong).clamp(0, s.keys) : key_lengths;
    c.lengths = c.lengths.to(at::kInt).contiguous();
  }
  return c;
}

// output, and what a backward pass will want: the logarithms of the softmax's sums, and what rounding took from the output
struct AttentionResult {
  Tensor output, lse, low;
};

AttentionResult attention_forward(const AttentionCall &c, double scale, bool train) {
  const c10::DeviceGuard guard(c.q.device());
  const mv_attention_shape &s = c.shape;
  const Tensor output = at::empty({s.batch, s.queries, s.heads, s.dim}, c.q.options());
  const Tensor lse = train ? at::empty({2, s.batch, s.heads, s.queries}, c.q.options().dtype(at::kFloat)) : Tensor();
  const Tensor low = train && c.code != MV_F32 ? at::empty_like(output) : Tensor();
  const size_t bytes = mv_cross_attention_forward_workspace_bytes(&s, c.code);
  const Tensor ws = bytes_on(c.q, bytes);
  check(mv_cross_attention_forward(ptr(c.q), ptr(c.k), ptr(c.v), ptr(c.mask), ptr(c.lengths), ptr(output), ptr(low), ptr(lse), &s,
                                   static_cast<float>(scale), c.code, ptr(ws), bytes, stream_of(c.q)));
  return {output, lse, low};
}

// Gradients of the query, and of key and value, as far as they are wanted
variable_list attention_backward(const AttentionCall &c, const Tensor &output, const Tensor &lse, const Tensor &low, const Tensor &grad_in, double scale,
                                 bool for_query, bool for_keys) {
  const c10::DeviceGuard guard(c.q.device());
  const mv_attention_shape &s = c.shape;
  same_device(c.q, grad_in, "grad_output");
  MVB_CHECK(grad_in.sizes() == output.sizes(), "grad_output has shape ", shape_text(grad_in.sizes()), ", expected ", shape_text(output.sizes()));
  const Tensor grad = grad_in.to(output.scalar_type()).contiguous();
  Tensor gq, gk, gv;
  if (for_query) gq = at::empty({s.batch, s.queries, s.heads, s.dim}, c.q.options());
  if (for_keys) gk = at::empty({s.batch, s.keys, s.key_heads, s.dim}, c.q.options()), gv = at::empty_like(gk);
  const size_t bytes = mv_cross_attention_backward_workspace_bytes_for(&s, c.code, for_query, for_keys);
  const Tensor ws = bytes_on(c.q, bytes);
  check(mv_cross_attention_backward(ptr(c.q), ptr(c.k), ptr(c.v), ptr(c.mask), ptr(c.lengths), ptr(output), ptr(low), ptr(lse), ptr(grad),
                                    ptr(gq), ptr(gk), ptr(gv), &s, static_cast<float>(scale), c.code, ptr(ws), bytes, stream_of(c.q)));
  return {gq, gk, gv};
}

struct CrossAttentionFunction : torch::autograd::Function<CrossAttentionFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &query, const Tensor &key, const Tensor &value,
                        const std::optional<Tensor> &key_mask, const std::optional<Tensor> &key_lengths, double scale) {
    const AttentionCall c = attention_call(query, key, value, key_mask.value_or(Tensor()), key_lengths.value_or(Tensor()));
    const AttentionResult r = attention_forward(c, scale, true);
    ctx->save_for_backward({query, key, value, c.mask, c.lengths, r.output, r.lse, r.low});
    ctx->saved_data["scale"] = scale;
    return r.output;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    variable_list out(6);
    if (!grads[0].defined()) return out;
    {
      const at::NoGradGuard no_grad;
      const auto t = ctx->get_saved_variables();
      const bool wanted[3] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2)};
      const variable_list g = attention_backward(attention_call(t[0], t[1], t[2], t[3], t[4]), t[5], t[6], t[7], grads[0],
                                                 ctx->saved_data["scale"].toDouble(), wanted[0], wanted[1] || wanted[2]);
      for (int i = 0; i < 3; ++i)
        if (wanted[i]) out[i] = g[i];
    }
    differentiable_once(grads, out);
    return out;
  }
};

double attention_scale(const Tensor &query, const std::optional<double> &scale) {
  return scale ? *scale : 1.0 / std::sqrt(static_cast<double>(query.dim() == 4 ? query.size(3) : 1));
}

Tensor cross_attention(const Tensor &query, const Tensor &key, const Tensor &value, const std::optional<Tensor> &key_mask,
                       const std::optional<Tensor> &key_lengths, const std::optional<double> &scale) {
  for (const Tensor &t : {query, key, value}) no_forward_mode(t);
  const py::gil_scoped_release no_gil;
  if (wants_gradient({query, key, value}))
    return CrossAttentionFunction::apply(query, key, value, key_mask, key_lengths, attention_scale(query, scale));
  const at::NoGradGuard no_grad;
  return attention_forward(attention_call(query, key, value, key_mask.value_or(Tensor()), key_lengths.value_or(Tensor())),
                           attention_scale(query, scale), false).output;
}

// The two halves for the Python form of the node
std::tuple<Tensor, Tensor, std::optional<Tensor>> cross_attention_forward(const Tensor &query, const Tensor &key, const Tensor &value, const std::optional<Tensor> &key_mask,
                                                  const std::optional<Tensor> &key_lengths, const std::optional<double> &scale) {
  const py::gil_scoped_release no_gil;
  const at::NoGradGuard no_grad;
  const AttentionResult r = attention_forward(attention_call(query, key, value, key_mask.value_or(Tensor()), key_lengths.value_or(Tensor())),
                                              attention_scale(query, scale), true);
  return {r.output, r.lse, r.low.defined() ? std::optional<Tensor>(r.low) : std::nullopt};
}

std::vector<std::optional<Tensor>> cross_attention_backward(const Tensor &query, const Tensor &key, const Tensor &value,
                                                            const std::optional<Tensor> &key_mask, const std::optional<Tensor> &key_lengths,
                                                            const Tensor &output, const Tensor &lse, const std::optional<Tensor> &low, const Tensor &grad,
                                                            const std::optional<double> &scale, bool for_query, bool for_keys) {
  const py::gil_scoped_release no_gil;
  const at::NoGradGuard no_grad;
  const auto g = attention_backward(attention_call(query, key, value, key_mask.value_or(Tensor()), key_lengths.value_or(Tensor())), output, lse,
                                    low.value_or(Tensor()), grad, attention_scale(query, scale), for_query, for_keys);
  return {maybe(g[0]), maybe(g[1]), maybe(g[2])};
}

struct NormCall {
  Tensor x, residual, weight;
  int64_t rows;
  int columns, code, weight_code;
};

NormCall norm_call(const Tensor &x, const Tensor &residual, const Tensor &weight, const char *what) {
  MVB_CHECK(x.is_cuda(), what, " is not implemented on CPU");
  NormCall c;
  c.code = float_code(x, what);
  MVB_CHECK(x.dim() >= 1 && x.size(-1) >= 1, what, " takes rows of at least one column, got shape ", shape_text(x.sizes()));
  same_device(x, residual, "residual");
  same_device(x, weight, "weight");
  MVB_CHECK(weight.dim() == 1 && weight.size(0) == x.size(-1), "weight has shape ", shape_text(weight.sizes()), ", expected (", x.size(-1), ")");
  MVB_CHECK(weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat, "weight has dtype ", dtype_name(weight),
            ", expected float32 or that of the input");
  MVB_CHECK(!residual.defined() || (residual.sizes() == x.sizes() && residual.scalar_type() == x.scalar_type()),
            "the residual must have the input's shape and dtype");
  c.weight_code = dtype_code(weight);
  c.x = x.contiguous();
  c.residual = residual.defined() ? residual.contiguous() : residual;
  c.weight = weight.contiguous();
  c.columns = to_int(x.size(-1), "a row");
  c.rows = x.numel() / c.columns;
  return c;
}

// y, and the sum where there is a residual
std::pair<Tensor, Tensor> norm_forward(const NormCall &c, double eps) {
  const c10::DeviceGuard guard(c.x.device());
  const Tensor y = at::empty_like(c.x);
  const Tensor sum = c.residual.defined() ? at::empty_like(c.x) : Tensor();
  check(mv_add_rms_norm(ptr(c.x), ptr(c.residual), ptr(c.weight), ptr(y), ptr(sum), c.rows, c.columns, static_cast<float>(eps), c.code,
                        c.weight_code, stream_of(c.x)));
  return {y, sum};
}

// gradients of the sum and of the weight, as far as they are wanted
std::pair<Tensor, Tensor> norm_backward(const Tensor &h, const Tensor &weight, const Tensor &grad_y, const Tensor &grad_sum, double eps,
                                        bool for_sum, bool for_weight) {
  const NormCall c = norm_call(h, Tensor(), weight, "add_rms_norm");
  const c10::DeviceGuard guard(c.x.device());
  same_device(c.x, grad_y, "grad_output");
  same_device(c.x, grad_sum, "grad_output");
  const Tensor gy = grad_y.defined() ? grad_y.to(h.scalar_type()).contiguous() : at::zeros_like(c.x);
  const Tensor gs = grad_sum.defined() ? grad_sum.to(h.scalar_type()).contiguous() : grad_sum;
  MVB_CHECK(gy.sizes() == h.sizes() && (!gs.defined() || gs.sizes() == h.sizes()), "grad_output must have the shape ", shape_text(h.sizes()));
  Tensor gx, gw;
  if (for_sum) gx = at::empty_like(c.x);
  if (for_weight) gw = at::empty_like(c.weight);
  const size_t bytes = for_weight ? mv_add_rms_norm_backward_workspace_bytes(c.rows, c.columns) : 0;
  const Tensor ws = bytes_on(c.x, bytes);
  check(mv_add_rms_norm_backward(ptr(c.x), ptr(c.weight), ptr(gy), ptr(gs), ptr(gx), ptr(gw), c.rows, c.columns, static_cast<float>(eps),
                                 c.code, c.weight_code, ptr(ws), bytes, stream_of(c.x)));
  return {gx, gw};
}

struct AddRmsNormFunction : torch::autograd::Function<AddRmsNormFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const std::optional<Tensor> &residual, const Tensor &weight, double eps) {
    const NormCall c = norm_call(x, residual.value_or(Tensor()), weight, "add_rms_norm");
    const auto [y, sum] = norm_forward(c, eps);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({sum.defined() ? sum : x, weight});
    ctx->saved_data["eps"] = eps;
    if (sum.defined()) return {y, sum};
    return {y};
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    variable_list out(4);
    const Tensor none, &gs = grads.size() > 1 ? grads[1] : none;
    if (!grads[0].defined() && !gs.defined()) return out;
    {
      const at::NoGradGuard no_grad;
      const auto t = ctx->get_saved_variables();
      // (inputs that are tensors: x, the residual where there is one, the weight)
      const bool added = grads.size() > 1, for_x = ctx->needs_input_grad(0), for_residual = added && ctx->needs_input_grad(1);
      const auto [gx, gw] = norm_backward(t[0], t[1], grads[0], gs, ctx->saved_data["eps"].toDouble(), for_x || for_residual,
                                          ctx->needs_input_grad(added ? 2 : 1));
      if (for_x) out[0] = gx;
      if (for_residual) out[1] = gx;
      out[2] = gw;
    }
    differentiable_once(grads, out);
    return out;
  }
};

// (y, sum); without a residual the sum is x itself
std::pair<Tensor, Tensor> add_rms_norm(const Tensor &x, const std::optional<Tensor> &residual, const Tensor &weight, double eps) {
  for (const Tensor &t : {x, residual.value_or(Tensor()), weight}) no_forward_mode(t);
  const py::gil_scoped_release no_gil;
  if (wants_gradient({x, residual.value_or(Tensor()), weight})) {
    const variable_list out = AddRmsNormFunction::apply(x, residual, weight, eps);
    return {out[0], out.size() > 1 ? out[1] : x};
  }
  const at::NoGradGuard no_grad;
  auto out = norm_forward(norm_call(x, residual.value_or(Tensor()), weight, "add_rms_norm"), eps);
  if (!out.second.defined()) out.second = x;
  return out;
}

std::pair<Tensor, std::optional<Tensor>> add_rms_norm_forward(const Tensor &x, const std::optional<Tensor> &residual, const Tensor &weight, double eps) {
  const py::gil_scoped_release no_gil;
  const at::NoGradGuard no_grad;
  const auto out = norm_forward(norm_call(x, residual.value_or(Tensor()), weight, "add_rms_norm"), eps);
  return {out.first, out.second.defined() ? std::optional<Tensor>(out.second) : std::nullopt};
}

std::pair<std::optional<Tensor>, std::optional<Tensor>> add_rms_norm_backward(const Tensor &h, const Tensor &weight, const std::optional<Tensor> &grad_y,
                                                                             const std::optional<Tensor> &grad_sum, double eps, bool for_sum,
                                                                             bool for_weight) {
  const py::gil_scoped_release no_gil;
  const at::NoGradGuard no_grad;
  const auto [gx, gw] = norm_backward(h, weight, grad_y.value_or(Tensor()), grad_sum.value_or(Tensor()), eps, for_sum, for_weight);
  return {maybe(gx), maybe(gw)};
}

// 8-bit values of rows of `columns` and their scales
std::pair<Tensor, Tensor> empty_blocks(const Tensor &x) {
  std::vector<int64_t> q = x.sizes().vec(), s = q;
  s.back() = (q.back() + 127) / 128;
  q.back() = 128 * s.back();
  return {at::empty(q, x.options().dtype(at::kFloat8_e4m3fn)), at::empty(s, x.options().dtype(at::kFloat))};
}

void no_gradient(std::initializer_list<Tensor> tensors, const char *what) {
  for (const Tensor &t : tensors) no_forward_mode(t);
  MVB_CHECK(!wants_gradient(tensors), what, " has no gradient: call it under torch.no_grad()");
}

std::tuple<Tensor, Tensor, Tensor> add_rms_norm_quantized(const Tensor &x, const std::optional<Tensor> &residual, const Tensor &weight, double eps) {
  no_gradient({x, residual.value_or(Tensor()), weight}, "add_rms_norm_quantized");
  const py::gil_scoped_release no_gil;
  const at::NoGradGuard no_grad;
  const NormCall c = norm_call(x, residual.value_or(Tensor()), weight, "add_rms_norm_quantized");
  const c10::DeviceGuard guard(c.x.device());
  const auto [q, scales] = empty_blocks(c.x);
  const Tensor sum = c.residual.defined() ? at::empty_like(c.x) : Tensor();
  check(mv_add_rms_norm_quantized(ptr(c.x), ptr(c.residual), ptr(c.weight), ptr(q), ptr(scales), ptr(sum), c.rows, c.columns,
                                  static_cast<float>(eps), c.code, c.weight_code, stream_of(c.x)));
  return {q, scales, sum.defined() ? sum : x};
}

std::pair<Tensor, Tensor> quantize_blocks(const Tensor &given, int64_t block_rows) {
  no_gradient({given}, "quantize_blocks");
  const py::gil_scoped_release no_gil;
  const at::NoGradGuard no_grad;
  MVB_CHECK(given.is_cuda(), "quantize_blocks is not implemented on CPU");
  const int code = float_code(given, "quantize_blocks");
  MVB_CHECK(block_rows == 1 || block_rows == 128, "block_rows ", block_rows, ": 1 or 128 are possible");
  MVB_CHECK(given.dim() >= 1 && given.size(-1) >= 1, "quantize_blocks takes rows of at least one column, got shape ", shape_text(given.sizes()));
  MVB_CHECK(block_rows == 1 || given.dim() == 2, "blocks of 128 rows are those of a matrix, got shape ", shape_text(given.sizes()));
  const c10::DeviceGuard guard(given.device());
  const Tensor x = given.contiguous();
  auto [q, scales] = empty_blocks(x);
  if (block_rows != 1) scales = at::empty({(x.size(0) + 127) / 128, scales.size(1)}, scales.options());
  const int columns = to_int(x.size(-1), "a row");
  check(mv_quantize_blocks(ptr(x), ptr(q), ptr(scales), x.numel() / columns, columns, static_cast<int>(block_rows), code, stream_of(x)));
  return {q, scales};
}

Tensor aligned_rows(const Tensor &t) {
  const Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}

Tensor block_linear(const Tensor &q_in, const Tensor &q_scales, const Tensor &weight_in, const Tensor &weight_scales,
                    const std::optional<Tensor> &bias_in, at::ScalarType out_dtype) {
  const Tensor bias_given = bias_in.value_or(Tensor());
  no_gradient({q_scales, weight_scales, bias_given}, "block_linear");
  const py::gil_scoped_release no_gil;
  const at::NoGradGuard no_grad;
  MVB_CHECK(q_in.is_cuda(), "block_linear is not implemented on CPU");
  MVB_CHECK(q_in.scalar_type() == at::kFloat8_e4m3fn && weight_in.scalar_type() == at::kFloat8_e4m3fn, "q and weight have to be float8_e4m3fn, got ",
            dtype_name(q_in), " and ", dtype_name(weight_in));
  MVB_CHECK(out_dtype == at::kHalf || out_dtype == at::kBFloat16, "out_dtype has to be float16 or bfloat16");
  same_device(q_in, q_scales, "q_scales");
  same_device(q_in, weight_in, "weight");
  same_device(q_in, weight_scales, "weight_scales");
  same_device(q_in, bias_given, "bias");
  MVB_CHECK(q_in.dim() >= 1 && weight_in.dim() == 2 && q_in.size(-1) == weight_in.size(1), "q has shape ", shape_text(q_in.sizes()), ", weight ",
            shape_text(weight_in.sizes()), ": the last dimensions have to be alike");
  const int inputs = to_int(weight_in.size(1), "a row"), outputs = to_int(weight_in.size(0), "the number of outputs");
  MVB_CHECK(inputs > 0 && inputs % 128 == 0, inputs, " inputs: whole blocks of 128 are needed (quantize_blocks pads)");
  std::vector<int64_t> want = q_in.sizes().vec();
  want.back() = inputs / 128;
  MVB_CHECK(q_scales.scalar_type() == at::kFloat && weight_scales.scalar_type() == at::kFloat, "scales have to be float32");
  MVB_CHECK(q_scales.sizes() == at::IntArrayRef(want), "q_scales has shape ", shape_text(q_scales.sizes()), ", expected ", shape_text(want));
  const std::vector<int64_t> want_w{(outputs + 127) / 128, inputs / 128};
  MVB_CHECK(weight_scales.sizes() == at::IntArrayRef(want_w), "weight_scales has shape ", shape_text(weight_scales.sizes()), ", expected ", shape_text(want_w));
  MVB_CHECK(!bias_given.defined() || (bias_given.dim() == 1 && bias_given.size(0) == outputs), "bias has shape ",
            bias_given.defined() ? shape_text(bias_given.sizes()) : "", ", expected (", outputs, ")");
  const c10::DeviceGuard guard(q_in.device());
  const Tensor q = aligned_rows(q_in), w = aligned_rows(weight_in), qs = q_scales.contiguous(), ws = weight_scales.contiguous();
  const Tensor bias = bias_given.defined() ? bias_given.to(out_dtype).contiguous() : bias_given;
  const int64_t rows = q.numel() / inputs;
  want.back() = outputs;
  const Tensor y = at::empty(want, q.options().dtype(out_dtype));
  const size_t bytes = mv_block_linear_workspace_bytes(rows, inputs, outputs);
  const Tensor work = bytes_on(q, bytes);
  check(mv_block_linear(ptr(q), ptr(qs), ptr(w), ptr(ws), ptr(bias), ptr(y), rows, inputs, outputs, dtype_code(y), ptr(work), bytes, stream_of(q)));
  return y;
}

// ---- group norm with an activation ------------------------------------------------------------------------------------
int activation_code(const std::optional<std::string> &name) {
  static const char *const names[] = {"none", "relu", "leaky_relu", "silu", "gelu"};
  if (!name) return MV_NO_ACTIVATION;
  for (int i = 0; i < 5; ++i)
    if (*name == names[i]) return i;
  throw std::runtime_error(c10::str("activation '", *name, "': 'relu', 'leaky_relu', 'silu', 'gelu' or None are possible"));
}

struct GroupNormCall {
  Tensor x, weight, bias;
  int64_t cells;
  int batch, channels, groups, code, weight_code, activation;
  float low;
};

GroupNormCall group_norm_call(const Tensor &x, int64_t groups, const Tensor &weight, const Tensor &bias, int activation, double low) {
  MVB_CHECK(x.is_cuda(), "group_norm_act is not implemented on CPU");
  GroupNormCall c;
  c.code = float_code(x, "group_norm_act");
  MVB_CHECK(x.dim() >= 2 && x.size(-1) >= 1, "group_norm_act takes [batch, ..., channels], got shape ", shape_text(x.sizes()));
  MVB_CHECK(groups >= 1 && x.size(-1) % groups == 0, x.size(-1), " channels in ", groups, " groups");
  const std::pair<const Tensor *, const char *> vectors[] = {{&weight, "weight"}, {&bias, "bias"}};
  for (const auto &[t, name] : vectors) {
    if (!t->defined()) continue;
    same_device(x, *t, name);
    MVB_CHECK(t->dim() == 1 && t->size(0) == x.size(-1), name, " has shape ", shape_text(t->sizes()), ", expected (", x.size(-1), ")");
    MVB_CHECK(t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat, name, " has dtype ", dtype_name(*t),
              ", expected float32 or that of the input");
  }
  MVB_CHECK(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(), "weight and bias must share one dtype");
  c.weight_code = weight.defined() ? dtype_code(weight) : bias.defined() ? dtype_code(bias) : c.code;
  c.x = x.contiguous();
  c.weight = weight.defined() ? weight.contiguous() : weight;
  c.bias = bias.defined() ? bias.contiguous() : bias;
  c.batch = to_int(x.size(0), "the batch"), c.channels = to_int(x.size(-1), "a row"), c.groups = static_cast<int>(groups);
  c.cells = 1;
  for (int64_t d = 1; d + 1 < x.dim(); ++d) c.cells *= x.size(d);
  c.activation = activation, c.low = static_cast<float>(low);
  return c;
}

// y, and the groups' means and inverse deviations
std::pair<Tensor, Tensor> group_norm_run(const GroupNormCall &c, double eps) {
  const c10::DeviceGuard guard(c.x.device());
  const Tensor y = at::empty_like(c.x), stats = at::empty({3, c.batch, c.groups}, c.x.options().dtype(at::kFloat));
  const size_t bytes = mv_group_norm_workspace_bytes(c.batch, c.cells, c.channels, c.groups);
  const Tensor ws = bytes_on(c.x, bytes);
  check(mv_group_norm(ptr(c.x), ptr(c.weight), ptr(c.bias), ptr(y), ptr(stats), c.batch, c.cells, c.channels, c.groups, static_cast<float>(eps),
                      c.activation, c.low, c.code, c.weight_code, ptr(ws), bytes, stream_of(c.x)));
  return {y, stats};
}

// gradients of the cells, the weight and the bias, as far as they are wanted
variable_list group_norm_grads(const GroupNormCall &c, const Tensor &stats, const Tensor &grad_in, bool for_x, bool for_weight, bool for_bias) {
  const c10::DeviceGuard guard(c.x.device());
  same_device(c.x, grad_in, "grad_output");
  MVB_CHECK(grad_in.sizes() == c.x.sizes(), "grad_output has shape ", shape_text(grad_in.sizes()), ", expected ", shape_text(c.x.sizes()));
  MVB_CHECK(stats.scalar_type() == at::kFloat && stats.is_contiguous() && stats.device() == c.x.device() &&
            stats.numel() == int64_t{3} * c.batch * c.groups, "stats are not those of the forward pass");
  const Tensor grad = grad_in.to(c.x.scalar_type()).contiguous();
  Tensor gx, gw, gb;
  if (for_x) gx = at::empty_like(c.x);
  if (for_weight && c.weight.defined()) gw = at::empty_like(c.weight);
  if (for_bias && c.bias.defined()) gb = at::empty_like(c.bias);
  const size_t bytes = mv_group_norm_backward_workspace_bytes(c.batch, c.cells, c.channels, c.groups);
  const Tensor ws = bytes_on(c.x, bytes);
  check(mv_group_norm_backward(ptr(c.x), ptr(c.weight), ptr(c.bias), ptr(stats), ptr(grad), ptr(gx), ptr(gw), ptr(gb), c.batch, c.cells,
                               c.channels, c.groups, c.activation, c.low, c.code, c.weight_code, ptr(ws), bytes, stream_of(c.x)));
  return {gx, gw, gb};
}

struct GroupNormActFunction : torch::autograd::Function<GroupNormActFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, int64_t groups, const std::optional<Tensor> &weight, const std::optional<Tensor> &bias,
                        double eps, int64_t activation, double low) {
    const GroupNormCall c = group_norm_call(x, groups, weight.value_or(Tensor()), bias.value_or(Tensor()), static_cast<int>(activation), low);
    const auto [y, stats] = group_norm_run(c, eps);
    // (the copy of cells that are not in this order is not made twice)
    ctx->save_for_backward({x.is_contiguous() ? x : c.x, weight.value_or(Tensor()), bias.value_or(Tensor()), stats});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["low"] = low;
    return y;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    variable_list out(7);
    if (!grads[0].defined()) return out;
    {
      const at::NoGradGuard no_grad;
      const auto t = ctx->get_saved_variables();
      // (inputs that are tensors: x, the weight and the bias where there are some)
      const bool weighted = t[1].defined(), biased = t[2].defined();
      const bool for_x = ctx->needs_input_grad(0), for_weight = weighted && ctx->needs_input_grad(1), for_bias = biased && ctx->needs_input_grad(weighted ? 2 : 1);
      const GroupNormCall c = group_norm_call(t[0], ctx->saved_data["groups"].toInt(), t[1], t[2], static_cast<int>(ctx->saved_data["activation"].toInt()),
                                              ctx->saved_data["low"].toDouble());
      const variable_list g = group_norm_grads(c, t[3], grads[0], for_x, for_weight, for_bias);
      out[0] = g[0], out[2] = g[1], out[3] = g[2];
    }
    differentiable_once(grads, out);
    return out;
  }
};

Tensor group_norm_act(const Tensor &x, int64_t groups, const std::optional<Tensor> &weight, const std::optional<Tensor> &bias, double eps,
                      const std::optional<std::string> &activation, double low) {
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  for (const Tensor &t : {x, w, b}) no_forward_mode(t);
  const py::gil_scoped_release no_gil;
  const int kind = activation_code(activation);
  if (wants_gradient({x, w, b})) return GroupNormActFunction::apply(x, groups, weight, bias, eps, static_cast<int64_t>(kind), low);
  const at::NoGradGuard no_grad;
  return group_norm_run(group_norm_call(x, groups, w, b, kind, low), eps).first;
}

std::pair<Tensor, Tensor> group_norm_act_forward(const Tensor &x, int64_t groups, const std::optional<Tensor> &weight, const std::optional<Tensor> &bias,
                                                 double eps, const std::optional<std::string> &activation, double low) {
  const py::gil_scoped_release no_gil;
  const at::NoGradGuard no_grad;
  return group_norm_run(group_norm_call(x, groups, weight.value_or(Tensor()), bias.value_or(Tensor()), activation_code(activation), low), eps);
}

std::vector<std::optional<Tensor>> group_norm_act_backward(const Tensor &x, int64_t groups, const std::optional<Tensor> &weight,
                                                           const std::optional<Tensor> &bias, const Tensor &stats, const Tensor &grad,
                                                           const std::optional<std::string> &activation, double low, bool for_x, bool for_weight,
                                                           bool for_bias) {
  const py::gil_scoped_release no_gil;
  const at::NoGradGuard no_grad;
  const auto g = group_norm_grads(group_norm_call(x, groups, weight.value_or(Tensor()), bias.value_or(Tensor()), activation_code(activation), low), stats,
                                  grad, for_x, for_weight, for_bias);
  return {maybe(g[0]), maybe(g[1]), maybe(g[2])};
}

// ---- rotary positions ---------------------------------------------------------------------------------------------------
struct RotaryCall {
  Tensor x, places, frequencies;
  mv_rotary_shape shape;
  int code, place_code;
};

RotaryCall rotary_call(const Tensor &x, const Tensor &positions, const Tensor &frequencies) {
  MVB_CHECK(x.is_cuda(), "rotary_positions is not implemented on CPU");
  MVB_CHECK(x.dim() == 4, "rotary_positions takes [batch, rows, heads, channels], got shape ", shape_text(x.sizes()));
  RotaryCall c;
  c.code = float_code(x, "rotary_positions");
  same_device(x, positions, "positions");
  same_device(x, frequencies, "frequencies");
  MVB_CHECK(frequencies.dim() == 2 && frequencies.size(0) >= 1 && frequencies.size(0) <= 8 && 2 * frequencies.size(1) <= x.size(3),
            "frequencies have shape ", shape_text(frequencies.sizes()), ", expected (axes, pairs) of 1 to 8 axes and up to ", x.size(3) / 2, " pairs");
  MVB_CHECK(x.size(3) >= 1 && x.size(3) <= 1024, "heads of ", x.size(3), " channels: 1 to 1024 are possible");
  MVB_CHECK(frequencies.scalar_type() == at::kFloat || frequencies.scalar_type() == at::kDouble, "frequencies have to be float32 or float64, got ", dtype_name(frequencies));
  const auto type = positions.scalar_type();
  MVB_CHECK(type == at::kFloat || type == at::kDouble || type == at::kHalf || type == at::kBFloat16 || (at::isIntegralType(type, false) && type != at::kUInt64),
            "positions have to be whole or floating numbers, got ", dtype_name(positions));
  const bool shared = positions.dim() == 2;
  MVB_CHECK((shared || (positions.dim() == 3 && positions.size(0) == x.size(0))) && positions.size(-2) == x.size(1) && positions.size(-1) == frequencies.size(0),
            "positions have shape ", shape_text(positions.sizes()), ", expected (", x.size(0), ", ", x.size(1), ", ", frequencies.size(0), ") or (", x.size(1), ", ", frequencies.size(0), ")");
  c.x = rows_of_heads(x);
  c.places = type == at::kFloat || type == at::kDouble || type == at::kInt ? positions
             : at::isIntegralType(type, false) ? positions.to(at::kDouble) : positions.to(at::kFloat);
  c.place_code = c.places.scalar_type() == at::kInt ? static_cast<int>(MV_I32) : dtype_code(c.places);
  c.frequencies = frequencies.to(at::kDouble).contiguous();
  c.shape = {to_int(x.size(0), "the batch"), to_int(x.size(1), "the number of rows"), to_int(x.size(2), "the number of heads"), static_cast<int>(x.size(3)),
             static_cast<int>(frequencies.size(0)), static_cast<int>(frequencies.size(1)), {}, {}};
  for (int a = 0; a < 3; ++a) c.shape.x_strides[a] = c.x.stride(a), c.shape.place_strides[a] = shared ? (a ? c.places.stride(a - 1) : 0) : c.places.stride(a);
  return c;
}

Tensor rotary_run(const RotaryCall &c, bool neighbours, bool back) {
  const c10::DeviceGuard guard(c.x.device());
  const Tensor y = at::empty(c.x.sizes(), c.x.options());
  check(mv_rotary_positions(ptr(c.x), ptr(c.places), ptr(c.frequencies), ptr(y), &c.shape, neighbours, back, c.code, c.place_code, stream_of(c.x)));
  return y;
}

struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &positions, const Tensor &frequencies, bool neighbours) {
    const RotaryCall c = rotary_call(x, positions, frequencies);
    ctx->save_for_backward({positions, frequencies});
    ctx->saved_data["neighbours"] = neighbours;
    ctx->saved_data["dtype"] = x.scalar_type();
    return rotary_run(c, neighbours, false);
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    variable_list out(4);
    if (!grads[0].defined()) return out;
    {
      const at::NoGradGuard no_grad;
      const auto t = ctx->get_saved_variables();
      out[0] = rotary_run(rotary_call(grads[0].to(ctx->saved_data["dtype"].toScalarType()), t[0], t[1]), ctx->saved_data["neighbours"].toBool(), true);
    }
    differentiable_once(grads, out);
    return out;
  }
};

Tensor rotary_positions(const Tensor &x, const Tensor &positions, const Tensor &frequencies, bool neighbours) {
  for (const Tensor &t : {x, positions, frequencies}) no_forward_mode(t);
  MVB_CHECK(!wants_gradient({positions, frequencies}), "rotary_positions has no gradient for positions and frequencies: detach them");
  const py::gil_scoped_release no_gil;
  if (wants_gradient({x})) return RotaryFunction::apply(x, positions, frequencies, neighbours);
  const at::NoGradGuard no_grad;
  return rotary_run(rotary_call(x, positions, frequencies), neighbours, false);
}

Tensor rotary_positions_turn(const Tensor &x, const Tensor &positions, const Tensor &frequencies, bool neighbours, bool back) {
  const py::gil_scoped_release no_gil;
  const at::NoGradGuard no_grad;
  return rotary_run(rotary_call(x, positions, frequencies), neighbours, back);
}

// ---- linear layers with weights in 4 bits --------------------------------------------------------------------------------
void check_group(int64_t group) { MVB_CHECK(group == 32 || group == 64 || group == 128, "groups of ", group, " columns: 32, 64 or 128 are possible"); }

std::pair<Tensor, Tensor> quantize_groups(const Tensor &given, int64_t group) {
  no_gradient({given}, "quantize_groups");
  const py::gil_scoped_release no_gil;
  const at::NoGradGuard no_grad;
  MVB_CHECK(given.is_cuda(), "quantize_groups is not implemented on CPU");
  const int code = float_code(given, "quantize_groups");
  check_group(group);
  MVB_CHECK(given.dim() == 2 && given.size(1) >= 1, "quantize_groups takes a matrix of at least one column, got shape ", shape_text(given.sizes()));
  const c10::DeviceGuard guard(given.device());
  const Tensor w = given.contiguous();
  const int64_t blocks = (w.size(1) + 127) / 128;
  const Tensor q = at::empty({w.size(0), 64 * blocks}, w.options().dtype(at::kByte));
  const Tensor scales = at::empty({w.size(0), 128 / group * blocks}, w.options().dtype(at::kFloat));
  check(mv_quantize_groups(ptr(w), ptr(q), ptr(scales), w.size(0), to_int(w.size(1), "a row"), static_cast<int>(group), code, stream_of(w)));
  return {q, scales};
}

Tensor group_linear(const Tensor &x_in, const Tensor &weight_in, const Tensor &scales_in, const std::optional<Tensor> &bias_in) {
  const Tensor bias_given = bias_in.value_or(Tensor());
  no_gradient({x_in, scales_in, bias_given}, "group_linear");
  const py::gil_scoped_release no_gil;
  const at::NoGradGuard no_grad;
  MVB_CHECK(x_in.is_cuda(), "group_linear is not implemented on CPU");
  MVB_CHECK(x_in.scalar_type() == at::kHalf || x_in.scalar_type() == at::kBFloat16, "group_linear takes float16 or bfloat16, got ", dtype_name(x_in));
  MVB_CHECK(weight_in.scalar_type() == at::kByte && scales_in.scalar_type() == at::kFloat, "weight and scales have to be uint8 and float32, got ",
            dtype_name(weight_in), " and ", dtype_name(scales_in));
  same_device(x_in, weight_in, "weight");
  same_device(x_in, scales_in, "scales");
  same_device(x_in, bias_given, "bias");
  MVB_CHECK(x_in.dim() >= 1 && x_in.size(-1) >= 1, "group_linear takes rows of at least one column, got shape ", shape_text(x_in.sizes()));
  const int inputs = to_int(x_in.size(-1), "a row");
  const int64_t blocks = (int64_t{inputs} + 127) / 128;
  MVB_CHECK(weight_in.dim() == 2 && weight_in.size(1) == 64 * blocks, "weight has shape ", shape_text(weight_in.sizes()), ", expected (outputs, ", 64 * blocks,
            ") for rows of ", inputs);
  const int outputs = to_int(weight_in.size(0), "the number of outputs");
  MVB_CHECK(scales_in.dim() == 2 && scales_in.size(0) == outputs && (scales_in.size(1) == blocks || scales_in.size(1) == 2 * blocks || scales_in.size(1) == 4 * blocks),
            "scales have shape ", shape_text(scales_in.sizes()), ", expected (", outputs, ", ", 4 * blocks, "), (", outputs, ", ", 2 * blocks, ") or (", outputs, ", ",
            blocks, ")");
  MVB_CHECK(!bias_given.defined() || (bias_given.dim() == 1 && bias_given.size(0) == outputs), "bias has shape ",
            bias_given.defined() ? shape_text(bias_given.sizes()) : "", ", expected (", outputs, ")");
  const c10::DeviceGuard guard(x_in.device());
  const Tensor x = aligned_rows(x_in), w = aligned_rows(weight_in), scales = scales_in.contiguous();
  const Tensor bias = bias_given.defined() ? bias_given.to(x.scalar_type()).contiguous() : bias_given;
  const int64_t rows = x.numel() / inputs;
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = outputs;
  const Tensor y = at::empty(shape, x.options());
  const size_t bytes = mv_group_linear_workspace_bytes(rows, inputs, outputs);
  const Tensor work = bytes_on(x, bytes);
  check(mv_group_linear(ptr(x), ptr(w), ptr(scales), ptr(bias), ptr(y), rows, inputs, outputs, static_cast<int>(128 * blocks / scales.size(1)), dtype_code(x),
                        ptr(work), bytes, stream_of(x)));
  return y;
}

// ---- helpers of the augmentation stages ----------------------------------------------------------------------------
// A host array (rois, a control grid) on the device, without waiting for what is queued there.  float64 stays float64,
// every other type becomes float32.
Tensor upload(const py::array &given, const at::Device &device) {
  const bool wide = py::isinstance<py::array_t<double>>(given);
  const py::array array = wide ? py::array(py::array_t<double, py::array::c_style | py::array::forcecast>(given))
                               : py::array(py::array_t<float, py::array::c_style | py::array::forcecast>(given));
  const auto type = wide ? at::kDouble : at::kFloat;
  const std::vector<int64_t> shape(array.shape(), array.shape() + array.ndim());
  const size_t bytes = static_cast<size_t>(array.nbytes());
  const void *data = array.data();
  const py::gil_scoped_release no_gil;
  const at::NoGradGuard no_grad;
  if (!device.is_cuda() || bytes > MV_UPLOAD_MAX_BYTES)
    return at::from_blob(const_cast<void *>(data), shape, type).to(device, type, false, true);
  const c10::DeviceGuard guard(device);
  const Tensor out = at::empty(shape, at::TensorOptions().dtype(type).device(device));
  check(mv_upload(data, ptr(out), bytes, stream_of(out)));
  return out;
}

// The roi of one window of one sample, as geometry.window_rois has it (its float32 arithmetic, in its order), on the device
Tensor window_roi(int dim, const std::vector<double> &start, const std::vector<double> &end, const std::vector<double> &scales,
                  const std::vector<double> &shifts, double rotate, const at::Device &device) {
  const size_t n = static_cast<size_t>(dim);
  MVB_CHECK((dim == 2 || dim == 3) && start.size() == n && end.size() == n && scales.size() == n && shifts.size() == n,
            "expected one value per axis");
  float row[10] = {};
  const int columns = dim == 2 ? 6 : 10;
  for (size_t a = 0; a < n; a++) {
    const float s = static_cast<float>(start[a]), e = static_cast<float>(end[a]), scale = static_cast<float>(scales[a]), shift = static_cast<float>(shifts[a]);
    const float extent = e - s, middle = (s + e) / 2.f, moved = extent * shift;
    row[1 + a] = middle - moved / scale;
    row[1 + n + a] = extent / scale;
  }
  row[columns - 1] = static_cast<float>(rotate);
  const py::gil_scoped_release no_gil;
  const at::NoGradGuard no_grad;
  const c10::OptionalDeviceGuard guard(device.is_cuda() ? std::optional<at::Device>(device) : std::nullopt);
  const Tensor out = at::empty({1, columns}, at::TensorOptions().dtype(at::kFloat).device(device));
  if (device.is_cuda()) check(mv_upload(row, ptr(out), columns * sizeof(float), stream_of(out)));
  else std::memcpy(out.data_ptr(), row, columns * sizeof(float));
  return out;
}

// torch.cuda.max_memory_allocated() in MiB, without building the whole tree of statistics (18 us)
double peak_mib() {
  auto *allocator = c10::hip::HIPCachingAllocator::get();
  if (!allocator->initialized()) return 0.0;
  return allocator->getDeviceStats(c10::hip::current_device()).allocated_bytes[0].peak / 1048576.0;
}

}  // namespace

PYBIND11_MODULE(_native, m) {
  m.def("roi_align", &roi_align);
  m.def("affine", &affine);
  m.def("affine_sample", &affine_sample);
  m.def("modulated_deform_conv", &modulated_deform_conv);
  m.def("deform_conv", &deform_conv);
  m.def("deform_warp", &deform_warp);
  m.def("elastic_warp", &elastic_warp);
  m.def("cross_attention", &cross_attention);
  m.def("cross_attention_forward", &cross_attention_forward);
  m.def("cross_attention_backward", &cross_attention_backward);
  m.def("add_rms_norm", &add_rms_norm);
  m.def("add_rms_norm_forward", &add_rms_norm_forward);
  m.def("add_rms_norm_backward", &add_rms_norm_backward);
  m.def("add_rms_norm_quantized", &add_rms_norm_quantized);
  m.def("quantize_blocks", &quantize_blocks);
  m.def("block_linear", &block_linear);
  m.def("group_norm_act", &group_norm_act);
  m.def("group_norm_act_forward", &group_norm_act_forward);
  m.def("group_norm_act_backward", &group_norm_act_backward);
  m.def("rotary_positions", &rotary_positions);
  m.def("rotary_positions_turn", &rotary_positions_turn);
  m.def("quantize_groups", &quantize_groups);
  m.def("group_linear", &group_linear);
  m.def("upload", &upload);
  m.def("window_roi", &window_roi);
  m.def("peak_mib", &peak_mib);
}
