// Host side of the short calls: argument checks, allocation and launch of the MXFP4 and AdamW entry points of libcltmi355.so
// for torch tensors.  What a kernel of a few microseconds costs from Python is mostly this, so it is compiled; the library's
// functions are handed over as addresses (bind), so that there is one loader (_lib.py) and one library.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/extension.h>

#include <algorithm>
#include <string>
#include <vector>

#include "../../include/clt_mi355.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

decltype(&clt_last_error) last_error = nullptr;
decltype(&clt_mxfp4_quantize) quantize_fn = nullptr;
decltype(&clt_mxfp4_dequantize) dequantize_fn = nullptr;
decltype(&clt_mxfp4_linear) linear_fn = nullptr;
decltype(&clt_mxfp4_linear_x) linear_x_fn = nullptr;
decltype(&clt_mxfp4_linear_x_workspace_bytes) linear_x_bytes_fn = nullptr;
decltype(&clt_adamw_step) adamw_fn = nullptr;

void bind(const py::dict& address) {
  auto take = [&](auto& fn, const char* name) {
    fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(address[name].cast<uintptr_t>());
  };
  take(last_error, "clt_last_error");
  take(quantize_fn, "clt_mxfp4_quantize");
  take(dequantize_fn, "clt_mxfp4_dequantize");
  take(linear_fn, "clt_mxfp4_linear");
  take(linear_x_fn, "clt_mxfp4_linear_x");
  take(linear_x_bytes_fn, "clt_mxfp4_linear_x_workspace_bytes");
  take(adamw_fn, "clt_adamw_step");
}

void check(int rc, const char* name) {
  TORCH_CHECK(rc == 0, name, " failed (status ", rc, "): ", last_error());
}

int code_of(at::ScalarType t) {
  TORCH_CHECK_TYPE(t == at::kFloat || t == at::kBFloat16, "unsupported dtype ", t, ": only float32 / bfloat16");
  return t == at::kFloat ? CLT_F32 : CLT_BF16;
}
void on_gpu(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "clt_training_amd ops need tensors on an MI355X GPU (there is no CPU fallback)");
}
void same_device(const Tensor& a, const Tensor& b) {
  TORCH_CHECK_VALUE(a.device() == b.device(), "tensors on different devices: ", a.device(), " and ", b.device());
}
int64_t padded(int64_t K) { return (K + 127) / 128 * 128; }

// the device of `t` for the calls below, and its current stream
struct On {
  c10::DeviceIndex before, now;
  void* stream;
  explicit On(const Tensor& t) : before(c10::hip::current_device()), now(t.device().index()) {
    if (now != before) c10::hip::set_device(now);
    stream = c10::hip::getCurrentHIPStream(now).stream();
  }
  ~On() {
    if (now != before) c10::hip::set_device(before);
  }
};

// torch's allocation without its dispatcher (0.4 us less a tensor)
Tensor empty(at::IntArrayRef size, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(size, type, like.device(), std::nullopt);
}
// memory for the length of a call, on its stream (not kept: a captured graph then holds its own)
struct Scratch {
  void* p;
  Scratch(size_t bytes, const On& on)
      : p(bytes ? c10::hip::HIPCachingAllocator::raw_alloc_with_stream(bytes, (hipStream_t)on.stream) : nullptr) {}
  Scratch(const Scratch&) = delete;
  ~Scratch() {
    if (p) c10::hip::HIPCachingAllocator::raw_delete(p);
  }
};

// A tensor was written in place: autograd sees that a saved value is no longer there.  (Inference tensors have no count.)
void written(c10::TensorImpl* t) {
  if (!t->is_inference()) t->bump_version();
}

// rows of unit stride (a copy if they have another)
Tensor rows_of(const Tensor& x) { return x.size(1) > 1 && x.stride(1) != 1 ? x.contiguous() : x; }
int64_t row_stride(const Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }

void check_codes(const Tensor& codes, const Tensor& scales, int64_t cols) {
  TORCH_CHECK_TYPE(codes.scalar_type() == at::kByte && scales.scalar_type() == at::kByte && codes.dim() == 2 && scales.dim() == 2,
                   "MXFP4Tensor: codes and scales are uint8 matrices");
  const int64_t kp = padded(cols);
  TORCH_CHECK_VALUE(cols >= 1 && codes.size(1) == kp / 2 && scales.size(0) == codes.size(0) && scales.size(1) == kp / 32,
                    "MXFP4Tensor: ", cols, " columns need codes [rows, ", kp / 2, "] and scales [rows, ", kp / 32, "], got ",
                    codes.sizes(), " and ", scales.sizes());
  TORCH_CHECK_VALUE(codes.is_contiguous() && scales.is_contiguous() && codes.device() == scales.device(),
                    "MXFP4Tensor: codes and scales are contiguous and on one device");
}

std::tuple<Tensor, Tensor> mxfp4_quantize(const Tensor& x_) {
  TORCH_CHECK_VALUE(x_.dim() == 2, "mxfp4_quantize: a matrix is needed, got shape ", x_.sizes());
  const int dt = code_of(x_.scalar_type());
  on_gpu(x_);
  TORCH_CHECK_VALUE(x_.size(1) >= 1, "mxfp4_quantize: no columns");
  const Tensor x = rows_of(x_);
  const int64_t R = x.size(0), K = x.size(1), kp = padded(K);
  Tensor codes = empty({R, kp / 2}, at::kByte, x), scales = empty({R, kp / 32}, at::kByte, x);
  if (R) {
    const On on(x);
    check(quantize_fn(x.const_data_ptr(), dt, row_stride(x), R, K, codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(),
                      on.stream),
          "clt_mxfp4_quantize");
  }
  return {codes, scales};
}

Tensor mxfp4_dequantize(const Tensor& codes, const Tensor& scales, int64_t cols, at::ScalarType dtype) {
  const int dt = code_of(dtype);
  on_gpu(codes);
  check_codes(codes, scales, cols);
  Tensor out = empty({codes.size(0), cols}, dtype, codes);
  if (out.numel()) {
    const On on(out);
    check(dequantize_fn(codes.const_data_ptr<uint8_t>(), scales.const_data_ptr<uint8_t>(), codes.size(0), cols,
                        out.mutable_data_ptr(), dt, on.stream),
          "clt_mxfp4_dequantize");
  }
  return out;
}

// Rows of equal length, equally far apart, in bytes.  (at::assert_no_overlap accepts what is not dense unseen.)
struct Rows {
  uintptr_t first;
  int64_t count, pitch, width;
  explicit Rows(const Tensor& t)  // (of unit stride in a row; a vector or what is contiguous is one row)
      : first((uintptr_t)t.const_data_ptr()), count(1), pitch(0), width(t.numel() * t.element_size()) {
    if (t.numel() && !t.is_contiguous()) count = t.size(0), pitch = t.stride(0) * t.element_size(), width = t.size(1) * t.element_size();
  }
  uintptr_t end() const { return first + (count - 1) * pitch + width; }
  bool meets(const Rows& o) const {
    if (!width || !o.width || first >= o.end() || o.first >= end()) return false;
    for (int64_t n = 0; n < count; ++n) {
      const uintptr_t low = first + n * pitch, high = low + width;
      if (high <= o.first) continue;
      const int64_t last = o.pitch ? std::min<int64_t>(o.count - 1, (high - 1 - o.first) / o.pitch) : 0;  // that begins below high
      if (o.first + last * o.pitch + o.width > low) return true;
    }
    return false;
  }
};

// x: a matrix, or codes with their scales
Tensor mxfp4_linear(const Tensor& x_, const OptTensor& x_scales, const Tensor& codes, const Tensor& scales, int64_t cols,
                    const OptTensor& bias_, bool relu, std::optional<at::ScalarType> dtype, const OptTensor& out_) {
  const bool packed = x_scales.has_value();
  const auto odt = dtype ? *dtype : out_ ? out_->scalar_type() : packed ? at::kFloat : x_.scalar_type();
  const int oc = code_of(odt);
  check_codes(codes, scales, cols);
  if (packed) check_codes(x_, *x_scales, cols);
  TORCH_CHECK_VALUE(x_.dim() == 2 && (packed || x_.size(1) == cols), "mxfp4_linear: x ", x_.sizes(), " does not fit W [",
                    codes.size(0), ", ", cols, "]");
  const int64_t N = x_.size(0), M = codes.size(0);
  Tensor bias;
  int bc = 0;
  if (bias_) {
    TORCH_CHECK_VALUE(bias_->dim() == 1 && bias_->size(0) == M, "mxfp4_linear: bias ", bias_->sizes(), " for ", M, " rows of W");
    bc = code_of(bias_->scalar_type());
    bias = bias_->contiguous();
  }
  const int xc = packed ? 0 : code_of(x_.scalar_type());
  same_device(codes, x_);
  if (bias_) same_device(codes, bias);
  Tensor out;
  if (out_) {
    out = *out_;
    same_device(codes, out);
    TORCH_CHECK_VALUE(out.dim() == 2 && out.size(0) == N && out.size(1) == M && out.scalar_type() == odt &&
                          (M <= 1 || out.stride(1) == 1) && (N <= 1 || out.stride(0) >= M),
                      "mxfp4_linear: out must be [", N, ", ", M, "] ", odt, " with rows that do not overlap");
    for (const Tensor* t : {&x_, packed ? &*x_scales : nullptr, &codes, &scales, bias_ ? &*bias_ : nullptr}) {
      if (!t) continue;
      at::assert_no_overlap(out, *t);
      const bool in_place = t->dim() == 1 ? t->is_contiguous() : t->size(1) <= 1 || t->stride(1) == 1;  // (else a copy is read)
      TORCH_CHECK(!in_place || !Rows(out).meets(Rows(*t)), "mxfp4_linear: out shares memory with another argument");
    }
  }
  on_gpu(codes);
  if (!out_) out = empty({N, M}, odt, codes);
  if (N == 0 || M == 0) return out;
  const On on(out);
  const int64_t ldo = N > 1 ? out.stride(0) : M;
  const uint8_t *wc = codes.const_data_ptr<uint8_t>(), *ws = scales.const_data_ptr<uint8_t>();
  const void* bp = bias_ ? bias.const_data_ptr() : nullptr;
  if (packed) {
    check(linear_fn(x_.const_data_ptr<uint8_t>(), x_scales->const_data_ptr<uint8_t>(), wc, ws, bp, bc, N, M, cols, relu,
                    out.mutable_data_ptr(), oc, ldo, on.stream),
          "clt_mxfp4_linear");
    if (out_) written(out.unsafeGetTensorImpl());
    return out;
  }
  const Tensor x = rows_of(x_);
  const size_t bytes = linear_x_bytes_fn(N, cols);
  const Scratch scratch(bytes, on);
  check(linear_x_fn(x.const_data_ptr(), xc, row_stride(x), wc, ws, bp, bc, N, M, cols, relu, out.mutable_data_ptr(), oc, ldo,
                    scratch.p, bytes, on.stream),
        "clt_mxfp4_linear_x");
  if (out_) written(out.unsafeGetTensorImpl());
  return out;
}

// Memory that a call writes must be no other argument's.
struct Ranges {
  struct Range {
    uintptr_t first, end;
    bool written;
  };
  std::vector<Range> all;
  void add(const void* p, int64_t bytes, bool written) {
    if (bytes) all.push_back({(uintptr_t)p, (uintptr_t)p + bytes, written});
  }
  bool clash() {
    std::sort(all.begin(), all.end(), [](const Range& a, const Range& b) { return a.first < b.first; });
    uintptr_t any = 0, written = 0;  // where what has been seen ends
    for (const Range& r : all) {
      if (r.first < (r.written ? any : written)) return true;
      any = std::max(any, r.end);
      if (r.written) written = std::max(written, r.end);
    }
    return false;
  }
};

// a number, or one per tensor
std::vector<double> per_tensor(const py::object& v, size_t n, const char* name) {
  if (py::isinstance<py::list>(v) || py::isinstance<py::tuple>(v)) {
    auto r = v.cast<std::vector<double>>();
    TORCH_CHECK_VALUE(r.size() == n, "adamw_step: ", name, " is a number or one number per tensor");
    return r;
  }
  return std::vector<double>(n, v.cast<double>());
}

// the items of a list, a tuple or what can be iterated
struct Items {
  py::object held;
  explicit Items(const py::object& o) : held(py::reinterpret_steal<py::object>(PySequence_Fast(o.ptr(), "adamw_step: lists of tensors"))) {
    if (!held) throw py::error_already_set();
  }
  size_t size() const { return PySequence_Fast_GET_SIZE(held.ptr()); }
  PyObject* operator[](size_t i) const { return PySequence_Fast_GET_ITEM(held.ptr(), i); }
  const Tensor& tensor(size_t i) const {
    TORCH_CHECK_TYPE(THPVariable_Check((*this)[i]), "adamw_step: item ", i, " of the parameters or gradients is no tensor");
    return THPVariable_Unpack((*this)[i]);
  }
};

void adamw_step(const py::object& params_, const py::object& grads_, const py::object& first_, const py::object& second_,
                int64_t step, const py::object& lr, std::pair<double, double> betas, double eps, const py::object& weight_decay,
                int64_t seed) {
  const Items params(params_), grads(grads_), first(first_), second(second_);
  const size_t n = params.size();
  const auto lrs = per_tensor(lr, n, "lr"), wds = per_tensor(weight_decay, n, "weight_decay");
  TORCH_CHECK_VALUE(params.size() == n && grads.size() == n && first.size() == n && second.size() == n,
                    "adamw_step: one gradient and two moments for every parameter");
  if (!n) return;
  on_gpu(params.tensor(0));
  const auto dev = params.tensor(0).device();
  const On on(params.tensor(0));
  {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    TORCH_CHECK(hipStreamIsCapturing((hipStream_t)on.stream, &status) == hipSuccess, "adamw_step: stream state");
    TORCH_CHECK(status == hipStreamCaptureStatusNone, "adamw_step cannot be captured into a graph: the step count is a number "
                "of the call, and every replay would repeat the same step");
  }
  std::vector<clt_adamw_tensor> table(n);
  std::vector<Tensor> keep;  // contiguous copies outlive the launch
  Ranges memory;
  memory.all.reserve(6 * n);
  std::vector<std::pair<Tensor, Tensor>> pairs;  // (a sequence may make its items when it is asked for them)
  std::vector<c10::TensorImpl*> changed;         // (held by the lists and by `pairs`)
  changed.reserve(5 * n);
  for (size_t i = 0; i < n; ++i) {
    const Tensor& p = params.tensor(i);
    const bool dense = grads.tensor(i).is_contiguous();
    if (!dense) keep.push_back(grads.tensor(i).contiguous());
    const Tensor& g = dense ? grads.tensor(i) : keep.back();
    clt_adamw_tensor& r = table[i];
    r = {};
    TORCH_CHECK_TYPE((p.scalar_type() == at::kFloat || p.scalar_type() == at::kBFloat16) &&
                         (g.scalar_type() == at::kFloat || g.scalar_type() == at::kBFloat16),
                     "adamw_step: tensor ", i, ": only float32 / bfloat16, got ", p.scalar_type(), " and ", g.scalar_type());
    TORCH_CHECK_VALUE(p.device() == dev && g.device() == dev && g.sizes() == p.sizes() && p.is_contiguous(),
                      "adamw_step: tensor ", i, ": a contiguous parameter and a gradient of its shape, on ", dev);
    const int64_t numel = p.numel();
    const bool eight = !THPVariable_Check(first[i]);
    TORCH_CHECK_VALUE(eight != THPVariable_Check(second[i]), "adamw_step: tensor ", i, ": both moments in 32 bits or both in 8");
    void* ptr[2];
    for (int k = 0; k < 2; ++k) {
      PyObject* o = k ? second[i] : first[i];
      if (!eight) {
        const Tensor& c = THPVariable_Unpack(o);
        TORCH_CHECK_TYPE(c.scalar_type() == at::kFloat, "adamw_step: tensor ", i, ": moments are float32 or 8-bit pairs, got ",
                         c.scalar_type());
        TORCH_CHECK_VALUE(c.sizes() == p.sizes() && c.is_contiguous() && c.device() == dev, "adamw_step: tensor ", i,
                          ": moments of the parameter's shape, contiguous, on ", dev);
        ptr[k] = c.mutable_data_ptr();
        memory.add(ptr[k], 4 * numel, true);
        changed.push_back(c.unsafeGetTensorImpl());
      } else {
        pairs.push_back(py::handle(o).cast<std::pair<Tensor, Tensor>>());
        const auto& pair = pairs.back();
        const auto ct = pair.first.scalar_type(), st = pair.second.scalar_type();
        TORCH_CHECK_TYPE((ct == at::kByte || ct == at::kFloat8_e4m3fn) && (st == at::kByte || st == at::kFloat8_e8m0fnu),
                         "adamw_step: tensor ", i, ": 8-bit moments are uint8 / float8_e4m3fn codes with uint8 / "
                         "float8_e8m0fnu scales, got ", ct, " and ", st);
        TORCH_CHECK_VALUE(pair.first.numel() == numel && pair.second.numel() == (numel + 127) / 128 &&
                              pair.first.is_contiguous() && pair.second.is_contiguous() && pair.first.device() == dev &&
                              pair.second.device() == dev,
                          "adamw_step: tensor ", i, ": one code per element and one scale per 128, contiguous, on ", dev);
        ptr[k] = pair.first.mutable_data_ptr();
        (k ? r.v_scale : r.m_scale) = static_cast<uint8_t*>(pair.second.mutable_data_ptr());
        changed.push_back(pair.first.unsafeGetTensorImpl());
        changed.push_back(pair.second.unsafeGetTensorImpl());
        memory.add(ptr[k], numel, true);
        memory.add(k ? r.v_scale : r.m_scale, (numel + 127) / 128, true);
      }
    }
    r.p = p.mutable_data_ptr(), r.g = g.const_data_ptr(), r.m = ptr[0], r.v = ptr[1];
    r.numel = numel, r.lr = lrs[i], r.weight_decay = wds[i];
    r.p_dtype = p.scalar_type() == at::kFloat ? CLT_F32 : CLT_BF16;
    r.g_dtype = g.scalar_type() == at::kFloat ? CLT_F32 : CLT_BF16;
    changed.push_back(p.unsafeGetTensorImpl());
    memory.add(r.p, numel * p.element_size(), true);
    memory.add(r.g, numel * g.element_size(), false);
  }
  TORCH_CHECK_VALUE(!memory.clash(), "adamw_step: a tensor is given twice, or two share memory (parameters and moments are "
                    "updated in place)");
  check(adamw_fn(table.data(), (int)n, betas.first, betas.second, eps, step, (uint32_t)seed, on.stream), "clt_adamw_step");
  for (c10::TensorImpl* t : changed) written(t);
}

}  // namespace

PYBIND11_MODULE(_clthost, m) {
  m.def("bind", &bind);
  m.def("check_codes", &check_codes);
  m.def("mxfp4_quantize", &mxfp4_quantize);
  m.def("mxfp4_dequantize", &mxfp4_dequantize);
  m.def("mxfp4_linear", &mxfp4_linear);
  m.def("adamw_step", &adamw_step);
}
