// Python bindings of the 8-bit operators (kernels/int8_ops.h).  Arguments are
// checked here; kunserve_b200/ops/int8.py documents them.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>
#include <cmath>

#include "kernels/int8_ops.h"
#include "messages.h"

namespace py = pybind11;
using namespace kus;

namespace {

using OptTensor = c10::optional<torch::Tensor>;

int value_type(torch::ScalarType t, bool fp32, const char* what) {
  KUS_CHECK(t == torch::kBFloat16 || t == torch::kFloat16 || (fp32 && t == torch::kFloat32), what,
            fp32 ? " must be bfloat16, float16 or float32, got " : " must be bfloat16 or float16, got ", t);
  return t == torch::kBFloat16 ? kInt8TypeBF16 : t == torch::kFloat16 ? kInt8TypeFP16 : kInt8TypeFP32;
}

void no_gradient(const torch::Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(!(t.requires_grad() && at::GradMode::is_enabled()), what,
                    " requires a gradient, but 8-bit results carry none (call under torch.no_grad())");
  TORCH_CHECK_VALUE(!t._fw_grad(0).defined(), what,
                    " carries a forward-mode tangent, but 8-bit results carry none (detach it)");
}

// [T, K] on a GPU, the elements of a row next to one another.
void check_rows(const torch::Tensor& t, const char* what) {
  KUS_CHECK(t.is_cuda() && t.dim() == 2 && t.size(1) > 0 && (t.size(1) == 1 || t.stride(1) == 1), what,
            " must be a CUDA tensor [rows, columns] with contiguous rows of at least one column, got ", t.device(), " ",
            t.sizes(), " strides ", t.strides());
  // (a tile of 256 that ends behind the last row still counts in 32 bits)
  KUS_CHECK(t.size(0) <= (1LL << 31) - 512 && t.size(1) < (1LL << 30), what, " has too many rows or columns");
}
void check_like(const torch::Tensor& t, const torch::Tensor& like, const char* what) {
  check_rows(t, what);
  KUS_CHECK(t.device() == like.device() && t.scalar_type() == like.scalar_type() && t.sizes() == like.sizes(), what,
            " must be a ", like.scalar_type(), " tensor ", like.sizes(), " on ", like.device(), ", got ",
            t.scalar_type(), " ", t.sizes(), " on ", t.device());
}
void check_vector(const torch::Tensor& t, int64_t n, torch::ScalarType type, const torch::Device& device,
                  const char* what) {
  KUS_CHECK(t.device() == device && t.scalar_type() == type && t.dim() == 1 && t.size(0) == n && t.is_contiguous(),
            what, " must be a contiguous ", type, " tensor of ", n, " on ", device, ", got ", t.scalar_type(), " ",
            t.sizes(), " on ", t.device());
}

// First byte and the one behind the last of a tensor's rows.
std::pair<uintptr_t, uintptr_t> span(const torch::Tensor& t) {
  const auto at = reinterpret_cast<uintptr_t>(t.data_ptr());
  int64_t last = t.numel() ? 1 : 0;
  for (int d = 0; t.numel() && d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  return {at, at + last * t.element_size()};
}
bool apart(const torch::Tensor& a, const torch::Tensor& b) {
  const auto x = span(a), y = span(b);
  return x.first == x.second || y.first == y.second || x.second <= y.first || y.second <= x.first;
}
// A kernel writes over `t`: what gradients were recorded with it shows as changed.
void changed(const torch::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// A written tensor's rows lie apart from one another.
void check_written(const torch::Tensor& t, const char* what) {
  KUS_CHECK(t.size(0) <= 1 || t.stride(0) >= t.size(1), what, "'s rows overlap: sizes ", t.sizes(), " strides ",
            t.strides());
}
// `out` is `in` itself, or shares no element with it (other columns of one
// buffer, say): each element is written by the thread that read it.
void check_in_place(const torch::Tensor& out, const torch::Tensor& in, const char* what) {
  if (apart(out, in)) return;
  bool fine = out.data_ptr() == in.data_ptr() && (out.size(0) <= 1 || out.stride(0) == in.stride(0));
  if (!fine && out.element_size() == in.element_size() && out.stride(0) == in.stride(0) && out.stride(0) > 0) {
    const int64_t el = out.element_size(), s = out.stride(0);
    const int64_t d = reinterpret_cast<intptr_t>(out.data_ptr()) - reinterpret_cast<intptr_t>(in.data_ptr());
    const int64_t m = ((d / el) % s + s) % s;
    fine = d % el == 0 && m >= out.size(1) && s - m >= out.size(1);
  }
  KUS_CHECK(fine, "out overlaps ", what, " without being it");
}

torch::Tensor empty(at::IntArrayRef sizes, torch::ScalarType type, const torch::Device& device) {
  return torch::Tensor(at::detail::empty_cuda(sizes, type, device, {}));
}
// 8-bit rows that start on 16 bytes, as the matrix product reads them, and
// their scales, behind them in one block of memory, and behind
// those a tensor of the rows' sizes where `total` asks for one and it is small
// (64 KB: it may outlive the integers, whose memory it then keeps).  An
// allocation takes a tenth of a small call.
constexpr int64_t kSmallTotal = 64 << 10;
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> empty_quantized(const torch::Tensor& like, bool total) {
  const int64_t rows = like.size(0), columns = like.size(1), wide = (columns + 15) / 16 * 16;
  const int64_t scales_at = rows * wide, total_at = (scales_at + 4 * rows + 15) / 16 * 16;
  const int64_t total_bytes = rows * columns * like.element_size();
  const bool together = total && total_bytes <= kSmallTotal;
  const torch::Tensor block = empty({together ? total_at + total_bytes : total_at}, torch::kInt8, like.device());
  auto view = [&](torch::ScalarType type, at::IntArrayRef sizes, at::IntArrayRef strides, int64_t at_byte) {
    torch::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(block.storage()),
                                                               c10::DispatchKeySet(c10::DispatchKey::CUDA),
                                                               c10::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_sizes_and_strides(sizes, strides, at_byte / (int64_t)c10::elementSize(type));
    return t;
  };
  torch::Tensor sum;
  if (total)
    sum = together ? view(like.scalar_type(), {rows, columns}, {columns, 1}, total_at)
                   : empty(like.sizes(), like.scalar_type(), like.device());
  return {view(torch::kInt8, {rows, columns}, {wide, 1}, 0), view(torch::kFloat32, {rows}, {1}, scales_at), sum};
}

// `total`: where the sum goes; asked for one (a.other) and given none, it is made.
std::tuple<torch::Tensor, torch::Tensor> run_rows(Int8Rows a, const torch::Tensor& x, torch::Tensor* total = nullptr) {
  auto [q, scales, sum] = empty_quantized(x, total && !total->defined());
  if (total) {
    if (!total->defined()) *total = sum;
    a.total = total->data_ptr();
    a.ts = total->stride(0);
  }
  a.x = x.data_ptr();
  a.xs = x.stride(0);
  a.q = q.data_ptr<int8_t>();
  a.qs = q.stride(0);
  a.scales = scales.data_ptr<float>();
  a.T = (int)x.size(0);
  a.K = (int)x.size(1);
  int8_rows(a, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {q, scales};
}

std::tuple<torch::Tensor, torch::Tensor> quantize_int8_op(const torch::Tensor& x) {
  check_rows(x, "x");
  no_gradient(x, "x");
  c10::cuda::CUDAGuard guard(x.device());
  Int8Rows a{};
  a.op = kRowsQuantize;
  a.type = value_type(x.scalar_type(), true, "x");
  return run_rows(a, x);
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> add_rms_norm_int8_op(const torch::Tensor& x,
                                                                            const torch::Tensor& weight, double eps,
                                                                            const OptTensor& residual,
                                                                            const OptTensor& out) {
  check_rows(x, "x");
  Int8Rows a{};
  a.op = kRowsNorm;
  a.type = value_type(x.scalar_type(), false, "x");
  check_vector(weight, x.size(1), x.scalar_type(), x.device(), "weight");
  KUS_CHECK((float)eps > 0 && std::isfinite((float)eps), "eps must be positive");
  no_gradient(x, "x");
  no_gradient(weight, "weight");
  c10::cuda::CUDAGuard guard(x.device());
  a.weight = weight.data_ptr();
  a.eps = (float)eps;
  if (!residual.has_value()) {
    KUS_CHECK(!out.has_value(), "out takes the sum of x and residual: without a residual there is none");
    auto [q, scales] = run_rows(a, x);
    return {q, scales, x};
  }
  check_like(*residual, x, "residual");
  no_gradient(*residual, "residual");
  a.other = residual->data_ptr();
  a.os = residual->stride(0);
  torch::Tensor total;
  if (out.has_value()) {
    total = *out;
    check_like(total, x, "out");
    no_gradient(total, "out");
    check_written(total, "out");
    check_in_place(total, x, "x");
    check_in_place(total, *residual, "residual");
    KUS_CHECK(apart(total, weight), "out overlaps weight");
  }
  auto [q, scales] = run_rows(a, x, &total);
  if (out.has_value()) changed(total);
  return {q, scales, total};
}

std::tuple<torch::Tensor, torch::Tensor> silu_mul_int8_op(const torch::Tensor& gate, const torch::Tensor& up) {
  check_rows(gate, "gate");
  Int8Rows a{};
  a.op = kRowsSilu;
  a.type = value_type(gate.scalar_type(), false, "gate");
  check_like(up, gate, "up");
  no_gradient(gate, "gate");
  no_gradient(up, "up");
  c10::cuda::CUDAGuard guard(gate.device());
  a.other = up.data_ptr();
  a.os = up.stride(0);
  return run_rows(a, gate);
}

void check_quantized(const torch::Tensor& q, const torch::Tensor& scales) {
  KUS_CHECK(q.scalar_type() == torch::kInt8, "q must be int8, got ", q.scalar_type());
  check_rows(q, "q");
  check_vector(scales, q.size(0), torch::kFloat32, q.device(), "scales");
  no_gradient(scales, "scales");
}

torch::Tensor dequantize_int8_op(const torch::Tensor& q, const torch::Tensor& scales, torch::ScalarType dtype,
                                 const OptTensor& out) {
  check_quantized(q, scales);
  Int8Values a{};
  c10::cuda::CUDAGuard guard(q.device());
  torch::Tensor o = out.has_value() ? *out : empty(q.sizes(), dtype, q.device());
  a.type = value_type(o.scalar_type(), true, "out");
  check_rows(o, "out");
  KUS_CHECK(o.device() == q.device() && o.sizes() == q.sizes(), "out must have q's sizes ", q.sizes(), ", got ",
            o.sizes());
  no_gradient(o, "out");
  check_written(o, "out");
  KUS_CHECK(apart(o, q) && apart(o, scales), "out overlaps q or scales");
  a.q = q.data_ptr<int8_t>();
  a.qs = q.stride(0);
  a.scales = scales.data_ptr<float>();
  a.out = o.data_ptr();
  a.os = o.stride(0);
  a.T = (int)q.size(0);
  a.K = (int)q.size(1);
  int8_values(a, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (out.has_value()) changed(o);
  return o;
}

// A projection's weights as the kernel reads them, and their scales.
struct Int8Weight {
  torch::Tensor packed, scales;
  c10::cuda::CUDAStream made_on;
  CUtensorMap map;
  int N, K;
  // plans of the numbers of tokens met last (choosing one takes 1 to 3 us)
  struct Recent {
    int M = -1, element = 0;
    Int8Plan plan;
  };
  mutable Recent recent[32];

  const Int8Plan& plan_of(int M, int element) const {
    Recent& r = recent[M % 32];
    if (r.M != M || r.element != element) {
      r.plan = int8_plan(M, N, K, element, int8_slots());
      r.M = M;
      r.element = element;
    }
    return r.plan;
  }

  static c10::cuda::CUDAStream stream_of(const torch::Tensor& q, const torch::Tensor& s) {
    check_quantized(q, s);
    return c10::cuda::getCurrentCUDAStream(q.get_device());
  }
  Int8Weight(const torch::Tensor& q, const torch::Tensor& s) : made_on(stream_of(q, s)) {
    KUS_CHECK(q.size(0) > 0, "a weight needs channels");
    KUS_CHECK(q.size(1) <= kInt8MaxK, "at most ", (int64_t)kInt8MaxK, " columns: their products' sum must fit 32 bits");
    c10::cuda::CUDAGuard guard(q.device());
    N = (int)q.size(0);
    K = (int)q.size(1);
    const int64_t blocks = int8_blocks(N) * int8_blocks(K);
    packed = empty({blocks, kInt8Block, kInt8Block}, torch::kInt8, q.device());
    scales = empty({N}, torch::kFloat32, q.device());
    KUS_CHECK(int8_weight_map(&map, packed.data_ptr<int8_t>(), N, K), "the weight is too large");
    int8_pack(q.data_ptr<int8_t>(), q.stride(0), N, K, packed.data_ptr<int8_t>(), made_on);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    // Behind the packing, and no kernel: it begins once the packing has ended
    // and its writes are seen, and what comes after it begins no earlier.  A
    // product behind the packing itself could start as soon as the last of its
    // blocks had left, and reads its first weights before it waits.
    C10_CUDA_CHECK(cudaMemcpyAsync(scales.data_ptr<float>(), s.data_ptr<float>(), N * sizeof(float),
                                   cudaMemcpyDeviceToDevice, made_on));
  }
  // The weights outlive the work queued on `st`.
  void use(const c10::cuda::CUDAStream& st) const {
    if (st == made_on) return;
    packed.record_stream(st);
    scales.record_stream(st);
  }
};

torch::Tensor int8_linear_op(const torch::Tensor& q, const torch::Tensor& scales, const Int8Weight* weight,
                             const OptTensor& bias, torch::ScalarType dtype, const OptTensor& out) {
  KUS_CHECK(weight != nullptr, "weight must be an Int8Weight");
  check_quantized(q, scales);
  KUS_CHECK(weight->packed.device() == q.device(), "the weight is on ", weight->packed.device(), ", q on ", q.device());
  KUS_CHECK(q.size(1) == weight->K, "q has ", q.size(1), " columns, the weight ", (int64_t)weight->K);
  c10::cuda::CUDAGuard guard(q.device());
  const int64_t M = q.size(0), N = weight->N;
  torch::Tensor o = out.has_value() ? *out : empty({M, N}, dtype, q.device());
  Int8Gemm a{};
  a.type = value_type(o.scalar_type(), true, "out");
  check_rows(o, "out");
  KUS_CHECK(o.device() == q.device() && o.size(0) == M && o.size(1) == N, "out must be [", M, ", ", N, "] on ",
            q.device(), ", got ", o.sizes());
  no_gradient(o, "out");
  check_written(o, "out");
  KUS_CHECK(apart(o, q) && apart(o, scales), "out overlaps q or scales");
  if (bias.has_value()) {
    check_vector(*bias, N, o.scalar_type(), q.device(), "bias");
    no_gradient(*bias, "bias");
    KUS_CHECK(apart(o, *bias), "out overlaps bias");
    a.bias = bias->data_ptr();
  }
  const auto st = at::cuda::getCurrentCUDAStream();
  weight->use(st);
  if (M == 0) return o;
  // the kernel reads rows that start on 16 bytes
  const int8_t* x = q.data_ptr<int8_t>();
  int64_t stride = (weight->K + 15) / 16 * 16;
  c10::DataPtr copied;
  if (reinterpret_cast<uintptr_t>(x) % 16 == 0 && (M == 1 || (q.stride(0) % 16 == 0 && q.stride(0) >= weight->K))) {
    if (M > 1) stride = q.stride(0);
  } else {
    copied = c10::cuda::CUDACachingAllocator::get()->allocate(M * stride);
    int8_align(x, q.stride(0), (int)M, weight->K, static_cast<int8_t*>(copied.get()), st);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    x = static_cast<const int8_t*>(copied.get());
  }
  a.M = (int)M;
  a.N = (int)N;
  a.K = weight->K;
  a.x_scales = scales.data_ptr<float>();
  a.w_scales = weight->scales.data_ptr<float>();
  a.out = o.data_ptr();
  a.ldc = o.stride(0);
  KUS_CHECK(int8_blocks(M) * int8_blocks(N) < (1LL << 28), "the product is too large for one launch");
  const Int8Plan& plan = weight->plan_of(a.M, (int)o.element_size());
  CUtensorMap tokens;
  KUS_CHECK(int8_token_map(&tokens, x, stride, a.M, a.K, plan), "q cannot be mapped");
  int8_gemm(a, plan, weight->map, tokens, st);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (out.has_value()) changed(o);
  return o;
}

}  // namespace

void bind_int8_ops(py::module& m) {
  py::class_<Int8Weight>(m, "Int8Weight")
      .def(py::init<const torch::Tensor&, const torch::Tensor&>())
      .def_readonly("out_features", &Int8Weight::N)
      .def_readonly("in_features", &Int8Weight::K)
      .def_readonly("scales", &Int8Weight::scales)
      .def_property_readonly("device", [](const Int8Weight& w) { return w.packed.device(); });
  m.def("quantize_int8", &quantize_int8_op);
  m.def("add_rms_norm_int8", &add_rms_norm_int8_op);
  m.def("silu_mul_int8", &silu_mul_int8_op);
  m.def("dequantize_int8", &dequantize_int8_op);
  m.def("int8_linear", &int8_linear_op);
  m.def("int8_slots", [] {
    const Int8Slots s = int8_slots();
    return std::vector<int>(s.clusters, s.clusters + 9);
  });
  m.def("int8_plan", [](int M, int N, int K, int element, const std::vector<int>& slots) {
    Int8Slots s{};
    for (int c = 0; c < 9; ++c) s.clusters[c] = slots.at(c);
    const Int8Plan p = int8_plan(M, N, K, element, s);
    return std::map<std::string, int>{{"pair", p.pair},     {"width", p.width}, {"token_tiles", p.token_tiles},
                                      {"channel_tiles", p.channel_tiles},       {"splits", p.splits}, {"alone", p.alone}, {"apart", p.apart},
                                      {"group", p.group},   {"grid", p.grid},   {"stages", p.stages},
                                      {"tmem_columns", p.tmem_columns},         {"smem", p.smem}};
  });
}
