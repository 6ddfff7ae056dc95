// Torch-facing wrappers of the mixture-of-experts block operators (norm_mx.cu, expert_dispatch.cu,
// expert_mm.cu): argument validation, output allocation, then the plain launchers.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <string>

#include "launchers.h"

namespace {
using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

cudaStream_t stream() { return at::cuda::getCurrentCUDAStream(); }
int sms(const Tensor& t) { return at::cuda::getDeviceProperties(t.get_device())->multiProcessorCount; }
Tensor make(at::IntArrayRef size, const Tensor& like, torch::ScalarType type) {
  return at::detail::empty_cuda(size, type, like.device(), c10::nullopt);
}
Tensor make(at::IntArrayRef size, const Tensor& like) { return make(size, like, like.scalar_type()); }
// A contiguous tensor of its own inside `whole`'s memory, `at` bytes in: tensors that live and die together (the
// tables of an order; codes and their scales) come from one allocation, which is most of a small call's cost.
Tensor part_of(const Tensor& whole, int64_t at, at::IntArrayRef size, torch::ScalarType type) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(),
                                                      c10::scalarTypeToTypeMeta(type));
  t.unsafeGetTensorImpl()->set_storage_offset(at / (int64_t)c10::elementSize(type));
  t.unsafeGetTensorImpl()->set_sizes_contiguous(size);
  return t;
}
int64_t up16(int64_t bytes) { return (bytes + 15) / 16 * 16; }
bool is16(const Tensor& t) { return t.scalar_type() == torch::kBFloat16 || t.scalar_type() == torch::kFloat16; }
bool on16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
// a row of a two-dimensional tensor that has one row may report any stride
int64_t row_stride(const Tensor& t) { return t.size(0) == 1 ? t.size(1) : t.stride(0); }

// Numbers in messages go through std::to_string: c10::str streams integers, which crashes where the extension
// and torch were linked with different C++ runtimes.
std::string num(int64_t v) { return std::to_string(v); }

// Rows of adjacent elements: a column of one element may report any stride.
bool dense_rows(const Tensor& t) { return t.numel() == 0 || t.size(1) == 1 || t.stride(1) == 1; }

// The operators have no forward-mode derivative: a tangent is refused, where the bare kernels would drop it.
void check_tangent(const Tensor& t) {
  TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), "the expert block operators have no forward-mode derivative");
}
void check_tangent(const OptTensor& t) {
  if (t) check_tangent(*t);
}
template <typename... T>
void check_tangents(const T&... t) {
  (check_tangent(t), ...);
}

void check_device(const Tensor& like, const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be on ", like.device());
}
void check_rows(const Tensor& like, const Tensor& t, int64_t rows, int64_t n, torch::ScalarType type, const char* name) {
  check_device(like, t, name);
  TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == n, name, " must be [", num(rows), ", ", num(n), "]");
  TORCH_CHECK(t.scalar_type() == type, name, " must be ", type);
  TORCH_CHECK(dense_rows(t), name, " rows must be contiguous");
}
void check_rows16(const Tensor& like, const Tensor& t, int64_t rows, int64_t n, torch::ScalarType type, const char* name) {
  check_rows(like, t, rows, n, type, name);
  TORCH_CHECK(t.numel() == 0 || (on16(t) && row_stride(t) * t.element_size() % 16 == 0), name,
              " rows must start on 16-byte boundaries");
}
// t itself if its rows are contiguous, apart from one another and on 16-byte boundaries, else a copy whose rows are
Tensor rows16(const Tensor& t) {
  if (t.dim() != 2 || t.numel() == 0 ||
      (t.stride(1) == 1 && on16(t) && row_stride(t) >= t.size(1) && row_stride(t) * t.element_size() % 16 == 0))
    return t;
  return t.is_contiguous() ? t.clone() : t.contiguous();
}
OptTensor rows16(const OptTensor& t) { return t ? OptTensor(rows16(*t)) : t; }
// t itself if its rows are contiguous, else a copy
Tensor packed_rows(const Tensor& t) { return t.dim() != 2 || dense_rows(t) ? t : t.contiguous(); }
OptTensor packed_rows(const OptTensor& t) { return t ? OptTensor(packed_rows(*t)) : t; }
void check_err(const Tensor& like, const Tensor& err) {
  check_device(like, err, "err");
  TORCH_CHECK(err.scalar_type() == torch::kInt32 && err.numel() >= 4, "err must be CUDA int32[4]");
}

void check_weight(const Tensor& like, const Tensor& w, int64_t n) {
  check_device(like, w, "w");
  TORCH_CHECK(w.scalar_type() == torch::kFloat32 && w.dim() == 1 && w.size(0) == n && w.is_contiguous() && on16(w),
              "w must be contiguous fp32 [", num(n), "]");
}
// Memory that rows of x and of t share: kNo and kYes are exact.
enum class Shared { kNo, kYes, kUnknown };
Shared shared_rows(const Tensor& x, const Tensor& t) {
  if (x.numel() == 0 || t.numel() == 0) return Shared::kNo;
  const int64_t xb = x.size(1) * x.element_size(), tb = t.size(1) * t.element_size();
  const int64_t step = row_stride(x) * x.element_size(), tstep = row_stride(t) * t.element_size();
  const int64_t apart = reinterpret_cast<intptr_t>(t.data_ptr()) - reinterpret_cast<intptr_t>(x.data_ptr());
  if (apart >= (x.size(0) - 1) * step + xb || -apart >= (t.size(0) - 1) * tstep + tb) return Shared::kNo;
  if (x.size(0) == 1 && t.size(0) == 1) return Shared::kYes;
  if (step != tstep || step < xb || step < tb) return Shared::kUnknown;
  // rows of one step: t's lie `at` bytes into x's period, between x's columns or not
  const int64_t at = (apart % step + step) % step;
  return at >= xb && at + tb <= step ? Shared::kNo : Shared::kYes;
}
// An operand of a call that writes over x, as rows that no thread can find written by another: t itself if it is x
// or shares no memory with it, a copy where the strides do not tell.
Tensor beside(const Tensor& x, const Tensor& t, const char* name) {
  if (t.data_ptr() == x.data_ptr() && t.scalar_type() == x.scalar_type() && t.sizes() == x.sizes() && row_stride(t) == row_stride(x))
    return t;
  const Shared s = shared_rows(x, t.dim() == 1 ? t.unsqueeze(0) : t);
  TORCH_CHECK(s != Shared::kYes, "add_rmsnorm_mx: ", name, " and the x that is written over overlap in part");
  return s == Shared::kNo ? t : t.clone(at::MemoryFormat::Contiguous);
}

void check_norm(const Tensor& x, const char* op) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && is16(x), op, ": x must be a CUDA BF16 or FP16 [rows, n] tensor");
  TORCH_CHECK(x.size(1) >= 32 && x.size(1) % 32 == 0 && x.size(1) <= 8192, op,
              ": n must be a multiple of 32 and at most 8192");
}
}  // namespace

// -> (stream, codes, scales, h or None); stream is x itself without addends or in place
std::tuple<Tensor, Tensor, Tensor, OptTensor> add_rmsnorm_mx(const Tensor& x_in, const Tensor& w_in, double eps,
                                                             const OptTensor& d_in, const OptTensor& df_in, bool inplace,
                                                             bool return_h) {
  check_norm(x_in, "add_rmsnorm_mx");
  check_tangents(x_in, w_in, d_in, df_in);
  const Tensor x = inplace ? x_in : rows16(x_in);
  OptTensor d = rows16(d_in), df = rows16(df_in);
  Tensor w = w_in;
  const int64_t rows = x.size(0), n = x.size(1);
  check_rows16(x, x, rows, n, x.scalar_type(), "x");
  check_weight(x, w, n);
  if (d) check_rows16(x, *d, rows, n, x.scalar_type(), "d");
  if (df) check_rows16(x, *df, rows, n, torch::kFloat32, "dfp32");
  const bool add = d || df;
  const c10::cuda::CUDAGuard g(x.device());
  if (inplace && add) {
    TORCH_CHECK(rows <= 1 || row_stride(x) >= n, "add_rmsnorm_mx: inplace needs rows apart from one another");
    if (d) d = beside(x, *d, "d");
    if (df) df = beside(x, *df, "dfp32");
    w = beside(x, w, "w");
    x.unsafeGetTensorImpl()->bump_version();  // a gradient that saved x's old values must not use the new ones
  }
  Tensor s = add && !inplace ? make({rows, n}, x) : x_in;
  const Tensor mx = make({rows * n + rows * (n / 32)}, x, torch::kUInt8);
  Tensor codes = part_of(mx, 0, {rows, n}, torch::kUInt8);
  Tensor scales = part_of(mx, rows * n, {rows, n / 32}, torch::kUInt8);
  OptTensor h;
  if (return_h) h = make({rows, n}, x);
  NormMxArgs a{};
  a.rows = rows;
  a.n = (int)n;
  a.half = x.scalar_type() == torch::kFloat16;
  a.x = x.data_ptr();
  a.xs = row_stride(x);
  if (d) { a.d = d->data_ptr(); a.ds = row_stride(*d); }
  if (df) { a.df = df->data_ptr<float>(); a.dfs = row_stride(*df); }
  if (add) { a.x_out = s.data_ptr(); a.xos = row_stride(s); }
  a.w = w.data_ptr<float>();
  a.eps = (float)eps;
  if (h) a.h = h->data_ptr();
  a.codes = codes.data_ptr<uint8_t>();
  a.scales = scales.data_ptr<uint8_t>();
  launch_add_rmsnorm_mx(a, stream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {s, codes, scales, h};
}

// -> (dx in x's type, dw fp32, dx in fp32 or None)
std::tuple<Tensor, Tensor, OptTensor> rmsnorm_backward(const Tensor& dh_in, const Tensor& x_in, const Tensor& w,
                                                       double eps, const OptTensor& dres_in, bool fp32_dx) {
  check_norm(x_in, "add_rmsnorm_backward");
  check_tangents(dh_in, x_in, w, dres_in);
  const Tensor x = rows16(x_in), dh = rows16(dh_in);
  const OptTensor dres = rows16(dres_in);
  const int64_t rows = x.size(0), n = x.size(1);
  check_rows16(x, x, rows, n, x.scalar_type(), "x");
  check_rows16(x, dh, rows, n, x.scalar_type(), "dh");
  check_weight(x, w, n);
  if (dres) check_rows16(x, *dres, rows, n, x.scalar_type(), "dres");
  const c10::cuda::CUDAGuard g(x.device());
  const int slots = rmsnorm_bwd_slots(rows, (int)n, sms(x));
  Tensor dx = make({rows, n}, x), dw = make({n}, x, torch::kFloat32);
  Tensor part = make({slots, n}, x, torch::kFloat32);
  OptTensor dxf;
  if (fp32_dx) dxf = make({rows, n}, x, torch::kFloat32);
  NormBwdArgs a{};
  a.rows = rows;
  a.n = (int)n;
  a.half = x.scalar_type() == torch::kFloat16;
  a.x = x.data_ptr();
  a.xs = row_stride(x);
  a.dh = dh.data_ptr();
  a.dhs = row_stride(dh);
  if (dres) { a.dres = dres->data_ptr(); a.drs = row_stride(*dres); }
  a.w = w.data_ptr<float>();
  a.eps = (float)eps;
  a.dx = dx.data_ptr();
  if (dxf) a.dxf = dxf->data_ptr<float>();
  a.part = part.data_ptr<float>();
  a.dw = dw.data_ptr<float>();
  launch_rmsnorm_bwd(a, slots, stream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {dx, dw, dxf};
}

Tensor mx_dequantize(const Tensor& codes_in, const Tensor& scales_in) {
  const Tensor codes = codes_in.contiguous(), scales = scales_in.contiguous();
  TORCH_CHECK(codes.is_cuda() && codes.dim() == 2 && codes.scalar_type() == torch::kUInt8 && codes.size(1) % 32 == 0,
              "mx_dequantize: codes must be a CUDA uint8 [rows, n] tensor, n a multiple of 32");
  check_rows(codes, scales, codes.size(0), codes.size(1) / 32, torch::kUInt8, "scales");
  TORCH_CHECK(codes.numel() == 0 || on16(codes), "mx_dequantize: codes must start on a 16-byte boundary");
  const c10::cuda::CUDAGuard g(codes.device());
  Tensor out = make({codes.size(0), codes.size(1)}, codes, torch::kBFloat16);
  launch_mx_dequantize(codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(), codes.numel(), out.data_ptr(), stream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

// -> (offsets [E + 1], slots [T, k], pairs [T k])
std::tuple<Tensor, Tensor, Tensor> expert_order(const Tensor& ids_in, int64_t num_experts, int64_t expert_base) {
  const Tensor ids = ids_in.contiguous();
  TORCH_CHECK(ids.is_cuda() && ids.dim() == 2 &&
              (ids.scalar_type() == torch::kInt32 || ids.scalar_type() == torch::kInt64),
              "expert_order: ids must be a CUDA int32 or int64 [tokens, topk] tensor");
  TORCH_CHECK(num_experts >= 1 && num_experts <= 4096, "expert_order: num_experts must be in [1, 4096]");
  TORCH_CHECK(ids.numel() < (1 << 30) && ids.size(1) <= 1024, "expert_order: at most 2^30 pairs and 1024 choices");
  const c10::cuda::CUDAGuard g(ids.device());
  const int64_t T = ids.size(0), k = ids.size(1);
  const auto i32 = ids.options().dtype(torch::kInt32);
  if (T * k == 0) return {torch::zeros({num_experts + 1}, i32), torch::empty({T, k}, i32), torch::empty({0}, i32)};
  const int64_t table = up16(T * k * 4);
  const Tensor whole = make({2 * table + (num_experts + 1) * 4}, ids, torch::kUInt8);
  Tensor slots = part_of(whole, 0, {T, k}, torch::kInt32), pairs = part_of(whole, table, {T * k}, torch::kInt32);
  Tensor offsets = part_of(whole, 2 * table, {num_experts + 1}, torch::kInt32);
  const int rc = launch_expert_order(ids.data_ptr(), ids.scalar_type() == torch::kInt64, T * k, expert_base,
                                     (int)num_experts, offsets.data_ptr<int32_t>(),
                                     slots.data_ptr<int32_t>(), pairs.data_ptr<int32_t>(), stream());
  TORCH_CHECK(rc == 0, "expert_order: launch failed (", num(rc), ")");
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {offsets, slots, pairs};
}

namespace {
void check_order(const Tensor& like, const Tensor& offsets, const Tensor& slots) {
  check_device(like, offsets, "offsets");
  check_device(like, slots, "slots");
  TORCH_CHECK(offsets.scalar_type() == torch::kInt32 && offsets.dim() == 1 && offsets.size(0) >= 2 &&
              offsets.is_contiguous(), "offsets must be contiguous int32 [experts + 1]");
  TORCH_CHECK(slots.scalar_type() == torch::kInt32 && slots.dim() == 2 && slots.is_contiguous() &&
              slots.size(1) <= 1024, "slots must be contiguous int32 [tokens, topk], topk at most 1024");
}
}  // namespace

// x [T, width] (and scales [T, ...], uint8) -> the same for the sorted rows
std::tuple<Tensor, OptTensor> expert_gather(const Tensor& x_in, const OptTensor& scales_in, const Tensor& slots,
                                            const Tensor& offsets) {
  check_tangents(x_in);
  const Tensor x = packed_rows(x_in);
  const OptTensor scales = packed_rows(scales_in);
  TORCH_CHECK(x.is_cuda() && x.dim() == 2, "gather: x must be a CUDA [tokens, width] tensor");
  check_order(x, offsets, slots);
  const int64_t T = slots.size(0), k = slots.size(1);
  check_rows(x, x, T, x.size(1), x.scalar_type(), "x");
  if (scales) check_rows(x, *scales, T, scales->size(1), torch::kUInt8, "scales");
  const c10::cuda::CUDAGuard g(x.device());
  Tensor out = make({T * k, x.size(1)}, x);
  OptTensor sout;
  if (scales) sout = make({T * k, scales->size(1)}, *scales);
  GatherArgs a{};
  a.T = T;
  a.k = (int)k;
  a.E = (int)offsets.size(0) - 1;
  a.num_sms = sms(x);
  a.slots = slots.data_ptr<int32_t>();
  a.offsets = offsets.data_ptr<int32_t>();
  a.src = x.data_ptr();
  a.row_bytes = x.size(1) * x.element_size();
  a.src_stride = row_stride(x) * x.element_size();
  a.dst = out.data_ptr();
  if (scales && scales->size(1) > 0) {
    a.scales = scales->data_ptr();
    a.scale_bytes = scales->size(1);
    a.scales_stride = row_stride(*scales);
    a.scales_dst = sout->data_ptr();
  }
  launch_expert_gather(a, stream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {out, sout};
}

namespace {
int row_type(const Tensor& y, const char* op) {
  TORCH_CHECK(y.is_cuda() && y.dim() == 2 && (is16(y) || y.scalar_type() == torch::kFloat32), op,
              ": rows must be a CUDA BF16, FP16 or FP32 [rows, width] tensor");
  return y.scalar_type() == torch::kFloat32 ? 2 : y.scalar_type() == torch::kFloat16 ? 1 : 0;
}
bool wide(const Tensor& t) { return t.size(1) % 8 == 0 && on16(t) && row_stride(t) * t.element_size() % 16 == 0; }
}  // namespace

Tensor expert_combine(const Tensor& y_in, const OptTensor& weights_in, const OptTensor& residual_in,
                      const Tensor& slots, const Tensor& offsets, bool out_f32) {
  check_tangents(y_in, weights_in, residual_in);
  const Tensor y = packed_rows(y_in);
  const OptTensor weights = packed_rows(weights_in), residual = packed_rows(residual_in);
  const int type = row_type(y, "combine");
  check_order(y, offsets, slots);
  const int64_t T = slots.size(0), k = slots.size(1), width = y.size(1);
  check_rows(y, y, T * k, width, y.scalar_type(), "y");
  const auto out_type = out_f32 ? torch::kFloat32 : y.scalar_type();
  if (weights) check_rows(y, *weights, T, k, torch::kFloat32, "weights");
  if (residual) check_rows(y, *residual, T, width, out_type, "residual");
  const c10::cuda::CUDAGuard g(y.device());
  Tensor out = make({T, width}, y, out_type);
  CombineArgs a{};
  a.T = T;
  a.k = (int)k;
  a.width = (int)width;
  a.num_sms = sms(y);
  a.slots = slots.data_ptr<int32_t>();
  if (weights) { a.weights = weights->data_ptr<float>(); a.ws = row_stride(*weights); }
  a.y = y.data_ptr();
  a.ys = row_stride(y);
  if (residual) { a.residual = residual->data_ptr(); a.rs = row_stride(*residual); }
  a.out = out.data_ptr();
  launch_expert_combine(a, type, out_f32, wide(y) && (!residual || wide(*residual)), stream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

// -> (dy or None, dweights or None)
std::tuple<OptTensor, OptTensor> expert_combine_backward(const Tensor& dout_in, const Tensor& y_in,
                                                         const Tensor& weights_in, const Tensor& slots,
                                                         const Tensor& offsets, bool need_dy, bool need_dw) {
  check_tangents(dout_in, y_in, weights_in);
  const Tensor dout = packed_rows(dout_in), y = packed_rows(y_in), weights = packed_rows(weights_in);
  const int type = row_type(y, "combine_backward");
  check_order(y, offsets, slots);
  const int64_t T = slots.size(0), k = slots.size(1), width = y.size(1);
  check_rows(y, y, T * k, width, y.scalar_type(), "y");
  check_rows(y, weights, T, k, torch::kFloat32, "weights");
  TORCH_CHECK(dout.scalar_type() == y.scalar_type() || dout.scalar_type() == torch::kFloat32,
              "combine_backward: dout must be fp32 or have y's type");
  check_rows(y, dout, T, width, dout.scalar_type(), "dout");
  const c10::cuda::CUDAGuard g(y.device());
  OptTensor dy, dw;
  if (need_dy) dy = make({T * k, width}, y);
  if (need_dw) dw = make({T, k}, weights);
  CombineBwdArgs a{};
  a.T = T;
  a.k = (int)k;
  a.width = (int)width;
  a.E = (int)offsets.size(0) - 1;
  a.slots = slots.data_ptr<int32_t>();
  a.offsets = offsets.data_ptr<int32_t>();
  a.weights = weights.data_ptr<float>();
  a.ws = row_stride(weights);
  a.y = y.data_ptr();
  a.ys = row_stride(y);
  a.dout = dout.data_ptr();
  a.gs = row_stride(dout);
  if (dy) a.dy = dy->data_ptr();
  if (dw) a.dw = dw->data_ptr<float>();
  if (need_dy || need_dw)
    launch_expert_combine_bwd(a, type, dout.scalar_type() == torch::kFloat32, wide(y) && wide(dout), stream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {dy, dw};
}

namespace {
void check_mm(const Tensor& w, const Tensor& offsets, const Tensor& err, const char* op) {
  TORCH_CHECK(w.is_cuda() && w.dim() == 3 && is16(w), op, ": w must be a CUDA BF16 or FP16 [experts, n, k] tensor");
  TORCH_CHECK(w.is_contiguous() && on16(w), op, ": w must be contiguous and start on a 16-byte boundary");
  TORCH_CHECK(w.size(0) >= 1 && w.size(0) <= 1024, op, ": 1 to 1024 experts");
  TORCH_CHECK(w.size(1) >= 8 && w.size(1) % 8 == 0 && w.size(2) >= 8 && w.size(2) % 8 == 0, op,
              ": n and k must be multiples of 8");
  check_device(w, offsets, "offsets");
  TORCH_CHECK(offsets.scalar_type() == torch::kInt32 && offsets.dim() == 1 && offsets.size(0) == w.size(0) + 1 &&
              offsets.is_contiguous(), op, ": offsets must be contiguous int32 [experts + 1]");
  check_err(w, err);
}
ExpertMmCall mm_call(const Tensor& w, const Tensor& offsets, const Tensor& err, int64_t P) {
  TORCH_CHECK(P < (1 << 30), "at most 2^30 rows");
  ExpertMmCall c{};
  c.w = w.data_ptr();
  c.offsets = offsets.data_ptr<int32_t>();
  c.P = P;
  c.E = (int)w.size(0);
  c.N = (int)w.size(1);
  c.K = (int)w.size(2);
  c.half = w.scalar_type() == torch::kFloat16;
  c.num_sms = sms(w);
  c.err = err.data_ptr<int>();
  return c;
}
void run_mm(int mode, const ExpertMmCall& c) {
  const int rc = launch_expert_mm(mode, c, stream());
  TORCH_CHECK(rc == 0, "expert products: tensor map or shared memory refused (", num(rc), ")");
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}
}  // namespace

// -> (y, the products z or None); gated: y = silu(z[:, :n / 2]) z[:, n / 2:]
std::tuple<Tensor, OptTensor> expert_mm(const Tensor& x_in, const Tensor& w, const Tensor& offsets, bool gated,
                                        bool save_pre, const Tensor& err) {
  check_mm(w, offsets, err, "expert_linear");
  check_tangents(x_in, w);
  const Tensor x = rows16(x_in);
  const int64_t P = x.size(0), N = w.size(1), K = w.size(2);
  check_rows16(w, x, P, K, w.scalar_type(), "x");
  TORCH_CHECK(!gated || N % 16 == 0, "expert_linear: a gated product needs n a multiple of 16");
  TORCH_CHECK(gated || !save_pre, "expert_linear: only a gated product keeps its operands");
  const c10::cuda::CUDAGuard g(w.device());
  Tensor y = make({P, gated ? N / 2 : N}, x);
  OptTensor pre;
  if (save_pre) pre = make({P, N}, x);
  if (P > 0) {
    ExpertMmCall c = mm_call(w, offsets, err, P);
    c.x = x.data_ptr();
    c.xs = row_stride(x);
    c.out = y.data_ptr();
    c.pre = pre ? pre->data_ptr() : nullptr;
    c.gated = gated;
    run_mm(0, c);
  }
  return {y, pre};
}

// -> (dx or None, dw or None)
std::tuple<OptTensor, OptTensor> expert_mm_backward(const Tensor& dz_in, const Tensor& x_in, const Tensor& w,
                                                    const Tensor& offsets, bool need_dx, bool need_dw,
                                                    const Tensor& err) {
  check_mm(w, offsets, err, "expert_linear_backward");
  check_tangents(dz_in, x_in, w);
  const Tensor x = rows16(x_in), dz = rows16(dz_in);
  const int64_t P = x.size(0), N = w.size(1), K = w.size(2);
  check_rows16(w, x, P, K, w.scalar_type(), "x");
  check_rows16(w, dz, P, N, w.scalar_type(), "dy");
  const c10::cuda::CUDAGuard g(w.device());
  OptTensor dx, dw;
  if (need_dx) dx = make({P, K}, x);
  if (need_dw) dw = P > 0 ? make(w.sizes(), w) : torch::zeros_like(w);
  if (P > 0) {
    ExpertMmCall c = mm_call(w, offsets, err, P);
    c.x = x.data_ptr();
    c.xs = row_stride(x);
    c.dz = dz.data_ptr();
    c.dzs = row_stride(dz);
    if (dx) { c.out = dx->data_ptr(); run_mm(1, c); }
    if (dw) { c.out = dw->data_ptr(); run_mm(2, c); }
  }
  return {dx, dw};
}

Tensor swiglu_backward(const Tensor& da_in, const Tensor& pre_in, const Tensor& offsets) {
  check_tangents(da_in, pre_in);
  const Tensor da = rows16(da_in), pre = rows16(pre_in);
  TORCH_CHECK(pre.is_cuda() && pre.dim() == 2 && is16(pre) && pre.size(1) >= 16 && pre.size(1) % 16 == 0,
              "swiglu_backward: pre must be a CUDA BF16 or FP16 [rows, n] tensor, n a multiple of 16");
  const int64_t P = pre.size(0), N = pre.size(1);
  check_rows16(pre, pre, P, N, pre.scalar_type(), "pre");
  check_rows16(pre, da, P, N / 2, pre.scalar_type(), "dy");
  check_device(pre, offsets, "offsets");
  TORCH_CHECK(offsets.scalar_type() == torch::kInt32 && offsets.dim() == 1 && offsets.size(0) >= 2 &&
              offsets.is_contiguous(), "swiglu_backward: offsets must be contiguous int32 [experts + 1]");
  const c10::cuda::CUDAGuard g(pre.device());
  Tensor dz = make({P, N}, pre);
  launch_swiglu_bwd(da.data_ptr(), row_stride(da), pre.data_ptr(), row_stride(pre), dz.data_ptr(), P, (int)(N / 2),
                    offsets.data_ptr<int32_t>(), (int)offsets.size(0) - 1, pre.scalar_type() == torch::kFloat16,
                    sms(pre), stream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return dz;
}

// ----------------------------------------------------------------------------- autograd
// The differentiable entry points: where a gradient is recorded they run as autograd nodes, else directly.
namespace {
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

bool wanted(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t && t->defined() && t->requires_grad()) return true;
  return false;
}
const Tensor* at_or_null(const OptTensor& t) { return t ? &*t : nullptr; }
void check_once() { TORCH_CHECK(!at::GradMode::is_enabled(), "the expert block operators have no second derivative"); }
OptTensor some(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

struct AddRmsNormMx : Function<AddRmsNormMx> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& d,
                               const OptTensor& df, double eps, bool return_h) {
    auto [s, codes, scales, h] = add_rmsnorm_mx(x, w, eps, d, df, false, return_h);
    ctx->save_for_backward({s, w});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["d"] = d.has_value();
    ctx->saved_data["df"] = df.has_value();
    ctx->mark_non_differentiable({codes, scales});
    ctx->set_materialize_grads(false);
    variable_list out{s, codes, scales};
    if (h) out.push_back(*h);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_once();
    const auto saved = ctx->get_saved_variables();
    const bool has_d = ctx->saved_data["d"].toBool(), has_f = ctx->saved_data["df"].toBool();
    const Tensor ds = g[0], dh = g.size() > 3 ? g[3] : Tensor();
    Tensor dx = ds, dw, dxf;
    if (dh.defined()) {
      auto [a, b, c] = rmsnorm_backward(dh, saved[0], saved[1], ctx->saved_data["eps"].toDouble(), some(ds), has_f);
      dx = a;
      dw = b;
      if (c) dxf = *c;
    } else if (has_f && ds.defined()) {
      dxf = ds.to(torch::kFloat32);  // only the stream was used
    }
    return {dx, dw, has_d ? dx : Tensor(), dxf, Tensor(), Tensor()};
  }
};

struct Gather : Function<Gather> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& slots, const Tensor& offsets) {
    ctx->save_for_backward({slots, offsets});
    return std::get<0>(expert_gather(x, c10::nullopt, slots, offsets));
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_once();
    const auto saved = ctx->get_saved_variables();
    return {expert_combine(g[0], c10::nullopt, c10::nullopt, saved[0], saved[1], false), Tensor(), Tensor()};
  }
};

struct Combine : Function<Combine> {
  static Tensor forward(AutogradContext* ctx, const Tensor& y, const OptTensor& weights, const OptTensor& residual,
                        const Tensor& slots, const Tensor& offsets, bool out_f32) {
    // without weights no gradient reads the rows
    ctx->save_for_backward({weights ? y : Tensor(), weights ? *weights : Tensor(), slots, offsets});
    ctx->saved_data["type"] = static_cast<int64_t>(y.scalar_type());
    ctx->saved_data["res"] = residual.has_value();
    return expert_combine(y, weights, residual, slots, offsets, out_f32);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_once();
    const auto saved = ctx->get_saved_variables();
    const Tensor& y = saved[0];
    const Tensor& weights = saved[1];
    const bool need_dy = ctx->needs_input_grad(0), need_dw = weights.defined() && ctx->needs_input_grad(1);
    Tensor dy, dw;
    if (!weights.defined()) {
      if (need_dy) dy = std::get<0>(expert_gather(g[0], c10::nullopt, saved[2], saved[3])).to(static_cast<torch::ScalarType>(ctx->saved_data["type"].toInt()));
    } else {
      auto [a, b] = expert_combine_backward(g[0], y, weights, saved[2], saved[3], need_dy, need_dw);
      if (a) dy = *a;
      if (b) dw = *b;
    }
    return {dy, dw, ctx->saved_data["res"].toBool() ? g[0] : Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

struct ExpertLinear : Function<ExpertLinear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& offsets, bool gated,
                        const Tensor& err) {
    auto [y, pre] = expert_mm(x, w, offsets, gated, gated, err);
    ctx->save_for_backward({x, w, offsets, pre ? *pre : Tensor()});
    ctx->saved_data["err"] = err;  // not a saved variable: the host clears it in place between the passes
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_once();
    const auto saved = ctx->get_saved_variables();
    const Tensor dz = saved[3].defined() ? swiglu_backward(g[0], saved[3], saved[2]) : g[0];
    auto [dx, dw] = expert_mm_backward(dz, saved[0], saved[1], saved[2], ctx->needs_input_grad(0),
                                       ctx->needs_input_grad(1), ctx->saved_data["err"].toTensor());
    return {dx ? *dx : Tensor(), dw ? *dw : Tensor(), Tensor(), Tensor(), Tensor()};
  }
};
}  // namespace

std::tuple<Tensor, Tensor, Tensor, OptTensor> add_rmsnorm_mx_op(const Tensor& x, const Tensor& w, double eps,
                                                                const OptTensor& d, const OptTensor& df, bool inplace,
                                                                bool return_h) {
  if (!wanted({&x, &w, at_or_null(d), at_or_null(df)})) return add_rmsnorm_mx(x, w, eps, d, df, inplace, return_h);
  TORCH_CHECK(!inplace, "add_rmsnorm_mx: inplace is not available where a gradient is recorded");
  variable_list o = AddRmsNormMx::apply(x, w, d, df, eps, return_h);
  return {o[0], o[1], o[2], return_h ? OptTensor(o[3]) : OptTensor()};
}
Tensor gather_op(const Tensor& x, const Tensor& slots, const Tensor& offsets) {
  if (!wanted({&x})) return std::get<0>(expert_gather(x, c10::nullopt, slots, offsets));
  return Gather::apply(x, slots, offsets);
}
Tensor combine_op(const Tensor& y, const OptTensor& weights, const OptTensor& residual, const Tensor& slots,
                  const Tensor& offsets, bool out_f32) {
  if (!wanted({&y, at_or_null(weights), at_or_null(residual)}))
    return expert_combine(y, weights, residual, slots, offsets, out_f32);
  return Combine::apply(y, weights, residual, slots, offsets, out_f32);
}
Tensor expert_linear_op(const Tensor& x, const Tensor& w, const Tensor& offsets, bool gated, const Tensor& err) {
  if (!wanted({&x, &w})) return std::get<0>(expert_mm(x, w, offsets, gated, false, err));
  return ExpertLinear::apply(x, w, offsets, gated, err);
}

void bind_block_ops(pybind11::module_& m) {
  const auto unlocked = pybind11::call_guard<pybind11::gil_scoped_release>();
  m.def("add_rmsnorm_mx", &add_rmsnorm_mx_op, "residual add + RMSNorm -> MXFP8 rows", unlocked);
  m.def("rmsnorm_backward", &rmsnorm_backward, "gradient of residual add + RMSNorm", unlocked);
  m.def("mx_dequantize", &mx_dequantize, "MXFP8 rows -> BF16", unlocked);
  m.def("expert_order", &expert_order, "stable sort of (token, choice) pairs by expert", unlocked);
  m.def("expert_gather", &gather_op, "token rows -> rows sorted by expert", unlocked);
  m.def("expert_gather_mx", &expert_gather, "MXFP8 token rows -> rows sorted by expert", unlocked);
  m.def("expert_combine", &combine_op, "rows sorted by expert -> weighted sums per token", unlocked);
  m.def("expert_combine_backward", &expert_combine_backward, "gradients of expert_combine", unlocked);
  m.def("expert_linear", &expert_linear_op, "every expert's matrix product (tcgen05), optionally gated", unlocked);
  m.def("expert_linear_backward", &expert_mm_backward, "gradients of the ungated expert_linear (tcgen05)", unlocked);
  m.def("swiglu_backward", &swiglu_backward, "gradient of silu(gate) * up over sorted rows", unlocked);
}
