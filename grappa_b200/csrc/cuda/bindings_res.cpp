// torch bindings of the residual layer's operators: RMS norm, linear with its epilogue,
// rows in 8 bits.  Every argument is checked before the device is touched (so a refused
// call is refused the same way on CPU tensors), then the kernels run on the current
// stream of the tensors' device.  Work areas come from torch's caching allocator on that
// stream: two streams, or two captured graphs, never share one.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <limits>
#include <optional>
#include <string>
#include <vector>

#include "cuda_check.h"
#include "kernels.h"

namespace d = grappa::dev;
using at::Tensor;
using OptT = std::optional<Tensor>;

namespace {

// Numbers of a message as text: formatting them through a stream inside the extension
// crashes with this toolchain's C++ runtime.
std::string num(int64_t v) { return std::to_string(v); }
int64_t up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }
bool has(const OptT& t) { return t.has_value() && t->defined(); }
bool f32(const Tensor& t) { return t.scalar_type() == at::kFloat; }

// A matrix argument: where it lies and what it spans.
struct Mat {
  char* p = nullptr;
  int64_t rows = 0, cols = 0, ld = 0;  // elements
  int64_t es = 0;
  const char* name = "";
  template <typename T>
  T* as() const { return reinterpret_cast<T*>(p); }
  int64_t width() const { return cols * es; }
  int64_t pitch() const { return ld * es; }
  int64_t bytes() const { return rows > 0 && cols > 0 ? (rows - 1) * pitch() + width() : 0; }
};

enum Use { kRead, kReadTma, kWrite };

// 2-D, contiguous columns, at least rows x cols, rows that start on 16 bytes (align)
Mat mat(const Tensor& t, const char* name, std::initializer_list<at::ScalarType> types, int64_t rows, int64_t cols,
        Use use, bool align = true) {
  bool typed = false;
  for (auto s : types) typed = typed || t.scalar_type() == s;
  TORCH_CHECK(typed, name, " has dtype ", t.scalar_type(), ", which this operator does not take");
  TORCH_CHECK(t.dim() == 2 && (t.stride(1) == 1 || t.size(1) <= 1), name, " must be 2-D with contiguous rows");
  TORCH_CHECK(t.size(0) >= rows, name, " has ", num(t.size(0)), " rows, ", num(rows), " are needed");
  TORCH_CHECK(t.size(1) >= cols, name, " has ", num(t.size(1)), " columns, ", num(cols), " are needed (rows padded)");
  Mat m;
  m.p = static_cast<char*>(t.data_ptr());
  m.rows = t.size(0);
  m.cols = t.size(1);
  m.es = t.element_size();
  m.ld = t.size(0) > 1 ? t.stride(0) : up(t.size(1), 16);
  m.name = name;
  if (use != kRead) TORCH_CHECK(m.ld >= m.cols, name, " has rows that overlap (stride ", num(m.ld), ")");
  if (align)
    TORCH_CHECK(reinterpret_cast<uintptr_t>(m.p) % 16 == 0 && m.pitch() % 16 == 0, name,
                ": rows must start on 16-byte boundaries");
  return m;
}

float* vec(const Tensor& t, const char* name, int64_t n) {
  TORCH_CHECK(t.scalar_type() == at::kFloat && t.is_contiguous(), name, " must be contiguous float32");
  TORCH_CHECK(t.numel() >= n, name, " has ", num(t.numel()), " elements, ", num(n), " are needed");
  return t.data_ptr<float>();
}

const int32_t* count(const OptT& t, const char* name) {
  if (!has(t)) return nullptr;
  TORCH_CHECK(t->scalar_type() == at::kInt && t->numel() >= 1, name, " must be int32 with one element");
  return t->data_ptr<int32_t>();
}

int32_t* word(const Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.numel() >= 1, name, " must be int32 with one element");
  return t.data_ptr<int32_t>();
}

// Codes and exponent bytes, both or neither.
d::Rows8 rows8(const OptT& q, const OptT& e, int64_t rows, int64_t dim, Use use, std::vector<Mat>* mats) {
  TORCH_CHECK(has(q) == has(e), "q and q_exp are given together");
  d::Rows8 r;
  if (!has(q)) return r;
  const Mat mq = mat(*q, "q", {at::kChar}, rows, up(dim, 32), use);
  const Mat me = mat(*e, "q_exp", {at::kByte}, rows, up(dim, 32) / 32, use, false);
  r.q = mq.as<int8_t>();
  r.ldq = mq.ld;
  r.e = me.as<uint8_t>();
  r.lde = e->size(0) > 1 ? e->stride(0) : e->size(1);
  mats->push_back(mq);
  mats->push_back(me);
  return r;
}

// An output shares no bytes with another argument, unless it is the very same matrix and
// the operator allows that (it reads each element before it writes it).
void apart(const Mat& out, const Mat& other, bool same_ok = false) {
  if (!out.p || !other.p || out.bytes() == 0 || other.bytes() == 0) return;
  if (out.p + out.bytes() <= other.p || other.p + other.bytes() <= out.p) return;
  if (same_ok && out.p == other.p && out.pitch() == other.pitch() && out.es == other.es) return;
  // column windows of one buffer
  if (out.pitch() == other.pitch()) {
    const int64_t pitch = out.pitch();
    const int64_t off = ((other.p - out.p) % pitch + pitch) % pitch;
    if (off >= out.width() && off + other.width() <= pitch) return;
  }
  TORCH_CHECK(false, out.name, " overlaps ", other.name);
}
void all_apart(const Mat& out, const std::vector<Mat>& others) {
  for (const Mat& o : others) apart(out, o);
}

// A vector argument as a matrix of one row, for the overlap checks.
Mat line(float* p, int64_t n, const char* name) {
  Mat m;
  m.p = reinterpret_cast<char*>(p);
  m.rows = 1;
  m.cols = m.ld = n;
  m.es = sizeof(float);
  m.name = name;
  return m;
}

int32_t rows_cap(int64_t cap) {
  TORCH_CHECK(cap >= 0 && cap <= std::numeric_limits<int32_t>::max() - 256, "cap must be in [0, 2^31 - 256)");
  return static_cast<int32_t>(cap);
}
int32_t columns(int64_t dim, int64_t most, const char* what) {
  TORCH_CHECK(dim >= 1 && dim <= most, what, " must be in [1, ", num(most), "], got ", num(dim));
  return static_cast<int32_t>(dim);
}
constexpr int64_t kMostColumns = 1 << 20;

// All tensors on one CUDA device (checked last).
c10::Device on_device(std::initializer_list<const Tensor*> ts, std::initializer_list<const OptT*> os) {
  const Tensor& a = **ts.begin();
  TORCH_CHECK(a.is_cuda(), "the operator's tensors must be CUDA tensors");
  for (const Tensor* t : ts) TORCH_CHECK(t->device() == a.device(), "the operator's tensors are on different devices");
  for (const OptT* t : os)
    if (has(*t)) TORCH_CHECK((*t)->device() == a.device(), "the operator's tensors are on different devices");
  return a.device();
}

cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }
int sms() { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }
Tensor work_area(int64_t floats, c10::Device dev) {
  return floats > 0 ? at::empty({floats}, at::TensorOptions().dtype(at::kFloat).device(dev)) : Tensor();
}

void dropout_args(double p, const OptT& counters, float* out_p, const int64_t** out_c) {
  TORCH_CHECK(p >= 0.0 && p < 1.0, "dropout_p must be in [0, 1)");
  *out_p = static_cast<float>(p);
  if (p == 0.0) return;
  TORCH_CHECK(has(counters) && counters->scalar_type() == at::kLong && counters->numel() >= 3,
              "dropout needs the int64 step counters");
  *out_c = counters->data_ptr<int64_t>();
}

void rmsnorm_fwd(Tensor x, int64_t dim, OptT n_dev, int64_t cap, Tensor gamma, double eps, Tensor y, Tensor rstd,
                 OptT residual, OptT s_out, OptT q, OptT q_exp) {
  d::RmsNormArgs a;
  a.dim = columns(dim, d::kRmsNormMaxDim, "dim");
  a.cap = rows_cap(cap);
  const int64_t w = up(dim, 8);
  const Mat mx = mat(x, "x", {at::kBFloat16, at::kFloat}, cap, w, kRead);
  const Mat my = mat(y, "y", {at::kBFloat16}, cap, w, kWrite);
  a.gamma = vec(gamma, "gamma", dim);
  std::vector<Mat> others{mx, line(const_cast<float*>(a.gamma), dim, "gamma")};
  a.x = mx.p;
  a.f32 = f32(x);
  a.ldx = mx.ld;
  TORCH_CHECK(has(residual) || !has(s_out), "s_out is the sum x + residual: it needs the residual");
  Mat mr, ms;
  if (has(residual)) {
    mr = mat(*residual, "residual", {x.scalar_type()}, cap, w, kRead);
    a.residual = mr.p;
    a.ldr = mr.ld;
    others.push_back(mr);
  }
  if (has(s_out)) {
    ms = mat(*s_out, "s_out", {x.scalar_type()}, cap, w, kWrite);
    a.s_out = ms.p;
    a.lds = ms.ld;
    apart(ms, mx, true);
    apart(ms, others[1]);
    apart(ms, mr, true);
  }
  std::vector<Mat> coded;
  a.q8 = rows8(q, q_exp, cap, dim, kWrite, &coded);
  all_apart(my, others);
  apart(my, ms);
  for (const Mat& m : coded) {
    all_apart(m, others);
    apart(m, ms);
    apart(m, my);
  }
  if (coded.size() == 2) apart(coded[0], coded[1]);
  a.eps = static_cast<float>(eps);
  TORCH_CHECK(a.eps >= 0.f, "eps must not be negative");
  a.y = my.as<__nv_bfloat16>();
  a.ldy = my.ld;
  a.rstd = vec(rstd, "rstd", cap);
  const Mat mstd = line(a.rstd, cap, "rstd");
  all_apart(mstd, others);
  all_apart(mstd, coded);
  apart(mstd, ms);
  apart(mstd, my);
  a.n_ptr = count(n_dev, "n_dev");
  const auto dev = on_device({&x, &gamma, &y, &rstd}, {&n_dev, &residual, &s_out, &q, &q_exp});
  c10::cuda::CUDAGuard g(dev);
  d::launch_rmsnorm_fwd(a, sms(), stream());
}

void rmsnorm_bwd(Tensor dy, OptT x, Tensor rstd, Tensor gamma, int64_t dim, OptT n_dev, int64_t cap, Tensor dx,
                 Tensor dgamma, OptT dres, OptT n_res_dev, bool clear_dy, OptT q, OptT q_exp, bool accumulate) {
  d::RmsNormBwdArgs a;
  a.dim = columns(dim, d::kRmsNormMaxDim, "dim");
  a.cap = rows_cap(cap);
  const int64_t w = up(dim, 8);
  TORCH_CHECK(has(x) != has(q), "give the normalised rows' input x or its 8-bit form (q, q_exp), one of them");
  const Mat my = mat(dy, "dy", {at::kBFloat16, at::kFloat}, cap, w, clear_dy ? kWrite : kRead);
  const Mat md = mat(dx, "dx", {at::kBFloat16, at::kFloat}, cap, w, kWrite);
  std::vector<Mat> others;
  a.dy = my.p;
  a.dy_f32 = f32(dy);
  a.lddy = my.ld;
  a.clear_dy = clear_dy;
  if (has(x)) {
    const Mat mx = mat(*x, "x", {at::kBFloat16, at::kFloat}, cap, w, kRead);
    a.x = mx.p;
    a.x_f32 = f32(*x);
    a.ldx = mx.ld;
    others.push_back(mx);
  }
  a.q8 = rows8(q, q_exp, cap, dim, kRead, &others);
  Mat mr;
  a.n_res_ptr = count(n_res_dev, "n_res_dev");
  if (has(dres)) {
    // with a row count of its own it may have fewer rows (the kernel reads below both counts)
    mr = mat(*dres, "dres", {dx.scalar_type()}, a.n_res_ptr ? 0 : cap, w, kRead);
    a.dres = mr.p;
    a.lddr = mr.ld;
    a.res_cap = static_cast<int32_t>(std::min<int64_t>(mr.rows, cap));
  }
  TORCH_CHECK(has(dres) || !has(n_res_dev), "n_res_dev counts the rows of dres");
  all_apart(md, others);
  apart(md, mr, true);
  apart(md, my, !clear_dy);
  if (clear_dy) {
    all_apart(my, others);
    apart(my, mr);
  }
  a.dx = md.p;
  a.dx_f32 = f32(dx);
  a.lddx = md.ld;
  a.rstd = vec(rstd, "rstd", cap);
  a.gamma = vec(gamma, "gamma", dim);
  a.dgamma = vec(dgamma, "dgamma", dim);
  const Mat mgam = line(a.dgamma, dim, "dgamma");
  all_apart(mgam, others);
  apart(mgam, my);
  apart(mgam, mr);
  apart(mgam, md);
  apart(mgam, line(const_cast<float*>(a.rstd), cap, "rstd"));
  apart(md, line(const_cast<float*>(a.rstd), cap, "rstd"));
  apart(md, line(const_cast<float*>(a.gamma), dim, "gamma"));
  a.accumulate = accumulate;
  a.n_ptr = count(n_dev, "n_dev");
  const auto dev = on_device({&dy, &rstd, &gamma, &dx, &dgamma}, {&x, &n_dev, &dres, &n_res_dev, &q, &q_exp});
  c10::cuda::CUDAGuard g(dev);
  const Tensor work = work_area(d::rmsnorm_bwd_work_floats(a.dim, a.cap, sms()), dev);
  a.work = work.defined() ? work.data_ptr<float>() : nullptr;
  d::launch_rmsnorm_bwd(a, sms(), stream());
}

void linear_fwd(Tensor A, Tensor W, OptT n_dev, int64_t cap, Tensor out, Tensor err, OptT bias, int64_t act,
                OptT residual, OptT z, OptT q, OptT q_exp, double dropout_p, OptT counters, int64_t salt) {
  d::LinearArgs a;
  a.cap = rows_cap(cap);
  TORCH_CHECK(W.dim() == 2 && A.dim() == 2 && W.size(1) == A.size(1), "A [rows, K] and W [N, K] share K");
  const int64_t N = W.size(0), K = W.size(1);
  a.N = columns(N, kMostColumns, "N");
  a.K = columns(K, kMostColumns, "K");
  const Mat ma = mat(A, "A", {at::kBFloat16}, cap, K, kReadTma);
  const Mat mw = mat(W, "W", {at::kBFloat16}, N, K, kReadTma);
  const Mat mo = mat(out, "out", {at::kBFloat16}, cap, up(N, 8), kWrite);
  std::vector<Mat> others{ma, mw};
  a.A = ma.as<__nv_bfloat16>();
  a.a_rows = ma.rows;
  a.lda = ma.ld;
  a.W = mw.as<__nv_bfloat16>();
  a.ldw = mw.ld;
  a.out = mo.as<__nv_bfloat16>();
  a.out_rows = mo.rows;
  a.ldo = mo.ld;
  TORCH_CHECK(act >= 0 && act <= 3, "act must be 0 (none), 1 (ReLU), 2 (GELU) or 3 (SiLU)");
  a.act = static_cast<int32_t>(act);
  if (has(bias)) {
    a.bias = vec(*bias, "bias", N);
    others.push_back(line(const_cast<float*>(a.bias), N, "bias"));
  }
  Mat mr, mz;
  if (has(residual)) {
    mr = mat(*residual, "residual", {at::kBFloat16}, cap, up(N, 8), kReadTma);
    a.residual = mr.as<__nv_bfloat16>();
    a.r_rows = mr.rows;
    a.ldr = mr.ld;
  }
  if (has(z)) {
    mz = mat(*z, "z", {at::kBFloat16}, cap, up(N, 8), kWrite);
    a.z = mz.as<__nv_bfloat16>();
    a.ldz = mz.ld;
    all_apart(mz, others);
    apart(mz, mr);
    apart(mz, mo);
  }
  std::vector<Mat> coded;
  a.q8 = rows8(q, q_exp, cap, N, kWrite, &coded);
  if (!coded.empty()) a.q_rows = coded[0].rows;
  for (const Mat& m : coded) {
    all_apart(m, others);
    apart(m, mr);
    apart(m, mz);
    apart(m, mo);
  }
  if (coded.size() == 2) apart(coded[0], coded[1]);
  all_apart(mo, others);
  apart(mo, mr, true);
  dropout_args(dropout_p, counters, &a.dropout_p, &a.counters);
  a.dropout_salt = static_cast<uint32_t>(salt);
  a.err = word(err, "err");
  a.n_ptr = count(n_dev, "n_dev");
  const auto dev = on_device({&A, &W, &out, &err}, {&n_dev, &bias, &residual, &z, &q, &q_exp, &counters});
  c10::cuda::CUDAGuard g(dev);
  d::launch_linear_fwd(a, stream());
}

void linear_act_bwd(Tensor dout, int64_t dim, OptT n_dev, int64_t cap, int64_t act, Tensor dz, OptT dbias, OptT z,
                    OptT q, OptT q_exp, bool clear_dout, double dropout_p, OptT counters, int64_t salt,
                    std::optional<int64_t> ld_mask, bool accumulate) {
  d::LinearActBwdArgs a;
  a.dim = columns(dim, kMostColumns, "dim");
  a.cap = rows_cap(cap);
  const int64_t w = up(dim, 8);
  TORCH_CHECK(act >= 0 && act <= 3, "act must be 0 (none), 1 (ReLU), 2 (GELU) or 3 (SiLU)");
  a.act = static_cast<int32_t>(act);
  TORCH_CHECK(!(has(z) && has(q)), "give z or its 8-bit form (q, q_exp), not both");
  TORCH_CHECK(act == 0 || has(z) || has(q), "the activation's backward needs z or its 8-bit form (q, q_exp)");
  const Mat mg = mat(dout, "dout", {at::kBFloat16, at::kFloat}, cap, w, clear_dout ? kWrite : kRead);
  const Mat md = mat(dz, "dz", {at::kBFloat16}, cap, w, kWrite);
  std::vector<Mat> others;
  a.dout = mg.p;
  a.dout_f32 = f32(dout);
  a.lddo = mg.ld;
  a.clear_dout = clear_dout;
  if (has(z)) {
    const Mat mz = mat(*z, "z", {at::kBFloat16}, cap, w, kRead);
    a.z = mz.as<__nv_bfloat16>();
    a.ldz = mz.ld;
    others.push_back(mz);
  }
  a.q8 = rows8(q, q_exp, cap, dim, kRead, &others);
  all_apart(md, others);
  apart(md, mg, !clear_dout);
  if (clear_dout) all_apart(mg, others);
  a.dz = md.as<__nv_bfloat16>();
  a.lddz = md.ld;
  dropout_args(dropout_p, counters, &a.dropout_p, &a.counters);
  a.dropout_salt = static_cast<uint32_t>(salt);
  a.ld_mask = ld_mask.has_value() ? *ld_mask : md.ld;
  TORCH_CHECK(a.ld_mask >= 0, "ld_mask must not be negative");
  if (has(dbias)) {
    a.dbias = vec(*dbias, "dbias", dim);
    const Mat mb = line(a.dbias, dim, "dbias");
    all_apart(mb, others);
    apart(mb, mg);
    apart(mb, md);
  }
  a.accumulate = accumulate;
  a.n_ptr = count(n_dev, "n_dev");
  const auto dev = on_device({&dout, &dz}, {&n_dev, &dbias, &z, &q, &q_exp, &counters});
  c10::cuda::CUDAGuard g(dev);
  Tensor work;
  if (a.dbias) {
    work = work_area(d::linear_act_bwd_work_floats(a.dim, a.cap, sms()), dev);
    a.work = work.defined() ? work.data_ptr<float>() : nullptr;
  }
  d::launch_linear_act_bwd(a, sms(), stream());
}

void ckpt8_store(Tensor x, int64_t dim, OptT n_dev, int64_t cap, Tensor q, Tensor q_exp) {
  d::Ckpt8Args a;
  a.dim = columns(dim, kMostColumns, "dim");
  a.cap = rows_cap(cap);
  const Mat mx = mat(x, "x", {at::kBFloat16, at::kFloat}, cap, up(dim, 8), kRead);
  a.x = mx.p;
  a.f32 = f32(x);
  a.ld = mx.ld;
  std::vector<Mat> coded;
  a.q8 = rows8(q, q_exp, cap, dim, kWrite, &coded);
  apart(coded[0], mx);
  apart(coded[1], mx);
  apart(coded[0], coded[1]);
  a.n_ptr = count(n_dev, "n_dev");
  const auto dev = on_device({&x, &q, &q_exp}, {&n_dev});
  c10::cuda::CUDAGuard g(dev);
  d::launch_ckpt8_store(a, stream());
}

void ckpt8_load(Tensor q, Tensor q_exp, int64_t dim, OptT n_dev, int64_t cap, Tensor out) {
  d::Ckpt8Args a;
  a.dim = columns(dim, kMostColumns, "dim");
  a.cap = rows_cap(cap);
  std::vector<Mat> coded;
  a.q8 = rows8(q, q_exp, cap, dim, kRead, &coded);
  const Mat mo = mat(out, "out", {at::kBFloat16, at::kFloat}, cap, up(dim, 8), kWrite);
  all_apart(mo, coded);
  a.out = mo.p;
  a.f32 = f32(out);
  a.ld = mo.ld;
  a.n_ptr = count(n_dev, "n_dev");
  const auto dev = on_device({&q, &q_exp, &out}, {&n_dev});
  c10::cuda::CUDAGuard g(dev);
  d::launch_ckpt8_load(a, stream());
}

void ckpt8_dw(Tensor dy, Tensor q, Tensor q_exp, OptT n_dev, int64_t cap, Tensor gw, Tensor err, bool accumulate) {
  d::Ckpt8DwArgs a;
  a.cap = rows_cap(cap);
  TORCH_CHECK(gw.dim() == 2, "gw must be 2-D");
  a.M = columns(gw.size(0), kMostColumns, "gw rows");
  a.N = columns(gw.size(1), kMostColumns, "gw columns");
  const Mat my = mat(dy, "dy", {at::kBFloat16}, cap, gw.size(0), kReadTma);
  const Mat mg = mat(gw, "gw", {at::kFloat}, gw.size(0), gw.size(1), kWrite, false);
  std::vector<Mat> coded;
  a.q8 = rows8(q, q_exp, cap, gw.size(1), kReadTma, &coded);
  apart(mg, my);
  all_apart(mg, coded);
  a.dy = my.as<__nv_bfloat16>();
  a.dy_rows = my.rows;
  a.dy_cols = my.cols;
  a.lddy = my.ld;
  a.q_rows = coded[0].rows;
  a.q_cols = coded[0].cols;
  a.groups = static_cast<int32_t>(up(gw.size(1), 32) / 32);
  a.gw = mg.as<float>();
  a.ldg = gw.size(0) > 1 ? gw.stride(0) : gw.size(1);
  a.accumulate = accumulate;
  a.err = word(err, "err");
  a.n_ptr = count(n_dev, "n_dev");
  const auto dev = on_device({&dy, &q, &q_exp, &gw, &err}, {&n_dev});
  c10::cuda::CUDAGuard g(dev);
  const Tensor work = work_area(d::ckpt8_dw_work_floats(a.M, a.N, a.cap, sms()), dev);
  a.work = work.defined() ? work.data_ptr<float>() : nullptr;
  d::launch_ckpt8_dw(a, sms(), stream());
}

}  // namespace

void bind_residual(pybind11::module_& m) {
  namespace py = pybind11;
  const auto none = py::none();
  m.def("rmsnorm_fwd", &rmsnorm_fwd, py::arg("x"), py::arg("dim"), py::arg("n_dev"), py::arg("cap"), py::arg("gamma"),
        py::arg("eps"), py::arg("y"), py::arg("rstd"), py::arg("residual") = none, py::arg("s_out") = none,
        py::arg("q") = none, py::arg("q_exp") = none,
        R"(RMS norm of rows, with the residual's addition.

s = x + residual (rounded to their type, bf16 or float32; kept in s_out when given),
rstd[r] = 1 / sqrt(mean(s[r, :dim]^2) + eps), y = s rstd gamma in bf16; q / q_exp: the rows
s rstd (before gamma) in 8 bits (see ckpt8_store).  Rows [0, n) with n = min(*n_dev, cap)
(cap without n_dev); later rows are left as they were.  Matrices are [>= cap, >= dim rounded
up to 8] (q: to 32) with rows on 16-byte boundaries; columns between dim and that width are
not read and are written as zeros.  s_out may be x or residual itself.  dim <= 8192.)");
  m.def("rmsnorm_bwd", &rmsnorm_bwd, py::arg("dy"), py::arg("x"), py::arg("rstd"), py::arg("gamma"), py::arg("dim"),
        py::arg("n_dev"), py::arg("cap"), py::arg("dx"), py::arg("dgamma"), py::arg("dres") = none,
        py::arg("n_res_dev") = none, py::arg("clear_dy") = false, py::arg("q") = none, py::arg("q_exp") = none,
        py::arg("accumulate") = true,
        R"(Backward of rmsnorm_fwd.

dx = rstd (gamma dy - xh mean(gamma dy xh)) + dres,  dgamma (+)= sum over the rows of dy xh
(+= unless accumulate is False), with xh = x rstd (x: the rows that were normalised, s_out
where there was a residual) or, with x None, the 8-bit rows q / q_exp.  dy, x and dx are
bf16 or float32 each, dres as dx.  dres (the gradient that reaches the residual stream from above) has
min(*n_res_dev, n) rows when n_res_dev is given; rows past them get none.  clear_dy zeroes
dy after reading it.  dx may be dres, or dy without clear_dy.  dgamma has the same bits on
every run.)");
  m.def("linear_fwd", &linear_fwd, py::arg("A"), py::arg("W"), py::arg("n_dev"), py::arg("cap"), py::arg("out"),
        py::arg("err"), py::arg("bias") = none, py::arg("act") = 0, py::arg("residual") = none, py::arg("z") = none,
        py::arg("q") = none, py::arg("q_exp") = none, py::arg("dropout_p") = 0.0, py::arg("counters") = none,
        py::arg("salt") = 0,
        R"(out = dropout(act(z)) + residual with z = A W^T + bias, in one kernel.

A [>= cap, K] and W [N, K] bf16, bias [N] float32, out and residual bf16 rows of N columns
(padded to 8; out may be the residual itself).  act: 0 none, 1 ReLU, 2 GELU (tanh form),
3 SiLU.  The pre-activation is kept for linear_act_bwd as bf16 rows (z) and / or in 8 bits
(q / q_exp; with ReLU a positive value keeps a code of at least 1).  z is summed in fp32 by the
tensor core, which truncates: it is short by about 8e-10 K of itself (1e-6 at K = 1024), so that
a value that close to the middle between two codes may get the other one (3 of 100000 there);
both stand for it equally well.  Same bits on every run.  Dropout draws the Philox mask of
element r * out.stride(0) + c, as gemm does.  Rows past n = min(*n_dev, cap) are left as they
were.  err: the engine's error word.)");
  m.def("linear_act_bwd", &linear_act_bwd, py::arg("dout"), py::arg("dim"), py::arg("n_dev"), py::arg("cap"),
        py::arg("act"), py::arg("dz"), py::arg("dbias") = none, py::arg("z") = none, py::arg("q") = none,
        py::arg("q_exp") = none, py::arg("clear_dout") = false, py::arg("dropout_p") = 0.0, py::arg("counters") = none,
        py::arg("salt") = 0, py::arg("ld_mask") = none, py::arg("accumulate") = true,
        R"(Backward of linear_fwd's epilogue: dz = mask(dout) act'(z) in bf16, dbias (+)= its column
sums before that rounding (same bits on every run).

dout bf16 or float32 (the residual's gradient is dout itself); z bf16 rows or q / q_exp.
ld_mask: the row stride of linear_fwd's out, when dropout is on (default: dz's).  Rows
[n, n rounded up to 64) of dz below cap are zeroed, as the weight-gradient GEMM wants them.
The layer's other gradients: gemm(dz, W) and ckpt8_dw(dz, ...) or gemm(dz^T, A).)");
  m.def("ckpt8_store", &ckpt8_store, py::arg("x"), py::arg("dim"), py::arg("n_dev"), py::arg("cap"), py::arg("q"),
        py::arg("q_exp"),
        R"(Rows (bf16 or float32) to 8 bits.

Columns in groups of 32: q[r, 32 g + j] = round(x / 2^E) (ties to even), q_exp[r, g] = E + 127
with E >= -126 the smallest integer with max|x| <= 127 * 2^E in the group.  q: int8, columns
of dim rounded up to 32 (zeros past dim), rows on 16-byte boundaries; q_exp: uint8, one
column a group.  A group with a NaN or an infinity gets the byte 255 and reads back as NaN.)");
  m.def("ckpt8_load", &ckpt8_load, py::arg("q"), py::arg("q_exp"), py::arg("dim"), py::arg("n_dev"), py::arg("cap"),
        py::arg("out"), "The rows that 8-bit rows stand for (exact in bf16 and float32), zeros from dim to the next multiple of 8.");
  m.def("ckpt8_dw", &ckpt8_dw, py::arg("dy"), py::arg("q"), py::arg("q_exp"), py::arg("n_dev"), py::arg("cap"),
        py::arg("gw"), py::arg("err"), py::arg("accumulate") = true,
        R"(Weight gradient from 8-bit rows: gw[M, N] (+)= dy[:n, :M]^T xh[:n, :N].

dy bf16 [>= cap, >= M], xh the rows that q / q_exp stand for, gw float32 (any row stride).
Rows past n may hold anything.  Sums in fp32 in a fixed order: the same bits on every run.)");
}
