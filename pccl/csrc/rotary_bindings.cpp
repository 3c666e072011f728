// Python bindings of the query/key norms with rotation.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cmath>
#include <cstring>
#include <optional>
#include <tuple>

#include "comm.h"
#include "fresh.h"
#include "overlap.h"
#include "rotary.h"

namespace py = pybind11;
using namespace pccl;

namespace {

struct Shape {
  bool flat;                       // [rows, heads, dim]
  int64_t B, S, D;
};

RotaryTensor view(const at::Tensor& t, const char* name, const at::Tensor& q, const Shape& s, int64_t H) {
  TORCH_CHECK(t.is_cuda() && t.device() == q.device() && t.scalar_type() == q.scalar_type(), name, " must have the device and dtype of q");
  TORCH_CHECK(t.dim() == (s.flat ? 3 : 4) && t.size(-1) == s.D && t.size(-2) == H && t.size(-3) == s.S && (s.flat || t.size(0) == s.B), name,
              " has the wrong shape");
  RotaryTensor v;
  v.p = t.data_ptr();
  v.sb = s.flat ? 0 : t.stride(0);
  v.ss = t.stride(-3);
  v.sh = t.stride(-2);
  if (t.numel() == 0) return v;
  TORCH_CHECK(t.stride(-1) == 1, "the last dimension of ", name, " must be contiguous");
  TORCH_CHECK((reinterpret_cast<uintptr_t>(v.p) & 15u) == 0, name, " must start on a 16-byte boundary");
  TORCH_CHECK((s.S <= 1 || v.ss % 8 == 0) && (H <= 1 || v.sh % 8 == 0) && (s.flat || s.B <= 1 || v.sb % 8 == 0), "the strides of ", name,
              " must be multiples of 8 elements");
  return v;
}

// An output: the caller's tensor, which may be exactly one of its own inputs (a row is read before it is written) but shares nothing
// with those of the other heads nor with what every row reads (weights, tables, positions), or a new one.
at::Tensor output(const std::optional<at::Tensor>& given, const at::Tensor& like, const char* name, std::initializer_list<at::Tensor> own,
                  std::initializer_list<at::Tensor> others) {
  if (!given.has_value()) return fresh(like.sizes(), like.scalar_type(), like);
  TORCH_CHECK(distinct(*given), name, " must not overlap itself");
  for (const at::Tensor& t : own) TORCH_CHECK(share(*given, t) != Share::kSome, name, " must not partly overlap an input");
  for (const at::Tensor& t : others) TORCH_CHECK(share(*given, t) == Share::kNone, name, " must not overlap an input of the other heads");
  return *given;
}
// The weights, tables and positions of a call beside an output that the caller gave.
void check_apart(const at::Tensor& out, const char* name, std::initializer_list<at::Tensor> shared, const std::optional<at::Tensor>& positions) {
  for (const at::Tensor& t : shared) TORCH_CHECK(share(out, t) == Share::kNone, name, " must not overlap the weights or the tables");
  TORCH_CHECK(!positions.has_value() || share(out, *positions) == Share::kNone, name, " must not overlap the positions");
}

Shape fill(RotaryArgs& a, const at::Tensor& q, const at::Tensor& k, const at::Tensor& qw, const at::Tensor& kw, const at::Tensor& cos,
           const at::Tensor& sin, const std::optional<at::Tensor>& positions, double eps, bool interleaved) {
  std::memset(&a, 0, sizeof(a));
  TORCH_CHECK(q.is_cuda() && (q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf), "q must be a bfloat16 or float16 CUDA tensor");
  TORCH_CHECK(q.dim() == 3 || q.dim() == 4, "q must be [rows, heads, dim] or [batch, rows, heads, dim]");
  TORCH_CHECK(k.dim() == q.dim(), "k must have as many dimensions as q");
  Shape s;
  s.flat = q.dim() == 3;
  s.B = s.flat ? 1 : q.size(0);
  s.S = q.size(-3);
  s.D = q.size(-1);
  TORCH_CHECK(s.D >= 8 && s.D <= kRotaryMaxDim && s.D % 8 == 0, "the head size must be a multiple of 8 up to ", kRotaryMaxDim);
  TORCH_CHECK(s.B * s.S < ((int64_t)1 << 31) && q.size(-2) < (1 << 20) && k.size(-2) < (1 << 20), "too many rows or heads");
  a.B = (int)s.B;
  a.S = (int)s.S;
  a.D = (int)s.D;
  a.H[0] = (int)q.size(-2);
  a.H[1] = (int)k.size(-2);
  a.x[0] = view(q, "q", q, s, a.H[0]);
  a.x[1] = view(k, "k", q, s, a.H[1]);
  a.is_bf16 = q.scalar_type() == at::kBFloat16;
  TORCH_CHECK(qw.scalar_type() == q.scalar_type() || qw.scalar_type() == at::kFloat, "the weights must have the dtype of q, or be float32");
  for (const at::Tensor* w : {&qw, &kw})
    TORCH_CHECK(w->is_cuda() && w->device() == q.device() && w->is_contiguous() && w->dim() == 1 && w->numel() == s.D &&
                    w->scalar_type() == qw.scalar_type(),
                "q_weight and k_weight must be contiguous, of one dtype, and hold one number per column of a head");
  a.w[0] = qw.data_ptr();
  a.w[1] = kw.data_ptr();
  a.w_type = qw.scalar_type() == at::kFloat ? 2 : (a.is_bf16 ? 0 : 1);
  for (const at::Tensor* t : {&cos, &sin})
    TORCH_CHECK(t->is_cuda() && t->device() == q.device() && t->is_contiguous() && t->scalar_type() == at::kFloat && t->dim() == 2 &&
                    t->sizes() == cos.sizes() && (reinterpret_cast<uintptr_t>(t->data_ptr()) & 15u) == 0,
                "cos and sin must be contiguous float32 [positions, rotated columns / 2], on 16-byte boundaries");
  TORCH_CHECK(cos.size(1) >= 4 && cos.size(1) % 4 == 0 && 2 * cos.size(1) <= s.D, "the rotated columns must be a multiple of 8, at most the head size");
  a.cos = cos.data_ptr<float>();
  a.sin = sin.data_ptr<float>();
  a.table = cos.size(0);
  a.half = (int)cos.size(1);
  a.interleaved = interleaved;
  if (positions.has_value()) {
    TORCH_CHECK(positions->is_cuda() && positions->device() == q.device() && positions->is_contiguous() &&
                    (positions->scalar_type() == at::kLong || positions->scalar_type() == at::kInt) && positions->dim() == (s.flat ? 1 : 2) &&
                    positions->size(-1) == s.S && (s.flat || positions->size(0) == s.B),
                "positions must be contiguous int32 or int64, one for each row");
    a.positions = positions->data_ptr();
    a.positions64 = positions->scalar_type() == at::kLong;
  } else {
    TORCH_CHECK(s.S <= a.table, "the table holds ", a.table, " positions, q has ", s.S, " rows");
  }
  TORCH_CHECK(std::isfinite(eps) && eps >= 0, "eps must be finite and not negative");
  a.eps = (float)eps;
  return s;
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rope_forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& qw, const at::Tensor& kw,
                                                        const at::Tensor& cos, const at::Tensor& sin, std::optional<at::Tensor> positions,
                                                        double eps, bool interleaved, std::optional<at::Tensor> q_out,
                                                        std::optional<at::Tensor> k_out) {
  RotaryArgs a;
  const Shape s = fill(a, q, k, qw, kw, cos, sin, positions, eps, interleaved);
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor qo = output(q_out, q, "q_out", {q}, {k}), ko = output(k_out, k, "k_out", {k}, {q});
  TORCH_CHECK(share(qo, ko) == Share::kNone, "q_out and k_out must not overlap");
  if (q_out.has_value()) check_apart(qo, "q_out", {qw, kw, cos, sin}, positions);
  if (k_out.has_value()) check_apart(ko, "k_out", {qw, kw, cos, sin}, positions);
  a.y[0] = view(qo, "q_out", q, s, a.H[0]);
  a.y[1] = view(ko, "k_out", q, s, a.H[1]);
  if (s.B * s.S == 0 || a.H[0] + a.H[1] == 0) return {qo, ko};
  const int blocks = rotary_blocks(a, false, at::cuda::getCurrentDeviceProperties()->multiProcessorCount);
  PCCL_CUDA(launch_rotary_forward(a, blocks, at::cuda::getCurrentCUDAStream().stream()));
  return {qo, ko};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> qk_norm_rope_backward(
    const at::Tensor& dq, const at::Tensor& dk, const at::Tensor& q, const at::Tensor& k, const at::Tensor& qw, const at::Tensor& kw,
    const at::Tensor& cos, const at::Tensor& sin, std::optional<at::Tensor> positions, double eps, bool interleaved,
    std::optional<at::Tensor> dq_in, std::optional<at::Tensor> dk_in, std::optional<at::Tensor> dqw_, std::optional<at::Tensor> dkw_) {
  RotaryArgs a;
  const Shape s = fill(a, q, k, qw, kw, cos, sin, positions, eps, interleaved);
  c10::cuda::CUDAGuard guard(q.device());
  a.dy[0] = view(dq, "dq", q, s, a.H[0]);
  a.dy[1] = view(dk, "dk", q, s, a.H[1]);
  at::Tensor qo = output(dq_in, q, "dq_in", {dq, q}, {dk, k}), ko = output(dk_in, k, "dk_in", {dk, k}, {dq, q});
  TORCH_CHECK(share(qo, ko) == Share::kNone, "dq_in and dk_in must not overlap");
  if (dq_in.has_value()) check_apart(qo, "dq_in", {qw, kw, cos, sin}, positions);
  if (dk_in.has_value()) check_apart(ko, "dk_in", {qw, kw, cos, sin}, positions);
  a.y[0] = view(qo, "dq_in", q, s, a.H[0]);
  a.y[1] = view(ko, "dk_in", q, s, a.H[1]);
  at::Tensor dqw = dqw_.has_value() ? *dqw_ : fresh(qw.sizes(), qw.scalar_type(), q), dkw = dkw_.has_value() ? *dkw_ : fresh(kw.sizes(), kw.scalar_type(), q);
  for (const at::Tensor* w : {&dqw, &dkw})
    TORCH_CHECK(w->is_cuda() && w->device() == q.device() && w->is_contiguous() && w->dim() == 1 && w->numel() == s.D &&
                    w->scalar_type() == qw.scalar_type(),
                "dq_weight and dk_weight must look like the weights");
  TORCH_CHECK(share(dqw, dkw) == Share::kNone, "dq_weight and dk_weight must not overlap");
  for (const at::Tensor* w : {&dqw, &dkw})
    TORCH_CHECK(share(*w, qo) == Share::kNone && share(*w, ko) == Share::kNone, "dq_weight and dk_weight must not overlap dq_in or dk_in");
  a.dw[0] = dqw.data_ptr();
  a.dw[1] = dkw.data_ptr();
  if (s.B * s.S == 0 || a.H[0] + a.H[1] == 0) {
    dqw.zero_();
    dkw.zero_();
    return {qo, ko, dqw, dkw};
  }
  const int blocks = rotary_blocks(a, true, at::cuda::getCurrentDeviceProperties()->multiProcessorCount);
  at::Tensor partial = fresh({(int64_t)blocks * s.D}, at::kFloat, q);
  a.partial = partial.data_ptr<float>();
  PCCL_CUDA(launch_rotary_backward(a, blocks, at::cuda::getCurrentCUDAStream().stream()));
  return {qo, ko, dqw, dkw};
}

}  // namespace

void bind_rotary(py::module_& m) {
  m.def("qk_norm_rope_forward", &qk_norm_rope_forward, py::arg("q"), py::arg("k"), py::arg("q_weight"), py::arg("k_weight"), py::arg("cos"),
        py::arg("sin"), py::arg("positions") = py::none(), py::arg("eps") = 1e-6, py::arg("interleaved") = false,
        py::arg("q_out") = py::none(), py::arg("k_out") = py::none(), "norm of each head and rotation: returns (q, k)");
  m.def("qk_norm_rope_backward", &qk_norm_rope_backward, py::arg("dq"), py::arg("dk"), py::arg("q"), py::arg("k"), py::arg("q_weight"),
        py::arg("k_weight"), py::arg("cos"), py::arg("sin"), py::arg("positions") = py::none(), py::arg("eps") = 1e-6,
        py::arg("interleaved") = false, py::arg("dq_in") = py::none(), py::arg("dk_in") = py::none(), py::arg("dq_weight") = py::none(),
        py::arg("dk_weight") = py::none(), "its gradients: returns (dq, dk, dq_weight, dk_weight)");
}
