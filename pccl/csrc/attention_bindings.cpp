// Python bindings of attention.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <atomic>
#include <cmath>
#include <cstring>
#include <mutex>
#include <optional>
#include <tuple>

#include "attention.h"
#include "comm.h"
#include "fresh.h"
#include "overlap.h"

namespace py = pybind11;
using namespace pccl;

namespace {

// One word per device, in host memory that the device can write: 0 until a bounded wait of some launch runs out.  It is
// allocated outside of any capture's rules, because the first call of a process may be a captured one.
volatile int* error_word(int device) {
  static int* words = nullptr;
  static std::once_flag once;
  TORCH_CHECK(device >= 0 && device < 64, "device number out of range");
  std::call_once(once, [] {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    PCCL_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
    void* p = nullptr;
    const cudaError_t e = cudaHostAlloc(&p, 64 * sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable);
    const cudaError_t back = cudaThreadExchangeStreamCaptureMode(&mode);
    PCCL_CUDA(e);
    PCCL_CUDA(back);
    std::memset(p, 0, 64 * sizeof(int));
    words = static_cast<int*>(p);
  });
  return words + device;
}

std::atomic<int64_t> g_kernels{0};         // launched since the process began

struct Shape {
  bool packed;
  int64_t B, Sq, Sk, H, Hk, D;
};

AttnTensor view(const at::Tensor& t, const char* name, const at::Tensor& like, int64_t B, int64_t S, int64_t H, int64_t D) {
  const bool packed = t.dim() == 3;
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be a CUDA tensor on the device of q");
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, " must have the dtype of q");
  TORCH_CHECK(t.dim() == like.dim() && t.size(-1) == D && t.size(-2) == H && t.size(-3) == S && (packed || t.size(0) == B), name,
              " has the wrong shape");
  AttnTensor v;
  v.p = t.data_ptr();
  v.sb = packed ? 0 : t.stride(0);
  v.ss = t.stride(-3);
  v.sh = t.stride(-2);
  if (t.numel() == 0) return v;
  TORCH_CHECK(t.stride(-1) == 1, "the last dimension of ", name, " must be contiguous");
  TORCH_CHECK((reinterpret_cast<uintptr_t>(v.p) & 15u) == 0, name, " must start on a 16-byte boundary");
  auto fits = [](int64_t n, int64_t stride) { return n <= 1 || (stride > 0 && stride % 8 == 0 && stride < ((int64_t)1 << 38)); };
  TORCH_CHECK(fits(S, v.ss) && fits(H, v.sh) && (packed || fits(B, v.sb)), "the strides of ", name,
              " must be positive multiples of 8 elements (an expanded dimension is not one)");
  return v;
}

void check_cu(const at::Tensor& t, const char* name, const at::Tensor& q) {
  TORCH_CHECK(t.is_cuda() && t.device() == q.device() && t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() && t.numel() >= 2,
              name, " must be a contiguous 1-D int32 tensor of at least two starts, on the device of q");
  TORCH_CHECK(t.numel() <= (1 << 24), name, " names too many sequences");
}

// Fills in what both passes share and returns the shape.
Shape fill(AttnArgs& a, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, bool causal, std::optional<double> scale,
           const std::optional<at::Tensor>& cu_q, const std::optional<at::Tensor>& cu_k) {
  std::memset(&a, 0, sizeof(a));
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf, "q must be bfloat16 or float16");
  Shape s;
  s.packed = cu_q.has_value();
  TORCH_CHECK(s.packed || !cu_k.has_value(), "cu_seqlens_k needs cu_seqlens_q");
  TORCH_CHECK(q.dim() == (s.packed ? 3 : 4), s.packed ? "packed sequences: q must be [rows, heads, dim]" : "q must be [batch, rows, heads, dim]");
  TORCH_CHECK(k.dim() == q.dim(), "k must have as many dimensions as q");
  s.B = s.packed ? 1 : q.size(0);
  s.Sq = q.size(-3);
  s.Sk = k.size(-3);
  s.H = q.size(-2);
  s.Hk = k.size(-2);
  s.D = q.size(-1);
  TORCH_CHECK(s.D >= 8 && s.D <= kAttnMaxDim && s.D % 8 == 0, "the head size must be a multiple of 8 up to ", kAttnMaxDim);
  TORCH_CHECK(s.H > 0 && s.Hk > 0 && s.H % s.Hk == 0, "the number of query heads must be a multiple of that of key heads");
  TORCH_CHECK(s.Sq < (1 << 30) && s.Sk < (1 << 30) && s.H <= 65535 && s.B < (1 << 24), "too many rows, heads or batch entries");
  a.q = view(q, "q", q, s.B, s.Sq, s.H, s.D);
  a.k = view(k, "k", q, s.B, s.Sk, s.Hk, s.D);
  a.v = view(v, "v", q, s.B, s.Sk, s.Hk, s.D);
  a.is_bf16 = q.scalar_type() == at::kBFloat16;
  a.B = (int)s.B;
  a.H = (int)s.H;
  a.Hk = (int)s.Hk;
  a.D = (int)s.D;
  a.Sq = (int)s.Sq;
  a.Sk = (int)s.Sk;
  if (s.packed) {
    check_cu(*cu_q, "cu_seqlens_q", q);
    a.cu_q = cu_q->data_ptr<int>();
    a.nseq = (int)cu_q->numel() - 1;
    if (cu_k.has_value()) {
      check_cu(*cu_k, "cu_seqlens_k", q);
      TORCH_CHECK(cu_k->numel() == cu_q->numel(), "cu_seqlens_q and cu_seqlens_k must name equally many sequences");
      a.cu_k = cu_k->data_ptr<int>();
    } else {
      TORCH_CHECK(s.Sq == s.Sk, "cu_seqlens_k may be left out only where k has as many rows as q");
      a.cu_k = a.cu_q;
    }
  }
  a.causal = causal;
  const double sc = scale.has_value() ? *scale : 1.0 / std::sqrt((double)s.D);
  TORCH_CHECK(std::isfinite(sc) && sc > 0 && (float)sc > 1e-30f && (float)sc < 1e30f, "scale must be positive and finite");
  a.scale = (float)sc;
  a.error = const_cast<int*>(error_word(q.get_device()));
  return s;
}

// An output: the caller's tensor, or a new one.
at::Tensor output(const std::optional<at::Tensor>& given, const at::Tensor& like, const char* name, std::initializer_list<at::Tensor> inputs,
                  const std::optional<at::Tensor>& cu_q, const std::optional<at::Tensor>& cu_k) {
  if (!given.has_value()) return fresh(like.sizes(), like.scalar_type(), like);
  TORCH_CHECK(distinct(*given), name, " must not overlap itself");
  for (const at::Tensor& t : inputs) TORCH_CHECK(share(*given, t) == Share::kNone, name, " must not overlap an input");
  for (const std::optional<at::Tensor>* t : {&cu_q, &cu_k})
    TORCH_CHECK(!t->has_value() || share(*given, **t) == Share::kNone, name, " must not overlap the starts of the sequences");
  return *given;
}

std::tuple<at::Tensor, at::Tensor> attention_forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, bool causal,
                                                     std::optional<double> scale, std::optional<at::Tensor> cu_q,
                                                     std::optional<at::Tensor> cu_k, std::optional<at::Tensor> out_) {
  AttnArgs a;
  const Shape s = fill(a, q, k, v, causal, scale, cu_q, cu_k);
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor out = output(out_, q, "out", {q, k, v}, cu_q, cu_k);
  a.o = view(out, "out", q, s.B, s.Sq, s.H, s.D);
  at::Tensor lse = s.packed ? fresh({s.H, s.Sq}, at::kFloat, q) : fresh({s.B, s.H, s.Sq}, at::kFloat, q);
  a.lse = lse.data_ptr<float>();
  a.zero_tail = !out_.has_value();
  const AttnScratch need = plan_attention_forward(a, at::cuda::getCurrentDeviceProperties()->multiProcessorCount);
  at::Tensor partial, partial_lse, order;
  if (need.order_q > 0) {
    order = fresh({2 * need.order_q}, at::kInt, q);
    a.order_q = reinterpret_cast<int2*>(order.data_ptr<int>());
  }
  if (need.partial > 0) {
    partial = fresh({need.partial}, at::kFloat, q);
    partial_lse = fresh({need.partial_lse}, at::kFloat, q);
    a.partial = partial.data_ptr<float>();
    a.partial_lse = partial_lse.data_ptr<float>();
  }
  int64_t kernels = 0;
  const cudaError_t e = launch_attention_forward(a, at::cuda::getCurrentCUDAStream().stream(), kernels);
  g_kernels += kernels;
  PCCL_CUDA(e);
  return {out, lse};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> attention_backward(const at::Tensor& dout, const at::Tensor& q, const at::Tensor& k,
                                                                  const at::Tensor& v, const at::Tensor& out, const at::Tensor& lse,
                                                                  bool causal, std::optional<double> scale,
                                                                  std::optional<at::Tensor> cu_q, std::optional<at::Tensor> cu_k,
                                                                  std::optional<at::Tensor> dq_, std::optional<at::Tensor> dk_,
                                                                  std::optional<at::Tensor> dv_) {
  AttnArgs a;
  const Shape s = fill(a, q, k, v, causal, scale, cu_q, cu_k);
  c10::cuda::CUDAGuard guard(q.device());
  a.dout = view(dout, "dout", q, s.B, s.Sq, s.H, s.D);
  a.o = view(out, "out", q, s.B, s.Sq, s.H, s.D);
  TORCH_CHECK(lse.is_cuda() && lse.device() == q.device() && lse.scalar_type() == at::kFloat && lse.is_contiguous() &&
                  lse.dim() == (s.packed ? 2 : 3) && lse.size(-1) == s.Sq && lse.size(-2) == s.H && (s.packed || lse.size(0) == s.B),
              "lse must be what the forward pass returned");
  TORCH_CHECK(dq_.has_value() == dk_.has_value() && dq_.has_value() == dv_.has_value(), "dq, dk and dv are given together or not at all");
  const std::initializer_list<at::Tensor> inputs = {dout, q, k, v, out, lse};
  at::Tensor dq = output(dq_, q, "dq", inputs, cu_q, cu_k), dk = output(dk_, k, "dk", inputs, cu_q, cu_k),
             dv = output(dv_, v, "dv", inputs, cu_q, cu_k);
  TORCH_CHECK(share(dq, dk) == Share::kNone && share(dq, dv) == Share::kNone && share(dk, dv) == Share::kNone,
              "dq, dk and dv must not overlap each other");
  TORCH_CHECK(s.B <= 65535, "the backward pass takes up to 65535 batch entries");
  a.dq = view(dq, "dq", q, s.B, s.Sq, s.H, s.D);
  a.dk = view(dk, "dk", q, s.B, s.Sk, s.Hk, s.D);
  a.dv = view(dv, "dv", q, s.B, s.Sk, s.Hk, s.D);
  a.lse = lse.data_ptr<float>();
  at::Tensor delta = fresh(lse.sizes(), at::kFloat, q);
  a.delta = delta.data_ptr<float>();
  a.zero_tail = !dq_.has_value();
  const AttnScratch need = plan_attention_backward(a, at::cuda::getCurrentDeviceProperties()->multiProcessorCount);
  at::Tensor partial, order;
  if (need.order_q > 0) {
    order = fresh({2 * (need.order_q + need.order_k)}, at::kInt, q);
    a.order_q = reinterpret_cast<int2*>(order.data_ptr<int>());
    a.order_k = a.order_q + need.order_q;
  }
  if (need.partial > 0) {
    partial = fresh({need.partial}, at::kFloat, q);
    a.partial = partial.data_ptr<float>();
  }
  int64_t kernels = 0;
  const cudaError_t e = launch_attention_backward(a, at::cuda::getCurrentCUDAStream().stream(), kernels);
  g_kernels += kernels;
  PCCL_CUDA(e);
  return {dq, dk, dv};
}

}  // namespace

void bind_attention(py::module_& m) {
  m.def("attention_forward", &attention_forward, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("causal") = true,
        py::arg("scale") = py::none(), py::arg("cu_seqlens_q") = py::none(), py::arg("cu_seqlens_k") = py::none(),
        py::arg("out") = py::none(), "softmax(scale q k^T) v: returns (out, lse)");
  m.def("attention_backward", &attention_backward, py::arg("dout"), py::arg("q"), py::arg("k"), py::arg("v"), py::arg("out"), py::arg("lse"),
        py::arg("causal") = true, py::arg("scale") = py::none(), py::arg("cu_seqlens_q") = py::none(),
        py::arg("cu_seqlens_k") = py::none(), py::arg("dq") = py::none(), py::arg("dk") = py::none(), py::arg("dv") = py::none(),
        "gradients of attention: returns (dq, dk, dv)");
  m.def("attention_kernels_launched", [] { return g_kernels.load(); }, "kernels of attention launched since the process began");
  m.def("attention_error", [](int device) { return (int)*error_word(device); }, "0, or why a bounded wait of an attention kernel gave up");
  m.def("attention_reset_error", [](int device) { *error_word(device) = 0; });
}
