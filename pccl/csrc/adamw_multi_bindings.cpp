// Python bindings of AdamW over a list of tensors.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <pybind11/stl.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <tuple>
#include <vector>

#include "adamw_multi.h"
#include "comm.h"

namespace py = pybind11;
using namespace pccl;

namespace {

int type_of(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return kAdamBf16;
    case at::kHalf: return kAdamF16;
    case at::kFloat: return kAdamF32;
    default: TORCH_CHECK(false, name, " must be bfloat16, float16 or float32");
  }
}

struct Range {
  uintptr_t lo, hi;
  bool written;
};
void add_range(std::vector<Range>& r, const at::Tensor& t, bool written) {
  if (t.numel() == 0) return;
  const uintptr_t lo = reinterpret_cast<uintptr_t>(t.data_ptr());
  r.push_back({lo, lo + t.nbytes(), written});
}

// The state: fp32 m and v, or codes with their scales.
bool check_state(const at::Tensor& m, const at::Tensor& v, const std::optional<at::Tensor>& ms, const std::optional<at::Tensor>& vs,
                 const c10::Device& device) {
  const bool bits8 = ms.has_value() || vs.has_value();
  TORCH_CHECK(ms.has_value() == vs.has_value(), "8-bit states have a scale tensor each");
  TORCH_CHECK(m.is_cuda() && m.device() == device && v.device() == device && m.is_contiguous() && v.is_contiguous() && m.dim() == 1 && v.dim() == 1,
              "the states must be contiguous 1-D CUDA tensors on the device of the parameters");
  TORCH_CHECK(m.numel() == v.numel() && m.numel() % kAdamBlock == 0, "the states must hold as many elements as each other, a multiple of ", kAdamBlock);
  TORCH_CHECK(((reinterpret_cast<uintptr_t>(m.data_ptr()) | reinterpret_cast<uintptr_t>(v.data_ptr())) & 31u) == 0,
              "the states must start on 32-byte boundaries");
  if (bits8) {
    TORCH_CHECK(m.scalar_type() == at::kChar && v.scalar_type() == at::kByte, "8-bit states: exp_avg is int8, exp_avg_sq uint8");
    for (const at::Tensor* t : {&*ms, &*vs})
      TORCH_CHECK(t->is_cuda() && t->device() == device && t->is_contiguous() && t->scalar_type() == at::kFloat && t->dim() == 1 &&
                      t->numel() == m.numel() / kAdamBlock,
                  "8-bit states: a float32 scale for every ", kAdamBlock, " elements");
  } else {
    TORCH_CHECK(m.scalar_type() == at::kFloat && v.scalar_type() == at::kFloat, "states without scales are float32");
  }
  return bits8;
}

void adamw_multi(const std::vector<at::Tensor>& params, const std::vector<at::Tensor>& grads,
                 const std::optional<std::vector<at::Tensor>>& masters, at::Tensor& m, at::Tensor& v, std::optional<at::Tensor> m_scale,
                 std::optional<at::Tensor> v_scale, const std::vector<double>& decay, int64_t step, double lr, double beta1, double beta2,
                 double eps, double grad_scale, double max_grad_norm, std::optional<at::Tensor> total_sq_norm, uint64_t seed) {
  const size_t n = params.size();
  TORCH_CHECK(grads.size() == n && (!masters.has_value() || masters->size() == n), "as many gradients (and masters) as parameters are needed");
  TORCH_CHECK(decay.size() == n || decay.size() == 1, "weight_decay: one number, or one for each parameter");
  TORCH_CHECK(step >= 1, "step counts from 1");
  TORCH_CHECK(std::isfinite(lr) && beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0 && std::isfinite(eps),
              "lr and eps must be finite, eps not negative, beta1 and beta2 in [0, 1)");
  TORCH_CHECK(!std::isnan(max_grad_norm), "max_grad_norm must be a number: NaN would switch clipping off");
  TORCH_CHECK(!(m_scale.has_value() || v_scale.has_value()) || eps >= adamw_least_eps(beta2), "8-bit states need an eps of at least ",
              adamw_least_eps(beta2), " at this beta2: they hold second moments below 2^-80 as zeros");
  if (n == 0) return;
  const c10::Device device = params[0].device();
  const int pt = type_of(params[0], "a parameter"), gt = type_of(grads[0], "a gradient");
  TORCH_CHECK(masters.has_value() == (pt != kAdamF32), "16-bit parameters need a float32 master each, float32 parameters have none");
  const bool bits8 = check_state(m, v, m_scale, v_scale, device);
  std::vector<AdamTensor> table;
  std::vector<uint64_t> blocks;            // of each entry
  std::vector<Range> ranges;
  table.reserve(n);
  blocks.reserve(n);
  ranges.reserve(3 * n + 5);
  uint64_t total = 0;
  for (size_t i = 0; i < n; ++i) {
    const at::Tensor &p = params[i], &g = grads[i];
    TORCH_CHECK(p.is_cuda() && p.device() == device && g.device() == device && p.is_contiguous() && g.is_contiguous() && p.numel() == g.numel(),
                "parameter ", i, ": parameter and gradient must be contiguous CUDA tensors of one size, all on one device");
    TORCH_CHECK(p.scalar_type() == params[0].scalar_type() && g.scalar_type() == grads[0].scalar_type(),
                "parameter ", i, ": all parameters must have one dtype, all gradients one");
    AdamTensor t;
    t.param = p.data_ptr();
    t.master = nullptr;
    t.grad = g.data_ptr();
    t.n = p.numel();
    t.decay = (float)(decay.size() == 1 ? decay[0] : decay[i]);
    t.first = 0;
    add_range(ranges, p, true);
    add_range(ranges, g, false);
    if (masters.has_value()) {
      const at::Tensor& w = (*masters)[i];
      TORCH_CHECK(w.is_cuda() && w.device() == device && w.is_contiguous() && w.scalar_type() == at::kFloat && w.numel() == t.n, "parameter ", i,
                  ": its master must be a contiguous float32 CUDA tensor of its size");
      t.master = w.data_ptr<float>();
      add_range(ranges, w, true);
    }
    const uint64_t nb = ((uint64_t)t.n + kAdamBlock - 1) / kAdamBlock;
    if (nb == 0) continue;
    table.push_back(t);
    blocks.push_back(nb);
    total += nb;
  }
  TORCH_CHECK(total * kAdamBlock == (uint64_t)m.numel(), "the states hold ", m.numel(), " elements, these parameters need ", total * kAdamBlock);
  TORCH_CHECK(total < ((uint64_t)1 << 32), "too many parameters for one call");
  if (max_grad_norm > 0) {
    TORCH_CHECK(total_sq_norm.has_value(), "max_grad_norm needs total_sq_norm");
    TORCH_CHECK(total_sq_norm->device() == device && total_sq_norm->scalar_type() == at::kFloat && total_sq_norm->numel() == 1,
                "total_sq_norm must hold one float32 on the device of the parameters");
    add_range(ranges, *total_sq_norm, false);
  }
  // two blocks of the grid that update the same memory would race, and every block reads the norm
  for (const at::Tensor* t : {static_cast<const at::Tensor*>(&m), static_cast<const at::Tensor*>(&v)}) add_range(ranges, *t, true);
  if (bits8) {
    add_range(ranges, *m_scale, true);
    add_range(ranges, *v_scale, true);
  }
  std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; });
  uintptr_t end_any = 0, end_written = 0;
  for (const Range& r : ranges) {
    TORCH_CHECK(r.lo >= (r.written ? end_any : end_written), "a tensor that the step writes overlaps another one of the call");
    end_any = std::max(end_any, r.hi);
    if (r.written) end_written = std::max(end_written, r.hi);
  }
  AdamMultiArgs a;
  a.m = m.data_ptr();
  a.v = v.data_ptr();
  a.m_scale = bits8 ? m_scale->data_ptr<float>() : nullptr;
  a.v_scale = bits8 ? v_scale->data_ptr<float>() : nullptr;
  a.key = adamw_noise_key(seed, step);
  a.lr = (float)lr;
  a.beta1 = (float)beta1;
  a.beta2 = (float)beta2;
  a.one_minus_beta1 = (float)(1.0 - beta1);
  a.one_minus_beta2 = (float)(1.0 - beta2);
  a.eps = (float)eps;
  a.bias1 = (float)(1.0 / (1.0 - std::pow(beta1, (double)step)));
  a.bias2 = (float)(1.0 / (1.0 - std::pow(beta2, (double)step)));
  a.grad_scale = (float)grad_scale;
  a.max_grad_norm = (float)max_grad_norm;
  a.total_sq_norm = max_grad_norm > 0 ? total_sq_norm->data_ptr<float>() : nullptr;
  c10::cuda::CUDAGuard guard(device);
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  uint64_t first = 0;
  for (size_t i = 0; i < table.size(); i += kAdamTensors) {
    const size_t count = std::min<size_t>(kAdamTensors, table.size() - i);
    uint64_t here = 0;
    for (size_t j = i; j < i + count; ++j) {
      table[j].first = (uint32_t)here;
      here += blocks[j];
    }
    a.first_block = first;
    a.blocks = (uint32_t)here;
    PCCL_CUDA(launch_adamw_multi(a, table.data() + i, (int)count, pt, gt, bits8, sms, stream));
    first += here;
  }
}

std::tuple<at::Tensor, at::Tensor> adamw_dequantize(const at::Tensor& m, const at::Tensor& v, const at::Tensor& m_scale, const at::Tensor& v_scale) {
  TORCH_CHECK(m.is_cuda(), "the states must be CUDA tensors");
  check_state(m, v, m_scale, v_scale, m.device());
  c10::cuda::CUDAGuard guard(m.device());
  at::Tensor mo = at::empty({m.numel()}, m.options().dtype(at::kFloat)), vo = at::empty({m.numel()}, m.options().dtype(at::kFloat));
  PCCL_CUDA(launch_adamw_dequantize(m.data_ptr<int8_t>(), m_scale.data_ptr<float>(), v.data_ptr<uint8_t>(), v_scale.data_ptr<float>(),
                                    mo.data_ptr<float>(), vo.data_ptr<float>(), m.numel(), at::cuda::getCurrentCUDAStream().stream()));
  return {mo, vo};
}

}  // namespace

void bind_adamw_multi(py::module_& m) {
  m.attr("adamw_block") = kAdamBlock;
  m.def("adamw_least_eps", &adamw_least_eps, py::arg("beta2"), "the smallest eps that 8-bit states take");
  m.def("adamw_multi", &adamw_multi, py::arg("params"), py::arg("grads"), py::arg("masters"), py::arg("exp_avg"), py::arg("exp_avg_sq"),
        py::arg("exp_avg_scale"), py::arg("exp_avg_sq_scale"), py::arg("weight_decay"), py::arg("step"), py::arg("lr"), py::arg("beta1"),
        py::arg("beta2"), py::arg("eps"), py::arg("grad_scale") = 1.0, py::arg("max_grad_norm") = 0.0,
        py::arg("total_sq_norm") = py::none(), py::arg("seed") = 0, "one AdamW step over a list of tensors");
  m.def("adamw_dequantize", &adamw_dequantize, py::arg("exp_avg"), py::arg("exp_avg_sq"), py::arg("exp_avg_scale"),
        py::arg("exp_avg_sq_scale"), "the values that 8-bit states stand for, in fp32");
}
