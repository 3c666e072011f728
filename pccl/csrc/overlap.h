// Whether strided tensors share memory, for the checks of outputs.
#pragma once
#include <ATen/core/Tensor.h>

#include <algorithm>
#include <cstdint>
#include <vector>

namespace pccl {

enum class Share { kNone, kSame, kSome };

namespace overlap {

struct Dim {
  int64_t stride, low, high;        // difference of two indexes along this dimension: low <= i - j <= high
};

// Whether the sum of difference * stride can be `delta`; dims from the largest stride down.  Where the strides nest, two or three
// differences are possible at each level; where they do not and many are, the answer is the cautious one.
inline bool reaches(const std::vector<Dim>& dims, size_t at, int64_t delta) {
  if (at == dims.size()) return delta == 0;
  int64_t low = 0, high = 0;
  for (size_t i = at + 1; i < dims.size(); ++i) low += dims[i].low * dims[i].stride, high += dims[i].high * dims[i].stride;
  const int64_t s = dims[at].stride;
  auto down = [s](int64_t x) { return x >= 0 ? x / s : -((-x + s - 1) / s); };
  const int64_t first = std::max(dims[at].low, -down(high - delta)), last = std::min(dims[at].high, down(delta - low));
  if (last - first >= 8) return true;
  for (int64_t d = first; d <= last; ++d)
    if (reaches(dims, at + 1, delta - d * s)) return true;
  return false;
}

}  // namespace overlap

// kSame: one and the same elements in the same order.  Two views of equal strides (parts of a packed projection) are compared
// exactly; others that lie in one another's range count as sharing.
inline Share share(const at::Tensor& a, const at::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return Share::kNone;
  auto span = [](const at::Tensor& t) {
    int64_t n = 1;
    for (int64_t i = 0; i < t.dim(); ++i) n += (t.size(i) - 1) * t.stride(i);
    return n * t.element_size();
  };
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.data_ptr()), pb = reinterpret_cast<uintptr_t>(b.data_ptr());
  if (pa + (uintptr_t)span(a) <= pb || pb + (uintptr_t)span(b) <= pa) return Share::kNone;
  if (a.dim() != b.dim() || a.element_size() != b.element_size() || (pa > pb ? pa - pb : pb - pa) % (uintptr_t)a.element_size() != 0)
    return Share::kSome;
  bool same = pa == pb;
  std::vector<overlap::Dim> dims;
  for (int64_t i = 0; i < a.dim(); ++i) {
    same = same && a.size(i) == b.size(i);
    if (a.size(i) > 1 && b.size(i) > 1 && a.stride(i) != b.stride(i)) return Share::kSome;
    const int64_t s = a.size(i) > 1 ? a.stride(i) : b.stride(i);
    if ((a.size(i) > 1 || b.size(i) > 1) && s > 0) dims.push_back({s, -(b.size(i) - 1), a.size(i) - 1});
  }
  if (same) return Share::kSame;
  std::sort(dims.begin(), dims.end(), [](const overlap::Dim& x, const overlap::Dim& y) { return x.stride > y.stride; });
  const int64_t delta = ((int64_t)pb - (int64_t)pa) / (int64_t)a.element_size();
  return overlap::reaches(dims, 0, delta) ? Share::kSome : Share::kNone;
}

// Whether no two elements of a tensor lie on one another: each stride steps over all that smaller strides reach.
inline bool distinct(const at::Tensor& t) {
  std::vector<std::pair<int64_t, int64_t>> dims;
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1) dims.emplace_back(t.stride(i), t.size(i));
  std::sort(dims.begin(), dims.end());
  int64_t reach = 0;
  for (const auto& [stride, size] : dims) {
    if (stride <= reach) return false;
    reach += stride * (size - 1);
  }
  return true;
}

}  // namespace pccl
