// What the bindings of the paged caches check and convert alike.
#pragma once
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <string>

#include "bindings.h"
#include "kernels.h"

namespace {

// Messages are put together as plain strings: c10's own, which goes by a stream as soon as it has more than one part, ends the process here.
#define CHECK_ARG(cond, msg) TORCH_CHECK_VALUE(cond, std::string(msg))

std::string list(at::IntArrayRef sizes) {
  std::string s = "[";
  for (size_t i = 0; i < sizes.size(); ++i) s += (i ? ", " : "") + std::to_string(sizes[i]);
  return s + "]";
}

int dt_code(const Tensor& t) { return t.scalar_type() == at::kFloat ? nxd::kF32 : t.scalar_type() == at::kBFloat16 ? nxd::kBF16 : nxd::kF16; }
bool half_type(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }
cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }

// Last dimension contiguous, everything else whole 16-byte packets apart, and so the address
bool packets(const Tensor& t) {
  const int64_t per = 16 / t.element_size();
  bool ok = t.stride(-1) == 1 && (uintptr_t)t.data_ptr() % 16 == 0 && t.size(-1) % per == 0;
  for (int64_t d = 0; d + 1 < t.dim(); ++d) ok = ok && (t.size(d) <= 1 || t.stride(d) % per == 0);
  return ok;
}
Tensor as_packets(const Tensor& t) { return packets(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

void check_ints(const Tensor& t, const char* name, at::ScalarType type, int64_t n, const Tensor& like) {
  CHECK_ARG(t.scalar_type() == type && t.dim() == 1 && t.size(0) == n && t.is_contiguous() && t.device() == like.device(),
            std::string(name) + " must be a contiguous " + c10::toString(type) + " tensor of " + std::to_string(n) + " numbers on the queries' device");
}

// Numbers of another type, or not one after the other, are converted
Tensor ints(const Tensor& t, at::ScalarType type) { return t.scalar_type() == type && t.is_contiguous() ? t : t.to(type).contiguous(); }
c10::optional<Tensor> ints(const c10::optional<Tensor>& t, at::ScalarType type) { return t.has_value() ? c10::optional<Tensor>(ints(*t, type)) : t; }
Tensor as_table(const Tensor& t) {
  return t.scalar_type() == at::kInt && (t.dim() != 2 || t.size(1) <= 1 || t.stride(1) == 1) ? t : t.to(at::kInt).contiguous();
}

// Memory of a GPU without a walk through the dispatcher, which costs these calls 0.5 us of 7 for each tensor that they return
Tensor empty_on(at::IntArrayRef sizes, at::ScalarType type, const at::Device& device) { return Tensor(at::detail::empty_cuda(sizes, type, device, c10::nullopt)); }

// [B, W, H, D] with tokens first in memory, as the layers around take and leave it
Tensor rows_out(const Tensor& q) {
  const int64_t B = q.size(0), W = q.size(1), H = q.size(2), D = q.size(3);
  return Tensor(at::detail::empty_strided_cuda({B, W, H, D}, {H * D, B * H * D, D, 1}, q.scalar_type(), q.device()));
}

}  // namespace
