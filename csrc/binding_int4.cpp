// Torch binding of the o_proj with 4-bit weights.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cstdlib>
#include <string>

#include "exchange.h"
#include "oproj_int4.h"

namespace {

// x [tokens, K]; packed uint8 (hidden * K / 2 bytes), scales [hidden / 16, K / group, 8, 2], zeros uint8 of that shape or none, as made
// by helix_a2a_b200.ops.oproj.pack_weight_int4
torch::Tensor oproj_int4(torch::Tensor x, torch::Tensor packed, torch::Tensor scales, const c10::optional<torch::Tensor>& zeros,
                         int64_t hidden, int64_t K, int64_t group) {
  TORCH_CHECK(x.is_cuda(), "inputs must be on CUDA");
  const torch::Device dev = x.device();
  TORCH_CHECK(packed.device() == dev && scales.device() == dev && (!zeros || zeros->device() == dev), "x and the weight must be on one device");
  const auto type = x.scalar_type();
  TORCH_CHECK((type == at::ScalarType::BFloat16 || type == at::ScalarType::Half) && scales.scalar_type() == type,
              "x and the scales must both be bfloat16 or both float16");
  TORCH_CHECK(group == 32 || group == 64 || group == 128, "group must be 32, 64 or 128");
  TORCH_CHECK(hidden > 0 && hidden % 16 == 0 && K > 0 && K % 64 == 0 && K % group == 0, "hidden must be a multiple of 16, K of 64 and of the group");
  TORCH_CHECK(K <= helix::kInt4MaxK && hidden <= 0x7fffffff, "K must be at most ", helix::kInt4MaxK);
  TORCH_CHECK(x.dim() == 2 && x.size(1) == K && x.stride(1) == 1, "x must be [tokens, K]");
  const int64_t tokens = x.size(0);
  TORCH_CHECK(tokens == 0 || (reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 && (tokens == 1 || x.stride(0) % 8 == 0)),
              "rows of x must start on 16-byte boundaries");
  TORCH_CHECK(packed.scalar_type() == at::ScalarType::Byte && packed.is_contiguous() && packed.numel() == hidden * K / 2 &&
                  reinterpret_cast<uintptr_t>(packed.data_ptr()) % 16 == 0,
              "packed weight has the wrong size or alignment for [", hidden, ", ", K, "]");
  TORCH_CHECK(scales.is_contiguous() && scales.numel() == hidden * (K / group) && reinterpret_cast<uintptr_t>(scales.data_ptr()) % 4 == 0,
              "scales have the wrong size or alignment");
  TORCH_CHECK(!zeros || (zeros->scalar_type() == at::ScalarType::Byte && zeros->is_contiguous() && zeros->numel() == scales.numel() &&
                         reinterpret_cast<uintptr_t>(zeros->data_ptr()) % 2 == 0),
              "zeros must be uint8 of the scales' size");
  c10::cuda::CUDAGuard guard(dev);
  auto stream = at::cuda::getCurrentCUDAStream();
  torch::Tensor y = torch::empty({tokens, hidden}, x.options());
  const char* v = std::getenv("HELIX_A2A_ENABLE_PDL");
  const bool pdl = v && std::string(v) == "1";
  for (int64_t t0 = 0; t0 < tokens; t0 += helix::kInt4MaxTokens) {
    helix::OprojInt4Params p{};
    p.x = reinterpret_cast<const uint16_t*>(x.data_ptr()) + t0 * x.stride(0);
    p.x_stride = x.stride(0);
    p.w = reinterpret_cast<const uint4*>(packed.data_ptr());
    p.scales = reinterpret_cast<const uint32_t*>(scales.data_ptr());
    p.zeros = zeros ? reinterpret_cast<const uint16_t*>(zeros->data_ptr()) : nullptr;
    p.y = reinterpret_cast<uint16_t*>(y.data_ptr()) + t0 * hidden;
    p.y_stride = hidden;
    p.tokens = (int)std::min<int64_t>(tokens - t0, helix::kInt4MaxTokens);
    p.hidden = (int)hidden; p.K = (int)K; p.group = (int)group;
    p.is_bf16 = type == at::ScalarType::BFloat16;
    const cudaError_t e = helix::launch_oproj_int4(p, pdl, helix::device_sm_count(), stream);
    TORCH_CHECK(e == cudaSuccess, "helix: o_proj (4-bit) launch failed: ", cudaGetErrorString(e));
  }
  return y;
}

}  // namespace

void register_int4_ops(torch::Library& m) {
  m.def("oproj_int4(Tensor x, Tensor packed, Tensor scales, Tensor? zeros, int hidden, int K, int group) -> Tensor", &oproj_int4);
}
