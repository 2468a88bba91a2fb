// Products grouped by expert (bf16, both gradients, block-scaled e4m3) and the
// dense block-scaled e4m3 products, which are the same with a single group.
#include "gemm_grouped_simt.cuh"

namespace {

using col::simt::GroupedSimtParams;

constexpr std::uint64_t kIntMax = 0x7fffffffull;

// Sizes every entry point shares: rows and widths below 2^31 (rounded up to
// whole tiles), at most kMaxGroups groups.
inline bool sizes_ok(std::uint64_t rows, std::uint64_t k, std::uint64_t columns,
                     std::uint64_t groups) {
  return rows <= kIntMax - 1024 && k != 0 && k <= kIntMax - 1024 && columns <= kIntMax - 1024 &&
         groups <= static_cast<std::uint64_t>(col::kMaxGroups);
}

GroupedSimtParams simt_params(const void* a, const void* b, const std::int32_t* offsets, void* out,
                              std::uint64_t rows, std::uint64_t k, std::uint64_t n,
                              std::uint64_t w_rows, std::uint64_t groups) {
  GroupedSimtParams p = {};
  p.a = a;
  p.b = b;
  p.offsets = offsets;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.rows = static_cast<int>(rows);
  p.k = static_cast<int>(k);
  p.n = static_cast<int>(n);
  p.w_rows = static_cast<int>(w_rows);
  p.groups = static_cast<int>(groups);
  return p;
}

template <bool SWIGLU>
int grouped_forward_bf16(const void* x, const void* w, const std::int32_t* offsets, void* out,
                         std::uint64_t t, std::uint64_t k, std::uint64_t n, std::uint64_t experts,
                         void* stream) {
  if (t == 0 || n == 0 || experts == 0) return 0;
  const std::uint64_t w_rows = SWIGLU ? 2 * n : n;
  if (!x || !w || !offsets || !out || !sizes_ok(t, k, n, experts) || w_rows > kIntMax - 1024) {
    return static_cast<int>(cudaErrorInvalidValue);
  }
  const GroupedSimtParams p = simt_params(x, w, offsets, out, t, k, n, w_rows, experts);
  return col::simt::launch_grouped_simt<__nv_bfloat16, col::simt::kForward, SWIGLU>(
      p, col::as_stream(stream));
}

template <bool SWIGLU>
int forward_fp8(const void* x, const float* xs, const void* w, const float* ws,
                const std::int32_t* offsets, void* out, std::uint64_t t, std::uint64_t k,
                std::uint64_t n, std::uint64_t experts, void* stream) {
  const std::uint64_t w_rows = SWIGLU ? 2 * n : n;
  if (!x || !xs || !w || !ws || !out || !sizes_ok(t, k, n, experts) || w_rows > kIntMax - 1024) {
    return static_cast<int>(cudaErrorInvalidValue);
  }
  // A tile of scales must not span gate and up rows.
  if (SWIGLU && n % 128 != 0) return static_cast<int>(cudaErrorInvalidValue);
  GroupedSimtParams p = simt_params(x, w, offsets, out, t, k, n, w_rows, experts);
  p.a_scale = xs;
  p.b_scale = ws;
  return col::simt::launch_grouped_simt<__nv_fp8_e4m3, col::simt::kForward, SWIGLU>(
      p, col::as_stream(stream));
}

}  // namespace

COL_API int cuda_operator_gemm_grouped_bf16(const void* input_bf16, const void* weight_bf16,
                                            const int32_t* offsets, void* output_bf16, uint64_t t,
                                            uint64_t k, uint64_t n, uint64_t experts,
                                            void* stream) {
  return grouped_forward_bf16<false>(input_bf16, weight_bf16, offsets, output_bf16, t, k, n,
                                     experts, stream);
}

COL_API int cuda_operator_gemm_grouped_swiglu_bf16(const void* input_bf16,
                                                   const void* packed_weight_bf16,
                                                   const int32_t* offsets, void* output_bf16,
                                                   uint64_t t, uint64_t k, uint64_t n,
                                                   uint64_t experts, void* stream) {
  return grouped_forward_bf16<true>(input_bf16, packed_weight_bf16, offsets, output_bf16, t, k, n,
                                    experts, stream);
}

COL_API int cuda_operator_gemm_grouped_bf16_grad_input(const void* grad_bf16,
                                                       const void* weight_bf16,
                                                       const int32_t* offsets,
                                                       void* grad_input_bf16, uint64_t t,
                                                       uint64_t k, uint64_t n, uint64_t experts,
                                                       void* stream) {
  if (t == 0 || k == 0 || experts == 0) return 0;
  if (!grad_bf16 || !weight_bf16 || !offsets || !grad_input_bf16 || n == 0 ||
      !sizes_ok(t, k, n, experts)) {
    return static_cast<int>(cudaErrorInvalidValue);
  }
  const GroupedSimtParams p =
      simt_params(grad_bf16, weight_bf16, offsets, grad_input_bf16, t, k, n, n, experts);
  return col::simt::launch_grouped_simt<__nv_bfloat16, col::simt::kGradX, false>(
      p, col::as_stream(stream));
}

COL_API int cuda_operator_gemm_grouped_bf16_grad_weight(const void* grad_bf16,
                                                        const void* input_bf16,
                                                        const int32_t* offsets,
                                                        void* grad_weight_bf16, uint64_t t,
                                                        uint64_t k, uint64_t n, uint64_t experts,
                                                        void* stream) {
  if (k == 0 || n == 0 || experts == 0) return 0;
  if (!offsets || !grad_weight_bf16 || (t != 0 && (!grad_bf16 || !input_bf16)) ||
      !sizes_ok(t, k, n, experts)) {
    return static_cast<int>(cudaErrorInvalidValue);
  }
  const GroupedSimtParams p =
      simt_params(grad_bf16, input_bf16, offsets, grad_weight_bf16, t, k, n, n, experts);
  return col::simt::launch_grouped_simt<__nv_bfloat16, col::simt::kGradW, false>(
      p, col::as_stream(stream));
}

COL_API int cuda_operator_gemm_fp8_block128(const void* input_fp8, const float* input_scale,
                                            const void* weight_fp8, const float* weight_scale,
                                            void* output_bf16, uint64_t m, uint64_t k, uint64_t n,
                                            void* stream) {
  if (m == 0 || n == 0) return 0;
  return forward_fp8<false>(input_fp8, input_scale, weight_fp8, weight_scale, nullptr, output_bf16,
                            m, k, n, 1, stream);
}

COL_API int cuda_operator_gemm_swiglu_fp8_block128(const void* input_fp8, const float* input_scale,
                                                   const void* packed_weight_fp8,
                                                   const float* weight_scale, void* output_bf16,
                                                   uint64_t m, uint64_t k, uint64_t n,
                                                   void* stream) {
  if (m == 0 || n == 0) return 0;
  return forward_fp8<true>(input_fp8, input_scale, packed_weight_fp8, weight_scale, nullptr,
                           output_bf16, m, k, n, 1, stream);
}

COL_API int cuda_operator_gemm_grouped_fp8_block128(const void* input_fp8,
                                                    const float* input_scale,
                                                    const void* weight_fp8,
                                                    const float* weight_scale,
                                                    const int32_t* offsets, void* output_bf16,
                                                    uint64_t t, uint64_t k, uint64_t n,
                                                    uint64_t experts, void* stream) {
  if (t == 0 || n == 0 || experts == 0) return 0;
  if (!offsets) return static_cast<int>(cudaErrorInvalidValue);
  return forward_fp8<false>(input_fp8, input_scale, weight_fp8, weight_scale, offsets, output_bf16,
                            t, k, n, experts, stream);
}

COL_API int cuda_operator_gemm_grouped_swiglu_fp8_block128(
    const void* input_fp8, const float* input_scale, const void* packed_weight_fp8,
    const float* weight_scale, const int32_t* offsets, void* output_bf16, uint64_t t, uint64_t k,
    uint64_t n, uint64_t experts, void* stream) {
  if (t == 0 || n == 0 || experts == 0) return 0;
  if (!offsets) return static_cast<int>(cudaErrorInvalidValue);
  return forward_fp8<true>(input_fp8, input_scale, packed_weight_fp8, weight_scale, offsets,
                           output_bf16, t, k, n, experts, stream);
}
