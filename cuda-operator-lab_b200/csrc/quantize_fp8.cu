// e4m3 quantisation with one fp32 scale for each block of 128 columns (rows)
// or 128 x 128 tile (weights).
//
//   a = max(max |x| over the block, 2^-100)
//   scale = a / 448        inverse = 448 / a      (fp32, IEEE division)
//   q = e4m3(x * inverse), to nearest even, saturating
//
// 448 is e4m3's largest value, so a block always uses the whole range.  The
// floor keeps the inverse finite: an all-zero block gives q = 0 with scale
// 2^-100 / 448.  A NaN in a block makes its scale and every q of it NaN; an
// infinity makes the scale infinite and q NaN there, 0 elsewhere (finite *
// 448 / inf), so a product over either block is NaN, never a plausible number.
// The maximum is taken over the bit patterns of |x| as integers, which order
// like the values and put NaN above infinity, where fmaxf would drop it.
// One division a block and one multiplication an element: the kernels are
// bound by memory, one read of x and one write of q.
#include <cuda_fp8.h>

#include "common.cuh"

namespace {

using col::grid_dependency_wait;
using col::unpack_bf16x8;

constexpr float kE4m3Max = 448.0f;
constexpr unsigned kAmaxFloorBits = (127u - 100u) << 23;  // 2^-100
constexpr int kThreads = 256;
constexpr int kLanes = 16;  // lanes of a 128-column block, 8 columns each

// 8 consecutive values as floats; `vec`: one 16-byte (bf16) or two 16-byte
// (fp32) loads, otherwise element by element, zeros behind the row's end.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int left, bool vec, float (&f)[8]) {
  if (left >= 8 && vec) {
    if constexpr (sizeof(T) == 2) {
      unpack_bf16x8(*reinterpret_cast<const uint4*>(p), f);
    } else {
      const float4 a = *reinterpret_cast<const float4*>(p);
      const float4 b = *reinterpret_cast<const float4*>(p + 4);
      f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
      f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 2) {
        f[i] = i < left ? __bfloat162float(p[i]) : 0.0f;
      } else {
        f[i] = i < left ? p[i] : 0.0f;
      }
    }
  }
}

__device__ __forceinline__ unsigned abs_bits_max(const float (&f)[8]) {
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
  return m;
}

__device__ __forceinline__ void store8(__nv_fp8_storage_t* q, int left, bool vec,
                                       const float (&f)[8], float inverse) {
  uint2 v;
  unsigned w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * i] * inverse, f[2 * i + 1] * inverse),
                                    __NV_SATFINITE, __NV_E4M3);
  }
  v.x = w[0] | (w[1] << 16);
  v.y = w[2] | (w[3] << 16);
  if (left >= 8 && vec) {
    *reinterpret_cast<uint2*>(q) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i < left) q[i] = static_cast<__nv_fp8_storage_t>(((i < 4 ? v.x : v.y) >> (8 * (i & 3))) & 0xffu);
    }
  }
}

// Rows: block b of all rows * kb blocks belongs to 16 lanes; a thread holds
// the values of UNROLL blocks at once so that their loads are in flight
// together.
template <typename T, int UNROLL>
__global__ void __launch_bounds__(kThreads)
    quantize_rows_kernel(const T* __restrict__ x, __nv_fp8_storage_t* __restrict__ q,
                         float* __restrict__ scale, unsigned long long blocks, unsigned kb,
                         unsigned k, int vec_in, int vec_out) {
  grid_dependency_wait();
  const unsigned lane = threadIdx.x % kLanes;
  const unsigned long long first =
      static_cast<unsigned long long>(blockIdx.x) * (kThreads / kLanes * UNROLL) + threadIdx.x / kLanes;
  float f[UNROLL][8];
  std::size_t at[UNROLL];
  int left[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const unsigned long long b = first + u * (kThreads / kLanes);
    if (k == kb * 128u) {  // whole blocks: no division
      at[u] = b * 128u + lane * 8u;
      left[u] = b < blocks ? 8 : 0;
    } else {
      const unsigned long long row =
          (b >> 32) == 0 ? static_cast<unsigned>(b) / kb : b / kb;
      const unsigned col = static_cast<unsigned>(b - row * kb) * 128u + lane * 8u;
      at[u] = row * k + col;
      left[u] = b < blocks ? static_cast<int>(k) - static_cast<int>(col) : 0;
    }
    load8(x + at[u], left[u], vec_in != 0, f[u]);
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    unsigned m = abs_bits_max(f[u]);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float amax = __uint_as_float(max(m, kAmaxFloorBits));
    const unsigned long long b = first + u * (kThreads / kLanes);
    if (left[u] > 0) store8(q + at[u], left[u], vec_out != 0, f[u], __fdiv_rn(kE4m3Max, amax));
    if (lane == 0 && b < blocks) scale[b] = __fdiv_rn(amax, kE4m3Max);
  }
}

// Weights: one CTA a 128 x 128 tile, held in registers between the maximum
// and the rounding (8 rows of 8 columns a thread).
template <typename T>
__global__ void __launch_bounds__(kThreads)
    quantize_tiles_kernel(const T* __restrict__ w, __nv_fp8_storage_t* __restrict__ q,
                          float* __restrict__ scale, unsigned n, unsigned k, unsigned nb,
                          unsigned kb, int vec_in, int vec_out) {
  grid_dependency_wait();
  __shared__ unsigned warp_max[kThreads / 32];
  constexpr int kRows = 128 / (kThreads / kLanes);
  const unsigned tile_k = blockIdx.x % kb;
  const unsigned rest = blockIdx.x / kb;
  const unsigned tile_n = rest % nb;
  const std::size_t base = static_cast<std::size_t>(rest / nb) * n;
  const unsigned col = tile_k * 128u + threadIdx.x % kLanes * 8u;
  const unsigned row0 = tile_n * 128u + threadIdx.x / kLanes;
  float f[kRows][8];
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const unsigned row = row0 + i * (kThreads / kLanes);
    const int left = row < n ? static_cast<int>(k) - static_cast<int>(col) : 0;
    load8(w + (base + row) * k + col, left, vec_in != 0, f[i]);
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) m = max(m, abs_bits_max(f[i]));
  m = __reduce_max_sync(0xffffffffu, m);
  if (threadIdx.x % 32 == 0) warp_max[threadIdx.x / 32] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) m = max(m, warp_max[i]);
  const float amax = __uint_as_float(max(m, kAmaxFloorBits));
  const float inverse = __fdiv_rn(kE4m3Max, amax);
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const unsigned row = row0 + i * (kThreads / kLanes);
    const int left = row < n ? static_cast<int>(k) - static_cast<int>(col) : 0;
    if (left > 0) store8(q + (base + row) * k + col, left, vec_out != 0, f[i], inverse);
  }
  if (threadIdx.x == 0) scale[blockIdx.x] = __fdiv_rn(amax, kE4m3Max);
}

inline bool aligned8(const void* p) { return (reinterpret_cast<std::uintptr_t>(p) & 7u) == 0u; }

template <typename T>
int quantize_rows(const void* x, void* q, float* scale, std::uint64_t m, std::uint64_t k,
                  void* stream) {
  if (m == 0 || k == 0) return 0;
  if (!x || !q || !scale || m > 0x7fffffffull || k > 0x7fffff00ull) {
    return static_cast<int>(cudaErrorInvalidValue);
  }
  const std::uint64_t kb = (k + 127) / 128;
  const std::uint64_t blocks = m * kb;
  const int vec_in = k % 8 == 0 && col::aligned16(x);
  const int vec_out = k % 8 == 0 && aligned8(q);
  constexpr int kUnroll = 4;
  const std::uint64_t per = kThreads / kLanes;
  const cudaStream_t s = col::as_stream(stream);
  // Four blocks a thread once that still leaves a CTA for every SM twice
  // over; a single row gets one, for the shorter chain.
  const bool wide = blocks >= per * kUnroll * 2 * 148;
  const std::uint64_t grid = (blocks + per * (wide ? kUnroll : 1) - 1) / (per * (wide ? kUnroll : 1));
  if (grid > 0x7fffffffull) return static_cast<int>(cudaErrorInvalidValue);
  return col::launch_serialised(
      wide ? quantize_rows_kernel<T, kUnroll> : quantize_rows_kernel<T, 1>,
      dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, s, static_cast<const T*>(x),
      static_cast<__nv_fp8_storage_t*>(q), scale, static_cast<unsigned long long>(blocks),
      static_cast<unsigned>(kb), static_cast<unsigned>(k), vec_in, vec_out);
}

template <typename T>
int quantize_tiles(const void* w, void* q, float* scale, std::uint64_t experts, std::uint64_t n,
                   std::uint64_t k, void* stream) {
  if (experts == 0 || n == 0 || k == 0) return 0;
  if (!w || !q || !scale || n > 0x7fffff00ull || k > 0x7fffff00ull) {
    return static_cast<int>(cudaErrorInvalidValue);
  }
  const std::uint64_t nb = (n + 127) / 128;
  const std::uint64_t kb = (k + 127) / 128;
  if (experts > 0x7fffffffull || nb * kb > 0x7fffffffull || experts * nb * kb > 0x7fffffffull) {
    return static_cast<int>(cudaErrorInvalidValue);
  }
  return col::launch_serialised(
      quantize_tiles_kernel<T>, dim3(static_cast<unsigned>(experts * nb * kb)), dim3(kThreads), 0,
      col::as_stream(stream), static_cast<const T*>(w), static_cast<__nv_fp8_storage_t*>(q), scale,
      static_cast<unsigned>(n), static_cast<unsigned>(k), static_cast<unsigned>(nb),
      static_cast<unsigned>(kb), static_cast<int>(k % 8 == 0 && col::aligned16(w)),
      static_cast<int>(k % 8 == 0 && aligned8(q)));
}

}  // namespace

COL_API int cuda_operator_quantize_fp8_block128_f32(const float* input, void* output_fp8,
                                                    float* scale, uint64_t m, uint64_t k,
                                                    void* stream) {
  return quantize_rows<float>(input, output_fp8, scale, m, k, stream);
}
COL_API int cuda_operator_quantize_fp8_block128_bf16(const void* input_bf16, void* output_fp8,
                                                     float* scale, uint64_t m, uint64_t k,
                                                     void* stream) {
  return quantize_rows<__nv_bfloat16>(input_bf16, output_fp8, scale, m, k, stream);
}
COL_API int cuda_operator_quantize_fp8_block128_weight_f32(const float* weight, void* output_fp8,
                                                           float* scale, uint64_t experts,
                                                           uint64_t n, uint64_t k, void* stream) {
  return quantize_tiles<float>(weight, output_fp8, scale, experts, n, k, stream);
}
COL_API int cuda_operator_quantize_fp8_block128_weight_bf16(const void* weight_bf16,
                                                            void* output_fp8, float* scale,
                                                            uint64_t experts, uint64_t n,
                                                            uint64_t k, void* stream) {
  return quantize_tiles<__nv_bfloat16>(weight_bf16, output_fp8, scale, experts, n, k, stream);
}
