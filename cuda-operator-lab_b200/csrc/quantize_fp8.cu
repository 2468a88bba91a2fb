// e4m3 quantisation with one fp32 scale for each block of 128 columns (rows)
// or 128 x 128 tile (weights).
//
//   a = max(max |x| over the block, 2^-100)
//   scale = a / 448                    (fp32, IEEE division)
//   q = e4m3(x * 448 / a), to nearest even of the exact quotient
//
// v = x * (448 / a) in fp32 is up to 2 units in its last place off the quotient
// and rounds wrongly where a tie of two e4m3 values lies between (with bf16
// inputs quotients that are ties are common: 3 in 10^4 values of a normal sample
// came out one step off).  One Newton step on the residual v a - 448 x gives the
// quotient correctly rounded: then v is on the quotient's side of every tie, or
// is a tie itself.  With bf16 inputs the quotient then is that tie (two 8-bit
// significands: any other quotient is at least 2^-13 away).  With fp32 inputs it
// may lie beside it, and the sign of t a - 448 x for the tie t decides.
//
// 448 is e4m3's largest value, so a block always uses the whole range.  The
// floor keeps the inverse finite: an all-zero block gives q = 0 with scale
// 2^-100 / 448.  A NaN in a block makes its scale and every q of it NaN; an
// infinity makes the scale infinite and q NaN there, 0 elsewhere (finite *
// 448 / inf), so a product over either block is NaN, never a plausible number.
// The maximum is taken over the bit patterns of |x| as integers, which order
// like the values and put NaN above infinity, where fmaxf would drop it.
// The kernels are bound by memory, one read of x and one write of q.
#include <cuda_fp8.h>

#include "common.cuh"

namespace {

using col::grid_dependency_wait;

constexpr float kE4m3Max = 448.0f;
constexpr unsigned kAmaxFloorBits = (127u - 100u) << 23;  // 2^-100
constexpr int kThreads = 256;
constexpr int kRowLanes = 8;  // lanes of a row's block
constexpr int kLanes = 16;    // lanes of a tile's row, 8 columns each

// 8 consecutive values as they are in memory: bf16 pairs or fp32 words.
template <typename T>
struct Raw8 {
  static constexpr int kWords = sizeof(T) * 2;
  unsigned w[kWords];
};

// VEC: one 16-byte (bf16) or two 16-byte loads, all or nothing (rows are whole
// multiples of 8); otherwise element by element, zeros behind the row's end.
template <typename T, bool VEC>
__device__ __forceinline__ Raw8<T> load8(const T* p, int left) {
  Raw8<T> r;
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < Raw8<T>::kWords; i += 4) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (left > 0) v = *(reinterpret_cast<const uint4*>(p) + i / 4);
      r.w[i] = v.x, r.w[i + 1] = v.y, r.w[i + 2] = v.z, r.w[i + 3] = v.w;
    }
  } else if constexpr (sizeof(T) == 2) {
    const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned lo = 2 * i < left ? h[2 * i] : 0u;
      const unsigned hi = 2 * i + 1 < left ? h[2 * i + 1] : 0u;
      r.w[i] = lo | (hi << 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = i < left ? __float_as_uint(p[i]) : 0u;
  }
  return r;
}

// Running maximum of |x| as bit patterns: for bf16 both halves of a word at
// once, taken apart at the end.
template <typename T>
__device__ __forceinline__ unsigned abs_max(unsigned m, const Raw8<T>& r) {
#pragma unroll
  for (int i = 0; i < Raw8<T>::kWords; ++i) {
    if constexpr (sizeof(T) == 2) {
      m = __vmaxu2(m, r.w[i] & 0x7fff7fffu);
    } else {
      m = max(m, r.w[i] & 0x7fffffffu);
    }
  }
  return m;
}
template <typename T>
__device__ __forceinline__ float block_amax(unsigned m) {
  if constexpr (sizeof(T) == 2) m = max(m & 0xffff0000u, m << 16);
  return __uint_as_float(max(m, kAmaxFloorBits));
}

// What the values of a block are multiplied by and corrected with.  The residual
// is taken of x * 448 and a both times 2^-10, against overflow.  A block with an
// infinity is not corrected: x * 0 is its result.
struct BlockScale {
  float inverse;   // 448 / a
  float a10;       // a 2^-10
  float step;      // 1 / a10
  __device__ __forceinline__ explicit BlockScale(float amax) {
    inverse = __fdiv_rn(kE4m3Max, amax);
    const bool finite = __float_as_uint(amax) < 0x7f800000u;
    a10 = finite ? amax * 0x1p-10f : 0.0f;
    step = finite ? inverse * (1024.0f / 448.0f) : 0.0f;
  }
};
constexpr float kE4m3Max10 = 0.4375f;  // 448 2^-10

// The correctly rounded quotient v, or where it is a tie its neighbour on the
// side of the exact one.
__device__ __forceinline__ float settle_tie(float x, float v, float a10) {
  const unsigned b = __float_as_uint(v) & 0x7fffffffu;
  const float t = __uint_as_float(b);
  // normal values: half of the 20 bits that e4m3 drops; below, where the ties are
  // multiples of 2^-10, as e4m3's values are, for which nothing changes
  const bool tie = b >= 0x3c800000u ? (b & 0xfffffu) == 0x80000u
                                    : __fsub_rn(__fadd_rn(t, 12288.0f), 12288.0f) == t;
  if (!tie) return v;
  // every step is exact: t has at most 5 significant bits
  const float hi = __fmul_rn(fabsf(x), kE4m3Max10);
  const float lo = __fmaf_rn(fabsf(x), kE4m3Max10, -hi);
  const float d = __fsub_rn(__fmaf_rn(t, a10, -hi), lo);
  unsigned r = b;
  if (d < 0.0f) r += 1u;
  if (d > 0.0f) r -= 1u;
  return __uint_as_float(r | (__float_as_uint(v) & 0x80000000u));
}

// x * 448 / a, on the right side of every tie.
template <typename T>
__device__ __forceinline__ float quotient(float x, const BlockScale& s) {
  const float v = x * s.inverse;
  const float hi = __fmul_rn(x, kE4m3Max10);  // exact for bf16
  float d = __fmaf_rn(v, s.a10, -hi);
  if constexpr (sizeof(T) == 4) d = __fsub_rn(d, __fmaf_rn(x, kE4m3Max10, -hi));
  return __fmaf_rn(-d, s.step, v);
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(__nv_fp8_storage_t* q, int left, const Raw8<T>& r,
                                       const BlockScale& s) {
  if (left <= 0) return;
  unsigned w[4];
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = __nv_cvt_float2_to_fp8x2(
          make_float2(quotient<T>(__uint_as_float(r.w[i] << 16), s),
                      quotient<T>(__uint_as_float(r.w[i] & 0xffff0000u), s)),
          __NV_SATFINITE, __NV_E4M3);
    }
  } else {
    // Bounds of the quotient, 2^-22 to either side: where both round alike, so
    // does the quotient.  Else (one value in 10^6) it is computed.
    const float below = s.inverse * (1.0f - 0x1p-22f);
    const float above = s.inverse * (1.0f + 0x1p-22f);
    unsigned differ = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x0 = __uint_as_float(r.w[2 * i]);
      const float x1 = __uint_as_float(r.w[2 * i + 1]);
      w[i] = __nv_cvt_float2_to_fp8x2(make_float2(x0 * below, x1 * below), __NV_SATFINITE, __NV_E4M3);
      differ |= w[i] ^ __nv_cvt_float2_to_fp8x2(make_float2(x0 * above, x1 * above),
                                                __NV_SATFINITE, __NV_E4M3);
    }
    if (differ != 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float x = __uint_as_float(r.w[2 * i + j]);
          v[j] = settle_tie(x, quotient<T>(x, s), s.a10);
        }
        w[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[0], v[1]), __NV_SATFINITE, __NV_E4M3);
      }
    }
  }
  const uint2 bytes = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
  if constexpr (VEC) {
    *reinterpret_cast<uint2*>(q) = bytes;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i < left) q[i] = static_cast<__nv_fp8_storage_t>(((i < 4 ? bytes.x : bytes.y) >> (8 * (i & 3))) & 0xffu);
    }
  }
}

// Rows: block b of all rows * kb blocks belongs to 8 lanes of two 16-byte loads
// (bf16) each, which read 128 contiguous bytes at a time.  bf16 [16384, 4096]
// takes 33.0 us, 6.1 TB/s, fp32 48.2 us, 7.0 TB/s.  Before the correction to exact
// quotients bf16 took 29.9 us; 16 lanes with one load 39.8 (twice the divisions
// and shuffles a byte), several blocks a thread 30.2 and more (fewer threads),
// values kept as floats instead of as loaded 42.4 (registers).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    quantize_rows_kernel(const T* x, __nv_fp8_storage_t* __restrict__ q,
                         float* __restrict__ scale, unsigned long long blocks, unsigned kb,
                         unsigned k) {
  grid_dependency_wait();
  const unsigned lane = threadIdx.x % kRowLanes;
  const unsigned long long b =
      static_cast<unsigned long long>(blockIdx.x) * (kThreads / kRowLanes) + threadIdx.x / kRowLanes;
  std::size_t at;
  int left;  // columns from this lane's first piece to the row's end
  if (k == kb * 128u) {  // whole blocks: no division
    at = b * 128u + lane * 8u;
    left = b < blocks ? 128 : 0;
  } else {
    const unsigned long long row = (b >> 32) == 0 ? static_cast<unsigned>(b) / kb : b / kb;
    const unsigned col = static_cast<unsigned>(b - row * kb) * 128u + lane * 8u;
    at = row * k + col;
    left = b < blocks ? static_cast<int>(k) - static_cast<int>(col) : 0;
  }
  constexpr int kPieces = 16 / kRowLanes;
  Raw8<T> raw[kPieces];
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    raw[i] = load8<T, VEC>(x + at + i * kRowLanes * 8, left - i * kRowLanes * 8);
  }
#pragma unroll
  for (int i = 0; i < kPieces; ++i) m = abs_max<T>(m, raw[i]);
#pragma unroll
  for (int o = kRowLanes / 2; o > 0; o >>= 1) {
    const unsigned other = __shfl_xor_sync(0xffffffffu, m, o);
    m = sizeof(T) == 2 ? __vmaxu2(m, other) : max(m, other);
  }
  const float amax = block_amax<T>(m);
  const BlockScale block(amax);
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    store8<T, VEC>(q + at + i * kRowLanes * 8, left - i * kRowLanes * 8, raw[i], block);
  }
  if (lane == 0 && b < blocks) scale[b] = __fdiv_rn(amax, kE4m3Max);
}

// Weights: one CTA a 128 x 128 tile, held in registers between the maximum
// and the rounding (8 rows of 8 columns a thread).
// Three CTAs an SM for bf16: [16, 2048, 4096] 78.2 -> 68.2 us, 5.9 TB/s (four
// spill: 84.6); two for fp32, whose values take twice the registers: 100.5 us, 6.7
// TB/s (three: 137.6).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 3 : 2)
    quantize_tiles_kernel(const T* w, __nv_fp8_storage_t* __restrict__ q,
                          float* __restrict__ scale, unsigned n, unsigned k, unsigned nb,
                          unsigned kb) {
  grid_dependency_wait();
  __shared__ unsigned warp_max[kThreads / 32];
  constexpr int kRows = 128 / (kThreads / kLanes);
  const unsigned tile_k = blockIdx.x % kb;
  const unsigned rest = blockIdx.x / kb;
  const unsigned tile_n = rest % nb;
  const std::size_t base = static_cast<std::size_t>(rest / nb) * n;
  const unsigned col = tile_k * 128u + threadIdx.x % kLanes * 8u;
  const unsigned row0 = tile_n * 128u + threadIdx.x / kLanes;
  Raw8<T> raw[kRows];
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const unsigned row = row0 + i * (kThreads / kLanes);
    const int left = row < n ? static_cast<int>(k) - static_cast<int>(col) : 0;
    raw[i] = load8<T, VEC>(w + (base + row) * k + col, left);
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) m = abs_max<T>(m, raw[i]);
  if constexpr (sizeof(T) == 2) m = max(m & 0xffffu, m >> 16) << 16;
  m = __reduce_max_sync(0xffffffffu, m);
  if (threadIdx.x % 32 == 0) warp_max[threadIdx.x / 32] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) m = max(m, warp_max[i]);
  const float amax = __uint_as_float(max(m, kAmaxFloorBits));
  const BlockScale block(amax);
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const unsigned row = row0 + i * (kThreads / kLanes);
    const int left = row < n ? static_cast<int>(k) - static_cast<int>(col) : 0;
    store8<T, VEC>(q + (base + row) * k + col, left, raw[i], block);
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
  const bool vec = k % 8 == 0 && col::aligned16(x) && aligned8(q);
  const cudaStream_t s = col::as_stream(stream);
  const std::uint64_t per = kThreads / kRowLanes;
  const std::uint64_t grid = (blocks + per - 1) / per;
  if (grid > 0x7fffffffull) return static_cast<int>(cudaErrorInvalidValue);
  return col::launch_serialised(
      vec ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>,
      dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, s, static_cast<const T*>(x),
      static_cast<__nv_fp8_storage_t*>(q), scale, static_cast<unsigned long long>(blocks),
      static_cast<unsigned>(kb), static_cast<unsigned>(k));
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
  const bool vec = k % 8 == 0 && col::aligned16(w) && aligned8(q);
  return col::launch_serialised(
      vec ? quantize_tiles_kernel<T, true> : quantize_tiles_kernel<T, false>,
      dim3(static_cast<unsigned>(experts * nb * kb)), dim3(kThreads), 0, col::as_stream(stream),
      static_cast<const T*>(w), static_cast<__nv_fp8_storage_t*>(q), scale,
      static_cast<unsigned>(n), static_cast<unsigned>(k), static_cast<unsigned>(nb),
      static_cast<unsigned>(kb));
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
