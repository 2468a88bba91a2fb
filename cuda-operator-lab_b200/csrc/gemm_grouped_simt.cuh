// CUDA-core products grouped by expert: the layouts that TMA cannot address
// (row strides that are not a multiple of 16 bytes, unaligned bases).
//
// The mathematics of all modes, for the rows r of group g:
//   kForward  out[r, j]   = sum_c x[r, c] w[g, j, c]        (SwiGLU: silu(gate) * up)
//   kGradX    dx[r, c]    = sum_j dy[r, j] w[g, j, c]
//   kGradW    dw[g, j, c] = sum_r dy[r, j] x[r, c]
// e4m3 operands: each block of 128 is summed by itself and added times its two
// scales, as on the tensor cores.
// 64 x 64 output tile per 256-thread CTA, 16-deep slices through shared
// memory, 4 x 4 fp32 sums a thread: bound by the fp32 FMA rate.
#pragma once

#include <cuda_fp8.h>

#include <cstdint>
#include <type_traits>

#include "block_scale.cuh"
#include "grouped_schedule.cuh"

namespace col {
namespace simt {

enum GroupedMode : int { kForward = 0, kGradX = 1, kGradW = 2 };

struct GroupedSimtParams {
  const void* a;         // x or dy
  const void* b;         // w, or x (kGradW)
  const float* a_scale;  // e4m3: [rows, ceil(k / 128)]
  const float* b_scale;  // e4m3: [groups, ceil(columns / 128), ceil(k / 128)]
  const int* offsets;
  __nv_bfloat16* out;
  int rows;
  int k;        // columns of x
  int n;        // output columns of the forward product (SwiGLU: half of w's rows)
  int w_rows;   // n, or 2 n with SwiGLU
  int groups;
};

template <typename T>
__device__ __forceinline__ float grouped_elem(const void* p, std::size_t i) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  } else {
    return static_cast<float>(static_cast<const __nv_fp8_e4m3*>(p)[i]);
  }
}

template <typename T, int MODE, bool SWIGLU>
__global__ void __launch_bounds__(256) grouped_simt_kernel(const GroupedSimtParams p) {
  constexpr int kTile = 64;
  constexpr int kSlice = 16;
  constexpr bool kScaled = !std::is_same<T, __nv_bfloat16>::value;
  static_assert(MODE == kForward || (!SWIGLU && !kScaled), "gradients: bf16, plain");
  __shared__ float As[kSlice][kTile + 4];
  __shared__ float Bs[kSlice][kTile + 4];
  __shared__ float Us[SWIGLU ? kSlice : 1][SWIGLU ? kTile + 4 : 1];
  grid_dependency_wait();
  const int kb_count = (p.k + 127) / 128;
  const int j0 = blockIdx.x * kTile;
  const int cols = MODE == kForward ? p.n : p.k;  // output columns
  // Row tiles of all groups, numbered group after group; a block takes every
  // gridDim.y-th.
  int next = blockIdx.y;
  int tiles_before = 0;
  struct {
    int begin;
    int end;
  } range = {0, p.offsets == nullptr ? 0 : min(max(p.offsets[0], 0), p.rows)};
  for (int g = 0; g < p.groups; ++g) {
    range.begin = range.end;
    range.end = p.offsets == nullptr ? p.rows : max(range.begin, min(max(p.offsets[g + 1], 0), p.rows));
    const int out_rows = MODE == kGradW ? p.n : range.end - range.begin;
    const int depth = MODE == kForward ? p.k : MODE == kGradX ? p.n : range.end - range.begin;
    const int tiles = (out_rows + kTile - 1) / kTile;
    for (; next < tiles_before + tiles; next += gridDim.y) {
      const int i0 = (next - tiles_before) * kTile;
      const int tx = threadIdx.x % 16;
      const int ty = threadIdx.x / 16;
      float acc[4][4] = {};
      float up[4][4] = {};
      const std::size_t wbase = static_cast<std::size_t>(g) * p.w_rows;
      auto load_w = [&](int row, int c) { return grouped_elem<T>(p.b, (wbase + row) * p.k + c); };
      // e4m3: the sums of finished blocks
      float total[kScaled ? 4 : 1][kScaled ? 4 : 1] = {};
      float total_up[kScaled && SWIGLU ? 4 : 1][kScaled && SWIGLU ? 4 : 1] = {};
      // The block with column c is summed.  64 columns of the tile lie in one
      // 128-row block of w.
      auto end_block = [&](int c) {
        if constexpr (kScaled) {
          const std::size_t sbase = static_cast<std::size_t>(g) * ((p.w_rows + 127) / 128);
          const float w_scale = p.b_scale[(sbase + j0 / 128) * kb_count + c / 128];
          float up_scale = 0.0f;
          if constexpr (SWIGLU) up_scale = p.b_scale[(sbase + (p.n + j0) / 128) * kb_count + c / 128];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const std::size_t row = range.begin + min(i0 + ty * 4 + i, out_rows - 1);
            const float x_scale = p.a_scale[row * kb_count + c / 128];
            const BlockScales two = block_scales(x_scale, w_scale);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              total[i][j] = fmaf(acc[i][j] * two.first, two.rest, total[i][j]);
              acc[i][j] = 0.0f;
            }
            if constexpr (SWIGLU) {
              const BlockScales up_two = block_scales(x_scale, up_scale);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                total_up[i][j] = fmaf(up[i][j] * up_two.first, up_two.rest, total_up[i][j]);
                up[i][j] = 0.0f;
              }
            }
          }
        }
      };
      for (int s0 = 0; s0 < depth; s0 += kSlice) {
        for (int e = threadIdx.x; e < kTile * kSlice; e += 256) {
          const int r = e / kSlice;
          const int d = s0 + e % kSlice;
          float a = 0.0f, b = 0.0f, u = 0.0f;
          if (d < depth) {
            if (i0 + r < out_rows) {
              if constexpr (MODE == kForward) {
                const std::size_t row = static_cast<std::size_t>(range.begin + i0 + r);
                a = grouped_elem<T>(p.a, row * p.k + d);
              } else if constexpr (MODE == kGradX) {
                a = grouped_elem<T>(p.a, static_cast<std::size_t>(range.begin + i0 + r) * p.n + d);
              } else {
                a = grouped_elem<T>(p.a, static_cast<std::size_t>(range.begin + d) * p.n + i0 + r);
              }
            }
            if (j0 + r < cols) {
              if constexpr (MODE == kForward) {
                b = load_w(j0 + r, d);
                if constexpr (SWIGLU) u = load_w(p.n + j0 + r, d);
              } else if constexpr (MODE == kGradX) {
                b = load_w(d, j0 + r);
              } else {
                b = grouped_elem<T>(p.b, static_cast<std::size_t>(range.begin + d) * p.k + j0 + r);
              }
            }
          }
          As[e % kSlice][r] = a;
          Bs[e % kSlice][r] = b;
          if constexpr (SWIGLU) Us[e % kSlice][r] = u;
        }
        __syncthreads();
#pragma unroll
        for (int d = 0; d < kSlice; ++d) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              acc[i][j] = fmaf(As[d][ty * 4 + i], Bs[d][tx * 4 + j], acc[i][j]);
              if constexpr (SWIGLU) up[i][j] = fmaf(As[d][ty * 4 + i], Us[d][tx * 4 + j], up[i][j]);
            }
          }
        }
        __syncthreads();
        if (kScaled && ((s0 + kSlice) % 128 == 0 || s0 + kSlice >= depth)) end_block(s0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = i0 + ty * 4 + i;
          const int c = j0 + tx * 4 + j;
          if (r < out_rows && c < cols) {
            const std::size_t row = MODE == kGradW ? static_cast<std::size_t>(g) * p.n + r
                                                   : static_cast<std::size_t>(range.begin + r);
            float v = acc[i][j];
            float u = up[i][j];
            if constexpr (kScaled) v = total[i][j];
            if constexpr (kScaled && SWIGLU) u = total_up[i][j];
            if constexpr (SWIGLU) v = silu_f(v) * u;
            p.out[row * cols + c] = __float2bfloat16_rn(v);
          }
        }
      }
    }
    tiles_before += tiles;
  }
}

template <typename T, int MODE, bool SWIGLU>
inline int launch_grouped_simt(const GroupedSimtParams& p, cudaStream_t s) {
  const int cols = MODE == kForward ? p.n : p.k;
  const long long row_tiles = MODE == kGradW
                                  ? static_cast<long long>(p.groups) * ((p.n + 63) / 64)
                                  : static_cast<long long>(p.rows) / 64 + p.groups;
  const dim3 grid((cols + 63) / 64, static_cast<unsigned>(row_tiles < 32768 ? row_tiles : 32768));
  return launch_serialised(grouped_simt_kernel<T, MODE, SWIGLU>, grid, dim3(256), 0, s, p);
}

}  // namespace simt
}  // namespace col
