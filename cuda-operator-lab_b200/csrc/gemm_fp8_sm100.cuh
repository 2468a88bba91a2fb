// Tensor-core (tcgen05) products of block-scaled e4m3 operands, dense or
// grouped by expert, fp32 sums:
//
//   out[r, j] = sum_b xs[r, b] ws[j / 128, b] sum_{c in block b} x[r, c] w[j, c]
//
// (SwiGLU: silu(gate) * up of two such sums).  The scales are fp32 numbers of
// any value, so they cannot go into the tensor core's own power-of-two scales:
// each block of 128 columns is summed by itself in TMEM (four MMAs of K = 32)
// and added, times its scale, to fp32 sums in registers.  The tile's partial
// sums rotate through 512 / BN accumulators, so the MMAs of the next blocks run
// while eight warps read one: a thread owns one row, whose activation scale is
// a scalar, and BN / 2 columns inside one 128-row block of w, whose weight
// scale is a scalar too, so a block costs one multiply-add an element.
//
// Roles, tiles, ragged edges and bounded waits are those of the bf16 kernel
// (gemm_grouped_sm100.cuh); a dense product is one group of all rows.
#pragma once

#include "gemm_grouped_sm100.cuh"

namespace col {
namespace sm100 {

struct __align__(64) Fp8Params {
  GroupedParams g;
  const float* a_scale;  // [rows, k_blocks]
  const float* b_scale;  // [groups, b_scale_rows, k_blocks]
  int b_scale_rows;
};

constexpr int kFp8BlockK = 128;  // e4m3 elements of a k-block: one swizzle row

// BN = 256: 128 sums a thread, with registers moved over from the control
// warps (setmaxnreg, shares as in gemm_sm100.cuh).
constexpr bool fp8_split_regs(int bn) { return bn == 256; }

template <int CG, int BN>
struct Fp8Cfg {
  static constexpr int kTileRows = kBlockM * CG;
  static constexpr uint32_t kABytes = kBlockM * kFp8BlockK;
  static constexpr uint32_t kBBytes = BN / CG * kFp8BlockK;
  static constexpr uint32_t kStageBytes = kABytes + kBBytes;
  static constexpr uint32_t kExtraBytes = 512 + kGroupedTableBytes;
  static constexpr int kStagesFit =
      static_cast<int>((kSmemLimit - 1024 - kExtraBytes) / kStageBytes);
  static constexpr int kStages = kStagesFit > 8 ? 8 : kStagesFit;
  static constexpr int kAccs = 512 / BN;  // partial sums in flight
  static constexpr uint32_t kSmemBytes = kStages * kStageBytes + 1024 + kExtraBytes;
  static_assert((2 * kStages + 2 * kAccs + 1) * 8 + 8 <= 512, "barrier space");
};

// Instruction descriptor, kind::f8f6f4: D fp32, A and B e4m3, both K-major.
__host__ __device__ constexpr uint32_t idesc_e4m3_f32(int m, int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

template <int CG>
__device__ __forceinline__ void umma_e4m3(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                          uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 2) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}

// tcgen05.ld of 32 columns without waiting; tmem_wait32 completes it and names
// the registers, so that no use of them is scheduled before it.
__device__ __forceinline__ void tmem_ld32_start(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_wait32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
                 "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// sums[i] += part[i] * scale, two at a time (one packed instruction).
__device__ __forceinline__ void add_scaled32(float* sums, const uint32_t (&part)[32], float scale) {
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    asm("{\n\t.reg .b64 s, a, c;\n\t"
        "mov.b64 s, {%4, %4};\n\t"
        "mov.b64 a, {%2, %3};\n\t"
        "mov.b64 c, {%0, %1};\n\t"
        "fma.rn.f32x2 c, a, s, c;\n\t"
        "mov.b64 {%0, %1}, c;\n\t}"
        : "+f"(sums[i]), "+f"(sums[i + 1])
        : "f"(__uint_as_float(part[i])), "f"(__uint_as_float(part[i + 1])), "f"(scale));
  }
}

template <bool SWIGLU, int CG, int BN>
__global__ void __cluster_dims__(CG, 1, 1) __launch_bounds__(kCtaThreads, 1)
    fp8_kernel(const __grid_constant__ Fp8Params fp) {
  using Cfg = Fp8Cfg<CG, BN>;
  const GroupedParams& p = fp.g;
  constexpr int kStages = Cfg::kStages;
  constexpr int kAccs = Cfg::kAccs;
  constexpr uint32_t kIdesc = idesc_e4m3_f32(Cfg::kTileRows, BN);
  constexpr int kABoxRows = CG == 1 ? 32 : kBlockM;
  constexpr bool kSplitRegs = fp8_split_regs(BN);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<std::uintptr_t>(smem_raw) + 1023) & ~static_cast<std::uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kStages * Cfg::kStageBytes);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + kStages;
  uint64_t* tfull_bar = bars + 2 * kStages;
  uint64_t* tempty_bar = tfull_bar + kAccs;
  uint64_t* drain_bar = tempty_bar + kAccs;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  int* prefix = reinterpret_cast<int*>(smem + kStages * Cfg::kStageBytes + 512);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = CG == 2 ? static_cast<int>(cluster_ctarank()) : 0;
  const bool leader = rank == 0;
  const int worker = blockIdx.x / CG;
  const int workers = gridDim.x / CG;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(full_bar + s), 1);
      mbar_init(smem_u32(empty_bar + s), 1);
    }
    for (int a = 0; a < kAccs; ++a) {
      mbar_init(smem_u32(tfull_bar + a), 1);
      mbar_init(smem_u32(tempty_bar + a), CG * kEpiWarps);
    }
    mbar_init(smem_u32(drain_bar), 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    grid_dependents_launch();
  }
  if (warp == 2) {
    if constexpr (CG == 2) {
      tmem_alloc_pair(smem_u32(tmem_holder), 512);
    } else {
      tmem_alloc(smem_u32(tmem_holder), 512);
    }
  }
  grid_dependency_wait();
  if (warp == 3) {
    fill_tile_prefix(prefix, p.offsets, p.groups, p.rows, Cfg::kTileRows, lane);
  }
  tc_fence_before();
  if constexpr (CG == 2) {
    cluster_sync();
  } else {
    __syncthreads();
  }
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  auto fail = [&](unsigned code) {
    atomicOr(p.status, code);
    *abort_flag = 1;
  };
  const int num_tiles = prefix[p.groups] * p.num_n_blocks;

  if (warp < 4) {
    if constexpr (kSplitRegs) regs_release<kRegsControl>();
    if (warp == 0) {
      if (lane == 0) {
        // ---------------- TMA producer
        prefetch_tmap(&p.map_a);
        prefetch_tmap(&p.map_b);
        int stage = 0;
        uint32_t phase = 0;
        uint32_t issued_mask = 0;
        uint32_t issued_phase = 0;
        int filled = 0;
        bool ok = true;
        for (int tile = worker; ok && tile < num_tiles; tile += workers) {
          const GroupedTile t = grouped_tile<kForward, SWIGLU, CG, BN>(p, prefix, tile, rank);
          int a_boxes = 1;
          if constexpr (CG == 1) {
            a_boxes = min(kBlockM / kABoxRows, (t.end - t.a_row + kABoxRows - 1) / kABoxRows);
          }
          for (int kb = 0; kb < t.k_blocks; ++kb) {
            if (filled >= kStages &&
                !mbar_wait(smem_u32(empty_bar + stage), phase ^ 1u, abort_flag)) {
              fail(kStatusProducer);
              ok = false;
              break;
            }
            const uint32_t bytes = a_boxes * kABoxRows * 128u + Cfg::kBBytes;
            const uint32_t fb_local = smem_u32(full_bar + stage);
            uint32_t fb = fb_local;
            if constexpr (CG == 2) fb = map_to_cta(fb_local, 0);
            if (leader) mbar_arrive_expect_tx(fb_local, CG * bytes);
            const uint32_t sa = smem_u32(smem + stage * Cfg::kStageBytes);
            const uint32_t sb = sa + Cfg::kABytes;
            const int kc = kb * kFp8BlockK;
            for (int i = 0; i < a_boxes; ++i) {
              grouped_load_2d<CG>(sa + i * (kABoxRows * 128), &p.map_a, fb, kc,
                                  t.a_row + i * kABoxRows);
            }
#pragma unroll
            for (int i = 0; i < 2 / CG; ++i) {
              const int h = CG == 2 ? rank : i;
              grouped_load_3d<CG>(sb + i * (BN / 2 * 128), &p.map_b, fb, kc,
                                  t.col + h * (SWIGLU ? p.up_offset : BN / 2), t.group);
            }
            if (filled < kStages) ++filled;
            issued_mask |= 1u << stage;
            issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
        if (!ok || *abort_flag) {
          if (leader) {
            for (int s = 0; s < kStages; ++s) {
              if ((issued_mask & (1u << s)) &&
                  !mbar_wait_drain(smem_u32(full_bar + s), (issued_phase >> s) & 1u)) {
                atomicOr(p.status, kStatusDrain);
              }
            }
          } else {
            // CTA 1 cannot observe CTA 0's barriers: give its copies time to land.
            for (int i = 0; i < 200; ++i) __nanosleep(1000);
          }
        }
      }
    } else if (warp == 1) {
      if (lane == 0 && leader) {
        // ---------------- MMA issuer
        int stage = 0;
        uint32_t phase = 0;
        int acc = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        bool issued_any = false;
        for (int tile = worker; ok && tile < num_tiles; tile += workers) {
          for (int kb = 0; kb < p.num_k_blocks; ++kb) {
            if (!mbar_wait(smem_u32(tempty_bar + acc), acc_phase ^ 1u, abort_flag) ||
                !mbar_wait(smem_u32(full_bar + stage), phase, abort_flag)) {
              fail(kStatusMma);
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t d_tmem = tmem_base + acc * BN;
            const uint32_t sa = smem_u32(smem + stage * Cfg::kStageBytes);
            const uint32_t sb = sa + Cfg::kABytes;
#pragma unroll
            for (int k = 0; k < kFp8BlockK / 32; ++k) {
              umma_e4m3<CG>(d_tmem, sdesc_kmajor_sw128(sa + k * 32), sdesc_kmajor_sw128(sb + k * 32),
                            kIdesc, k != 0 ? 1u : 0u);
            }
            issued_any = true;
            grouped_commit<CG>(smem_u32(empty_bar + stage));
            grouped_commit<CG>(smem_u32(tfull_bar + acc));
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1u;
            }
            if (++acc == kAccs) {
              acc = 0;
              acc_phase ^= 1u;
            }
          }
        }
        if (issued_any) {
          if constexpr (CG == 2) {
            umma_commit_pair_local(smem_u32(drain_bar));
          } else {
            umma_commit(smem_u32(drain_bar));
          }
          if (!mbar_wait_drain(smem_u32(drain_bar), 0)) atomicOr(p.status, kStatusDrain);
        }
      }
    }
  } else {
    // ---------------- sums and epilogue: this CTA's 128 rows, half the columns a warpgroup
    if constexpr (kSplitRegs) regs_acquire<kRegsEpilogue>();
    constexpr int kCols = BN / 2;  // accumulator columns of a thread
    const int q = warp & 3;
    const int half = (warp - 4) >> 2;
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
    const int kb_count = p.num_k_blocks;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int tile = worker; ok && tile < num_tiles; tile += workers) {
      const GroupedTile t = grouped_tile<kForward, SWIGLU, CG, BN>(p, prefix, tile, rank);
      const int row = t.a_row + q * 32 + lane;
      const bool row_ok = row < t.end;
      const bool warp_ok = __any_sync(0xffffffffu, row_ok);
      // the scales of this row and of this thread's rows of w (with SwiGLU the
      // gate rows' and the up rows')
      const float* xs = fp.a_scale + static_cast<std::size_t>(row_ok ? row : t.begin) * kb_count;
      const float* ws = fp.b_scale + static_cast<std::size_t>(t.group) * fp.b_scale_rows * kb_count;
      const float* wu = ws;
      if constexpr (SWIGLU) {
        wu = ws + static_cast<std::size_t>((p.up_offset + t.col) / 128) * kb_count;
        ws += static_cast<std::size_t>(t.col / 128) * kb_count;
      } else {
        ws += static_cast<std::size_t>(min((t.col + half * kCols) / 128, fp.b_scale_rows - 1)) * kb_count;
      }
      float sums[kCols];
#pragma unroll
      for (int i = 0; i < kCols; ++i) sums[i] = 0.0f;
      float next_x = 0.0f, next_w = 0.0f, next_u = 0.0f;
      if (warp_ok) {
        next_x = __ldg(xs);
        next_w = __ldg(ws);
        if constexpr (SWIGLU) next_u = __ldg(wu);
      }
#pragma unroll 1
      for (int kb = 0; kb < kb_count; ++kb) {
        const float sw = next_x * next_w;
        const float su = SWIGLU ? next_x * next_u : 0.0f;
        if (warp_ok && kb + 1 < kb_count) {
          next_x = __ldg(xs + kb + 1);
          next_w = __ldg(ws + kb + 1);
          if constexpr (SWIGLU) next_u = __ldg(wu + kb + 1);
        }
        if (!mbar_wait(smem_u32(tfull_bar + acc), acc_phase, abort_flag)) {
          if (lane == 0) fail(kStatusEpilogue);
          ok = false;
          break;
        }
        tc_fence_after();
        if (warp_ok) {
          // SwiGLU: this thread's gate columns, then the up columns of the same outputs
          constexpr int kChunks = kCols / 32;
          const uint32_t t_row = t_lane + acc * BN;
          auto chunk_col = [&](int c) {
            if constexpr (SWIGLU) {
              constexpr int kGate = kCols / 2;
              return c * 32 < kGate ? half * kGate + c * 32 : BN / 2 + half * kGate + c * 32 - kGate;
            } else {
              return half * kCols + c * 32;
            }
          };
          uint32_t part[2][32];
          tmem_ld32_start(t_row + chunk_col(0), part[0]);
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            tmem_wait32(part[c & 1]);
            if (c + 1 < kChunks) tmem_ld32_start(t_row + chunk_col(c + 1), part[(c + 1) & 1]);
            const bool is_up = SWIGLU && c * 32 >= kCols / 2;
            add_scaled32(sums + c * 32, part[c & 1], is_up ? su : sw);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 2) {
            mbar_arrive_cluster(map_to_cta(smem_u32(tempty_bar + acc), 0));
          } else {
            mbar_arrive(smem_u32(tempty_bar + acc));
          }
        }
        if (++acc == kAccs) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
      if (ok && row_ok) {
        constexpr int kOut = SWIGLU ? kCols / 2 : kCols;
        const int col0 = t.col + half * kOut;
#pragma unroll
        for (int c = 0; c < kOut; c += 16) {
          float o[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            o[j] = SWIGLU ? silu_fast(sums[c + j]) * sums[kOut + c + j] : sums[c + j];
          }
          grouped_store<16>(p, row, col0 + c, o);
        }
      }
    }
  }

  // No CTA leaves while its partner may still address its shared memory.
  __syncwarp();
  tc_fence_before();
  if constexpr (CG == 2) {
    cluster_sync();
  } else {
    __syncthreads();
  }
  if (warp == 2) {
    tc_fence_after();
    if constexpr (CG == 2) {
      tmem_dealloc_pair(tmem_base, 512);
    } else {
      tmem_dealloc(tmem_base, 512);
    }
  }
}

}  // namespace sm100
}  // namespace col
