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
// scale is a scalar too, so a block costs one multiply-add an element (where the
// scales' product is no normal number, two multiplications: block_scale.cuh).
//
// Roles, tiles, ragged edges and bounded waits are those of the bf16 kernel
// (gemm_grouped_sm100.cuh); a dense product is one group of all rows.
#pragma once

#include "block_scale.cuh"
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
// warps (setmaxnreg: 128 x 40 + 256 x 232 of the 384 x 168 that the CTA starts
// with).
constexpr bool fp8_split_regs(int bn) { return bn == 256; }
constexpr int kFp8RegsControl = 40;
constexpr int kFp8RegsReader = 232;
constexpr int kFp8RegsLaunch = 168;
static_assert(128 * kFp8RegsControl + 256 * kFp8RegsReader <= 384 * kFp8RegsLaunch, "register shares");

// ROWS = 32: tiles of at most 32 rows, of which only those are loaded and kept
// (as in GroupedCfg).  SPLIT: the CTAs of a cluster share a tile's k-blocks and
// add their sums up in the first one, for a few such tiles.
template <int CG, int BN, int ROWS, int SPLIT>
struct Fp8Cfg {
  static_assert((ROWS == kBlockM && SPLIT == 1) || (ROWS == 32 && CG == 1 && SPLIT > 1), "variants");
  static constexpr int kTileRows = ROWS * CG;
  static constexpr int kCols = BN / 2;  // accumulator columns of a reading thread
  static constexpr int kChunk = kCols < 64 ? kCols / 2 : 32;  // columns read at a time
  static constexpr uint32_t kABytes = ROWS * kFp8BlockK;
  static constexpr uint32_t kBBytes = BN / CG * kFp8BlockK;
  static constexpr uint32_t kKBlockBytes = kABytes + kBBytes;
  // k-blocks a stage
  static constexpr int kKps = CG == 2 || kKBlockBytes > 40 * 1024 ? 1 : (BN == 64 ? 4 : 2);
  static constexpr uint32_t kStageBytes = kKps * kKBlockBytes;
  // one warp's sums of 32 rows, from each other CTA, for two warps
  static constexpr uint32_t kSumBytes = 32 * kCols * 4;
  static constexpr uint32_t kExtraBytes = 512 + kGroupTableBytes + (SPLIT - 1) * 2 * kSumBytes;
  static constexpr int kStagesFit =
      static_cast<int>((kSmemLimit - 1024 - kExtraBytes) / kStageBytes);
  static constexpr int kStages = kStagesFit > 8 ? 8 : kStagesFit;
  // A stage's partial sums are handed over together: two waits and a commit.
  static constexpr int kAccs = 512 / BN / kKps;  // stages whose sums TMEM holds
  static constexpr uint32_t kSmemBytes = kStages * kStageBytes + 1024 + kExtraBytes;
  static_assert(kAccs >= 2 && kStages >= kAccs, "a stage outlives its partial sums");
  static_assert((2 * kStages + kAccs + 3) * 8 + 8 <= 512, "barrier space");
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

// tcgen05.ld of 16 or 32 columns without waiting; tmem_ld_wait completes it and
// names the registers, so that no use of them is scheduled before it.
__device__ __forceinline__ void tmem_ld_start(uint32_t taddr, uint32_t (&r)[16]) {
  tmem_ld16_start(taddr, r);
}
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[16]) { tmem_wait16(r); }
__device__ __forceinline__ void tmem_ld_start(uint32_t taddr, uint32_t (&r)[32]) {
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

__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[32]) {
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

// 16 columns back to TMEM; tmem_st_wait completes them.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ uint64_t pack2(float x, float y) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
  return v;
}

// sums += part * scale, two columns an instruction.
template <int W>
__device__ __forceinline__ void add_scaled(uint64_t* sums, const uint32_t (&part)[W], float scale) {
  uint64_t s;
  asm("mov.b64 %0, {%1, %1};" : "=l"(s) : "f"(scale));
#pragma unroll
  for (int i = 0; i < W; i += 2) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(part[i]), "r"(part[i + 1]));
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(sums[i / 2]) : "l"(v), "l"(s));
  }
}

__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}

template <bool SWIGLU, int CG, int BN, int ROWS, int SPLIT>
__global__ void __cluster_dims__(CG * SPLIT, 1, 1) __launch_bounds__(kCtaThreads, 1)
    fp8_kernel(const __grid_constant__ Fp8Params fp) {
  using Cfg = Fp8Cfg<CG, BN, ROWS, SPLIT>;
  const GroupedParams& p = fp.g;
  constexpr int kStages = Cfg::kStages;
  constexpr int kKps = Cfg::kKps;
  constexpr int kAccs = Cfg::kAccs;
  constexpr uint32_t kIdesc = idesc_e4m3_f32(kBlockM * CG, BN);
  constexpr bool kSplitRegs = fp8_split_regs(BN);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<std::uintptr_t>(smem_raw) + 1023) & ~static_cast<std::uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kStages * Cfg::kStageBytes);
  uint64_t* full_bar = bars;
  // One barrier a stage says that its MMAs are done: the warps that read the
  // partial sums wait for it, and the producer before it refills the stage.  (A
  // second commit for the producer cost ~0.1 us a block.)  No waiter can miss a
  // phase: a stage's MMAs are issued again only after its partial sums were
  // read, as there are at least as many stages as sets of accumulators.
  uint64_t* done_bar = bars + kStages;
  uint64_t* tempty_bar = done_bar + kStages;
  uint64_t* drain_bar = tempty_bar + kAccs;
  uint64_t* sums_bar = drain_bar + 1;  // the other CTAs' sums for each of two warps
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(sums_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  const GroupTables tables = group_tables(smem + kStages * Cfg::kStageBytes + 512);
  uint8_t* other_sums = smem + kStages * Cfg::kStageBytes + 512 + kGroupTableBytes;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = CG == 2 ? static_cast<int>(cluster_ctarank()) : 0;
  const bool leader = rank == 0;
  const int worker = blockIdx.x / (CG * SPLIT);
  const int workers = gridDim.x / (CG * SPLIT);  // SPLIT > 1: at least as many as tiles
  // this CTA's k-blocks
  const int share = SPLIT > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int kb_begin = p.num_k_blocks * share / SPLIT;
  const int kb_end = p.num_k_blocks * (share + 1) / SPLIT;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(full_bar + s), 1);
      mbar_init(smem_u32(done_bar + s), 1);
    }
    for (int a = 0; a < kAccs; ++a) mbar_init(smem_u32(tempty_bar + a), CG * kEpiWarps);
    mbar_init(smem_u32(drain_bar), 1);
    mbar_init(smem_u32(sums_bar), 1);
    mbar_init(smem_u32(sums_bar + 1), 1);
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
    fill_group_tables(tables, p.offsets, p.groups, p.rows, Cfg::kTileRows, lane);
  }
  tc_fence_before();
  if constexpr (CG * SPLIT > 1) {
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
  int num_tiles = tables.prefix[p.groups] * p.num_n_blocks;
  if constexpr (SPLIT > 1) num_tiles = min(num_tiles, workers);  // one tile a cluster

  if (warp < 4) {
    if constexpr (kSplitRegs) regs_release<kFp8RegsControl>();
    if (warp == 0) {
      // ---------------- TMA producer: the whole warp keeps the loop's state, so
      // that addresses and coordinates stay in uniform registers; one lane issues
      if (elect_one()) {
        prefetch_tmap(&p.map_a);
        prefetch_tmap(&p.map_b);
      }
      __syncwarp();
      int stage = 0;
      uint32_t phase = 0;
      uint32_t issued_mask = 0;
      uint32_t issued_phase = 0;
      int filled = 0;
      bool ok = true;
      for (int tile = worker; ok && tile < num_tiles; tile += workers) {
        const GroupedTile t = grouped_tile<kForward, SWIGLU, CG, BN, ROWS>(p, tables, tile, rank);
        // Single CTAs load A 32 rows at a time where the group ends early.
        const int rows = min(ROWS, (t.end - t.a_row + 31) & ~31);
        const bool whole = CG == 2 || rows == kBlockM;
        for (int kb = kb_begin; kb < kb_end; kb += kKps) {
          const int nk = min(kKps, kb_end - kb);
          if (filled >= kStages && !warp_wait(smem_u32(done_bar + stage), phase ^ 1u, abort_flag)) {
            if (lane == 0) fail(kStatusProducer);
            ok = false;
            break;
          }
          if (elect_one()) {
            const uint32_t bytes = nk * ((whole ? kBlockM : rows) * 128u + Cfg::kBBytes);
            const uint32_t fb_local = smem_u32(full_bar + stage);
            uint32_t fb = fb_local;
            if constexpr (CG == 2) fb = map_to_cta(fb_local, 0);
            if (leader) mbar_arrive_expect_tx(fb_local, CG * bytes);
#pragma unroll
            for (int j = 0; j < kKps; ++j) {
              if (j >= nk) break;
              const uint32_t sa = smem_u32(smem + stage * Cfg::kStageBytes + j * Cfg::kKBlockBytes);
              const uint32_t sb = sa + Cfg::kABytes;
              const int kc = (kb + j) * kFp8BlockK;
              if (whole) {
                grouped_load_2d<CG>(sa, &p.map_a, fb, kc, t.a_row);
              } else {
                for (int r = 0; r < rows; r += 32) {
                  grouped_load_2d<CG>(sa + r * 128, &p.map_a32, fb, kc, t.a_row + r);
                }
              }
              constexpr int kBoxRows = b_box_rows(SWIGLU, CG, BN);
#pragma unroll
              for (int i = 0; i < BN / CG / kBoxRows; ++i) {
                const int h = CG == 2 ? rank : i;
                grouped_load_3d<CG>(sb + i * (kBoxRows * 128), &p.map_b, fb, kc,
                                    t.col + h * (SWIGLU ? p.up_offset : BN / 2), t.group);
              }
            }
          }
          __syncwarp();
          if (filled < kStages) ++filled;
          issued_mask |= 1u << stage;
          issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (lane == 0 && (!ok || *abort_flag)) {
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
    } else if (warp == 1) {
      if (leader) {
        // ---------------- MMA issuer: the whole warp keeps the loop's state, so
        // that descriptors stay in uniform registers; one lane issues
        int stage = 0;
        uint32_t phase = 0;
        int acc = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        bool issued_any = false;
        for (int tile = worker; ok && tile < num_tiles; tile += workers) {
          for (int kb = kb_begin; kb < kb_end; kb += kKps) {
            if (!warp_wait(smem_u32(full_bar + stage), phase, abort_flag)) {
              if (lane == 0) fail(kStatusMma);
              ok = false;
              break;
            }
            if (!warp_wait(smem_u32(tempty_bar + acc), acc_phase ^ 1u, abort_flag)) {
              if (lane == 0) fail(kStatusMma);
              ok = false;
              break;
            }
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int j = 0; j < kKps; ++j) {
                if (j > 0 && kb + j >= kb_end) break;
                const uint32_t d_tmem = tmem_base + (acc * kKps + j) * BN;
                const uint32_t sa = smem_u32(smem + stage * Cfg::kStageBytes + j * Cfg::kKBlockBytes);
                const uint32_t sb = sa + Cfg::kABytes;
#pragma unroll
                for (int k = 0; k < kFp8BlockK / 32; ++k) {
                  umma_e4m3<CG>(d_tmem, sdesc_kmajor_sw128(sa + k * 32),
                                sdesc_kmajor_sw128(sb + k * 32), kIdesc, k != 0 ? 1u : 0u);
                }
              }
              grouped_commit<CG>(smem_u32(done_bar + stage));
            }
            __syncwarp();
            issued_any = true;
            if (++acc == kAccs) {
              acc = 0;
              acc_phase ^= 1u;
            }
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
        if (issued_any && elect_one()) {
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
    if constexpr (kSplitRegs) regs_acquire<kFp8RegsReader>();
    constexpr int kCols = Cfg::kCols;
    constexpr int kChunk = Cfg::kChunk;
    const int q = warp & 3;
    const int part_of = (warp - 4) >> 2;  // which half of them
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
    const int kb_count = p.num_k_blocks;
    int acc = 0;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = worker; ok && tile < num_tiles; tile += workers) {
      const GroupedTile t = grouped_tile<kForward, SWIGLU, CG, BN, ROWS>(p, tables, tile, rank);
      const int row = t.a_row + q * 32 + lane;
      const bool row_ok = row < t.end;
      // rows of this warp
      const int valid = ROWS == 32 && q != 0 ? 0 : min(t.end - (t.a_row + q * 32), 32);
      const bool warp_ok = valid > 0;
      // offsets of the scales of this row and of this thread's rows of w (with
      // SwiGLU the gate rows', and the up rows' a constant behind them)
      uint32_t xs = static_cast<uint32_t>(row_ok ? row : t.begin) * static_cast<uint32_t>(kb_count) + kb_begin;
      const int block = SWIGLU ? t.col / 128 : min((t.col + part_of * kCols) / 128, fp.b_scale_rows - 1);
      uint32_t ws = static_cast<uint32_t>(t.group * fp.b_scale_rows + block) * static_cast<uint32_t>(kb_count) + kb_begin;
      const uint32_t wu = SWIGLU ? static_cast<uint32_t>(p.up_offset / 128 * kb_count) : 0u;
      uint64_t sums[kCols / 2];  // two fp32 each
#pragma unroll
      for (int i = 0; i < kCols / 2; ++i) sums[i] = 0u;
      // The next stage's partial sums: waits until its MMAs are done.
      auto next_stage = [&]() {
        if (!warp_wait(smem_u32(done_bar + stage), phase, abort_flag)) return false;
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
        tc_fence_after();
        return true;
      };
      auto release = [&]() {
        const uint32_t bar = smem_u32(tempty_bar + acc);
        release_sum<CG>(CG == 2 ? map_to_cta(bar, 0) : bar, lane);
        if (++acc == kAccs) acc = 0;
      };
      if (!warp_ok) {
        for (int kb = kb_begin; kb < kb_end; kb += kKps) {
          ok = next_stage();
          if (!ok) break;
          release();
        }
      } else {
        constexpr int kChunks = kCols / kChunk;
        static_assert(kChunks % 2 == 0, "the chunks' registers alternate");
        int in_stage = 0;
        // TMEM address of this thread's column `mine` of the sum: with SWIGLU its
        // gate columns, then the up columns of the same outputs.
        auto column = [&](int mine) {
          constexpr int kGate = kCols / 2;
          const uint32_t col = !SWIGLU          ? part_of * kCols + mine
                               : mine < kGate   ? part_of * kGate + mine
                                                : BN / 2 + part_of * kGate + mine - kGate;
          return t_lane + (acc * kKps + in_stage) * BN + col;
        };
        auto chunk_addr = [&](int c) { return column(c * kChunk); };
        // Plain loads: the kernel that writes the scales may still have been running
        // when this one started, which non-coherent loads do not allow for.
        float next_x = fp.a_scale[xs];
        float next_w = fp.b_scale[ws];
        float next_u = SWIGLU ? fp.b_scale[ws + wu] : 0.0f;
        uint32_t part[2][kChunk];
        ok = next_stage();
        if (ok) tmem_ld_start(chunk_addr(0), part[0]);
#pragma unroll 1
        for (int kb = kb_begin; ok && kb < kb_end; ++kb) {
          float sw = next_x * next_w;
          float su = next_x * next_u;
          // One branch for the warp; a row's own result does not depend on it.
          // Rare: the sum is multiplied by the first scale where it lies.
          if (__any_sync(0xffffffffu, !normal_f32(sw) || (SWIGLU && !normal_f32(su)))) {
            const BlockScales two = block_scales(next_x, next_w);
            const BlockScales two_up = block_scales(next_x, next_u);
            tmem_ld_wait(part[0]);
            // (nothing to multiply where no scale but zeros, infinities and NaN is met)
            const bool some = __any_sync(0xffffffffu, two.first != 1.0f || (SWIGLU && two_up.first != 1.0f));
#pragma unroll 1
            for (int c = some ? 0 : kCols; c < kCols; c += 16) {
              const float first = SWIGLU && c >= kCols / 2 ? two_up.first : two.first;
              uint32_t piece[16];
              tmem_ld_start(column(c), piece);
              tmem_ld_wait(piece);
#pragma unroll
              for (int i = 0; i < 16; ++i) piece[i] = __float_as_uint(__uint_as_float(piece[i]) * first);
              tmem_st16(column(c), piece);
            }
            tmem_st_wait();
            sw = two.rest;
            su = two_up.rest;
            tmem_ld_start(chunk_addr(0), part[0]);
          }
          if (kb + 1 < kb_end) {
            next_x = fp.a_scale[++xs];
            next_w = fp.b_scale[++ws];
            if constexpr (SWIGLU) next_u = fp.b_scale[ws + wu];
          }
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            tmem_ld_wait(part[c & 1]);
            // the next load is under way while this chunk is added: the next
            // chunk of this sum, or the next sum's first, once this stage's are
            // released where they end
            if (c + 1 < kChunks) {
              tmem_ld_start(chunk_addr(c + 1), part[(c + 1) & 1]);
            } else if (kKps > 1 && in_stage + 1 < kKps && kb + 1 < kb_end) {
              ++in_stage;
              tmem_ld_start(chunk_addr(0), part[0]);
            } else {
              release();
              in_stage = 0;
              if (kb + 1 < kb_end) {
                ok = next_stage();
                if (ok) tmem_ld_start(chunk_addr(0), part[0]);
              }
            }
            add_scaled(sums + c * kChunk / 2, part[c & 1],
                       SWIGLU && c * kChunk >= kCols / 2 ? su : sw);
          }
        }
      }
      if constexpr (SPLIT > 1) {
        // The first CTA adds the others' sums in their order.  Word j of a lane's
        // sums from CTA s lies at ((s - 1) * 2 + part_of) * kSumBytes + (j / 4) *
        // 512 + lane * 16: whole rows of banks for both sides.
        if (ok && warp_ok) {
          if (share != 0) {
            const uint32_t to = map_to_cta(smem_u32(other_sums + ((share - 1) * 2 + part_of) * Cfg::kSumBytes), 0);
            const uint32_t bar = map_to_cta(smem_u32(sums_bar + part_of), 0);
            if (row_ok) {
#pragma unroll
              for (int j = 0; j < kCols; j += 4) {
                st_async_v4(to + j / 4 * 512 + lane * 16, static_cast<uint32_t>(sums[j / 2]),
                            static_cast<uint32_t>(sums[j / 2] >> 32),
                            static_cast<uint32_t>(sums[j / 2 + 1]),
                            static_cast<uint32_t>(sums[j / 2 + 1] >> 32), bar);
              }
            }
          } else {
            const uint32_t bar = smem_u32(sums_bar + part_of);
            if (lane == 0) mbar_arrive_expect_tx(bar, (SPLIT - 1) * valid * kCols * 4);
            __syncwarp();
            ok = warp_wait_cluster(bar, 0, abort_flag);
            if (ok && row_ok) {
#pragma unroll 1
              for (int from = 0; from < SPLIT - 1; ++from) {
                const uint8_t* src = other_sums + (from * 2 + part_of) * Cfg::kSumBytes + lane * 16;
#pragma unroll
                for (int j = 0; j < kCols; j += 4) {
                  const float4 v = *reinterpret_cast<const float4*>(src + j / 4 * 512);
                  const float2 a = unpack2(sums[j / 2]);
                  const float2 b = unpack2(sums[j / 2 + 1]);
                  sums[j / 2] = pack2(a.x + v.x, a.y + v.y);
                  sums[j / 2 + 1] = pack2(b.x + v.z, b.y + v.w);
                }
              }
            }
          }
        }
      }
      if (!ok && lane == 0) fail(kStatusEpilogue);
      if (ok && warp_ok && share == 0) {
        constexpr int kOut = SWIGLU ? kCols / 2 : kCols;
        constexpr int kRun = kOut < 64 ? kOut : 64;
#pragma unroll
        for (int c = 0; c < kOut; c += kRun) {
          uint32_t w[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (i >= kRun / 2) {
              w[i] = 0u;
            } else if constexpr (SWIGLU) {
              const float2 g = unpack2(sums[c / 2 + i]);
              const float2 u = unpack2(sums[(kOut / 2 + c / 2 + i) % (kCols / 2)]);
              w[i] = pack_bf16x2(silu_fast(g.x) * u.x, silu_fast(g.y) * u.y);
            } else {
              const float2 v = unpack2(sums[(c / 2 + i) % (kCols / 2)]);
              w[i] = pack_bf16x2(v.x, v.y);
            }
          }
          store_rows64(p, static_cast<std::size_t>(t.a_row) + q * 32, valid,
                       t.col + part_of * kOut + c, kRun, w, lane);
        }
      }
    }
  }

  // No CTA leaves while its partner may still address its shared memory.
  __syncwarp();
  tc_fence_before();
  if constexpr (CG * SPLIT > 1) {
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
