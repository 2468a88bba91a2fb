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
  GroupedParams g;       // map_a: boxes of 128 rows
  CUtensorMap map_a32;   // the same in boxes of 32 rows
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

template <int CG, int BN>
struct Fp8Cfg {
  static constexpr int kTileRows = kBlockM * CG;
  static constexpr uint32_t kABytes = kBlockM * kFp8BlockK;
  static constexpr uint32_t kBBytes = BN / CG * kFp8BlockK;
  static constexpr uint32_t kKBlockBytes = kABytes + kBBytes;
  static constexpr int kKps = kKBlockBytes > 40 * 1024 ? 1 : 2;  // k-blocks a stage
  static constexpr uint32_t kStageBytes = kKps * kKBlockBytes;
  static constexpr uint32_t kExtraBytes = 512 + kGroupedTableBytes;
  static constexpr int kStagesFit =
      static_cast<int>((kSmemLimit - 1024 - kExtraBytes) / kStageBytes);
  static constexpr int kStages = kStagesFit > 8 ? 8 : kStagesFit;
  static constexpr int kAccs = 512 / BN;  // partial sums in flight
  static constexpr uint32_t kSmemBytes = kStages * kStageBytes + 1024 + kExtraBytes;
  static constexpr int kSlots = kStages * kKps;  // k-blocks in the ring
  static_assert(kSlots >= kAccs && kSlots <= 32, "a slot outlives its partial sum");
  static_assert((kStages + kSlots + kAccs + 1) * 8 + 8 <= 512, "barrier space");
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

// tcgen05.ld of 32 columns without waiting; tmem_ld_wait completes it and names
// the registers, so that no use of them is scheduled before it.
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

constexpr int kChunk = 32;  // columns of a partial sum read at a time

template <bool SWIGLU, int CG, int BN>
__global__ void __cluster_dims__(CG, 1, 1) __launch_bounds__(kCtaThreads, 1)
    fp8_kernel(const __grid_constant__ Fp8Params fp) {
  using Cfg = Fp8Cfg<CG, BN>;
  const GroupedParams& p = fp.g;
  constexpr int kStages = Cfg::kStages;
  constexpr int kKps = Cfg::kKps;
  constexpr int kAccs = Cfg::kAccs;
  constexpr uint32_t kIdesc = idesc_e4m3_f32(Cfg::kTileRows, BN);
  constexpr bool kSplitRegs = fp8_split_regs(BN);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<std::uintptr_t>(smem_raw) + 1023) & ~static_cast<std::uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kStages * Cfg::kStageBytes);
  uint64_t* full_bar = bars;
  // One barrier a k-block in the ring says that its MMAs are done: the warps
  // that read the partial sum wait for it, and the producer before it refills
  // the slot.  (A second commit for the producer cost ~0.1 us a block.)  No
  // waiter can miss a phase: a slot is used again only after its partial sum
  // was read, as there are at least as many slots as accumulators.
  uint64_t* done_bar = bars + kStages;
  uint64_t* tempty_bar = done_bar + Cfg::kSlots;
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
    for (int s = 0; s < kStages; ++s) mbar_init(smem_u32(full_bar + s), 1);
    for (int s = 0; s < Cfg::kSlots; ++s) mbar_init(smem_u32(done_bar + s), 1);
    for (int a = 0; a < kAccs; ++a) mbar_init(smem_u32(tempty_bar + a), CG * kEpiWarps);
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
    if constexpr (kSplitRegs) regs_release<kFp8RegsControl>();
    if (warp == 0) {
      if (lane == 0) {
        // ---------------- TMA producer
        prefetch_tmap(&p.map_a);
        prefetch_tmap(&p.map_b);
        int stage = 0;
        uint32_t phase = 0;
        uint32_t issued_mask = 0;
        uint32_t issued_phase = 0;
        uint32_t slot_phase = 0;  // bit s: parity of slot s's next use
        uint32_t last_slots = 0;  // two bits a stage: its last k-block in use
        int filled = 0;
        bool ok = true;
        for (int tile = worker; ok && tile < num_tiles; tile += workers) {
          const GroupedTile t = grouped_tile<kForward, SWIGLU, CG, BN>(p, prefix, tile, rank);
          // Single CTAs load A 32 rows at a time where the group ends early.
          const int rows = min(kBlockM, (t.end - t.a_row + 31) & ~31);
          const bool whole = CG == 2 || rows == kBlockM;
          for (int kb = 0; kb < t.k_blocks; kb += kKps) {
            const int nk = min(kKps, t.k_blocks - kb);
            if (filled >= kStages) {
              const int last = last_slots >> (2 * stage) & 3;
              const int slot = stage * kKps + last;
              if (!mbar_wait(smem_u32(done_bar + slot), ((slot_phase >> slot) & 1u) ^ 1u, abort_flag)) {
                fail(kStatusProducer);
                ok = false;
                break;
              }
            } else {
              ++filled;
            }
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
                  grouped_load_2d<CG>(sa + r * 128, &fp.map_a32, fb, kc, t.a_row + r);
                }
              }
#pragma unroll
              for (int i = 0; i < 2 / CG; ++i) {
                const int h = CG == 2 ? rank : i;
                grouped_load_3d<CG>(sb + i * (BN / 2 * 128), &p.map_b, fb, kc,
                                    t.col + h * (SWIGLU ? p.up_offset : BN / 2), t.group);
              }
              slot_phase ^= 1u << (stage * kKps + j);
            }
            last_slots = (last_slots & ~(3u << (2 * stage))) | (static_cast<uint32_t>(nk - 1) << (2 * stage));
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
          for (int kb = 0; ok && kb < p.num_k_blocks; kb += kKps) {
            if (!warp_wait(smem_u32(full_bar + stage), phase, abort_flag)) {
              if (lane == 0) fail(kStatusMma);
              ok = false;
              break;
            }
#pragma unroll
            for (int j = 0; j < kKps; ++j) {
              if (kb + j >= p.num_k_blocks) break;
              if (!warp_wait(smem_u32(tempty_bar + acc), acc_phase ^ 1u, abort_flag)) {
                if (lane == 0) fail(kStatusMma);
                ok = false;
                break;
              }
              tc_fence_after();
              const uint32_t d_tmem = tmem_base + acc * BN;
              const uint32_t sa = smem_u32(smem + stage * Cfg::kStageBytes + j * Cfg::kKBlockBytes);
              const uint32_t sb = sa + Cfg::kABytes;
              if (elect_one()) {
#pragma unroll
                for (int k = 0; k < kFp8BlockK / 32; ++k) {
                  umma_e4m3<CG>(d_tmem, sdesc_kmajor_sw128(sa + k * 32),
                                sdesc_kmajor_sw128(sb + k * 32), kIdesc, k != 0 ? 1u : 0u);
                }
                grouped_commit<CG>(smem_u32(done_bar + stage * kKps + j));
              }
              __syncwarp();
              issued_any = true;
              if (++acc == kAccs) {
                acc = 0;
                acc_phase ^= 1u;
              }
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
    constexpr int kCols = BN / 2;  // accumulator columns of a thread
    const int q = warp & 3;
    const int part_of = (warp - 4) >> 2;  // which half of them
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
    const int kb_count = p.num_k_blocks;
    int acc = 0;
    int slot = 0;
    uint32_t slot_phase = 0;  // bit s: parity of slot s's next completion
    bool ok = true;
    for (int tile = worker; ok && tile < num_tiles; tile += workers) {
      const GroupedTile t = grouped_tile<kForward, SWIGLU, CG, BN>(p, prefix, tile, rank);
      const int row = t.a_row + q * 32 + lane;
      const bool row_ok = row < t.end;
      const int valid = min(t.end - (t.a_row + q * 32), 32);  // rows of this warp
      const bool warp_ok = valid > 0;
      // offsets of the scales of this row and of this thread's rows of w (with
      // SwiGLU the gate rows', and the up rows' a constant behind them)
      uint32_t xs = static_cast<uint32_t>(row_ok ? row : t.begin) * static_cast<uint32_t>(kb_count);
      const int block = SWIGLU ? t.col / 128 : min((t.col + part_of * kCols) / 128, fp.b_scale_rows - 1);
      uint32_t ws = static_cast<uint32_t>(t.group * fp.b_scale_rows + block) * static_cast<uint32_t>(kb_count);
      const uint32_t wu = SWIGLU ? static_cast<uint32_t>(p.up_offset / 128 * kb_count) : 0u;
      uint64_t sums[kCols / 2];  // two fp32 each
#pragma unroll
      for (int i = 0; i < kCols / 2; ++i) sums[i] = 0u;
      // The sum of the next k-block: waits until its MMAs are done.
      auto next_sum = [&](int kb) {
        if (!warp_wait(smem_u32(done_bar + slot), (slot_phase >> slot) & 1u, abort_flag)) return false;
        slot_phase ^= 1u << slot;
        // the next block's slot: the stage's other one, or the next stage's first
        if (kKps == 1 || (slot & 1) == 1 || kb + 1 == kb_count) {
          slot = slot / kKps * kKps + kKps;
          if (slot == Cfg::kSlots) slot = 0;
        } else {
          ++slot;
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
        for (int kb = 0; kb < kb_count; ++kb) {
          ok = next_sum(kb);
          if (!ok) break;
          release();
        }
      } else {
        constexpr int kChunks = kCols / kChunk;
        static_assert(kChunks % 2 == 0, "the chunks' registers alternate");
        auto chunk_addr = [&](int c) {
          uint32_t col;
          if constexpr (SWIGLU) {
            // this thread's gate columns, then the up columns of the same outputs
            constexpr int kGate = kCols / 2;
            col = c * kChunk < kGate ? part_of * kGate + c * kChunk
                                     : BN / 2 + part_of * kGate + c * kChunk - kGate;
          } else {
            col = part_of * kCols + c * kChunk;
          }
          return t_lane + acc * BN + col;
        };
        float next_x = __ldg(fp.a_scale + xs);
        float next_w = __ldg(fp.b_scale + ws);
        float next_u = SWIGLU ? __ldg(fp.b_scale + ws + wu) : 0.0f;
        uint32_t part[2][kChunk];
        ok = next_sum(0);
        if (ok) tmem_ld_start(chunk_addr(0), part[0]);
#pragma unroll 1
        for (int kb = 0; ok && kb < kb_count; ++kb) {
          const float sw = next_x * next_w;
          const float su = next_x * next_u;
          if (kb + 1 < kb_count) {
            next_x = __ldg(fp.a_scale + ++xs);
            next_w = __ldg(fp.b_scale + ++ws);
            if constexpr (SWIGLU) next_u = __ldg(fp.b_scale + ws + wu);
          }
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            tmem_ld_wait(part[c & 1]);
            // the next load is under way while this chunk is added: the next
            // chunk of this sum, or, once this sum is released, the next one's
            if (c + 1 < kChunks) {
              tmem_ld_start(chunk_addr(c + 1), part[(c + 1) & 1]);
            } else {
              release();
              if (kb + 1 < kb_count) {
                ok = next_sum(kb + 1);
                if (ok) tmem_ld_start(chunk_addr(0), part[0]);
              }
            }
            add_scaled(sums + c * kChunk / 2, part[c & 1],
                       SWIGLU && c * kChunk >= kCols / 2 ? su : sw);
          }
        }
      }
      if (!ok && lane == 0) fail(kStatusEpilogue);
      if (ok && warp_ok) {
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
