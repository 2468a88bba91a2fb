// Tensor-core (tcgen05) products grouped by expert: bf16 operands, fp32 sums.
//
// For the rows r of group g (grouped_schedule.cuh):
//   kForward  out[r, j]   = sum_c x[r, c] w[g, j, c]        (SwiGLU: silu(gate) * up)
//   kGradX    dx[r, c]    = sum_j dy[r, j] w[g, j, c]
//   kGradW    dw[g, j, c] = sum_r dy[r, j] x[r, c]
//
// Persistent and warp-specialised like the dense kernel (gemm_sm100.cuh):
// warp 0 loads, warp 1 issues the MMAs, warp 2 owns TMEM, warp 3 builds the
// table of row tiles and zeroes ragged tails (kGradW), warps 4..11 store.  CG =
// 1: a CTA computes 128 rows; CG = 2: a pair of CTAs computes 256 rows, each
// holding half of B (tcgen05 cta_group::2).  BN accumulator columns a tile, two
// accumulators in TMEM, so that storing a tile overlaps the next one's MMAs.
//
// Every operand is read in place.  Forward reads A and B along the summed
// index (K-major).  The gradients sum over an index that is not the
// contiguous one: w in kGradX and both operands in kGradW are loaded as boxes
// of 64 contiguous columns x 64 summed rows and multiplied as MN-major tiles,
// so nothing is transposed in memory.
//
// Ragged edges: a tile that reaches past its group's last row loads rows of
// the next group, which only reach accumulator rows that are not stored.  In
// kGradW the rows are summed over, so the last block of a group is cut to
// whole steps of 16 rows and the rest of its last step is set to zero in shared
// memory, in both operands (a NaN there times zero would be a NaN).  Edges of
// n and k are filled with zeros by TMA; w is a three-dimensional map, so that a
// box never runs into the next expert.
#pragma once

#include "gemm_sm100.cuh"
#include "gemm_sm100_2sm.cuh"
#include "gemm_sm100_sk.cuh"
#include "grouped_schedule.cuh"

namespace col {
namespace sm100 {

enum GroupedMode : int { kForward = 0, kGradX = 1, kGradW = 2 };

struct __align__(64) GroupedParams {
  CUtensorMap map_a;    // boxes of 128 rows (kGradW: 64)
  CUtensorMap map_a32;  // the same in boxes of 32 rows (single CTAs)
  CUtensorMap map_b;    // boxes of b_box_rows() rows (gradients: 64)
  const int* offsets;
  __nv_bfloat16* out;
  unsigned* status;
  int rows;          // t
  int groups;
  int out_cols;      // n (kForward), k (gradients)
  int out_rows;      // kGradW: n
  int num_n_blocks;  // tiles along out_cols
  int num_k_blocks;  // blocks of the summed index (kGradW: by group)
  int up_offset;     // SwiGLU: rows from gate to up in w
  int out_vec_ok;    // 16-byte stores allowed
};

// B is loaded in two boxes where gate and up rows or two CTAs share it.
constexpr int b_box_rows(bool swiglu, int cg, int bn) { return swiglu || cg == 2 ? bn / 2 : bn; }

// ROWS = 32: tiles of at most 32 rows, for products whose time is reading w.
// Only those rows of A are loaded and kept (the MMA's other 96 rows read
// whatever lies behind them; what they add up is not stored), which leaves the
// ring to w.
// SPLIT: the CTAs of a cluster share a tile's k-blocks and add their sums up in
// the first one, for a few tiles of few rows.
template <int CG, int BN, int ROWS, int SPLIT>
struct GroupedCfg {
  static_assert(BN == 128 || BN == 256, "tile width");
  static_assert(CG == 1 || CG == 2, "CTAs of a tile");
  static_assert(ROWS == kBlockM || (ROWS == 32 && CG == 1), "rows of a tile");
  static_assert(SPLIT == 1 || (ROWS == 32 && BN == 128), "shared sums");
  static constexpr int kTileRows = ROWS * CG;
  static constexpr uint32_t kABytes = ROWS * kBlockK * 2;
  static constexpr uint32_t kBBytes = BN / CG * kBlockK * 2;
  static constexpr uint32_t kKBlockBytes = kABytes + kBBytes;
  // k-blocks a stage: one for pairs (six stages; with three of two blocks 16384 rows
  // over 8 experts, gate/up 4096 x 4096, took 747-750 us instead of 738-745: fastest
  // of 12 runs of ten launches back to back on the same inputs, measured twice)
  static constexpr int kKps = CG == 2 || kKBlockBytes > 40 * 1024 ? 1 : 2;
  static constexpr uint32_t kStageBytes = kKps * kKBlockBytes;
  // 32 rows of 64 sums, from each other CTA, for two warps
  static constexpr uint32_t kSumBytes = 32 * 64 * 4;
  static constexpr uint32_t kExtraBytes = 256 + kGroupTableBytes + (SPLIT - 1) * 2 * kSumBytes;
  static constexpr int kStagesFit =
      static_cast<int>((kSmemLimit - 1024 - kExtraBytes) / kStageBytes);
  static constexpr int kStages = kStagesFit > 8 ? 8 : kStagesFit;
  static constexpr uint32_t kTmemCols = 2 * BN;
  static constexpr uint32_t kSmemBytes = kStages * kStageBytes + 1024 + kExtraBytes;
};

// MN-major tile with the 128-byte swizzle: chunks of 64 contiguous elements,
// `chunk_bytes` apart (leading offset), rows of the summed index 128 bytes
// apart in groups of 8 (stride offset 1024).  A step of 16 rows is 2048 bytes.
__device__ __forceinline__ uint64_t sdesc_mnmajor_sw128(uint32_t saddr, uint32_t chunk_bytes) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) |
         (static_cast<uint64_t>(chunk_bytes >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) |
         (static_cast<uint64_t>(2) << 61);
}

constexpr uint32_t kIdescAMnMajor = 1u << 15;
constexpr uint32_t kIdescBMnMajor = 1u << 16;

template <int CG>
__device__ __forceinline__ void grouped_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                                int x, int y) {
  if constexpr (CG == 2) {
    tma_load_2d_pair(dst, map, bar, x, y);
  } else {
    tma_load_2d(dst, map, bar, x, y);
  }
}

template <int CG>
__device__ __forceinline__ void grouped_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                                int x, int y, int z) {
  if constexpr (CG == 2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
  }
}

// All MMAs issued so far by this thread: arrive on `bar` (both CTAs of a pair).
template <int CG>
__device__ __forceinline__ void grouped_commit(uint32_t bar) {
  if constexpr (CG == 2) {
    umma_commit_pair_both(bar);
  } else {
    umma_commit(bar);
  }
}

// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(yes));
  return yes != 0;
}

// Bounded waits of a whole converged warp (mbar_wait is one thread's).  All
// lanes poll with one instruction and leave on one flag, so that they leave
// together; the time limit sets that flag.  A wait that does not pass at once
// keeps one 32-bit clock reading: the e4m3 kernel's readers have no registers
// to spare.
//
// warp_wait is for what ends within one k-block or the storing of tiles: at most
// the time of writing the whole output (~30 ms for all of the card's memory).
// 2^31 cycles are 1.1 s at the highest clock.
constexpr uint32_t kWarpWaitCycles = 1u << 31;

__device__ __forceinline__ uint32_t clock32() {
  uint32_t t;
  asm volatile("mov.u32 %0, %%clock;" : "=r"(t));
  return t;
}

__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint32_t start = clock32();
  while (!mbar_try_wait(bar, parity)) {
    if (*abort_flag) return false;
    if (clock32() - start > kWarpWaitCycles) *abort_flag = 1;
  }
  return true;
}

// warp_wait on data that other CTAs of the cluster wrote.
__device__ __forceinline__ bool warp_wait_cluster(uint32_t bar, uint32_t parity,
                                                  volatile int* abort_flag) {
  if (mbar_try_wait_cluster(bar, parity)) return true;
  const uint32_t start = clock32();
  while (!mbar_try_wait_cluster(bar, parity)) {
    if (*abort_flag) return false;
    if (clock32() - start > kWarpWaitCycles) *abort_flag = 1;
  }
  return true;
}

// Limit of a wait that spans the sums of whole tiles: a gradient by W sums over an
// expert's rows, of which there may be 2^31 (2^25 k-blocks, several seconds).  A
// k-block takes 0.3 to 0.8 us.
__host__ __device__ constexpr unsigned long long blocks_limit_ns(unsigned long long k_blocks) {
  return kWaitLimitNs + k_blocks * 20000ull;
}

// warp_wait over `k_blocks` k-blocks.
__device__ __forceinline__ bool warp_wait_blocks(uint32_t bar, uint32_t parity,
                                                 volatile int* abort_flag,
                                                 unsigned long long k_blocks) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t start = globaltimer_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (*abort_flag) return false;
    if (globaltimer_ns() - start > blocks_limit_ns(k_blocks)) *abort_flag = 1;
  }
  return true;
}

// Arrival on a barrier of the cluster that publishes no memory.
__device__ __forceinline__ void arrive_relaxed_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// This warp has read its part of a partial sum: one arrival for the MMA issuer
// (of CTA 0).  Only tensor-memory reads come before it, which the fence orders,
// so the arrival itself is relaxed: with release semantics at cluster scope a
// block took 0.8 us where this takes 0.5 (8192 x 4096 x 4096, CTA pairs).
template <int CG>
__device__ __forceinline__ void release_sum(uint32_t bar, int lane) {
  tc_fence_before();
  __syncwarp();
  if (lane == 0) {
    if constexpr (CG == 2) {
      arrive_relaxed_cluster(bar);
    } else {
      mbar_arrive(bar);
    }
  }
}

// What the roles share about one tile.
struct GroupedTile {
  int group;
  int a_row;    // first row of this CTA's half of the tile (kGradW: of n)
  int col;      // first output column
  int begin;    // the group's rows
  int end;
  int k_blocks;
};

// Tiles of few rows stream w from DRAM.  Started together, they would read the
// same columns of all their rows, addresses that agree in their low bits, and
// crowd on few channels; so each tile's sum starts at another (even, its stages
// read pairs) k-block and wraps around.  256 rows over 64 experts, gate/up 2048
// x 4096 in bf16, back to back on the same inputs: 161 -> 156 us.  It depends on
// the expert, the columns and the tile's width, not on a tile's other rows (the
// width is chosen from the sizes alone).
__device__ __forceinline__ int few_rows_first_k(int group, int n_block, int num_n, int k_blocks) {
  const unsigned tile = static_cast<unsigned>(group) * num_n + n_block;
  return static_cast<int>(2u * (tile * 5u % ((k_blocks + 1u) / 2u)));
}

template <int MODE, bool SWIGLU, int CG, int BN, int ROWS>
__device__ __forceinline__ GroupedTile grouped_tile(const GroupedParams& p, const GroupTables& tables,
                                                    int tile, int rank) {
  constexpr int kTileRows = ROWS * CG;
  GroupedTile t;
  TileCoords c;
  if constexpr (MODE == kGradW) {
    // every group has the same tiles
    const int m_blocks = (p.out_rows + kTileRows - 1) / kTileRows;
    const int per_group = m_blocks * p.num_n_blocks;
    c.group = tile / per_group;
    const int local = tile - c.group * per_group;
    c.m = local % m_blocks;
    c.n = local / m_blocks;
  } else {
    c = tile_of(tile, tables.prefix, p.groups, p.num_n_blocks);
  }
  t.group = c.group;
  t.begin = tables.starts[c.group];
  t.end = tables.starts[c.group + 1];
  t.a_row = (MODE == kGradW ? 0 : t.begin) + c.m * kTileRows + rank * ROWS;
  t.col = c.n * (SWIGLU ? BN / 2 : BN);
  t.k_blocks = MODE == kGradW ? (t.end - t.begin + kBlockK - 1) / kBlockK : p.num_k_blocks;
  return t;
}

// Rows of the summed index in the last block of a kGradW tile; 0: it is whole
// steps of 16 and needs no zeroing.
__device__ __forceinline__ int ragged_rows(const GroupedTile& t) {
  const int last = (t.end - t.begin) % kBlockK;
  return last % 16 == 0 ? 0 : last;
}

// ---------------------------------------------------------------- output
//
// A lane of an epilogue warp holds one output row, so storing straight from
// its registers would write 32 rows 16 bytes at a time: half sectors, 32 lines
// an instruction (an 8192 x 4096 x 4096 e4m3 product spent 36 of 167 us on
// it).  The lanes exchange words first, so that neighbouring lanes hold
// neighbouring columns of a row.

// Within each N lanes: unit i (UNIT words) of lane l to unit l of lane i.
template <int N, int UNIT>
__device__ __forceinline__ void lane_transpose(uint32_t (&w)[N * UNIT], int lane) {
#pragma unroll
  for (int bit = 1; bit < N; bit <<= 1) {
    const bool upper = (lane & bit) != 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i & bit) continue;
#pragma unroll
      for (int u = 0; u < UNIT; ++u) {
        uint32_t& lo = w[i * UNIT + u];
        uint32_t& hi = w[(i | bit) * UNIT + u];
        const uint32_t got = __shfl_xor_sync(0xffffffffu, upper ? lo : hi, bit);
        if (upper) {
          lo = got;
        } else {
          hi = got;
        }
      }
    }
  }
}

// 64 output columns (32 words of two) of the warp's 32 rows, from column col0:
// lane l holds row l; rows from `valid` on and columns from p.out_cols on are
// not stored.  All lanes call it.
__device__ __forceinline__ void store_rows64(const GroupedParams& p, std::size_t row0, int valid,
                                             int col0, int cols, uint32_t (&w)[32], int lane) {
  __nv_bfloat16* base = p.out + row0 * p.out_cols + col0;
  const int limit = min(cols, p.out_cols - col0);  // columns to store
  if (p.out_vec_ok) {
    // four lanes' 16-byte pieces of a row side by side: 64-byte runs
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      uint32_t v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = w[16 * g + i];
      lane_transpose<4, 4>(v, lane);
      const int c = 32 * g + 8 * (lane & 3);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = (lane & ~3) + j;
        if (r < valid && c < limit) {
          *reinterpret_cast<uint4*>(base + static_cast<std::size_t>(r) * p.out_cols + c) =
              make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        }
      }
    }
  } else {
    // rows of any alignment: a row's 64 columns over the 32 lanes
    lane_transpose<32, 1>(w, lane);
    const int c = 2 * lane;
#pragma unroll
    for (int r = 0; r < 32; ++r) {
      if (r < valid) {
        __nv_bfloat16* dst = base + static_cast<std::size_t>(r) * p.out_cols + c;
        const uint32_t v = w[r];
        if (c < limit) *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(v);
        if (c + 1 < limit) *reinterpret_cast<uint16_t*>(dst + 1) = static_cast<uint16_t>(v >> 16);
      }
    }
  }
}

// One CTA of a product; worker w of `workers` (CTAs, pairs or clusters) takes tiles
// w, w + workers, ...; SPLIT > 1: there are at least as many workers as tiles.
template <int MODE, bool SWIGLU, int CG, int BN, int ROWS, int SPLIT>
__device__ __forceinline__ void grouped_bf16_cta(const GroupedParams& p, int worker, int workers) {
  using Cfg = GroupedCfg<CG, BN, ROWS, SPLIT>;
  static_assert(MODE != kGradW || ROWS == kBlockM, "rows of w are not ragged");
  static_assert(MODE == kForward || !SWIGLU, "SwiGLU is a forward epilogue");
  constexpr int kStages = Cfg::kStages;
  constexpr int kKps = Cfg::kKps;
  constexpr uint32_t kIdesc = idesc_bf16_f32(kBlockM * CG, BN) |
                              (MODE == kGradW ? kIdescAMnMajor : 0u) |
                              (MODE != kForward ? kIdescBMnMajor : 0u);
  constexpr uint32_t kChunkBytes = 64 * kBlockK * 2;  // 64 columns x 64 rows

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<std::uintptr_t>(smem_raw) + 1023) & ~static_cast<std::uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kStages * Cfg::kStageBytes);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + kStages;
  uint64_t* tfull_bar = bars + 2 * kStages;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint64_t* drain_bar = tempty_bar + 2;
  uint64_t* tail_bar = drain_bar + 1;  // kStages of them
  uint64_t* sums_bar = tail_bar + kStages;  // the other CTAs' sums for each of two warps
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(sums_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  static_assert((3 * kStages + 7) * 8 + 8 <= 256, "barrier space");
  const GroupTables tables = group_tables(smem + kStages * Cfg::kStageBytes + 256);
  uint8_t* other_sums = smem + kStages * Cfg::kStageBytes + 256 + kGroupTableBytes;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = CG == 2 ? static_cast<int>(cluster_ctarank()) : 0;
  const bool leader = rank == 0;
  const int share = SPLIT > 1 ? static_cast<int>(cluster_ctarank()) : 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      // kGradW pairs: both CTAs arrive for a stage (see the tail below)
      mbar_init(smem_u32(full_bar + s), MODE == kGradW ? CG : 1);
      mbar_init(smem_u32(empty_bar + s), 1);
      mbar_init(smem_u32(tail_bar + s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(tfull_bar + a), 1);
      mbar_init(smem_u32(tempty_bar + a), CG * kEpiWarps);
    }
    mbar_init(smem_u32(drain_bar), 1);
    mbar_init(smem_u32(sums_bar), 1);
    mbar_init(smem_u32(sums_bar + 1), 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    grid_dependents_launch();
  }
  if (warp == 2) {
    if constexpr (CG == 2) {
      tmem_alloc_pair(smem_u32(tmem_holder), Cfg::kTmemCols);
    } else {
      tmem_alloc(smem_u32(tmem_holder), Cfg::kTmemCols);
    }
  }
  // The offsets may come from the kernel before this one.
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
  int num_tiles;
  if constexpr (MODE == kGradW) {
    num_tiles = p.groups * ((p.out_rows + Cfg::kTileRows - 1) / Cfg::kTileRows) * p.num_n_blocks;
  } else {
    num_tiles = tables.prefix[p.groups] * p.num_n_blocks;
    if constexpr (SPLIT > 1) num_tiles = min(num_tiles, workers);  // one tile a cluster
  }

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
      const GroupedTile t = grouped_tile<MODE, SWIGLU, CG, BN, ROWS>(p, tables, tile, rank);
      // Single CTAs load A 32 rows at a time where the group ends early.
      const int rows = min(ROWS, (t.end - t.a_row + 31) & ~31);
      const bool whole = MODE == kGradW || CG == 2 || rows == kBlockM;
      const bool ragged = MODE == kGradW && ragged_rows(t) != 0;
      const int kb_begin = t.k_blocks * share / SPLIT;
      const int kb_end = t.k_blocks * (share + 1) / SPLIT;
      const int first_k =
          ROWS == 32 ? few_rows_first_k(t.group, t.col / (SWIGLU ? BN / 2 : BN), p.num_n_blocks, t.k_blocks)
                     : 0;
      for (int kb = kb_begin; kb < kb_end; kb += kKps) {
        if (filled >= kStages && !warp_wait(smem_u32(empty_bar + stage), phase ^ 1u, abort_flag)) {
          if (lane == 0) fail(kStatusProducer);
          ok = false;
          break;
        }
        const int nk = min(kKps, kb_end - kb);
        if (elect_one()) {
          const uint32_t bytes = nk * ((whole ? Cfg::kABytes : rows * 128u) + Cfg::kBBytes);
          const uint32_t fb_local = smem_u32(full_bar + stage);
          uint32_t fb = fb_local;
          if constexpr (CG == 2) fb = map_to_cta(fb_local, 0);
          if (ragged && kb + nk == t.k_blocks) {
            // A tail that needs zeroing completes on this CTA's own barrier;
            // the zeroing warp then arrives on the stage's.
            fb = smem_u32(tail_bar + stage);
            mbar_arrive_expect_tx(fb, bytes);
            if constexpr (CG == 2) fb = map_to_cta(fb, rank);
          } else if (leader) {
            mbar_arrive_expect_tx(fb_local, CG * bytes);
          } else if constexpr (MODE == kGradW) {
            arrive_relaxed_cluster(fb);  // it orders nothing: the bytes are counted by CTA 0
          }
#pragma unroll
          for (int j = 0; j < kKps; ++j) {
            if (j >= nk) break;
            const uint32_t sa = smem_u32(smem + stage * Cfg::kStageBytes + j * Cfg::kKBlockBytes);
            const uint32_t sb = sa + Cfg::kABytes;
            int kc = kb + j + first_k;
            if (ROWS == 32 && kc >= t.k_blocks) kc -= t.k_blocks;
            kc *= kBlockK;
            if constexpr (MODE == kGradW) {
#pragma unroll
              for (int i = 0; i < kBlockM / 64; ++i) {
                grouped_load_2d<CG>(sa + i * kChunkBytes, &p.map_a, fb, t.a_row + 64 * i,
                                    t.begin + kc);
              }
            } else if (whole) {
              grouped_load_2d<CG>(sa, &p.map_a, fb, kc, t.a_row);
            } else {
              for (int r = 0; r < rows; r += 32) {
                grouped_load_2d<CG>(sa + r * 128, &p.map_a32, fb, kc, t.a_row + r);
              }
            }
            if constexpr (MODE == kForward) {
              // half h of B: rows n0 + h BN/2 of w, or gate (0) and up (1) rows
              constexpr int kBoxRows = b_box_rows(SWIGLU, CG, BN);
#pragma unroll
              for (int i = 0; i < BN / CG / kBoxRows; ++i) {
                const int h = CG == 2 ? rank : i;
                grouped_load_3d<CG>(sb + i * (kBoxRows * 128), &p.map_b, fb, kc,
                                    t.col + h * (SWIGLU ? p.up_offset : BN / 2), t.group);
              }
            } else {
#pragma unroll
              for (int i = 0; i < BN / CG / 64; ++i) {
                const int col = t.col + rank * (BN / CG) + 64 * i;
                if constexpr (MODE == kGradX) {
                  grouped_load_3d<CG>(sb + i * kChunkBytes, &p.map_b, fb, col, kc, t.group);
                } else {
                  grouped_load_2d<CG>(sb + i * kChunkBytes, &p.map_b, fb, col, t.begin + kc);
                }
              }
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
      // ---------------- MMA issuer: the whole warp keeps the loop's state, so that
      // the descriptors stay in uniform registers; one lane issues
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      bool ok = true;
      bool issued_any = false;
      for (int tile = worker; ok && tile < num_tiles; tile += workers) {
        const GroupedTile t = grouped_tile<MODE, SWIGLU, CG, BN, ROWS>(p, tables, tile, rank);
        if (MODE == kGradW && t.k_blocks == 0) continue;  // zeros, stored without a sum
        const int acc = local & 1;
        if (!warp_wait(smem_u32(tempty_bar + acc), ((local >> 1) & 1) ^ 1u, abort_flag)) {
          if (lane == 0) fail(kStatusMma);
          break;
        }
        ++local;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
        const int last_rows = MODE == kGradW ? t.end - t.begin - (t.k_blocks - 1) * kBlockK : 0;
        const int kb_begin = t.k_blocks * share / SPLIT;
        const int kb_end = t.k_blocks * (share + 1) / SPLIT;
        for (int kb = kb_begin; kb < kb_end; kb += kKps) {
          const int nk = min(kKps, kb_end - kb);
          // The rows behind a ragged tail are zeroed by ordinary stores of both CTAs
          // of a pair, so the wait that precedes their MMAs acquires at cluster scope.
          const bool zeroed = CG == 2 && MODE == kGradW && kb + nk == t.k_blocks && ragged_rows(t) != 0;
          const uint32_t full = smem_u32(full_bar + stage);
          if (zeroed ? !warp_wait_cluster(full, phase, abort_flag)
                     : !warp_wait(full, phase, abort_flag)) {
            if (lane == 0) fail(kStatusMma);
            ok = false;
            break;
          }
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < kKps; ++j) {
              if (j >= nk) break;
              const uint32_t sa = smem_u32(smem + stage * Cfg::kStageBytes + j * Cfg::kKBlockBytes);
              const uint32_t sb = sa + Cfg::kABytes;
              int steps = kBlockK / 16;
              if (MODE == kGradW && kb + j == t.k_blocks - 1) steps = (last_rows + 15) / 16;
#pragma unroll
              for (int k = 0; k < kBlockK / 16; ++k) {
                if (MODE == kGradW && k >= steps) break;
                const uint64_t ad = MODE == kGradW ? sdesc_mnmajor_sw128(sa + k * 2048, kChunkBytes)
                                                   : sdesc_kmajor_sw128(sa + k * 32);
                const uint64_t bd = MODE == kForward ? sdesc_kmajor_sw128(sb + k * 32)
                                                     : sdesc_mnmajor_sw128(sb + k * 2048, kChunkBytes);
                const uint32_t accumulate = (kb + j != kb_begin || k != 0) ? 1u : 0u;
                if constexpr (CG == 2) {
                  umma_bf16_pair(d_tmem, ad, bd, kIdesc, accumulate);
                } else {
                  umma_bf16(d_tmem, ad, bd, kIdesc, accumulate);
                }
              }
            }
            grouped_commit<CG>(smem_u32(empty_bar + stage));
          }
          __syncwarp();
          issued_any = true;
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if (elect_one()) grouped_commit<CG>(smem_u32(tfull_bar + acc));
        __syncwarp();
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
  } else if (warp == 3) {
    if constexpr (MODE == kGradW) {
      // ---------------- zeroes the rows behind a group's last one
      int stage = 0;  // slot of this tile's first stage
      uint32_t tail_phase = 0;  // bit s: parity of tail_bar[s]'s next completion
      unsigned long long ahead = 0;  // k-blocks since the last tail: tiles without one are passed over
      for (int tile = worker; tile < num_tiles; tile += workers) {
        const GroupedTile t = grouped_tile<MODE, SWIGLU, CG, BN, ROWS>(p, tables, tile, rank);
        const int stages = (t.k_blocks + kKps - 1) / kKps;
        const int first = ragged_rows(t);
        ahead += t.k_blocks + 1;  // one for storing the tile
        if (first != 0) {
          const int slot = (stage + stages - 1) % kStages;
          const bool got = warp_wait_blocks(smem_u32(tail_bar + slot), (tail_phase >> slot) & 1u,
                                            abort_flag, ahead);
          ahead = 0;
          tail_phase ^= 1u << slot;
          if (!got) {
            if (lane == 0) fail(kStatusProducer);
            break;
          }
          const int j = (t.k_blocks - 1) % kKps;
          uint8_t* block = smem + slot * Cfg::kStageBytes + j * Cfg::kKBlockBytes;
          const int count = ((first + 15) / 16 * 16 - first) * 8;  // 16-byte pieces a chunk
          constexpr int kChunks = static_cast<int>(Cfg::kKBlockBytes / kChunkBytes);
#pragma unroll 1
          for (int c = 0; c < kChunks; ++c) {
            uint4* rows = reinterpret_cast<uint4*>(block + c * kChunkBytes + first * 128);
            for (int i = lane; i < count; i += 32) rows[i] = make_uint4(0u, 0u, 0u, 0u);
          }
          // the MMAs read these rows through the async proxy
          asm volatile("fence.proxy.async;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            const uint32_t fb = smem_u32(full_bar + slot);
            if constexpr (CG == 2) {
              mbar_arrive_cluster(map_to_cta(fb, 0));
            } else {
              mbar_arrive(fb);
            }
          }
          __syncwarp();
        }
        stage = (stage + stages) % kStages;
      }
    }
  } else if (warp >= 4) {
    // ---------------- epilogue: this CTA's 128 rows of the tile
    const int q = warp & 3;
    const int half = (warp - 4) >> 2;
    int local = 0;
    for (int tile = worker; tile < num_tiles; tile += workers) {
      const GroupedTile t = grouped_tile<MODE, SWIGLU, CG, BN, ROWS>(p, tables, tile, rank);
      const int row0 = t.a_row + q * 32;
      // rows of this warp to store; none: they all lie behind the group's last
      const int valid = ROWS == 32 && q != 0
                            ? 0
                            : min((MODE == kGradW ? p.out_rows : t.end) - row0, 32);
      const std::size_t out_row =
          MODE == kGradW ? static_cast<std::size_t>(t.group) * p.out_rows + row0 : row0;
      // output columns of the tile and of this warp
      constexpr int kOut = SWIGLU ? BN / 2 : BN;
      constexpr int kMine = kOut / 2;
      constexpr int kRun = kMine < 64 ? kMine : 64;
      const int mine = half * kMine;
      if (MODE == kGradW && t.k_blocks == 0) {
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) w[i] = 0u;
        for (int c = mine; c < mine + kMine; c += kRun) {
          store_rows64(p, out_row, valid, t.col + c, kRun, w, lane);
        }
        continue;
      }
      const int acc = local & 1;
      if (!epi_wait(smem_u32(tfull_bar + acc), (local >> 1) & 1, abort_flag, lane,
                    blocks_limit_ns(t.k_blocks))) {
        if (lane == 0) fail(kStatusEpilogue);
        break;
      }
      ++local;
      tc_fence_after();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * BN;
      if constexpr (SPLIT > 1) {
        // This warp's 64 sums a row, 32 at a time: of its columns, or gate and up
        // ones of the same outputs.  The first CTA adds the others' in their order;
        // words j .. j + 3 of chunk i lie at (i * 8 + j / 4) * 512 + lane * 16, whole
        // rows of banks for both sides.
        auto chunk = [&](int i) { return t_row + mine + (SWIGLU ? i * (BN / 2) : i * 32); };
        bool got = true;
        if (valid > 0 && share != 0) {
          const uint32_t to =
              map_to_cta(smem_u32(other_sums + ((share - 1) * 2 + half) * Cfg::kSumBytes), 0) + lane * 16;
          const uint32_t bar = map_to_cta(smem_u32(sums_bar + half), 0);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t a[32];
            tmem_ld32(chunk(i), a);
            if (lane < valid) {
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                st_async_v4(to + (i * 8 + j / 4) * 512, a[j], a[j + 1], a[j + 2], a[j + 3], bar);
              }
            }
          }
        } else if (valid > 0) {
          const uint32_t bar = smem_u32(sums_bar + half);
          if (lane == 0) mbar_arrive_expect_tx(bar, (SPLIT - 1) * valid * 64 * 4);
          __syncwarp();
          got = warp_wait_cluster(bar, 0, abort_flag);
          if (got) {
            float f[2][32];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t a[32];
              tmem_ld32(chunk(i), a);
#pragma unroll
              for (int j = 0; j < 32; ++j) f[i][j] = __uint_as_float(a[j]);
              // rows behind the last one read what lies there, and are not stored
#pragma unroll 1
              for (int from = 0; from < SPLIT - 1; ++from) {
                const uint8_t* src = other_sums + (from * 2 + half) * Cfg::kSumBytes + lane * 16;
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                  const float4 v = *reinterpret_cast<const float4*>(src + (i * 8 + j / 4) * 512);
                  f[i][j] += v.x;
                  f[i][j + 1] += v.y;
                  f[i][j + 2] += v.z;
                  f[i][j + 3] += v.w;
                }
              }
            }
            uint32_t w[32];
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              if constexpr (SWIGLU) {
                w[j / 2] = pack_bf16x2(silu_fast(f[0][j]) * f[1][j], silu_fast(f[0][j + 1]) * f[1][j + 1]);
                w[16 + j / 2] = 0u;
              } else {
                w[j / 2] = pack_bf16x2(f[0][j], f[0][j + 1]);
                w[16 + j / 2] = pack_bf16x2(f[1][j], f[1][j + 1]);
              }
            }
            store_rows64(p, out_row, valid, t.col + mine, kRun, w, lane);
          }
        }
        if (!got) {
          if (lane == 0) fail(kStatusEpilogue);
          break;
        }
      } else if (valid > 0) {
#pragma unroll 1
        for (int c = mine; c < mine + kMine; c += kRun) {
          uint32_t w[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) w[i] = 0u;
          if constexpr (SWIGLU) {
#pragma unroll
            for (int h = 0; h < kRun; h += 16) {
              uint32_t g[16], u[16];
              tmem_ld16x2(t_row + c + h, t_row + BN / 2 + c + h, g, u);
#pragma unroll
              for (int j = 0; j < 16; j += 2) {
                w[(h + j) / 2] = pack_bf16x2(
                    silu_fast(__uint_as_float(g[j])) * __uint_as_float(u[j]),
                    silu_fast(__uint_as_float(g[j + 1])) * __uint_as_float(u[j + 1]));
              }
            }
          } else {
#pragma unroll
            for (int h = 0; h < kRun; h += 32) {
              static_assert(SWIGLU || kRun >= 32, "columns of a run");
              uint32_t a[32];
              tmem_ld32(t_row + c + h, a);
#pragma unroll
              for (int j = 0; j < 32; j += 2) {
                w[(h + j) / 2] = pack_bf16x2(__uint_as_float(a[j]), __uint_as_float(a[j + 1]));
              }
            }
          }
          store_rows64(p, out_row, valid, t.col + c, kRun, w, lane);
        }
      }
      const uint32_t bar = smem_u32(tempty_bar + acc);
      release_sum<CG>(CG == 2 ? map_to_cta(bar, 0) : bar, lane);
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
      tmem_dealloc_pair(tmem_base, Cfg::kTmemCols);
    } else {
      tmem_dealloc(tmem_base, Cfg::kTmemCols);
    }
  }
}

template <int MODE, bool SWIGLU, int CG, int BN, int ROWS, int SPLIT>
__global__ void __cluster_dims__(CG * SPLIT, 1, 1) __launch_bounds__(kCtaThreads, 1)
    grouped_bf16_kernel(const __grid_constant__ GroupedParams p) {
  grouped_bf16_cta<MODE, SWIGLU, CG, BN, ROWS, SPLIT>(p, blockIdx.x / (CG * SPLIT),
                                                      gridDim.x / (CG * SPLIT));
}

// Both gradients of a small product in one launch, side by side: the first
// input_ctas CTAs compute the one by x, the others the one by W.
template <int ROWS>
__global__ void __launch_bounds__(kCtaThreads, 1)
    grouped_bf16_backward_kernel(const __grid_constant__ GroupedParams by_x,
                                 const __grid_constant__ GroupedParams by_w, int input_ctas) {
  const int cta = blockIdx.x;
  if (cta < input_ctas) {
    grouped_bf16_cta<kGradX, false, 1, 128, ROWS, 1>(by_x, cta, input_ctas);
  } else {
    grouped_bf16_cta<kGradW, false, 1, 128, kBlockM, 1>(by_w, cta - input_ctas,
                                                        gridDim.x - input_ctas);
  }
}

}  // namespace sm100
}  // namespace col
