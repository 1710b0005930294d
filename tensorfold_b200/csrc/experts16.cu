// Grouped MoE experts on 16-bit weights (bf16 or fp16): matrix products grouped by expert with ragged sizes, on tcgen05.
//
//   gate_up   act[p, n] = f(sum_k x[p / slots, k] U[e(p), n, k])       f: SwiGLU of (gate, up) or relu^2 of up
//   down      y[p, n]   = sum_k act[p, k] D[e(p), n, k]
//
// over the (row, slot) pairs p that a plan has sorted by expert into items of at most `tile` pairs of one expert.  The
// WEIGHTS are the MMA's A operand (128 rows of one expert), an item's PAIRS the B operand (N = pairs rounded up to 16 or
// 32), so an expert with three pairs costs an N of 16 and no padded row is ever written.  One fp32 chain over K in order of
// inputs: a pair's bits do not depend on its item, on the tile or on the call.
//
// What bounds it.  Few pairs an expert: HBM - 64 tokens of 128 experts (2048 x 768, top 8), gate/up 119 us for 793 MB, 1.02 of
// the copy rate; one token 14 us for 50 MB, of which 9 stream and the rest is start, plan and end.  Some hundred pairs: HBM
// and the tensor pipe in turn - 1999 tokens 145 us, DRAM 73 % of its peak, tensor pipe 40 % busy.  Many: the tensor pipe, 79 %
// busy at 4096 tokens of 32 experts (160 us, 1290 TFLOP/s), and on long runs the clock that the power cap leaves it: 8192 tokens
// of 160 experts (4096 x 1536) run at 877 MHz and 873 TFLOP/s, 0.82 of what the pipe can do at that clock (a plain 8192-cubed
// library product holds 1327 MHz and 1380 TFLOP/s under the same cap, so an operation costs more energy here).

#include "api.h"
#include "common.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

namespace tfb {

// ---- packed weights --------------------------------------------------------------------------------------------------
// Per expert R rows (one matrix: its N columns, rounded up to 16 with zero rows; gate and up: alternating runs of 16 gate
// and the same 16 up columns) by KB blocks of 64 inputs (K rounded up with zeros).  Tile t = rows 128 t .. (the last may be
// shorter); within a tile the blocks of 64 inputs follow one another, each rows_of_tile x 128 bytes, already in the
// 128-byte swizzle (16-byte chunk c of row r at c ^ (r & 7)).  So a tile's block is ONE contiguous run of HBM that a bulk
// copy brings straight into an operand tile.
constexpr int W16_ROWS = 128;
constexpr int W16_K = 64;

__host__ __device__ __forceinline__ int w16_rows(int mats, int n) { return mats * ((n + 15) / 16 * 16); }
__host__ __device__ __forceinline__ int w16_kblocks(int k) { return (k + W16_K - 1) / W16_K; }

// The place of 16-byte chunk i of a packed expert, as (matrix, column, input); the inverse of the layout above.
__device__ __forceinline__ void w16_chunk(int64_t i, int mats, int rows, int kb, int& m, int& col, int& k) {
  const int64_t tile_chunks = (int64_t)W16_ROWS * kb * 8;
  const int t = (int)(i / tile_chunks);
  const int64_t in_tile = i - t * tile_chunks;
  const int rt = min(W16_ROWS, rows - t * W16_ROWS);
  const int b = (int)(in_tile / (rt * 8)), rest = (int)(in_tile - (int64_t)b * rt * 8);
  const int r = rest >> 3, c = (rest & 7) ^ (r & 7), row = t * W16_ROWS + r;
  m = mats == 2 ? (row >> 4) & 1 : 0;
  col = mats == 2 ? (row >> 5) * 16 + (row & 15) : row;
  k = b * W16_K + c * 8;
}

__global__ void __launch_bounds__(256)
pack16_kernel(const uint8_t* m0, const uint8_t* m1, uint4* out, int mats, int n, int k, int rows, int kb) {
  const int64_t per = (int64_t)rows * kb * 8;
  const int e = blockIdx.y;
  pdl_wait();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < per; i += (int64_t)gridDim.x * 256) {
    int m, col, kk;
    w16_chunk(i, mats, rows, kb, m, col, kk);
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (col < n && kk < k)
      v = *reinterpret_cast<const uint4*>((m ? m1 : m0) + 2 * (((int64_t)e * n + col) * k + kk));
    out[e * per + i] = v;
  }
}

__global__ void __launch_bounds__(256)
unpack16_kernel(const uint4* packed, uint8_t* m0, uint8_t* m1, int mats, int n, int k, int rows, int kb) {
  const int64_t per = (int64_t)rows * kb * 8;
  const int e = blockIdx.y;
  pdl_wait();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < per; i += (int64_t)gridDim.x * 256) {
    int m, col, kk;
    w16_chunk(i, mats, rows, kb, m, col, kk);
    if (col < n && kk < k)
      *reinterpret_cast<uint4*>((m ? m1 : m0) + 2 * (((int64_t)e * n + col) * k + kk)) = packed[e * per + i];
  }
}

// ---- the grouped product ---------------------------------------------------------------------------------------------
// Persistent: the CTAs (CG = 1), or pairs of CTAs whose tensor cores work as one (CG = 2), walk units = (item, 128 CG rows of
// its expert's weights).  A CTA's roles run apart, each through all of its units, so that the copies of the next unit
// travel while the last one is finished:
//   one warp   the weights' bulk copies: 128 rows;  four or eight warps the pairs' input rows by TMA gathers (four rows an
//              instruction, zeros behind the last input), of a pair of CTAs each one half; both into a ring of stages of
//              64 inputs, 16 KB of weights each;
//   one warp   (of a pair's first CTA, on whose barriers both CTAs' copies count) issues tcgen05.mma (M = 128 CG, N = pairs)
//              into one of two accumulators in tensor memory;
//   four or eight warps  read the other accumulator, apply the activation and store the pairs' rows: through shared memory,
//              where a lane's one column of many pairs becomes 16 bytes of a pair's row.  (Stored from the registers, 2
//              bytes a lane, a unit of 256 pairs took 14 us to finish where its products take 3 to 9.)
// A role's loop runs in all lanes of its warp with one lane elected for the issue: addresses and descriptors stay in uniform
// registers.  (In a loop of lane 0 alone an MMA took 80 cycles to issue, and at few pairs that was the kernel's time.)
constexpr int G16_MAXP = 256;                      // pairs an item may hold (MMA N)
constexpr int G16_FEW = 32;                        // pairs up to which a launch makes its own plan

template <int CG, int MAXP>
struct G16Shape {
  static constexpr int EPI_WARPS = 4 * CG, B_WARPS = 4 * CG;               // finishing, gathering
  static constexpr int MMA_WARP = EPI_WARPS, A_WARP = MMA_WARP + 1, B_WARP = A_WARP + 1;
  static constexpr int THREADS = (B_WARP + B_WARPS) * 32;
  static constexpr int A_BYTES = W16_ROWS * 128, B_BYTES = MAXP / CG * 128;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = (206 * 1024 / STAGE) < 10 ? (206 * 1024 / STAGE) : 10;
  static constexpr int TABLE_OFFSET = STAGES * STAGE;                      // int pair[2][MAXP]
  static constexpr int TURN_OFFSET = TABLE_OFFSET + 2 * MAXP * 4;          // the finishing warps' rows: 2 KB each
  static constexpr int FEW_OFFSET = TURN_OFFSET + EPI_WARPS * 2048;        // plan_few's items, members and item count
  static constexpr int BAR_OFFSET = FEW_OFFSET + (4 * G16_FEW + 2) * 4;
  static constexpr int TMEM_OFFSET = BAR_OFFSET + (2 * STAGES + 4) * 8;
  static constexpr int TOTAL = TMEM_OFFSET + 16 + 1024;                    // + slack to align the tiles to 1024 bytes
  static constexpr int ACC_COLS = MAXP;                                    // tensor memory: two accumulators
  static constexpr int STEP = 16 * CG;                                     // N is a multiple of it
  static constexpr int LANES = (MAXP / CG / 4 + B_WARPS - 1) / B_WARPS;    // lanes of a gathering warp with a group of rows
  static_assert(TOTAL <= 227 * 1024, "one CTA's shared memory");
  static_assert(ACC_COLS >= 32 && 2 * ACC_COLS <= 512 && LANES >= 1 && LANES <= 32, "tensor memory; the gathers");
};

template <bool F16>
__device__ __forceinline__ uint16_t to16(float v) {
  if constexpr (F16) return __half_as_ushort(__float2half_rn(v));
  else return __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

// SwiGLU on the fp32 sums: silu(g) u, clipped first when limit > 0; the only rounding is the caller's to 16 bits.  (The
// 4-bit experts round gate, up and silu to bf16 on the way, as their reference does; here nothing asks for it.)
__device__ __forceinline__ float swiglu32(float g, float u, float limit) {
  if (limit > 0.f) {
    g = g > limit ? limit : g;                      // comparisons, not fminf: a NaN stays one
    u = u > limit ? limit : u < -limit ? -limit : u;
  }
  return __fdividef(g, 1.f + __expf(-g)) * u;
}

template <int CG>
__device__ __forceinline__ void umma_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accum)
        : "memory");
  else
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accum)
        : "memory");
}

// kind::f16, D fp32, both operands K-major, bf16 or fp16, M = 128 CG, N = n
template <int CG, bool F16>
__device__ __forceinline__ uint32_t g16_idesc(int n) {
  const uint32_t type = F16 ? 0u : 1u;
  return (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(CG * W16_ROWS >> 4) << 24);
}

// The MMAs so far have retired: one arrival on the barrier, of a pair of CTAs on both CTAs' barriers in that place.
template <int CG>
__device__ __forceinline__ void g16_commit(uint64_t* bar) {
  if constexpr (CG == 1)
    umma_commit(bar);
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(
                     smem_addr(bar)),
                 "h"((uint16_t)3)
                 : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

template <int CG>
__device__ __forceinline__ void g16_alloc(uint32_t* dst_smem, uint32_t ncols) {
  if constexpr (CG == 1) {
    tmem_alloc(dst_smem, ncols);
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_addr(dst_smem)), "r"(ncols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void g16_dealloc(uint32_t taddr, uint32_t ncols) {
  if constexpr (CG == 1) tmem_dealloc(taddr, ncols);
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(taddr), "r"(ncols) : "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }

// The first CTA's barrier (or other shared memory) in the place of this CTA's, as a shared::cluster address.
__device__ __forceinline__ uint32_t leader_addr(const void* p) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;\n" : "=r"(at) : "r"(smem_addr(p)));
  return at;
}
__device__ __forceinline__ void mbar_arrive_leader(uint64_t* bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(leader_addr(bar)) : "memory");
}

__device__ __forceinline__ void mbar_expect_tx_at(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.relaxed.cluster.shared::cluster.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ bool elect_one() {
  uint32_t on;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(on));
  return on != 0;
}

// Four rows' 64 inputs from column `col` on into 512 bytes of a swizzled operand tile; zeros behind the map's columns.  `bar`:
// a shared::cluster address; of a pair of CTAs both count on the first one's barrier.
template <int CG>
__device__ __forceinline__ void tma_gather4(void* dst, const CUtensorMap* map, int col, int4 r, uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, "
        "%6}], [%7];\n" ::"r"(smem_addr(dst)),
        "l"(map), "r"(col), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, "
        "{%2, %3, %4, %5, %6}], [%7];\n" ::"r"(smem_addr(dst)),
        "l"(map), "r"(col), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w), "r"(bar)
        : "memory");
}

// A tile of whole rows of the packed weights, as they are, for one CTA of a pair.
__device__ __forceinline__ void tma_rows_pair(void* dst, const CUtensorMap* map, int row, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], "
      "[%4];\n" ::"r"(smem_addr(dst)),
      "l"(map), "r"(0), "r"(row), "r"(bar)
      : "memory");
}

__device__ __forceinline__ int ld_any(const int* p) {                      // ld_dep, of a table in global or in shared memory
  int v;
  asm volatile("ld.s32 %0, [%1];\n" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// The plan of at most 32 pairs, by one warp into shared memory: what tfb_plan writes, without its launch (3.5 us where one
// token goes through 128 experts).  A lane holds a pair; its place is the number of lanes with a lower expert, by a ballot a
// bit, and of earlier lanes with the same.  (With a shuffle a lane it took 2.3 us, all warps waiting.)
__device__ __forceinline__ void plan_few(const int* picks, int pairs, int experts, int tile, int* items, int* members, int* n_items) {
  constexpr unsigned ALL = 0xffffffffu;
  const int lane = threadIdx.x & 31, bits = 32 - __clz(experts - 1);       // one expert: __clz(0) = 32
  const int e = lane < pairs ? ld_dep(picks + lane) : -1;
  const bool live = e >= 0 && e < experts;
  unsigned same = __ballot_sync(ALL, live), lower = 0;
  for (int b = bits - 1; b >= 0; --b) {
    const bool set = (e >> b) & 1;
    const unsigned with = __ballot_sync(ALL, set);
    if (set) lower |= same & ~with;
    same &= set ? with : ~with;
  }
  const int mine = __popc(same & ((1u << lane) - 1)), first = __popc(lower), at = first + mine;
  const bool head = live && mine % tile == 0;                              // opens an item
  const unsigned heads = __reduce_or_sync(ALL, head ? 1u << at : 0u);      // by place
  if (live) members[at] = lane;
  if (head) {
    int* item = items + 3 * __popc(heads & ((1u << at) - 1));
    item[0] = e;
    item[1] = at;
    item[2] = min(tile, __popc(same) - mine);
  }
  if (lane == 0) *n_items = __popc(heads);
}

struct RingAt {                                     // a walk around the ring of stages
  int s = 0;
  uint32_t ph = 0;
  int steps = 0;
  __device__ __forceinline__ void next(int stages) {
    ++steps;
    if (++s == stages) {
      s = 0;
      ph ^= 1;
    }
  }
  // after a wait that ran out: gives the copies in flight of the last round a while to land (`here`: they count on this CTA's
  // barriers)
  __device__ __forceinline__ void drain(uint64_t* full, int stages, bool here) {
    const uint64_t start = global_ns();
    while (!here && global_ns() - start < 10000000ull) {
    }
    if (!here) return;
    for (int i = min(steps, stages); i > 0; --i) {
      ph ^= s == 0;
      s = s == 0 ? stages - 1 : s - 1;
      mbar_wait_for(full + s, ph, 10000000ull);
    }
  }
};

// Every role reads what it needs of the plan one unit ahead: behind the last copy of a unit the chain item -> members ->
// rows took 2 us in which the ring ran dry.
template <int CG, int M, int EPI, bool F16, int MAXP>
__global__ void __launch_bounds__(G16Shape<CG, MAXP>::THREADS, 1)
g16_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, int slots,
           const uint8_t* __restrict__ W, int K, int N, const int* items, const int* counts, const int* members, const int* picks,
           int pairs, int experts, int tile, void* __restrict__ out, float limit) {
  using SH = G16Shape<CG, MAXP>;
  constexpr int STAGES = SH::STAGES, B_WARPS = SH::B_WARPS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  int* table = reinterpret_cast<int*>(smem + SH::TABLE_OFFSET);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + SH::BAR_OFFSET);     // [STAGES] weights and inputs landed
  uint64_t* empty = full + STAGES;                                         // [STAGES] the MMAs that read them retired
  uint64_t* acc_full = empty + STAGES;                                     // [2] a unit's sums are complete
  uint64_t* acc_free = acc_full + 2;                                       // [2] and have been read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + SH::TMEM_OFFSET);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int cta = CG == 1 ? 0 : (int)cluster_rank();                       // of the pair; 0 issues the MMAs
  const int rows = w16_rows(M, N), KB = w16_kblocks(K), nct = (rows + CG * W16_ROWS - 1) / (CG * W16_ROWS);
  const int u0 = blockIdx.x / CG, du = gridDim.x / CG;

  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      // every warp that waits for `empty` arrives here: one that had no part in a stage could fall a round behind and mistake
      // the barrier's phase
      mbar_init(full + s, CG * (1 + B_WARPS));
      mbar_init(empty + s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(acc_full + s, 1);
      mbar_init(acc_free + s, SH::EPI_WARPS * CG);
    }
    mbar_fence_init();
    fence_async_smem();
  }
  if (warp == SH::MMA_WARP) g16_alloc<CG>(tmem_slot, 2 * SH::ACC_COLS);
  pdl_wait();
  pdl_launch_dependents();                          // what follows waits for this grid's end all the same: its start is hidden
  after_wait(items, counts, members, picks);
  if (picks != nullptr) {
    int* few = reinterpret_cast<int*>(smem + SH::FEW_OFFSET);
    if (warp == 0) plan_few(picks, pairs, experts, tile, few, few + 3 * G16_FEW, few + 4 * G16_FEW);
    items = few;
    members = few + 3 * G16_FEW;
    counts = few + 4 * G16_FEW;
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) {
    cluster_arrive();
    cluster_wait();
  }
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int units = __shfl_sync(0xffffffffu, ld_any(counts), 0) * nct;
  bool ok = true;
  auto item = [&](int u) { return min(u, units - 1) / nct; };              // of the next unit, or any where there is none
  auto known = [&](int p) { return p < pairs ? p : -1; };                  // a plan of more rows than this call has

  if (units == 0) {
  } else if (warp == SH::A_WARP) {
    RingAt at;
    int e = ld_any(items + 3 * item(u0));
    for (int u = u0; u < units && ok; u += du) {
      const int r0 = ((u - u / nct * nct) * CG + cta) * W16_ROWS, t0 = r0 < rows ? r0 : 0;   // a second CTA without rows: any
      const int rt = min(W16_ROWS, rows - t0);
      const int ee = __shfl_sync(0xffffffffu, e, 0);
      const uint8_t* src = W + ((size_t)ee * rows + t0) * KB * 128;
      const int row = (ee * rows + t0) * KB;
      e = ld_any(items + 3 * item(u + du));
      for (int f = 0; f < KB; ++f) {
        ok = mbar_wait_warp(empty + at.s, at.ph ^ 1);                      // the ring's first round finds every stage free
        if (!ok) break;
        uint8_t* dst = smem + at.s * SH::STAGE;
        if (elect_one()) {
          if constexpr (CG == 1) {
            mbar_expect_tx(full + at.s, (uint32_t)rt * 128);
            bulk_g2s(dst, src + (size_t)f * rt * 128, rt * 128, full + at.s);
          } else {                                                         // 128 rows: behind a shorter tile's, the next block's
            const uint32_t bar = leader_addr(full + at.s);
            mbar_expect_tx_at(bar, SH::A_BYTES);
            tma_rows_pair(dst, &wmap, row + f * rt, bar);
          }
        }
        __syncwarp();
        at.next(STAGES);
      }
    }
    // once around: the last MMAs' arrivals on `empty` land before the CTA's shared memory goes to another
    for (int i = 0; i < STAGES && ok; ++i) {
      ok = mbar_wait_warp(empty + at.s, at.ph ^ 1);
      at.next(STAGES);
    }
    if (!ok) at.drain(full, STAGES, cta == 0);
    __syncwarp();
  } else if (warp >= SH::B_WARP) {
    // Lane l of warp w takes group l * B_WARPS + w of four rows.  A warp's gathers follow one another every 130 cycles,
    // whichever lanes issue them, hence the warps.
    const int g = lane * B_WARPS + warp - SH::B_WARP;
    RingAt at;
    int4 next;
    int next_cnt;
    auto fetch = [&](int u) {
      const int it = item(u);
      const int first = ld_any(items + 3 * it + 1);
      next_cnt = min(ld_any(items + 3 * it + 2), MAXP);
      const int half = (next_cnt + SH::STEP - 1) / SH::STEP * SH::STEP / CG;   // pairs of this CTA
      const int p = cta * half + 4 * g;                                    // rows past the last pair repeat it: never stored
      if (lane < SH::LANES) {
        next.x = ld_any(members + first + min(p, next_cnt - 1));
        next.y = ld_any(members + first + min(p + 1, next_cnt - 1));
        next.z = ld_any(members + first + min(p + 2, next_cnt - 1));
        next.w = ld_any(members + first + min(p + 3, next_cnt - 1));
      }
    };
    fetch(u0);
    for (int u = u0; u < units && ok; u += du) {
      int4 r = next;
      if (slots) r = make_int4(r.x / slots, r.y / slots, r.z / slots, r.w / slots);
      const int groups = (next_cnt + SH::STEP - 1) / SH::STEP * SH::STEP / CG / 4;     // of this CTA
      const int here = max(0, (groups - (warp - SH::B_WARP) + B_WARPS - 1) / B_WARPS);   // of this warp
      fetch(u + du);
      for (int f = 0; f < KB; ++f) {
        ok = mbar_wait_warp(empty + at.s, at.ph ^ 1);
        if (!ok) break;
        uint8_t* dst = smem + at.s * SH::STAGE + SH::A_BYTES + g * 512;
        const uint32_t bar = CG == 1 ? smem_addr(full + at.s) : leader_addr(full + at.s);
        if (lane == 0) {
          if constexpr (CG == 1) mbar_expect_tx(full + at.s, (uint32_t)here * 512);
          else mbar_expect_tx_at(bar, (uint32_t)here * 512);
        }
        __syncwarp();
        if (lane < SH::LANES && g < groups)
          tma_gather4<CG>(dst, &xmap, f * W16_K, r, bar);
        __syncwarp();
        at.next(STAGES);
      }
    }
    if (!ok) at.drain(full, STAGES, cta == 0);
    __syncwarp();
  } else if (warp == SH::MMA_WARP) {
    if (cta == 0) {
      const uint64_t a0 = umma_desc(smem_addr(smem)), b0 = umma_desc(smem_addr(smem + SH::A_BYTES));
      RingAt at;
      int n = 0;                                                           // the CTA's n-th unit
      int next_cnt = ld_any(items + 3 * item(u0) + 2);
      for (int u = u0; u < units && ok; u += du, ++n) {
        const int cnt = min(__shfl_sync(0xffffffffu, next_cnt, 0), MAXP);
        next_cnt = ld_any(items + 3 * item(u + du) + 2);
        const uint32_t idesc = g16_idesc<CG, F16>((cnt + SH::STEP - 1) / SH::STEP * SH::STEP);
        const uint32_t acc = tmem_base + (n & 1) * SH::ACC_COLS;
        ok = mbar_wait_warp(acc_free + (n & 1), ((n >> 1) & 1) ^ 1);
        if (!ok) break;
        if constexpr (CG == 2) asm volatile("fence.acq_rel.cluster;\n" ::: "memory");   // the other CTA's arrivals
        tc_fence_after();
        for (int f = 0; f < KB; ++f) {
          ok = mbar_wait_warp(full + at.s, at.ph);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint32_t off = (uint32_t)(at.s * SH::STAGE) >> 4;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) umma_ss<CG>(acc, a0 + off + 2 * ks, b0 + off + 2 * ks, idesc, (f | ks) ? 1u : 0u);
            g16_commit<CG>(empty + at.s);
            if (f == KB - 1) g16_commit<CG>(acc_full + (n & 1));
          }
          __syncwarp();
          at.next(STAGES);
        }
      }
    }
  } else {
    // ---- the finishing warps: tensor-memory lane = weight row, column = pair ----
    const int q = warp & 3, part = warp >> 2;                              // quarter of the lanes; share of the pairs
    uint8_t* turn = smem + SH::TURN_OFFSET + warp * 2048;
    int n = 0;
    int first = ld_any(items + 3 * item(u0) + 1), cnt = ld_any(items + 3 * item(u0) + 2);
    for (int u = u0; u < units && ok; u += du, ++n) {
      const int r0 = ((u - u / nct * nct) * CG + cta) * W16_ROWS, have = min(cnt, MAXP);
      int* pair = table + (n & 1) * MAXP;
      for (int i = tid; i < ((have + 31) & ~31); i += SH::EPI_WARPS * 32) pair[i] = i < have ? known(ld_any(members + first + i)) : -1;
      first = ld_any(items + 3 * item(u + du) + 1);
      cnt = ld_any(items + 3 * item(u + du) + 2);
      asm volatile("bar.sync 1, %0;\n" ::"n"(SH::EPI_WARPS * 32) : "memory");
      ok = mbar_wait_warp(acc_full + (n & 1), (n >> 1) & 1);
      if (!ok) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + (n & 1) * SH::ACC_COLS + ((uint32_t)(q * 32) << 16);
      constexpr int OUT = EPI == EPI_F32 ? 4 : 2;                          // bytes of a value
      constexpr int COLS_W = M == 1 ? 32 : 16;                             // columns a warp holds
      constexpr int TURN = EPI == EPI_F32 ? 16 : 32;                       // pairs a turn: 2 KB or 1
      constexpr int CHUNKS = COLS_W * OUT / 16;                            // 16-byte pieces of a pair's row
      const int c0 = r0 / M + q * COLS_W;                                  // the warp's first column
      const bool wide = ((size_t)N * OUT) % 16 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
      for (int j0 = part * TURN; j0 < have && c0 < N; j0 += SH::EPI_WARPS / 4 * TURN) {
        uint32_t a[32];
        if constexpr (TURN == 32) tmem_ld32(taddr + j0, a);
        else tmem_ld16(taddr + j0, *reinterpret_cast<uint32_t(*)[16]>(a));
        tmem_ld_wait();
        __syncwarp();                                                      // the turn before this one has been read
        if constexpr (M == 2) {
          // a column's gate and up rows sit 16 lanes apart: of two neighbouring pairs the gate lane forms the first
          // and the up lane the second
          static_assert(EPI == EPI_SWIGLU, "two matrices: gate and up");
          const bool up_lane = lane >= 16;
#pragma unroll
          for (int j = 0; j < TURN / 2; ++j) {
            const float give = __uint_as_float(up_lane ? a[2 * j] : a[2 * j + 1]);
            const float keep = __uint_as_float(up_lane ? a[2 * j + 1] : a[2 * j]);
            const float got = __shfl_xor_sync(0xffffffffu, give, 16);
            reinterpret_cast<uint16_t*>(turn)[2 * j * COLS_W + lane] =
                to16<F16>(swiglu32(up_lane ? got : keep, up_lane ? keep : got, limit));
          }
        } else {
#pragma unroll
          for (int j = 0; j < TURN; ++j) {
            float v = __uint_as_float(a[j]);
            if constexpr (EPI == EPI_RELU2) v = v > 0.f ? v * v : v != v ? v : 0.f;      // NaN stays NaN
            if constexpr (EPI == EPI_F32) reinterpret_cast<float*>(turn)[j * COLS_W + lane] = v;
            else reinterpret_cast<uint16_t*>(turn)[j * COLS_W + lane] = to16<F16>(v);
          }
        }
        __syncwarp();
        if (wide) {
#pragma unroll
          for (int i = 0; i < TURN * CHUNKS / 32; ++i) {
            const int at = i * 32 + lane, p = pair[j0 + at / CHUNKS], c = c0 + at % CHUNKS * (16 / OUT);
            const uint4 v = *reinterpret_cast<const uint4*>(turn + at * 16);
            if (p >= 0 && c < N) *reinterpret_cast<uint4*>(static_cast<uint8_t*>(out) + ((size_t)p * N + c) * OUT) = v;
          }
        } else {
          for (int at = lane; at < TURN * COLS_W; at += 32) {
            const int p = pair[j0 + at / COLS_W], c = c0 + at % COLS_W;
            if (p < 0 || c >= N) continue;
            if constexpr (EPI == EPI_F32) static_cast<float*>(out)[(size_t)p * N + c] = reinterpret_cast<const float*>(turn)[at];
            else static_cast<uint16_t*>(out)[(size_t)p * N + c] = reinterpret_cast<const uint16_t*>(turn)[at];
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 1) mbar_arrive(acc_free + (n & 1));
        else mbar_arrive_leader(acc_free + (n & 1));
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) {                                                 // nobody arrives on this CTA's barriers any more
    cluster_arrive();
    cluster_wait();
  }
  if (warp == SH::MMA_WARP) g16_dealloc<CG>(tmem_base, 2 * SH::ACC_COLS);
}

// The driver's encoder of tensor maps, looked up once.
inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult got;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &got) != cudaSuccess ||
        got != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

template <int CG, int M, int EPI, bool F16, int MAXP>
int launch_g16(const void* x, int64_t x_stride, int64_t x_rows, int slots, const void* w, int experts, int k, int n, const int* items,
               const int* counts, const int* members, const int* picks, int pairs, int tile, void* out, float limit,
               int64_t max_items, cudaStream_t stream) {
  using SH = G16Shape<CG, MAXP>;
  auto* kern = g16_kernel<CG, M, EPI, F16, MAXP>;
  static bool configured[64] = {false};
  int dev = 0;
  TFB_CUDA(cudaGetDevice(&dev), "experts16: cudaGetDevice");
  if (dev < 0 || dev >= 64) return fail(TFB_ERR_ARG, "experts16: device index %d out of range", dev);
  if (!configured[dev]) {
    TFB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SH::TOTAL),
             "experts16: shared memory opt-in");
    configured[dev] = true;
  }
  auto* encode = tensor_map_encoder();
  if (encode == nullptr) return fail(TFB_ERR_CUDA, "experts16: the driver has no cuTensorMapEncodeTiled");
  CUtensorMap map;
  const cuuint64_t sizes[2] = {(cuuint64_t)k, (cuuint64_t)x_rows}, strides[1] = {(cuuint64_t)x_stride * 2};
  const cuuint32_t box[2] = {W16_K, 1}, steps[2] = {1, 1};
  const CUresult rc = encode(&map, F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                             const_cast<void*>(x), sizes, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) return fail(TFB_ERR_CUDA, "experts16: no tensor map of x (%d)", (int)rc);
  CUtensorMap wmap = map;                                                  // read by pairs of CTAs alone
  if (CG == 2) {
    const int64_t lines = (int64_t)experts * w16_rows(M, n) * w16_kblocks(k);
    if (lines >= (int64_t(1) << 31)) return fail(TFB_ERR_ARG, "experts16: weights of 2^31 lines of 64 inputs or more");
    const cuuint64_t w_sizes[2] = {W16_K, (cuuint64_t)lines}, w_strides[1] = {W16_K * 2};
    const cuuint32_t w_box[2] = {W16_K, W16_ROWS};
    const CUresult wrc = encode(&wmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(w), w_sizes, w_strides, w_box, steps,
                                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (wrc != CUDA_SUCCESS) return fail(TFB_ERR_CUDA, "experts16: no tensor map of the weights (%d)", (int)wrc);
  }
  const int64_t units = max_items * ((w16_rows(M, n) + CG * W16_ROWS - 1) / (CG * W16_ROWS));
  if (units >= (int64_t(1) << 30)) return fail(TFB_ERR_ARG, "experts16: too many units");
  const int64_t most = sm_count() / CG, walkers = units < most ? units : most;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(walkers * CG));
  cfg.blockDim = dim3(SH::THREADS);
  cfg.dynamicSmemBytes = SH::TOTAL;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = CG == 1 ? attr + 1 : attr;
  cfg.numAttrs = (CG == 1 ? 0 : 1) + (g_use_pdl ? 1 : 0);
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, map, wmap, slots, static_cast<const uint8_t*>(w), k, n, items, counts, members,
                                       picks, pairs, experts, tile, out, limit),
                    "experts16");
}

}  // namespace tfb

using namespace tfb;

static int pack16_check(const char* what, const void* packed, const void* m0, const void* m1, int experts, int n, int k) {
  TFB_REQUIRE(packed && m0, "%s: null pointer", what);
  TFB_REQUIRE(aligned16(packed) && aligned16(m0) && aligned16(m1), "%s: 16-byte aligned tensors", what);
  TFB_REQUIRE(experts >= 1 && experts <= 65535 && n >= 1 && k >= 8 && k % 8 == 0 && n < (1 << 24) && k < (1 << 24),
              "%s: [%d, %d, %d] does not pack (inputs in multiples of 8)", what, experts, n, k);
  return TFB_OK;
}

// 16-bit weights [E, n, k] (m1: the up matrix beside the gate m0, or null) into the layout the grouped kernel reads:
// out [E, mats * (n up to 16), k up to 64] in the same 16-bit type.
extern "C" int tfb_pack16(const void* m0, const void* m1, void* out, int experts, int n, int k, void* stream) {
  if (int rc = pack16_check("pack16", out, m0, m1, experts, n, k)) return rc;
  const int mats = m1 ? 2 : 1, rows = w16_rows(mats, n), kb = w16_kblocks(k);
  const int64_t blocks = ((int64_t)rows * kb * 8 + 1023) / 1024;
  return check_cuda(launch(pack16_kernel, dim3((unsigned)(blocks < 65536 ? blocks : 65536), experts), dim3(256), 0,
                           static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(m0), static_cast<const uint8_t*>(m1),
                           static_cast<uint4*>(out), mats, n, k, rows, kb),
                    "pack16");
}

// tfb_pack16's inverse
extern "C" int tfb_unpack16(const void* packed, void* m0, void* m1, int experts, int n, int k, void* stream) {
  if (int rc = pack16_check("unpack16", packed, m0, m1, experts, n, k)) return rc;
  const int mats = m1 ? 2 : 1, rows = w16_rows(mats, n), kb = w16_kblocks(k);
  const int64_t blocks = ((int64_t)rows * kb * 8 + 1023) / 1024;
  return check_cuda(launch(unpack16_kernel, dim3((unsigned)(blocks < 65536 ? blocks : 65536), experts), dim3(256), 0,
                           static_cast<cudaStream_t>(stream), static_cast<const uint4*>(packed), static_cast<uint8_t*>(m0),
                           static_cast<uint8_t*>(m1), mats, n, k, rows, kb),
                    "unpack16");
}

// `picks` null: over the plan in items, counts and members, the call's `pairs` of it; else these are not read and the launch
// sorts the `pairs` picks.
static int experts16_run(int epi, int fp16, const void* x, int64_t x_stride, int64_t x_rows, int slots, const void* w, int experts,
                         int k, int n, const int32_t* items, const int32_t* counts, const int32_t* members, const int32_t* picks,
                         int pairs, void* out, float limit, int64_t max_items, int tile, cudaStream_t st) {
#define TFB_G16_AT(CG_, EPI_, M_, F16_, MAXP_)                                                                              \
  return launch_g16<CG_, M_, EPI_, F16_, MAXP_>(x, x_stride, x_rows, slots, w, experts, k, n, items, counts, members, picks,  \
                                                pairs, tile, out, limit, max_items, st)
#define TFB_G16(EPI_, M_, F16_)                             \
  do {                                                      \
    if (tile > 128) TFB_G16_AT(2, EPI_, M_, F16_, 256);     \
    if (tile > 32) TFB_G16_AT(2, EPI_, M_, F16_, 128);      \
    TFB_G16_AT(1, EPI_, M_, F16_, 32);                      \
  } while (0)
#define TFB_G16_EPI(EPI_, M_)          \
  if (epi == EPI_) {                   \
    if (fp16) TFB_G16(EPI_, M_, true); \
    TFB_G16(EPI_, M_, false);          \
  }
  TFB_G16_EPI(EPI_F32, 1) TFB_G16_EPI(EPI_RELU2, 1) TFB_G16_EPI(EPI_SWIGLU, 2) TFB_G16_EPI(EPI_BF16, 1)
#undef TFB_G16
#undef TFB_G16_AT
#undef TFB_G16_EPI
  return fail(TFB_ERR_ARG, "experts16: no kernel for epilogue %d", epi);
}

static int experts16_check(const void* x, int64_t x_stride, int64_t x_rows, const void* w, int experts, int k, int n, int tile) {
  TFB_REQUIRE(k >= 8 && k % 8 == 0 && k < (1 << 24) && n >= 1 && n < (1 << 24),
              "experts16: %d columns of %d inputs (inputs in multiples of 8)", n, k);
  TFB_REQUIRE(aligned16(x) && x_stride % 8 == 0 && x_stride >= k && x_rows >= 0 && x_rows < (int64_t(1) << 31),
              "experts16: x rows of K inputs, 16-byte aligned");
  TFB_REQUIRE(aligned16(w), "experts16: w must be 16-byte aligned");
  TFB_REQUIRE(experts >= 1, "experts16: bad expert count");
  TFB_REQUIRE(tile >= 1 && tile <= G16_MAXP, "experts16: items of 1..%d pairs, not %d", G16_MAXP, tile);
  return TFB_OK;
}

// The grouped product of 16-bit experts over a plan.  epi: 0 fp32 out, 1 relu^2, 2 SwiGLU over (gate, up), 3 rounded to the
// weights' type; 1 and 2 round to it too.  x: [x_rows, k] rows `x_stride` elements apart; pair p reads row p / slots, or p
// when slots is 0.  out: [P, n], row p of pair p.  max_items: an upper bound of the plan's items, which hold at most `tile`
// pairs (1..256).
extern "C" int tfb_experts16(int epi, int fp16, const void* x, int64_t x_stride, int64_t x_rows, int slots, const void* w,
                             int experts, int k, int n, const int32_t* items, const int32_t* counts, const int32_t* members,
                             void* out, float limit, int64_t max_items, int tile, void* stream) {
  TFB_REQUIRE(x && w && items && counts && members && out, "experts16: null pointer");
  if (int rc = experts16_check(x, x_stride, x_rows, w, experts, k, n, tile)) return rc;
  TFB_REQUIRE(slots >= 0 && max_items >= 0, "experts16: bad slots or item count");
  TFB_REQUIRE(epi >= EPI_F32 && epi <= EPI_BF16, "experts16: no kernel for epilogue %d", epi);
  if (max_items == 0 || x_rows == 0) return TFB_OK;
  const int64_t pairs = slots ? x_rows * slots : x_rows;
  TFB_REQUIRE(pairs < (int64_t(1) << 31), "experts16: 2^31 pairs or more");
  return experts16_run(epi, fp16, x, x_stride, x_rows, slots, w, experts, k, n, items, counts, members, nullptr, (int)pairs, out,
                       limit, max_items, tile, static_cast<cudaStream_t>(stream));
}

// The whole routed block behind one call: plan, gate/up, down and the weighted sum over the slots whose pick names an expert.
extern "C" int tfb_experts16_block(int fp16, const void* x, int64_t x_stride, int rows, const int32_t* picks, int slots,
                                   const float* wts, const void* up, int swiglu, float limit, const void* down, int experts,
                                   int dims, int width, int32_t* members, int32_t* items, int32_t* counts, int64_t max_items,
                                   int tile, void* act, float* y, void* out, int out_f32, void* stream) {
  TFB_REQUIRE(x && picks && wts && up && down && members && items && counts && act && y && out, "experts16: null pointer");
  if (int rc = experts16_check(x, x_stride, rows, up, experts, dims, width, tile)) return rc;
  TFB_REQUIRE(slots >= 1 && (int64_t)rows * slots < (int64_t(1) << 30) && max_items >= 0, "experts16: bad slots or item count");
  TFB_REQUIRE(experts <= PLAN_EMAX, "experts16: at most %d experts, not %d", PLAN_EMAX, experts);
  if (int rc = experts16_check(act, width, (int64_t)rows * slots, down, experts, width, dims, tile)) return rc;
  if (rows == 0) return TFB_OK;
  auto st = static_cast<cudaStream_t>(stream);
  const int pairs = rows * slots;
  const int32_t* few = pairs <= G16_FEW ? picks : nullptr;
  if (few == nullptr)
    if (int rc = tfb_plan(picks, pairs, experts, tile, members, items, counts, stream)) return rc;
  if (int rc = experts16_run(swiglu ? EPI_SWIGLU : EPI_RELU2, fp16, x, x_stride, rows, slots, up, experts, dims, width, items,
                             counts, members, few, pairs, act, limit, max_items, tile, st))
    return rc;
  if (int rc = experts16_run(EPI_F32, fp16, act, width, pairs, 0, down, experts, width, dims, items, counts, members, few, pairs,
                             y, 0.f, max_items, tile, st))
    return rc;
  return tfb_combine_window(y, 0, wts, picks, 0, experts, out, out_f32, rows, slots, dims, stream);
}
