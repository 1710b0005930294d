// Grouped MoE experts on 16-bit weights (bf16 or fp16): matrix products grouped by expert with ragged sizes, on tcgen05.
//
//   gate_up   act[p, n] = f(sum_k x[p / slots, k] U[e(p), n, k])       f: SwiGLU of (gate, up) or relu^2 of up
//   down      y[p, n]   = sum_k act[p, k] D[e(p), n, k]
//
// over the (row, slot) pairs p that a plan has sorted by expert into items of at most `tile` pairs of one expert.  The
// WEIGHTS are the MMA's A operand (128 rows of one expert), an item's PAIRS the B operand (N = pairs rounded up to 16),
// so an expert with three pairs costs an N of 16 and no padded row is ever written.  One fp32 chain over K in order of
// inputs: a pair's bits do not depend on its item, on the tile or on the call.

#include "api.h"
#include "common.cuh"

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
constexpr int G16_MAXP = 256;                      // pairs an item may hold (MMA N)
constexpr int G16_THREADS = 192;                   // warps 0-3 gather and finish, 4 issues the MMAs, 5 copies the weights

template <int MAXP>
struct G16Smem {
  static constexpr int A_BYTES = W16_ROWS * 128, B_BYTES = MAXP * 128;
  static constexpr int STAGES = 4;
  static constexpr int TABLE_OFFSET = STAGES * (A_BYTES + B_BYTES);        // int pair[MAXP]
  static constexpr int BAR_OFFSET = TABLE_OFFSET + MAXP * 4;
  static constexpr int TMEM_OFFSET = BAR_OFFSET + (2 * STAGES + 1) * 8;
  static constexpr int TOTAL = TMEM_OFFSET + 16 + 1024;                    // + slack to align the tiles to 1024 bytes
  static_assert(TOTAL <= 227 * 1024, "one CTA's shared memory");
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

__device__ __forceinline__ void umma_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accum)
      : "memory");
}

// kind::f16, D fp32, both operands K-major, bf16 or fp16, M = 128, N = n
template <bool F16>
__device__ __forceinline__ uint32_t g16_idesc(int n) {
  const uint32_t type = F16 ? 0u : 1u;
  return (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(W16_ROWS >> 4) << 24);
}

__device__ __forceinline__ void cp_async16_or_zero(void* dst, const void* src, bool have) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_addr(dst)), "l"(src), "r"(have ? 16 : 0)
               : "memory");
}

template <int M, int EPI, bool F16, int MAXP>
__global__ void __launch_bounds__(G16_THREADS)
g16_kernel(const uint16_t* __restrict__ X, int64_t x_stride, int slots, const uint8_t* __restrict__ W, int K, int N,
           const int* __restrict__ items, const int* __restrict__ counts, const int* __restrict__ members,
           void* __restrict__ out, float limit) {
  using SM = G16Smem<MAXP>;
  constexpr int STAGES = SM::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* a_ring = smem;
  uint8_t* b_ring = smem + STAGES * SM::A_BYTES;
  int* pair = reinterpret_cast<int*>(smem + SM::TABLE_OFFSET);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + SM::BAR_OFFSET);     // [STAGES] weights and inputs landed
  uint64_t* empty = full + STAGES;                                         // [STAGES] the MMAs that read them retired
  uint64_t* done = empty + STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + SM::TMEM_OFFSET);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rows = w16_rows(M, N), KB = w16_kblocks(K), nct = (rows + W16_ROWS - 1) / W16_ROWS;
  const int it = blockIdx.x / nct, ct = blockIdx.x - it * nct;

  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full + s, 1 + 128);
      mbar_init(empty + s, 1);
    }
    mbar_init(done, 1);
    mbar_fence_init();
    fence_async_smem();
  }
  pdl_wait();
  after_wait(X, items, counts, members);
  const bool live = it < ld_dep(counts);                                   // uniform over the CTA
  if (live && warp == 4) tmem_alloc(tmem_slot, MAXP);
  int e = 0, cnt = 0;
  if (live) {
    e = ld_dep(items + 3 * it);
    const int first = ld_dep(items + 3 * it + 1);
    cnt = min(ld_dep(items + 3 * it + 2), MAXP);
    for (int i = tid; i < cnt; i += G16_THREADS) pair[i] = ld_dep(members + first + i);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (!live) return;
  const uint32_t tmem_base = *tmem_slot;
  const int nmma = (cnt + 15) & ~15;
  const int rt = min(W16_ROWS, rows - ct * W16_ROWS);
  bool ok = true;

  if (warp == 5) {
    const uint8_t* src = W + ((size_t)e * rows + (size_t)ct * W16_ROWS) * KB * 128;
    int g = 0;
    for (; g < KB; ++g) {
      const int s = g % STAGES;
      if (g >= STAGES) ok = mbar_wait_warp(empty + s, (g / STAGES - 1) & 1);
      if (!ok) break;
      if (lane == 0) {
        mbar_expect_tx(full + s, (uint32_t)rt * 128);
        bulk_g2s(a_ring + s * SM::A_BYTES, src + (size_t)g * rt * 128, rt * 128, full + s);
      }
    }
    if (!ok && lane == 0)                                                  // give the copies in flight a while to land
      for (int f = max(0, g - STAGES); f < g; ++f) mbar_wait_for(full + f % STAGES, (f / STAGES) & 1, 10000000ull);
    __syncwarp();
  } else if (warp == 4) {
    if (lane == 0) {
      const uint32_t idesc = g16_idesc<F16>(nmma);
      const uint64_t a0 = umma_desc(smem_addr(a_ring)), b0 = umma_desc(smem_addr(b_ring));
      for (int g = 0; g < KB; ++g) {
        const int s = g % STAGES;
        ok = mbar_wait(full + s, (g / STAGES) & 1);
        if (!ok) break;
        tc_fence_after();
        const uint64_t ad = a0 + (uint32_t)(s * (SM::A_BYTES >> 4)), bd = b0 + (uint32_t)(s * (SM::B_BYTES >> 4));
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) umma_ss(tmem_base, ad + 2 * ks, bd + 2 * ks, idesc, (g | ks) ? 1u : 0u);
        umma_commit(empty + s);
      }
      if (ok) umma_commit(done);
    }
    __syncwarp();
  } else {
    // thread -> chunk c of rows r0, r0 + 16, ...; rows past the last pair repeat it: their columns are never stored
    const int c = tid & 7, r0 = tid >> 3;
    const uint32_t at = (uint32_t)(r0 * 128 + ((c ^ (r0 & 7)) << 4));
    for (int g = 0; g < KB; ++g) {
      const int s = g % STAGES;
      if (g >= STAGES) ok = mbar_wait_warp(empty + s, (g / STAGES - 1) & 1);
      if (!ok) break;
      const int k = g * W16_K + c * 8;
      for (int r = r0, j = 0; r < nmma; r += 16, ++j) {
        const int p = pair[min(r, cnt - 1)];
        const uint16_t* src = X + (size_t)(slots ? p / slots : p) * x_stride;
        cp_async16_or_zero(b_ring + s * SM::B_BYTES + at + j * (16 * 128), src + (k < K ? k : 0), k < K);
      }
      cp_async_commit();
      if (g >= 1) {                                                        // the stage before this one has landed
        cp_async_wait<1>();
        fence_async_smem();
        mbar_arrive(full + (g - 1) % STAGES);
      }
    }
    cp_async_wait<0>();
    fence_async_smem();
    if (ok) mbar_arrive(full + (KB - 1) % STAGES);
    // ---- epilogue: tensor-memory lane = weight row, column = pair ----
    if (ok) ok = mbar_wait_warp(done, 0);
    if (ok) {
      tc_fence_after();
      const int q = warp;
      const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16);
      const int col = M == 1 ? ct * W16_ROWS + q * 32 + lane : ct * (W16_ROWS / 2) + q * 16 + (lane & 15);
      for (int j0 = 0; j0 < nmma; j0 += 16) {
        uint32_t a[16];
        tmem_ld16(taddr + j0, a);
        tmem_ld_wait();
        if constexpr (M == 2) {
          // a column's gate and up rows sit 16 lanes apart: of two neighbouring pairs the gate lane forms the first
          // and the up lane the second
          static_assert(EPI == EPI_SWIGLU, "two matrices: gate and up");
          const bool up_lane = lane >= 16;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float give = __uint_as_float(up_lane ? a[2 * j] : a[2 * j + 1]);
            const float keep = __uint_as_float(up_lane ? a[2 * j + 1] : a[2 * j]);
            const float got = __shfl_xor_sync(0xffffffffu, give, 16);
            const int pi = j0 + 2 * j + (up_lane ? 1 : 0);
            const float v = swiglu32(up_lane ? got : keep, up_lane ? keep : got, limit);
            if (pi < cnt && col < N) static_cast<uint16_t*>(out)[(size_t)pair[pi] * N + col] = to16<F16>(v);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (j0 + j >= cnt || col >= N) continue;
            float v = __uint_as_float(a[j]);
            const size_t o = (size_t)pair[j0 + j] * N + col;
            if constexpr (EPI == EPI_RELU2) {
              v = v > 0.f ? v * v : v != v ? v : 0.f;                      // NaN stays NaN
            }
            if constexpr (EPI == EPI_F32) static_cast<float*>(out)[o] = v;
            else static_cast<uint16_t*>(out)[o] = to16<F16>(v);
          }
        }
      }
    }
  }
  pdl_launch_dependents();
  tc_fence_before();
  __syncthreads();
  if (warp == 4) tmem_dealloc(tmem_base, MAXP);
}

template <int M, int EPI, bool F16, int MAXP>
int launch_g16(const void* x, int64_t x_stride, int slots, const void* w, int k, int n, const int* items, const int* counts,
               const int* members, void* out, float limit, int64_t max_items, cudaStream_t stream) {
  using SM = G16Smem<MAXP>;
  auto* kern = g16_kernel<M, EPI, F16, MAXP>;
  static bool configured[64] = {false};
  int dev = 0;
  TFB_CUDA(cudaGetDevice(&dev), "experts16: cudaGetDevice");
  if (dev < 0 || dev >= 64) return fail(TFB_ERR_ARG, "experts16: device index %d out of range", dev);
  if (!configured[dev]) {
    TFB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::TOTAL),
             "experts16: shared memory opt-in");
    configured[dev] = true;
  }
  const int64_t grid = max_items * ((w16_rows(M, n) + W16_ROWS - 1) / W16_ROWS);
  if (grid >= (int64_t(1) << 31)) return fail(TFB_ERR_ARG, "experts16: too many units");
  return check_cuda(launch(kern, dim3((unsigned)grid), dim3(G16_THREADS), (size_t)SM::TOTAL, stream,
                           static_cast<const uint16_t*>(x), x_stride, slots, static_cast<const uint8_t*>(w), k, n, items,
                           counts, members, out, limit),
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

// The grouped product of 16-bit experts over a plan.  epi: 0 fp32 out, 1 relu^2, 2 SwiGLU over (gate, up), 3 rounded to the
// weights' type; 1 and 2 round to it too.  x: [x_rows, k] rows `x_stride` elements apart; pair p reads row p / slots, or p
// when slots is 0.  out: [P, n], row p of pair p.  max_items: an upper bound of the plan's items, which hold at most `tile`
// pairs (1..256).
extern "C" int tfb_experts16(int epi, int fp16, const void* x, int64_t x_stride, int64_t x_rows, int slots, const void* w,
                             int k, int n, const int32_t* items, const int32_t* counts, const int32_t* members, void* out,
                             float limit, int64_t max_items, int tile, void* stream) {
  TFB_REQUIRE(x && w && items && counts && members && out, "experts16: null pointer");
  TFB_REQUIRE(k >= 8 && k % 8 == 0 && k < (1 << 24) && n >= 1 && n < (1 << 24),
              "experts16: %d columns of %d inputs (inputs in multiples of 8)", n, k);
  TFB_REQUIRE(aligned16(x) && x_stride % 8 == 0 && x_stride >= k && x_rows >= 0 && x_rows < (int64_t(1) << 31),
              "experts16: x rows of K inputs, 16-byte aligned");
  TFB_REQUIRE(aligned16(w), "experts16: w must be 16-byte aligned");
  TFB_REQUIRE(slots >= 0 && max_items >= 0, "experts16: bad slots or item count");
  TFB_REQUIRE(tile >= 1 && tile <= G16_MAXP, "experts16: items of 1..%d pairs, not %d", G16_MAXP, tile);
  if (max_items == 0 || x_rows == 0) return TFB_OK;
  auto st = static_cast<cudaStream_t>(stream);
#define TFB_G16(EPI_, M_, F16_)                                                                                             \
  return tile <= 64 ? launch_g16<M_, EPI_, F16_, 64>(x, x_stride, slots, w, k, n, items, counts, members, out, limit,        \
                                                     max_items, st)                                                         \
                    : launch_g16<M_, EPI_, F16_, 256>(x, x_stride, slots, w, k, n, items, counts, members, out, limit,       \
                                                      max_items, st)
#define TFB_G16_EPI(EPI_, M_)          \
  if (epi == EPI_) {                   \
    if (fp16) TFB_G16(EPI_, M_, true); \
    TFB_G16(EPI_, M_, false);          \
  }
  TFB_G16_EPI(EPI_F32, 1) TFB_G16_EPI(EPI_RELU2, 1) TFB_G16_EPI(EPI_SWIGLU, 2) TFB_G16_EPI(EPI_BF16, 1)
#undef TFB_G16
#undef TFB_G16_EPI
  return fail(TFB_ERR_ARG, "experts16: no kernel for epilogue %d", epi);
}
