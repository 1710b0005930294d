// Low-rank adapters of many requests on top of a shared projection's output, in one launch:
//
//   out[m] = round(base[m] + scale[i] * B[i] (A[i] x[m])),   i = ids[m]; out[m] = round(base[m]) where i is no adapter
//
// A cluster of eight CTAs owns an item = up to 8 NT rows of one adapter.  Every warp of the cluster forms the products
// A x of its own run of inputs (mma: ranks x rows), the CTAs add the 32 partial sums in warp order through distributed
// shared memory, and each CTA then forms an eighth of the columns (mma: rows x columns) on top of the base rows.  The cut
// of the inputs depends on K alone, so a row's bits depend neither on its item nor on the call.
// The low-rank row is split into 16-bit parts that add up to it (after an exact power-of-two scaling of the row): two, which keep
// 16 bits of it (bf16) or 22 (fp16) where one rounding would keep 8 or 11, and for bf16 adapters under fp32 rows a third.
// (With two those rows came out 1.2e-6 off where a computation in 32 bits is 5e-7; with three everywhere a prompt's rows took
// 5 to 12 % longer.)
//
// What bounds it.  Few rows: latency, the chain id -> inputs and A -> two meetings of the cluster -> columns: one row 4.9 us, 64
// rows of as many adapters (4096 x 4096, rank 32; 25 MB) 10 us.  Many: latency too, a block of columns a turn - 8192 rows of
// 4096 x 4096, rank 16, 68 us for 270 MB (DRAM 44 % of its peak, a warp ready in 0.38 of the cycles, 19 warps an SM).  What
// counts is the number of rows in flight: items of 64 rows (fewer blocks an SM) took 124 us; the base's values through a
// ring in shared memory 93 to 149 (the more of it, the fewer blocks); the columns in a launch of their own 88.

#include "api.h"
#include "common.cuh"

#include <cooperative_groups.h>

namespace tfb {

constexpr int AD_CTAS = 8;                 // a cluster
constexpr int AD_WARPS = 4;
constexpr int AD_TILE = 64;                // rows an item of a plan holds at most
constexpr int AD_MAX_RANK = 128;
enum AdType : int { AD_F32 = 0, AD_BF16 = 1, AD_F16 = 2 };

struct AdArgs {
  const uint16_t* x;       // [rows, K]
  const uint16_t* a;       // [count, R, K]
  const uint16_t* b;       // [count, N, R]
  const float* scale;      // [count]
  const int* ids;          // [rows]
  const int *items, *counts, *members;     // a plan of the ids, or null: every row an item of its own
  const void* base;        // [rows, N]
  void* out;               // [rows, N], may be base
  int64_t x_stride, base_stride, out_stride;
  int rows, count, K, N, R, base_type, out_type, clusters;      // clusters: those that items may take
};

template <bool F16>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    mma_bf16(d, a0, a1, a2, a3, b0, b1);
}

template <bool F16>
__device__ __forceinline__ float from16(uint16_t v) {
  if constexpr (F16) return __half2float(__ushort_as_half(v));
  else return __uint_as_float((uint32_t)v << 16);
}

__device__ __forceinline__ float ad_load(const void* p, int type, int64_t i) {
  if (type == AD_F32) return static_cast<const float*>(p)[i];
  const uint16_t v = static_cast<const uint16_t*>(p)[i];
  return type == AD_BF16 ? from16<false>(v) : from16<true>(v);
}

__device__ __forceinline__ void ad_store(void* p, int type, int64_t i, float v) {
  if (type == AD_F32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = type == AD_BF16 ? to16<false>(v) : to16<true>(v);
}

__device__ __forceinline__ uint2 ldg_nc2(const void* p) {
  uint2 r;
  asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];\n" : "=r"(r.x), "=r"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ uint4 ld_dep_u4(const void* p) {                // base may be out: not the read-only path
  uint4 r;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p) : "memory");
  return r;
}

// the float4 at `p` of this CTA's shared memory, in the same place of CTA `rank` of the cluster
__device__ __forceinline__ float4 ld_cluster4(const float* p, int rank) {
  uint32_t at;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(smem_addr(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}

__device__ __forceinline__ uint32_t cluster_addr(const void* p, int rank) {      // this CTA's `p`, in CTA `rank`
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(smem_addr(p)), "r"(rank));
  return at;
}
__device__ __forceinline__ void st_cluster2(uint32_t at, uint2 v) {
  asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};\n" ::"r"(at), "r"(v.x), "r"(v.y) : "memory");
}
__device__ __forceinline__ void st_cluster1(uint32_t at, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;\n" ::"r"(at), "f"(v) : "memory");
}

// Eight neighbouring values of a row, loaded as they are stored: in 16-byte pieces when `whole`, else the first `have` one by
// one (rows that do not start on 16 bytes, a row's end), each in a word of its own; in fp32; and their way back.
__device__ __forceinline__ bool ad_wide(const void* p, int type, int64_t stride) {
  return stride % (type == AD_F32 ? 4 : 8) == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}
__device__ __forceinline__ uint32_t ld_dep_u16(const uint16_t* p) {
  uint16_t v;
  asm volatile("ld.global.u16 %0, [%1];\n" : "=h"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void ad_load8(const void* p, int type, int64_t at, bool whole, int have, uint4 (&raw)[2]) {
  if (whole) {
    if (type == AD_F32) {
      raw[0] = ld_dep_u4(static_cast<const float*>(p) + at);
      raw[1] = ld_dep_u4(static_cast<const float*>(p) + at + 4);
    } else {
      raw[0] = ld_dep_u4(static_cast<const uint16_t*>(p) + at);
    }
    return;
  }
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    w[i] = 0u;
    if (i < have)
      w[i] = type == AD_F32 ? (uint32_t)ld_dep(static_cast<const int*>(p) + at + i) : ld_dep_u16(static_cast<const uint16_t*>(p) + at + i);
  }
  raw[0] = make_uint4(w[0], w[1], w[2], w[3]);
  raw[1] = make_uint4(w[4], w[5], w[6], w[7]);
}
__device__ __forceinline__ void ad_widen(const uint4 (&raw)[2], int type, bool whole, float (&v)[8]) {
  const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint16_t u = (uint16_t)(whole ? w[i >> 1] >> (16 * (i & 1)) : w[i]);
    v[i] = type == AD_F32 ? __uint_as_float(w[i]) : type == AD_BF16 ? from16<false>(u) : from16<true>(u);
  }
}
__device__ __forceinline__ void ad_store8(void* p, int type, bool wide, int64_t at, int have, const float (&v)[8]) {
  if (have < 8 || !wide) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < have) ad_store(p, type, at + i, v[i]);
  } else if (type == AD_F32) {
    float* o = static_cast<float*>(p) + at;
    *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(o + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a = type == AD_BF16 ? to16<false>(v[2 * i]) : to16<true>(v[2 * i]);
      const uint32_t b = type == AD_BF16 ? to16<false>(v[2 * i + 1]) : to16<true>(v[2 * i + 1]);
      w[i] = a | (b << 16);
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + at) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Rows r0 .. r0 + B - 1 whose bit is set in `take`, columns 8 `c8` and every `step` eights further: the base alone.
template <int B>
__device__ __forceinline__ void ad_copy_rows(const AdArgs& g, int r0, uint32_t take, int c8, int step) {
  const bool wide_base = ad_wide(g.base, g.base_type, g.base_stride), wide_out = ad_wide(g.out, g.out_type, g.out_stride);
  for (int c = 8 * c8; c < g.N; c += 8 * step) {
    const int have = min(8, g.N - c);
    const bool whole = have == 8 && wide_base;
    uint4 raw[B][2];
#pragma unroll
    for (int i = 0; i < B; ++i)                                            // the rows' loads are in flight together
      if (take >> i & 1) ad_load8(g.base, g.base_type, (int64_t)(r0 + i) * g.base_stride + c, whole, have, raw[i]);
#pragma unroll
    for (int i = 0; i < B; ++i) {
      if (!(take >> i & 1)) continue;
      float v[8];
      ad_widen(raw[i], g.base_type, whole, v);
      ad_store8(g.out, g.out_type, wide_out, (int64_t)(r0 + i) * g.out_stride + c, have, v);
    }
  }
}

// inputs a warp of the cluster takes: K / 32 rounded up to 64
__host__ __device__ __forceinline__ int ad_run(int k) {
  const int runs = AD_CTAS * AD_WARPS;
  return ((k + runs - 1) / runs + 63) / 64 * 64;
}

// RT: sixteens of ranks.  NT: eights of rows an item holds; 1 = every row an item of its own (its tile's other rows idle).
template <int RT, int NT>
struct AdShape {
  static constexpr bool ALONE = NT == 1;
  static constexpr int ROWS = 8 * NT, RP = 16 * RT, PITCH = RP + 4;        // + 4: the partial sums' columns spread over banks
  static constexpr int MT = (ROWS + 15) / 16;                              // row tiles of the second product
  static constexpr int QUADS = RP / 4;                                     // fours of a row's ranks
  static constexpr int SUM_ROWS = ALONE ? 1 : ROWS / AD_CTAS;              // rows a CTA adds up over the cluster
  static constexpr int KU = NT > 1 ? (RT <= 2 ? 2 : 1) : (RT <= 2 ? 4 : RT == 4 ? 2 : 1);   // steps of 32 inputs loaded at once
  static constexpr int CH = ALONE && RT <= 2 ? 2 : 1;   // blocks of columns loaded at once
  static constexpr int PART = AD_WARPS * ROWS * PITCH * 4;                 // float part[warp][row][PITCH]; the sum in warp 0's
  static constexpr int LP = RT == 1 ? RP : RP + 16;                        // a tile's rows then spread over the banks
  static constexpr int LOW = ROWS * LP * 2;                                // a part of the low-rank rows, [row][LP]
  static constexpr int LOW_OFFSET = PART;
  static constexpr int BACK_OFFSET = LOW_OFFSET + 3 * LOW;                 // float back[row]: the row's scaling undone
  static constexpr int ROW_OFFSET = BACK_OFFSET + ROWS * 4;                // int row[ROWS]
  static constexpr int TOTAL = ROW_OFFSET + ROWS * 4;
  static_assert(ALONE || ROWS % AD_CTAS == 0, "the cluster shares the rows out");
  static_assert(SUM_ROWS * QUADS <= AD_WARPS * 32 || SUM_ROWS * QUADS % (AD_WARPS * 32) == 0, "whole warps reduce");
};

template <int RT, int NT, bool F16>
__global__ void __launch_bounds__(AD_WARPS * 32, RT == 1 ? 5 : RT == 2 ? 4 : RT == 4 ? 3 : 1)
adapters_kernel(AdArgs g) {
  using SH = AdShape<RT, NT>;
  constexpr int ROWS = SH::ROWS, RP = SH::RP, PITCH = SH::PITCH, LP = SH::LP, MT = SH::MT, QUADS = SH::QUADS, KU = SH::KU, CH = SH::CH;
  constexpr bool ALONE = SH::ALONE;
  constexpr int THREADS = AD_WARPS * 32, STRIDE = AD_CTAS * AD_WARPS * 32;   // columns the cluster forms at a time
  extern __shared__ __align__(16) uint8_t ad_smem[];
  float* part = reinterpret_cast<float*>(ad_smem);
  constexpr int PARTS = F16 ? 2 : 3;                                       // at most
  const int parts = F16 || g.out_type != AD_F32 ? 2 : 3;
  uint16_t* low = reinterpret_cast<uint16_t*>(ad_smem + SH::LOW_OFFSET);
  float* back = reinterpret_cast<float*>(ad_smem + SH::BACK_OFFSET);
  int* row = reinterpret_cast<int*>(ad_smem + SH::ROW_OFFSET);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gq = lane >> 2, t = lane & 3;
  const int cta = blockIdx.x % AD_CTAS, unit = blockIdx.x / AD_CTAS;
  const int N = g.N, K = g.K, R = g.R;

  pdl_wait();
  pdl_launch_dependents();                                                 // what follows waits for this grid's end all the same
  // ---- which rows, whose adapter (the same for the whole cluster) ----
  int who = -1, first = unit, cnt = 1;
  if (ALONE) {
    who = ld_dep(g.ids + unit);
    if (who >= g.count) who = -1;
  } else if (unit < g.clusters) {
    constexpr int SUB = AD_TILE / ROWS;                                    // items of more rows than a cluster takes
    const int it = unit / SUB, sub = unit - it * SUB;
    if (it >= ld_dep(g.counts)) return;
    who = ld_dep(g.items + 3 * it);
    first = ld_dep(g.items + 3 * it + 1) + sub * ROWS;
    cnt = min(ld_dep(g.items + 3 * it + 2) - sub * ROWS, ROWS);
    if (cnt <= 0) return;
  } else {
    // rows without an adapter, which no item holds: the base alone; eight rows a CTA, looked at all at once
    const int r0 = (unit - g.clusters) * AD_TILE + cta * 8, id = r0 + lane < g.rows && lane < 8 ? ld_dep(g.ids + r0 + lane) : 0;
    const uint32_t take = __ballot_sync(0xffffffffu, id < 0 || id >= g.count);
#pragma unroll
    for (int half = 0; half < 8; half += 4)
      if (take >> half & 15) ad_copy_rows<4>(g, r0 + half, take >> half, tid, THREADS);
    return;
  }
  if (who < 0) {
    ad_copy_rows<1>(g, unit, 1, cta * THREADS + tid, AD_CTAS * THREADS);
    return;
  }
  for (int i = tid; i < ROWS; i += THREADS)
    row[i] = ALONE ? unit : ld_dep(g.members + first + min(i, cnt - 1));   // past the last: it again, never stored
  __syncthreads();

  // ---- the low-rank rows: this warp's run of inputs ----
  {
    float acc[RT][NT][4];
#pragma unroll
    for (int m = 0; m < RT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][n][i] = 0.f;
    const int run = ad_run(K), k0 = (cta * AD_WARPS + warp) * run, k1 = min(K, k0 + run);
    const uint16_t* ap = g.a + ((size_t)who * R + gq) * K + 8 * t;
    const uint16_t* xp[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) xp[n] = g.x + (size_t)row[8 * n + gq] * g.x_stride + 8 * t;
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    for (int k = k0; k < k1; k += 32 * KU) {                               // lane t: inputs k + 8 t .. + 7, in any one order
      uint4 al[KU][RT], ah[KU][RT], xv[KU][NT];
#pragma unroll
      for (int v = 0; v < KU; ++v) {                                       // all of a step's loads are in flight at once
        const int kv = k + 32 * v;
        const bool in = kv < k1 && kv + 8 * t < K;
#pragma unroll
        for (int n = 0; n < NT; ++n) xv[v][n] = in && 8 * n < cnt ? ldg_nc(xp[n] + kv) : zero;
#pragma unroll
        for (int m = 0; m < RT; ++m) {
          al[v][m] = in && 16 * m < R ? ldg_nc(ap + (size_t)(16 * m) * K + kv) : zero;
          ah[v][m] = in && 16 * m + 8 < R ? ldg_nc(ap + (size_t)(16 * m + 8) * K + kv) : zero;
        }
      }
#pragma unroll
      for (int v = 0; v < KU; ++v) {
        if (k + 32 * v >= k1) break;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (8 * n >= cnt) break;
#pragma unroll
          for (int m = 0; m < RT; ++m) {
            mma16<F16>(acc[m][n], al[v][m].x, ah[v][m].x, al[v][m].y, ah[v][m].y, xv[v][n].x, xv[v][n].y);
            mma16<F16>(acc[m][n], al[v][m].z, ah[v][m].z, al[v][m].w, ah[v][m].w, xv[v][n].z, xv[v][n].w);
          }
        }
      }
    }
#pragma unroll
    for (int m = 0; m < RT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float* p = part + (warp * ROWS + 8 * n + 2 * t) * PITCH + 16 * m + gq;
        p[0] = acc[m][n][0];
        p[PITCH] = acc[m][n][1];
        p[8] = acc[m][n][2];
        p[PITCH + 8] = acc[m][n][3];
      }
  }

  // ---- the columns' operands that do not hang on the low-rank rows: on their way before the cluster meets ----
  // a warp forms 32 columns at a time, lane t columns 8 t .. 8 t + 7 of rows gq and gq + 8 of each tile of 16
  const uint16_t* bp = g.b + (size_t)who * N * R;
  uint2 bv[CH][RT][4];
  auto load_b = [&](int c0) {                                              // lane t: ranks 16 ks + 4 t .. + 3
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int ks = 0; ks < RT; ++ks)
#pragma unroll
        for (int j = 0; j < 4; ++j) {                                      // mma column gq of tile j = column 8 (gq / 2) + 2 j + gq % 2
          const int col = c0 + c * STRIDE + (gq >> 1) * 8 + 2 * j + (gq & 1), r = 16 * ks + 4 * t;
          bv[c][ks][j] = make_uint2(0u, 0u);
          if (col < N && r < R) bv[c][ks][j] = ldg_nc2(bp + (size_t)col * R + r);
        }
  };
  const bool wide_base = ad_wide(g.base, g.base_type, g.base_stride), wide_out = ad_wide(g.out, g.out_type, g.out_stride);
  uint4 pb[CH][MT][2][2];                                                  // the base's values as they are
  auto load_base = [&](int c0) {
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = 16 * m + 8 * h + gq, cl = c0 + c * STRIDE + 8 * t;
          if (r < cnt && cl < N)
            ad_load8(g.base, g.base_type, row[r] * g.base_stride + cl, wide_base && cl + 8 <= N, N - cl, pb[c][m][h]);
        }
  };
  const int c_first = (cta * AD_WARPS + warp) * 32;
  load_b(c_first);
  load_base(c_first);

  __syncthreads();
  for (int i = tid; i < (ALONE ? QUADS : ROWS * QUADS); i += THREADS) {    // the CTA's four partial sums, in warp order
    float4* p = reinterpret_cast<float4*>(part + i / QUADS * PITCH + i % QUADS * 4);
    float4 v = p[0];
#pragma unroll
    for (int w = 1; w < AD_WARPS; ++w) {
      const float4 q = p[w * ROWS * PITCH / 4];
      v.x += q.x;
      v.y += q.y;
      v.z += q.z;
      v.w += q.w;
    }
    p[0] = v;
  }
  cluster_arrive();
  cluster_wait();
  // ---- the cluster's eight, in CTA order; scaled; split in two.  Each CTA its share of the rows for all eight (a row alone:
  // each CTA for itself) ----
  const float scale = g.scale[who];
  for (int i = tid; i < SH::SUM_ROWS * QUADS; i += THREADS) {
    const int r = (ALONE ? 0 : cta * SH::SUM_ROWS) + i / QUADS, j = i % QUADS * 4;
    float4 v[AD_CTAS];
#pragma unroll
    for (int c = 0; c < AD_CTAS; ++c) v[c] = ld_cluster4(part + r * PITCH + j, c);
    float s[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
    for (int c = 1; c < AD_CTAS; ++c) {
      s[0] += v[c].x;
      s[1] += v[c].y;
      s[2] += v[c].z;
      s[3] += v[c].w;
    }
    float most = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      s[q] = scale == 0.f ? 0.f : s[q] * scale;                            // an empty slot's row: whatever its inputs hold
      most = fmaxf(most, fabsf(s[q]));
    }
    constexpr unsigned lanes = SH::SUM_ROWS * QUADS >= 32 ? 0xffffffffu : (1u << (SH::SUM_ROWS * QUADS % 32)) - 1;   // a row's fours are neighbours
#pragma unroll
    for (int d = 1; d < QUADS; d *= 2) most = fmaxf(most, __shfl_xor_sync(lanes, most, d));
    // the row's largest value into [1, 4), or near 1 as far as a power of two goes (fp32's largest and least values); a row with
    // an infinity or NaN as it is
    int ex = 0;
    if (most > 0.f && most <= 3.402823466e38f) ex = max(-126, min(126, ilogbf(most)));
    const float down = __uint_as_float((uint32_t)(127 - ex) << 23);        // 2^-ex: exact
#pragma unroll
    for (int q = 0; q < 4; ++q) s[q] *= down;
    const float up = __uint_as_float((uint32_t)(127 + ex) << 23);
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      if (p >= parts) break;
      uint16_t h[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        h[q] = to16<F16>(s[q]);
        const float rest = s[q] - from16<F16>(h[q]);
        s[q] = fabsf(rest) < 1.f ? rest : 0.f;                             // an infinity or NaN stays in the first part alone
      }
      const uint2 hv = make_uint2(h[0] | ((uint32_t)h[1] << 16), h[2] | ((uint32_t)h[3] << 16));
      uint16_t* dst = low + (p * ROWS + r) * LP + j;
      if constexpr (ALONE) {
        *reinterpret_cast<uint2*>(dst) = hv;
      } else {
#pragma unroll
        for (int c = 0; c < AD_CTAS; ++c) st_cluster2(cluster_addr(dst, c), hv);
      }
    }
    if (j == 0) {
      if constexpr (ALONE) {
        back[0] = up;
      } else {
#pragma unroll
        for (int c = 0; c < AD_CTAS; ++c) st_cluster1(cluster_addr(back + r, c), up);
      }
    }
  }
  cluster_arrive();
  if constexpr (ALONE) __syncthreads();
  else cluster_wait();

  // ---- an eighth of the columns ----
  for (int c0 = c_first; c0 < N; c0 += CH * STRIDE) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float d[MT][4][4];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) d[m][j][i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < RT; ++ks)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          if (16 * m >= cnt) break;
          const int ra = (ALONE ? 0 : 16 * m + gq) * LP + 16 * ks + 4 * t, rb = ALONE ? ra : ra + 8 * LP;
#pragma unroll
          for (int p = PARTS - 1; p >= 0; --p) {                           // the smallest first
            if (p >= parts) continue;
            const uint2 sa = *reinterpret_cast<const uint2*>(low + p * ROWS * LP + ra), sb = *reinterpret_cast<const uint2*>(low + p * ROWS * LP + rb);
#pragma unroll
            for (int j = 0; j < 4; ++j) mma16<F16>(d[m][j], sa.x, sb.x, sa.y, sb.y, bv[c][ks][j].x, bv[c][ks][j].y);
          }
        }
      if (c == CH - 1 && c0 + CH * STRIDE < N) load_b(c0 + CH * STRIDE);
      const int cl = c0 + c * STRIDE + 8 * t;                              // the lane's eight columns
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = 16 * m + 8 * h + gq;
          if (r >= cnt || cl >= N) continue;
          const float bk = back[r];
          const int have = min(8, N - cl);
          float v[8];
          ad_widen(pb[c][m][h], g.base_type, wide_base && have == 8, v);
          if (!ALONE && cl + STRIDE < N)                                   // the next block's, as soon as its place is free
            ad_load8(g.base, g.base_type, row[r] * g.base_stride + cl + STRIDE, wide_base && cl + STRIDE + 8 <= N, N - cl - STRIDE, pb[c][m][h]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v[2 * j] = fmaf(d[m][j][2 * h], bk, v[2 * j]);
            v[2 * j + 1] = fmaf(d[m][j][2 * h + 1], bk, v[2 * j + 1]);
          }
          ad_store8(g.out, g.out_type, wide_out, row[r] * g.out_stride + cl, have, v);
        }
    }
    if (ALONE && c0 + CH * STRIDE < N) load_base(c0 + CH * STRIDE);
  }
  if constexpr (ALONE) cluster_wait();                                     // nobody reads this CTA's sums any more
}

template <int RT, int NT, bool F16>
int launch_adapters(const AdArgs& g, int64_t units, cudaStream_t stream) {
  using SH = AdShape<RT, NT>;
  auto* kern = adapters_kernel<RT, NT, F16>;
  if constexpr (SH::TOTAL > 48 * 1024) {
    static bool configured[64] = {false};
    int dev = 0;
    TFB_CUDA(cudaGetDevice(&dev), "adapters: cudaGetDevice");
    if (dev < 0 || dev >= 64) return fail(TFB_ERR_ARG, "adapters: device index %d out of range", dev);
    if (!configured[dev]) {
      TFB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SH::TOTAL),
               "adapters: shared memory opt-in");
      configured[dev] = true;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * AD_CTAS));
  cfg.blockDim = dim3(AD_WARPS * 32);
  cfg.dynamicSmemBytes = SH::TOTAL;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = AD_CTAS;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_use_pdl ? 2 : 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, g), "adapters");
}

}  // namespace tfb

using namespace tfb;

// out[m] = base[m] + scale[i] B[i] (A[i] x[m]), i = ids[m]; the base alone where i is outside 0..count-1.  x [rows, k], a
// [count, rank, k] and b [count, n, rank] in bf16 or fp16 (rank a multiple of 8, zero rows and columns behind an adapter's
// own); base and out fp32 (0), bf16 (1) or fp16 (2), rows *_stride elements apart; out may be base.  items, counts, members:
// tfb_plan's tables of the ids with items of at most 64 rows, or null: every row on its own.
extern "C" int tfb_adapters(int fp16, const void* x, int64_t x_stride, const void* a, const void* b, const float* scale,
                            int rank, int k, int n, const int32_t* ids, int rows, int count, const int32_t* items,
                            const int32_t* counts, const int32_t* members, int64_t max_items, const void* base,
                            int base_type, int64_t base_stride, void* out, int out_type, int64_t out_stride, void* stream) {
  TFB_REQUIRE(x && a && b && scale && ids && base && out, "adapters: null pointer");
  TFB_REQUIRE((items && counts && members) || (!items && !counts && !members), "adapters: a whole plan or none");
  TFB_REQUIRE(rank >= 8 && rank % 8 == 0 && rank <= AD_MAX_RANK, "adapters: ranks up to %d in multiples of 8, not %d",
              AD_MAX_RANK, rank);
  TFB_REQUIRE(k >= 8 && k % 8 == 0 && k < (1 << 24) && n >= 1 && n < (1 << 24),
              "adapters: %d columns of %d inputs (inputs in multiples of 8)", n, k);
  TFB_REQUIRE(aligned16(x) && x_stride % 8 == 0 && (x_stride >= k || rows <= 1) && aligned16(a) && aligned16(b),
              "adapters: x rows, a and b must be 16-byte aligned");
  TFB_REQUIRE(base_type >= 0 && base_type <= 2 && out_type >= 0 && out_type <= 2, "adapters: fp32 (0), bf16 (1) or fp16 (2) "
              "rows, not %d and %d", base_type, out_type);
  TFB_REQUIRE(rows >= 0 && count >= 1 && max_items >= 0 && (rows <= 1 || (base_stride >= n && out_stride >= n)),
              "adapters: bad sizes");
  TFB_REQUIRE(out != base || (out_type == base_type && out_stride == base_stride), "adapters: in place needs one layout");
  if (rows == 0) return TFB_OK;
  auto st = static_cast<cudaStream_t>(stream);
  AdArgs g{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(a), static_cast<const uint16_t*>(b), scale, ids,
           items, counts, members, base, out, x_stride, base_stride, out_stride, rows, count, k, n, rank, base_type,
           out_type, 0};
  const int64_t bare = out == base ? 0 : (rows + AD_TILE - 1) / AD_TILE;   // rows that no item holds
#define TFB_AD(RT_, NT_)                                                                        \
  do {                                                                                          \
    const int64_t units = items ? max_items * (AD_TILE / (8 * NT_)) + bare : rows;              \
    TFB_REQUIRE(units * AD_CTAS < (int64_t(1) << 31), "adapters: too many units");              \
    if (units == 0) return TFB_OK;                                                              \
    g.clusters = (int)(max_items * (AD_TILE / (8 * NT_)));                                      \
    return fp16 ? launch_adapters<RT_, NT_, true>(g, units, st) : launch_adapters<RT_, NT_, false>(g, units, st); \
  } while (0)
  if (items == nullptr) {
    if (rank <= 16) TFB_AD(1, 1);
    if (rank <= 32) TFB_AD(2, 1);
    if (rank <= 64) TFB_AD(4, 1);
    TFB_AD(8, 1);
  }
  if (rank <= 16) TFB_AD(1, 4);
  if (rank <= 32) TFB_AD(2, 4);
  if (rank <= 64) TFB_AD(4, 4);
  TFB_AD(8, 2);
#undef TFB_AD
}
