// Low-rank adapters of many requests on top of a shared projection's output, in one launch:
//
//   out[m] = round(base[m] + scale[i] * B[i] (A[i] x[m])),   i = ids[m]; out[m] = round(base[m]) where i is no adapter
//
// A cluster of eight CTAs owns an item = up to 8 NT rows of one adapter.  Every warp of the cluster forms the products
// A x of its own run of inputs (mma: ranks x rows), the CTAs add the 32 partial sums in warp order through distributed
// shared memory, and each CTA then forms an eighth of the columns (mma: rows x columns) on top of the base rows.  The cut
// of the inputs depends on K alone, so a row's bits depend neither on its item nor on the call.
// The low-rank row is split into two 16-bit parts (s = hi + lo, after an exact power-of-two scaling of the row), which
// keeps 16 bits of it or more where one rounding would keep 8: the second product costs nothing beside the bytes.

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

// the float4 at `p` of this CTA's shared memory, in the same place of CTA `rank` of the cluster
__device__ __forceinline__ float4 ld_cluster4(const float* p, int rank) {
  uint32_t at;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(smem_addr(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}

// inputs a warp of the cluster takes: K / 32 rounded up to 64
__host__ __device__ __forceinline__ int ad_run(int k) {
  const int runs = AD_CTAS * AD_WARPS;
  return ((k + runs - 1) / runs + 63) / 64 * 64;
}

template <int RT, int NT>
struct AdSmem {
  static constexpr int ROWS = 8 * NT, RP = 16 * RT, PITCH = RP + 4;        // + 4: the partial sums' columns spread over banks
  static constexpr int PART = AD_WARPS * ROWS * PITCH * 4;                 // float part[warp][row][PITCH]; the sum in warp 0's
  static constexpr int LOW = ROWS * RP * 2;                                // hi[row][RP], then lo
  static constexpr int HI_OFFSET = PART;
  static constexpr int BACK_OFFSET = HI_OFFSET + 2 * LOW;                  // float back[row]: the row's scaling undone
  static constexpr int ROW_OFFSET = BACK_OFFSET + ROWS * 4;                // int row[ROWS]
  static constexpr int TOTAL = ROW_OFFSET + ROWS * 4;
};

template <int RT, int NT, bool F16>
__global__ void __launch_bounds__(AD_WARPS * 32)
adapters_kernel(AdArgs g) {
  using SM = AdSmem<RT, NT>;
  constexpr int ROWS = SM::ROWS, RP = SM::RP, PITCH = SM::PITCH;
  constexpr int MT = (ROWS + 15) / 16;                                     // row tiles of the second product
  extern __shared__ __align__(16) uint8_t ad_smem[];
  float* part = reinterpret_cast<float*>(ad_smem);
  uint16_t* hi = reinterpret_cast<uint16_t*>(ad_smem + SM::HI_OFFSET);
  uint16_t* lo = hi + ROWS * RP;
  float* back = reinterpret_cast<float*>(ad_smem + SM::BACK_OFFSET);
  int* row = reinterpret_cast<int*>(ad_smem + SM::ROW_OFFSET);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gq = lane >> 2, t = lane & 3;
  const int cta = blockIdx.x % AD_CTAS, unit = blockIdx.x / AD_CTAS;
  const int N = g.N, K = g.K, R = g.R;

  pdl_wait();
  // ---- which rows, whose adapter (the same for the whole cluster) ----
  int who = -1, first = unit, cnt = 1;
  if (g.items == nullptr) {
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
    // rows without an adapter, which no item holds: the base alone
    const int r0 = (unit - g.clusters) * AD_TILE, r1 = min(g.rows, r0 + AD_TILE);
    for (int r = r0; r < r1; ++r) {
      const int id = ld_dep(g.ids + r);
      if (id >= 0 && id < g.count) continue;
      for (int n = cta * (AD_WARPS * 32) + tid; n < N; n += AD_CTAS * AD_WARPS * 32)
        ad_store(g.out, g.out_type, r * g.out_stride + n, ad_load(g.base, g.base_type, r * g.base_stride + n));
    }
    return;
  }
  if (who < 0) {
    for (int n = cta * (AD_WARPS * 32) + tid; n < N; n += AD_CTAS * AD_WARPS * 32)
      ad_store(g.out, g.out_type, unit * g.out_stride + n, ad_load(g.base, g.base_type, unit * g.base_stride + n));
    return;
  }
  for (int i = tid; i < ROWS; i += AD_WARPS * 32)
    row[i] = g.items == nullptr ? unit : ld_dep(g.members + first + min(i, cnt - 1));   // past the last: it again, never stored
  __syncthreads();

  // ---- the low-rank rows: this warp's run of inputs ----
  float acc[RT][NT][4];
#pragma unroll
  for (int m = 0; m < RT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][n][i] = 0.f;
  {
    const int run = ad_run(K), k0 = (cta * AD_WARPS + warp) * run, k1 = min(K, k0 + run);
    const uint16_t* ap = g.a + ((size_t)who * R + gq) * K + 8 * t;
    const uint16_t* xp[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) xp[n] = g.x + (size_t)row[8 * n + gq] * g.x_stride + 8 * t;
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    for (int k = k0; k < k1; k += 32) {                                    // lane t: inputs k + 8 t .. + 7, in any one order
      const bool in = k + 8 * t < K;
      uint4 al[RT], ah[RT], xv[NT];
#pragma unroll
      for (int m = 0; m < RT; ++m) {
        al[m] = in && 16 * m < R ? ldg_nc(ap + (size_t)(16 * m) * K + k) : zero;
        ah[m] = in && 16 * m + 8 < R ? ldg_nc(ap + (size_t)(16 * m + 8) * K + k) : zero;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) xv[n] = in && 8 * n < cnt ? ldg_nc(xp[n] + k) : zero;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (8 * n >= cnt) break;
#pragma unroll
        for (int m = 0; m < RT; ++m) {
          mma16<F16>(acc[m][n], al[m].x, ah[m].x, al[m].y, ah[m].y, xv[n].x, xv[n].y);
          mma16<F16>(acc[m][n], al[m].z, ah[m].z, al[m].w, ah[m].w, xv[n].z, xv[n].w);
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
  __syncthreads();
  for (int i = tid; i < ROWS * RP; i += AD_WARPS * 32) {                   // the CTA's four partial sums, in warp order
    float* p = part + (i / RP) * PITCH + i % RP;
    float v = p[0];
#pragma unroll
    for (int w = 1; w < AD_WARPS; ++w) v += p[w * ROWS * PITCH];
    p[0] = v;
  }
  cluster_arrive();
  cluster_wait();
  // ---- the cluster's eight, in CTA order, into warp 1's place (nobody reads it from outside); scaled; split in two ----
  float* sum = part + ROWS * PITCH;
  const float scale = g.scale[who];
  for (int i = tid; i < ROWS * (RP / 4); i += AD_WARPS * 32) {
    const int at = (i / (RP / 4)) * PITCH + (i % (RP / 4)) * 4;
    float4 v[AD_CTAS];
#pragma unroll
    for (int c = 0; c < AD_CTAS; ++c) v[c] = ld_cluster4(part + at, c);
    float4 s = v[0];
#pragma unroll
    for (int c = 1; c < AD_CTAS; ++c) {
      s.x += v[c].x;
      s.y += v[c].y;
      s.z += v[c].z;
      s.w += v[c].w;
    }
    sum[at] = s.x * scale;
    sum[at + 1] = s.y * scale;
    sum[at + 2] = s.z * scale;
    sum[at + 3] = s.w * scale;
  }
  cluster_arrive();                                                        // this CTA has read its neighbours' sums
  __syncthreads();
  for (int r = tid; r < ROWS; r += AD_WARPS * 32) {
    float most = 0.f;
    for (int j = 0; j < RP; ++j) most = fmaxf(most, fabsf(sum[r * PITCH + j]));
    int ex = 0;
    if (most > 0.f && most <= 3.0e38f) ex = max(-100, min(100, ilogbf(most)));
    const float down = __uint_as_float((uint32_t)(127 - ex) << 23);        // 2^-ex: exact
    back[r] = __uint_as_float((uint32_t)(127 + ex) << 23);
    for (int j = 0; j < RP; ++j) {
      const float v = sum[r * PITCH + j] * down;
      const uint16_t h = to16<F16>(v);
      const float rest = v - from16<F16>(h);
      hi[r * RP + j] = h;
      lo[r * RP + j] = to16<F16>(fabsf(rest) < 1.f ? rest : 0.f);          // an infinity or NaN stays in hi alone
    }
  }
  __syncthreads();

  // ---- an eighth of the columns, 32 a warp at a time: lane t holds columns 8 t .. 8 t + 7 of rows gq, gq + 8 of each tile ----
  const bool wide_base = (g.base_type == AD_F32 ? g.base_stride % 4 : g.base_stride % 8) == 0 && (reinterpret_cast<uintptr_t>(g.base) & 15) == 0;
  const bool wide_out = (g.out_type == AD_F32 ? g.out_stride % 4 : g.out_stride % 8) == 0 && (reinterpret_cast<uintptr_t>(g.out) & 15) == 0;
  const uint16_t* bp = g.b + (size_t)who * N * R;
  for (int c0 = (warp * AD_CTAS + cta) * 32; c0 < N; c0 += AD_CTAS * AD_WARPS * 32) {
    float d[MT][4][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) d[m][j][i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < RT; ++ks) {                                      // lane t: ranks 16 ks + 4 t .. + 3
      uint2 bv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {                                        // mma column gq of tile j = column 8 (gq / 2) + 2 j + gq % 2
        const int col = c0 + (gq >> 1) * 8 + 2 * j + (gq & 1), r = 16 * ks + 4 * t;
        bv[j] = col < N && r < R ? __ldg(reinterpret_cast<const uint2*>(bp + (size_t)col * R + r)) : make_uint2(0u, 0u);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (16 * m >= cnt) break;
        const int ra = (16 * m + gq) * RP + 16 * ks + 4 * t, rb = ROWS > 8 ? ra + 8 * RP : ra;
        const uint2 ha = *reinterpret_cast<const uint2*>(hi + ra), hb = *reinterpret_cast<const uint2*>(hi + rb);
        const uint2 la = *reinterpret_cast<const uint2*>(lo + ra), lb = *reinterpret_cast<const uint2*>(lo + rb);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          mma16<F16>(d[m][j], la.x, lb.x, la.y, lb.y, bv[j].x, bv[j].y);
          mma16<F16>(d[m][j], ha.x, hb.x, ha.y, hb.y, bv[j].x, bv[j].y);
        }
      }
    }
    const int cl = c0 + 8 * t;                                             // the lane's eight columns
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = 16 * m + 8 * h + gq;
        if (r >= cnt || cl >= N) continue;
        const float bk = back[r];
        const int64_t at_b = row[r] * g.base_stride + cl, at_o = row[r] * g.out_stride + cl;
        float v[8];
        if (cl + 8 <= N && wide_base) {
          if (g.base_type == AD_F32) {
            const float4 p = *reinterpret_cast<const float4*>(static_cast<const float*>(g.base) + at_b);
            const float4 q = *reinterpret_cast<const float4*>(static_cast<const float*>(g.base) + at_b + 4);
            v[0] = p.x; v[1] = p.y; v[2] = p.z; v[3] = p.w; v[4] = q.x; v[5] = q.y; v[6] = q.z; v[7] = q.w;
          } else {
            const uint4 p = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(g.base) + at_b);
            const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint16_t u = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
              v[i] = g.base_type == AD_BF16 ? from16<false>(u) : from16<true>(u);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = cl + i < N ? ad_load(g.base, g.base_type, at_b + i) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[2 * j] = fmaf(d[m][j][2 * h], bk, v[2 * j]);
          v[2 * j + 1] = fmaf(d[m][j][2 * h + 1], bk, v[2 * j + 1]);
        }
        if (cl + 8 <= N && wide_out) {
          if (g.out_type == AD_F32) {
            float* o = static_cast<float*>(g.out) + at_o;
            *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(o + 4) = make_float4(v[4], v[5], v[6], v[7]);
          } else {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t a16 = g.out_type == AD_BF16 ? to16<false>(v[2 * i]) : to16<true>(v[2 * i]);
              const uint32_t b16 = g.out_type == AD_BF16 ? to16<false>(v[2 * i + 1]) : to16<true>(v[2 * i + 1]);
              w[i] = a16 | (b16 << 16);
            }
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(g.out) + at_o) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (cl + i < N) ad_store(g.out, g.out_type, at_o + i, v[i]);
        }
      }
  }
  pdl_launch_dependents();
  cluster_wait();                                                          // nobody reads this CTA's sums any more
}

template <int RT, int NT, bool F16>
int launch_adapters(const AdArgs& g, int64_t units, cudaStream_t stream) {
  using SM = AdSmem<RT, NT>;
  auto* kern = adapters_kernel<RT, NT, F16>;
  if constexpr (SM::TOTAL > 48 * 1024) {
    static bool configured[64] = {false};
    int dev = 0;
    TFB_CUDA(cudaGetDevice(&dev), "adapters: cudaGetDevice");
    if (dev < 0 || dev >= 64) return fail(TFB_ERR_ARG, "adapters: device index %d out of range", dev);
    if (!configured[dev]) {
      TFB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::TOTAL),
               "adapters: shared memory opt-in");
      configured[dev] = true;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * AD_CTAS));
  cfg.blockDim = dim3(AD_WARPS * 32);
  cfg.dynamicSmemBytes = SM::TOTAL;
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
  if (rank <= 16) TFB_AD(1, 8);
  if (rank <= 32) TFB_AD(2, 8);
  if (rank <= 64) TFB_AD(4, 8);
  TFB_AD(8, 2);
#undef TFB_AD
}
