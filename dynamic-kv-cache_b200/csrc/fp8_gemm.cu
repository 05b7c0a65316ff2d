// Products of e4m3 rows with e4m3 weight blocks (sm_100a, tcgen05):
//
//   C[m, n] = sum_b sa[m, b] * sw[n / 128, b] * sum_{k in group b} qa[m, k] qw[n, k]
//
// over the column groups b of 128 (fp8.cuh). The inner sums are exact products summed by
// the tensor cores in fp32 (kind::f8f6f4, one 128-column group per accumulator); a scale
// cannot be applied there, so each group's accumulator is read from TMEM, multiplied by its
// two scales and added to the running sum in registers, in fp32, while the tensor cores
// work on the next groups.
//
// fp8_gemm_kernel puts the weights on the 128 lanes of the accumulator and NT tokens on its
// columns: the weights are what a decoder step has to stream, a tile holds 128 of their rows
// whatever the token count, and 16 to 64 tokens waste no tensor work on padding. The column
// groups of one tile are divided among the S blocks of a cluster when the tiles alone would
// leave SMs idle; their partial sums meet in distributed shared memory, added in rank order.
//
// GATE computes two products with the same rows, G and U, and writes silu(g) * u as e4m3
// rows: a tile of 128 intermediate columns is exactly one column group of the next product,
// so its scale is found in the tile.
#include <cuda.h>

#include <mutex>

#include "fp8.cuh"
#include "tc_ptx.cuh"

namespace dkv {

using namespace ptx;

constexpr long long kGemmWaitCycles = 400000000LL;  // ~0.2 s: a healthy wait is microseconds
constexpr int kGemmStages = 4;
constexpr int kGemmSlots = 4;      // accumulators in TMEM, one column group each
constexpr int kGemmThreads = 192;  // warps 0-3: scale and add; 4: copies; 5: MMA issue
constexpr int kTileRows = 128;     // weight rows of a tile

struct GemmArgs {
  const float* sa;         // [m, groups]
  const float* sw;         // [ceil(n / 128), groups]
  const float* su;         // GATE: the same for the up weights
  void* out;               // [m, n] bf16 / fp32, or e4m3 with GATE
  float* out_scale;        // GATE: [m, ceil(n / 128)]
  int m, n, groups, splits;
  int out_f32;
};

template <int NT, bool GATE>
struct GemmTile {
  static constexpr int kParts = GATE ? 2 : 1;
  static constexpr int kWeightBytes = kTileRows * kFp8Group;  // one operand tile of one group
  static constexpr int kTokenBytes = NT * kFp8Group;
  static constexpr int kStageBytes = kParts * kWeightBytes + kTokenBytes;
  static constexpr int kCols = NT * kParts;  // TMEM columns of one accumulator
  static constexpr int kTmemCols = kCols * kGemmSlots < 32 ? 32 : kCols * kGemmSlots;
  static constexpr int kRingBytes = kGemmStages * kStageBytes;
  static constexpr int kPartialBytes = kParts * NT * kTileRows * 4;  // reuses the ring
  static_assert(kPartialBytes <= kRingBytes, "partial sums fit the operand ring");
  static_assert(kTmemCols <= 512 && (kTmemCols & (kTmemCols - 1)) == 0, "TMEM allocation");
  static size_t smem(int groups_per_split) {
    return 1024 + kRingBytes + static_cast<size_t>(kParts) * groups_per_split * NT * 4;
  }
};

// silu(g) * u = g / (1 + 2^(-g log2 e)) * u on the special-function unit: 2^x and 1 / x are off
// by a few fp32 units, and the exponent's rounding by |g| of them, far under the 2^-4 of the
// rounding to e4m3 that follows (IEEE expf and division made the epilogue the bottleneck).
// Where 2^x overflows, 1 / inf = 0 and the result is the 0 that silu tends to.
__device__ __forceinline__ float silu_times(float g, float u) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(1.0f + ex2(-1.4426950408889634f * g)));
  return g * r * u;
}

template <int NT, bool GATE>
__global__ void __launch_bounds__(kGemmThreads, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap umap,
                const __grid_constant__ CUtensorMap amap, const GemmArgs a) {
  using T = GemmTile<NT, GATE>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * kGemmStages + 2 * kGemmSlots];
  __shared__ uint32_t tmem_slot;
  const uint32_t ring = (smem_addr(smem_raw) + 1023u) & ~1023u;
  float* scales = reinterpret_cast<float*>(smem_raw + (ring - smem_addr(smem_raw)) + T::kRingBytes);
  const uint32_t full = smem_addr(bars);
  const uint32_t empty = full + 8 * kGemmStages;
  const uint32_t done = empty + 8 * kGemmStages;  // an accumulator is complete
  const uint32_t freed = done + 8 * kGemmSlots;   // ... and read

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = blockIdx.x % a.splits;
  const int tile = blockIdx.x / a.splits;
  const int token0 = blockIdx.y * NT;
  const int per = (a.groups + a.splits - 1) / a.splits;
  const int group0 = rank * per;
  const int count = max(0, min(per, a.groups - group0));

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * kGemmStages + kGemmSlots; ++i) mbar_init(full + 8 * i, 1);
    for (int i = 0; i < kGemmSlots; ++i) mbar_init(freed + 8 * i, 128);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 4 && lane == 0) {
    prefetch_tensor_map(&wmap);
    if (GATE) prefetch_tensor_map(&umap);
    prefetch_tensor_map(&amap);
  }
  pdl_wait();  // operands are the previous kernels' output
  // TMEM is taken after the wait and before the trigger: a waiting block never holds what
  // the grid it waits for still needs, and no dependent starts before every block has it.
  if (warp == 5) {
    tmem_alloc(smem_addr(&tmem_slot), T::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();
  const uint32_t tmem = tmem_slot;

  if (warp == 4) {
    if (lane == 0) {
      int i = 0;
      for (; i < count; ++i) {
        const int s = i % kGemmStages;
        if (i >= kGemmStages && !mbar_wait(empty + 8 * s, ((i / kGemmStages) + 1) & 1, kGemmWaitCycles)) break;
        const uint32_t dst = ring + s * T::kStageBytes;
        const int x = (group0 + i) * kFp8Group;
        mbar_arrive_expect_tx(full + 8 * s, T::kStageBytes);
        tile2d_g2s(dst, &wmap, x, tile * kTileRows, full + 8 * s);
        if (GATE) tile2d_g2s(dst + T::kWeightBytes, &umap, x, tile * kTileRows, full + 8 * s);
        tile2d_g2s(dst + T::kParts * T::kWeightBytes, &amap, x, token0, full + 8 * s);
      }
      // a wait that ran out: the copies in flight still target this block's memory
      if (i < count)
        for (int j = max(0, i - kGemmStages); j < i; ++j)
          mbar_wait(full + 8 * (j % kGemmStages), (j / kGemmStages) & 1, kGemmWaitCycles);
    }
    __syncwarp();
  } else if (warp == 5) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_e4m3(kTileRows, NT);
      for (int i = 0; i < count; ++i) {
        const int s = i % kGemmStages;
        const int slot = i % kGemmSlots;
        bool ok = mbar_wait(full + 8 * s, (i / kGemmStages) & 1, kGemmWaitCycles);
        if (ok && i >= kGemmSlots) ok = mbar_wait(freed + 8 * slot, ((i / kGemmSlots) + 1) & 1, kGemmWaitCycles);
        if (!ok) break;
        tc_fence_after();
        const uint32_t src = ring + s * T::kStageBytes;
        const uint64_t wd = sw128_desc(src, 16, 1024);
        const uint64_t ud = sw128_desc(src + T::kWeightBytes, 16, 1024);
        const uint64_t ad = sw128_desc(src + T::kParts * T::kWeightBytes, 16, 1024);
#pragma unroll
        for (int j = 0; j < kFp8Group / 32; ++j) {  // 32 columns are 32 bytes: 2 descriptor units
          umma_f8(tmem + slot * T::kCols, wd + 2 * j, ad + 2 * j, idesc, j > 0);
          if (GATE) umma_f8(tmem + slot * T::kCols + NT, ud + 2 * j, ad + 2 * j, idesc, j > 0);
        }
        umma_commit(empty + 8 * s);
        umma_commit(done + 8 * slot);
      }
    }
    __syncwarp();
  } else {
    // the scale products of this block's groups: scales[part][group][token]
    for (int i = threadIdx.x; i < count * NT; i += 128) {
      const int token = i / count;
      const int g = i - token * count;
      const float s = token0 + token < a.m ? a.sa[static_cast<int64_t>(token0 + token) * a.groups + group0 + g] : 0.f;
      const int64_t block = static_cast<int64_t>(tile) * a.groups + group0 + g;
      scales[g * NT + token] = s * a.sw[block];
      if (GATE) scales[(count + g) * NT + token] = s * a.su[block];
    }
    named_bar_sync(1, 128);
    float acc[T::kCols];
#pragma unroll
    for (int j = 0; j < T::kCols; ++j) acc[j] = 0.f;
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    bool ok = true;
    for (int i = 0; i < count && ok; ++i) {
      const int slot = i % kGemmSlots;
      ok = __all_sync(0xffffffffu, mbar_wait(done + 8 * slot, (i / kGemmSlots) & 1, kGemmWaitCycles));
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < T::kCols; c += 16) {
        uint32_t p[16];
        tmem_ld16(tmem + lanes + slot * T::kCols + c, p);
        tmem_wait_ld();
        const float* sc = scales + (c < NT ? i * NT + c : (count + i) * NT + c - NT);
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const float4 f = *reinterpret_cast<const float4*>(sc + j);
          acc[c + j] = fmaf(__uint_as_float(p[j]), f.x, acc[c + j]);
          acc[c + j + 1] = fmaf(__uint_as_float(p[j + 1]), f.y, acc[c + j + 1]);
          acc[c + j + 2] = fmaf(__uint_as_float(p[j + 2]), f.z, acc[c + j + 2]);
          acc[c + j + 3] = fmaf(__uint_as_float(p[j + 3]), f.w, acc[c + j + 3]);
        }
      }
      tc_fence_before();
      mbar_arrive(freed + 8 * slot);
    }
    // partial sums [part][token][weight row]; a wait that ran out leaves NaN, not a stale tile
    float* partial = reinterpret_cast<float*>(smem_raw + (ring - smem_addr(smem_raw)));
#pragma unroll
    for (int j = 0; j < T::kCols; ++j) partial[j * kTileRows + threadIdx.x] = ok ? acc[j] : __int_as_float(0x7fc00000);
  }
  // TMEM goes back before this block waits for another one: what holds TMEM never depends
  // on a block that may still be waiting for some.
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, T::kTmemCols);
  }
  if (a.splits > 1) cluster_sync_all();

  // a warp per token, 4 weight rows (output columns) per lane
  const int col = tile * kTileRows + lane * 4;
  for (int t = rank + a.splits * warp; t < NT && token0 + t < a.m; t += a.splits * (kGemmThreads / 32)) {
    float4 sum[T::kParts];
#pragma unroll
    for (int p = 0; p < T::kParts; ++p) {
      const uint32_t at = ring + ((p * NT + t) * kTileRows + lane * 4) * 4;
      sum[p] = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int r = 0; r < a.splits; ++r) {
        float4 v;
        if (a.splits > 1) {
          v = ld_dsmem_f4(dsmem_addr(at, r));
        } else {
          v = *reinterpret_cast<const float4*>(smem_raw + (at - smem_addr(smem_raw)));
        }
        sum[p].x += v.x;
        sum[p].y += v.y;
        sum[p].z += v.z;
        sum[p].w += v.w;
      }
    }
    const int64_t row = token0 + t;
    if (GATE) {  // n is a multiple of 16: a lane's 4 columns are all inside or all outside
      const float4 g = sum[0], u = sum[T::kParts - 1];
      float4 h = make_float4(0.f, 0.f, 0.f, 0.f);
      if (col < a.n)
        h = make_float4(silu_times(g.x, u.x), silu_times(g.y, u.y), silu_times(g.z, u.z), silu_times(g.w, u.w));
      float amax = max_nan(max_nan(fabsf(h.x), fabsf(h.y)), max_nan(fabsf(h.z), fabsf(h.w)));
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, off));
      amax = max_nan(amax, kFp8Floor);
      const float inverse = __fdiv_rn(kFp8Max, amax);
      if (col < a.n)
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.out) + row * a.n + col) =
            e4m3x4(h.x * inverse, h.y * inverse, h.z * inverse, h.w * inverse);
      if (lane == 0) a.out_scale[row * ((a.n + kFp8Group - 1) / kFp8Group) + tile] = __fdiv_rn(amax, kFp8Max);
    } else {
      const float4 v = sum[0];
      const int64_t at = row * a.n + col;
      const bool whole = col + 4 <= a.n && (a.n & 3) == 0;
      if (a.out_f32) {
        float* o = static_cast<float*>(a.out) + at;
        if (whole) {
          *reinterpret_cast<float4*>(o) = v;
        } else {
          if (col < a.n) o[0] = v.x;
          if (col + 1 < a.n) o[1] = v.y;
          if (col + 2 < a.n) o[2] = v.z;
          if (col + 3 < a.n) o[3] = v.w;
        }
      } else {
        __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.out) + at;
        if (whole) {
          *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
        } else {
          if (col < a.n) o[0] = __float2bfloat16_rn(v.x);
          if (col + 1 < a.n) o[1] = __float2bfloat16_rn(v.y);
          if (col + 2 < a.n) o[2] = __float2bfloat16_rn(v.z);
          if (col + 3 < a.n) o[3] = __float2bfloat16_rn(v.w);
        }
      }
    }
  }
  if (a.splits > 1) cluster_sync_all();  // the other blocks may still be reading this one's partial sums
}

// ---- many tokens -----------------------------------------------------------------
// fp8_wide_kernel keeps the tensor cores busy when there are tokens for it: a pair of
// blocks works on a tile of 256 tokens x 256 weight rows, each block with 128 of the
// tokens on its accumulators' lanes and half of the weight rows in its shared memory (so
// per group and block 32 KB arrive for 2 x 128 x 256 x 128 products). A group's products go
// to two accumulators of 128 columns, one per weight block of 128 rows; TMEM holds four, so
// the tensor cores run up to two groups ahead of the eight epilogue warps that scale and
// add them. A thread owns one token and 64 columns of each half: a half costs it one scale
// product and 32 packed FMAs. The grid is persistent (one pair per two SMs): a tile's store
// overlaps the next tile's first groups.
// GATE makes the halves the gate and the up rows of the same 128 intermediate columns:
// each thread then holds matching columns of G and U.
constexpr int kWideThreads = 384;  // warps 0-7: scale and add; 8: copies; 9: MMA issue; 10, 11: none
constexpr int kWideStages = 6;
constexpr int kWideHalf = 128 * kFp8Group;  // bytes of one block's operand tile of one group
constexpr int kWideStageBytes = 2 * kWideHalf;
constexpr int kWideChunk = 16;  // groups whose scales are staged at a time
constexpr int kWideScales = kWideChunk * 128 + 2 * kWideChunk;  // [group][token], then [group][half] of the weights
constexpr int kWideSmem = 1024 + kWideStages * kWideStageBytes + 2 * kWideScales * 4;
constexpr int kWideCols = 256;
constexpr int kWideSlots = 2;
constexpr uint32_t kWideTmem = kWideSlots * kWideCols;

// `count` columns of one token (a multiple of 16), of which `columns` exist.
__device__ __forceinline__ void store_columns_bf16(__nv_bfloat16* p, int columns, bool vector, const float* v, int count) {
  if (vector && columns >= count) {
#pragma unroll
    for (int j = 0; j < count; j += 16) {
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = __uint_as_float(pack_bf16x2(v[j + 2 * i], v[j + 2 * i + 1]));
      st_global_v8(reinterpret_cast<float*>(p + j), w);
    }
  } else {
#pragma unroll
    for (int j = 0; j < count; ++j)
      if (j < columns) p[j] = __float2bfloat16_rn(v[j]);
  }
}

__device__ __forceinline__ void store_columns_f32(float* p, int columns, bool vector, const float* v, int count) {
  if (vector && columns >= count) {
#pragma unroll
    for (int j = 0; j < count; j += 8) st_global_v8(p + j, v + j);
  } else {
#pragma unroll
    for (int j = 0; j < count; ++j)
      if (j < columns) p[j] = v[j];
  }
}

template <bool GATE>
__global__ void __launch_bounds__(kWideThreads, 1)
fp8_wide_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap umap,
                const __grid_constant__ CUtensorMap amap, const GemmArgs a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * kWideStages + kWideSlots + 4];
  __shared__ uint32_t tmem_slot;
  __shared__ float amax_part[2][2][128];  // GATE: [tile parity][column part][token]
  const uint32_t ring = (smem_addr(smem_raw) + 1023u) & ~1023u;
  const uint32_t full = smem_addr(bars);         // rank 0's: both blocks' copies of a stage
  // each block's own: a stage's products are done, its accumulator complete and its buffers
  // empty (one commit for both: a commit costs the issuing thread ~0.15 us)
  const uint32_t done = full + 8 * kWideStages;
  const uint32_t freed = done + 8 * kWideStages;  // rank 0's: both blocks have read an accumulator
  const uint32_t staged = freed + 8 * kWideSlots;  // each block's own: a chunk of scales is there
  const uint32_t used = staged + 16;               // ... and no longer needed
  float* const scales = reinterpret_cast<float*>(smem_raw + (ring - smem_addr(smem_raw)) + kWideStages * kWideStageBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1;
  const int pair = blockIdx.x >> 1;
  const int pairs = gridDim.x >> 1;
  constexpr int kColumns = GATE ? 128 : 256;  // output columns of a tile
  const int tiles_m = (a.m + 255) / 256;
  const int tiles = tiles_m * ((a.n + kColumns - 1) / kColumns);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * kWideStages; ++i) mbar_init(full + 8 * i, 1);
    for (int i = 0; i < kWideSlots; ++i) mbar_init(freed + 8 * i, 8 + (rank == 0));  // the epilogue warps of both blocks
    for (int i = 0; i < 2; ++i) {
      mbar_init(staged + 8 * i, 64);
      mbar_init(used + 8 * i, 8);
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 8 && lane == 0) {
    prefetch_tensor_map(&wmap);
    if (GATE) prefetch_tensor_map(&umap);
    prefetch_tensor_map(&amap);
  }
  cluster_sync_all();  // both blocks' barriers exist
  pdl_wait();
  if (warp == 9) {  // after the wait, before the trigger: see fp8_gemm_kernel
    tmem_alloc_pair(smem_addr(&tmem_slot), kWideTmem);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_arrive_release();  // the copies need not wait for TMEM: their warps join at the end

  // 384 x 168 registers at launch = 128 x (56 + 224 + 224)
  if (warp >= 8) {
    regs_give<56>();
    if (warp == 9) {
      cluster_wait_acquire();
      tc_fence_after();
      pdl_trigger();  // after every block's allocation
    }
    if (warp == 8 && lane == 0) {
      const uint32_t full0 = dsmem_addr(full, 0);
      int i = 0;
      bool ok = true;
      for (int tile = pair; tile < tiles && ok; tile += pairs) {
        const int token0 = (tile % tiles_m) * 256 + rank * 128;
        const int row0 = (tile / tiles_m) * kColumns + (GATE ? 0 : rank * 128);
        for (int g = 0; g < a.groups; ++g, ++i) {
          const int s = i % kWideStages;
          if (i >= kWideStages && !mbar_wait(done + 8 * s, ((i / kWideStages) + 1) & 1, kGemmWaitCycles)) {
            ok = false;
            break;
          }
          const uint32_t dst = ring + s * kWideStageBytes;
          if (rank == 0) mbar_arrive_expect_tx(full + 8 * s, 2 * kWideStageBytes);
          tile2d_g2s_pair(dst, &amap, g * kFp8Group, token0, full0 + 8 * s);
          tile2d_g2s_pair(dst + kWideHalf, GATE && rank == 1 ? &umap : &wmap, g * kFp8Group, row0, full0 + 8 * s);
        }
      }
      if (!ok && rank == 0)  // a wait that ran out: the copies in flight still target shared memory
        for (int j = max(0, i - kWideStages); j < i; ++j)
          mbar_wait(full + 8 * (j % kWideStages), (j / kWideStages) & 1, kGemmWaitCycles);
    } else if (warp == 9 && rank == 1 && lane == 0) {
      const int total = (tiles - pair + pairs - 1) / pairs * a.groups;
      const uint32_t freed0 = dsmem_addr(freed, 0);
      for (int i = 0; i < total; ++i) {
        const int slot = i % kWideSlots;
        if (!mbar_wait(freed + 8 * slot, (i / kWideSlots) & 1, kGemmWaitCycles)) break;
        mbar_arrive_cluster(freed0 + 8 * slot);
      }
    } else if (warp == 9 && rank == 0 && lane == 0) {
      constexpr uint32_t idesc = idesc_e4m3(256, kWideCols);
      const uint32_t tmem = tmem_slot;
      const int total = (tiles - pair + pairs - 1) / pairs * a.groups;
      bool ok = true;
      for (int i = 0; i < total && ok; ++i) {
        const int s = i % kWideStages;
        ok = mbar_wait(full + 8 * s, (i / kWideStages) & 1, kGemmWaitCycles);
        const uint32_t src = ring + s * kWideStageBytes;
        const uint64_t ad = sw128_desc(src, 16, 1024);
        const uint64_t wd = sw128_desc(src + kWideHalf, 16, 1024);
        const int slot = i % kWideSlots;
        if (ok && i >= kWideSlots) ok = mbar_wait(freed + 8 * slot, ((i / kWideSlots) + 1) & 1, kGemmWaitCycles);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int j = 0; j < kFp8Group / 32; ++j)
          umma_f8_pair(tmem + slot * kWideCols, ad + 2 * j, wd + 2 * j, idesc, j > 0);
        umma_commit_pair(done + 8 * s);
      }
    }
    if (warp >= 10) {
      // The scales arrive as rows of groups, and each epilogue thread needs one row: read by
      // that thread, every group would be 32 cache lines per warp. Copied flat and turned
      // over in shared memory, it is one conflict-free load.
      const int t = threadIdx.x - 32 * 10;
      int c = 0;
      bool ok = true;
      for (int tile = pair; tile < tiles && ok; tile += pairs) {
        const int token0 = (tile % tiles_m) * 256 + rank * 128;
        const int tn = tile / tiles_m;
        const int tokens = min(128, a.m - token0);  // may be negative: nothing to read
        const float* sw0 = a.sw + static_cast<int64_t>(GATE ? tn : 2 * tn) * a.groups;
        const float* sw1 = GATE ? a.su + static_cast<int64_t>(tn) * a.groups
                                : a.sw + static_cast<int64_t>(min(2 * tn + 1, (a.n + 127) / 128 - 1)) * a.groups;
        for (int g0 = 0; g0 < a.groups; g0 += kWideChunk, ++c) {
          const int n = min(kWideChunk, a.groups - g0);
          if (c >= 2 && !mbar_wait(used + 8 * (c & 1), ((c >> 1) + 1) & 1, kGemmWaitCycles)) {
            ok = false;
            break;
          }
          float* dst = scales + (c & 1) * kWideScales;
          const float* src = a.sa + static_cast<int64_t>(token0) * a.groups + g0;
          const int g = t % kWideChunk;
          if (g < n)
            for (int token = t / kWideChunk; token < tokens; token += 64 / kWideChunk)
              dst[g * 128 + token] = __ldg(src + static_cast<int64_t>(token) * a.groups + g);
          if (t < 2 * n) dst[kWideChunk * 128 + t] = __ldg((t & 1 ? sw1 : sw0) + g0 + (t >> 1));
          mbar_arrive(staged + 8 * (c & 1));
        }
      }
    }
    __syncwarp();
    if (warp != 9) cluster_wait_acquire();
  } else {
    regs_take<224>();
    cluster_wait_acquire();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const int part = warp >> 2;
    const int token_in = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    int i = 0, chunk = 0;
    bool ok = true;
    const auto next_chunk = [&] {  // this warp is done with a chunk of scales
      __syncwarp();
      if (lane == 0) mbar_arrive(used + 8 * (chunk & 1));
      ++chunk;
    };
    for (int tile = pair, parity = 0; tile < tiles; tile += pairs, parity ^= 1) {
      const int token = (tile % tiles_m) * 256 + rank * 128 + token_in;
      const int tn = tile / tiles_m;
      const bool live = token < a.m;
      const int blocks = (a.n + 127) / 128;
      float acc[128];  // GATE: 64 columns of G, then the same of U
#pragma unroll
      for (int j = 0; j < 128; ++j) acc[j] = 0.f;
      for (int g = 0; g < a.groups; ++g, ++i) {
        if (g % kWideChunk == 0) {
          if (g > 0) next_chunk();
          ok = ok && __all_sync(0xffffffffu, mbar_wait(staged + 8 * (chunk & 1), (chunk >> 1) & 1, kGemmWaitCycles));
        }
        const float* sc = scales + (chunk & 1) * kWideScales + (g % kWideChunk) * 128;
        const float sa = sc[token_in];
        const float2 sw = *reinterpret_cast<const float2*>(scales + (chunk & 1) * kWideScales + kWideChunk * 128 +
                                                           2 * (g % kWideChunk));
        const float f0 = sa * (GATE || part == 0 ? sw.x : sw.y), f1 = sa * sw.y;
        const int slot = i % kWideSlots;
        const int s = i % kWideStages;
        ok = ok && __all_sync(0xffffffffu, mbar_wait(done + 8 * s, (i / kWideStages) & 1, kGemmWaitCycles));
        if (!ok) continue;
        tc_fence_after();
        // the next 32 columns are on their way from TMEM while these are added
        const uint32_t src = tmem + lanes + slot * kWideCols + part * (GATE ? 64 : 128);
        uint32_t p[2][32];
        tmem_ld32(src, p[0]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tmem_wait_ld();
          if (c < 3) {
            tmem_ld32(src + (GATE ? ((c + 1) >> 1) * 128 + ((c + 1) & 1) * 32 : (c + 1) * 32), p[(c + 1) & 1]);
          } else {  // every column is in registers
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(freed + 8 * slot);
          }
          const float2 f = GATE && c >= 2 ? make_float2(f1, f1) : make_float2(f0, f0);
          float2* ac = reinterpret_cast<float2*>(acc + c * 32);
#pragma unroll
          for (int j = 0; j < 16; ++j)
            ac[j] = fma2(make_float2(__uint_as_float(p[c & 1][2 * j]), __uint_as_float(p[c & 1][2 * j + 1])), f, ac[j]);
        }
      }
      next_chunk();
      if (!ok) {  // a wait that ran out leaves NaN, not a stale tile
#pragma unroll
        for (int j = 0; j < 128; ++j) acc[j] = __int_as_float(0x7fc00000);
      }
      if (GATE) {
        const int col0 = tn * 128 + part * 64;
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < 64; ++j) {
          acc[j] = silu_times(acc[j], acc[64 + j]);
          if (col0 + j < a.n) amax = max_nan(amax, fabsf(acc[j]));
        }
        amax_part[parity][part][token_in] = amax;
        named_bar_sync(1, 256);
        amax = max_nan(max_nan(amax, amax_part[parity][part ^ 1][token_in]), kFp8Floor);
        const float inverse = __fdiv_rn(kFp8Max, amax);
        if (live) {
          uint8_t* q = static_cast<uint8_t*>(a.out) + static_cast<int64_t>(token) * a.n + col0;
#pragma unroll
          for (int j = 0; j < 64; j += 16)  // n is a multiple of 16
            if (col0 + j < a.n) *reinterpret_cast<uint4*>(q + j) = codes16(acc + j, inverse);
          if (part == 0) a.out_scale[static_cast<int64_t>(token) * blocks + tn] = __fdiv_rn(amax, kFp8Max);
        }
      } else if (live) {
        const bool vector = (reinterpret_cast<uintptr_t>(a.out) & 31) == 0 && (a.n & (a.out_f32 ? 7 : 15)) == 0;
        const int col0 = tn * 256 + part * 128;
        const int64_t at = static_cast<int64_t>(token) * a.n + col0;
        if (a.out_f32)
          store_columns_f32(static_cast<float*>(a.out) + at, a.n - col0, vector, acc, 128);
        else
          store_columns_bf16(static_cast<__nv_bfloat16*>(a.out) + at, a.n - col0, vector, acc, 128);
      }
    }
  }
  tc_fence_before();
  cluster_sync_all();  // the other block's copies, arrivals and products are done with this one
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_slot, kWideTmem);
  }
}

namespace {

using FnEncode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

FnEncode encoder() {
  static const FnEncode fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<FnEncode>(p);
  }();
  return fn;
}

// Tiles of `box` rows x 128 columns of an 8-bit matrix [rows, cols], rows `stride` bytes
// apart, 128-byte swizzled.
bool encode_tiles(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t stride, int box) {
  const FnEncode fn = encoder();
  if (fn == nullptr) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride)};
  const cuuint32_t boxes[2] = {kFp8Group, static_cast<cuuint32_t>(box)};
  const cuuint32_t steps[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, boxes, steps,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct GemmCall {
  const void *a, *w, *u;
  int64_t as, ws, us;  // row strides in bytes
  int k;
  GemmArgs args;
};

template <int NT, bool GATE>
cudaError_t launch_gemm(const GemmCall& c, int splits, cudaStream_t stream) {
  using T = GemmTile<NT, GATE>;
  CUtensorMap wmap, umap, amap;
  if (!encode_tiles(&wmap, c.w, c.args.n, c.k, c.ws, kTileRows) || !encode_tiles(&amap, c.a, c.args.m, c.k, c.as, NT))
    return cudaErrorInvalidValue;
  umap = wmap;
  if (GATE && !encode_tiles(&umap, c.u, c.args.n, c.k, c.us, kTileRows)) return cudaErrorInvalidValue;
  GemmArgs args = c.args;
  args.splits = splits;
  const size_t smem = T::smem((args.groups + splits - 1) / splits);
  const cudaError_t e = cudaFuncSetAttribute(fp8_gemm_kernel<NT, GATE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((args.n + kTileRows - 1) / kTileRows * splits, (args.m + NT - 1) / NT);
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, fp8_gemm_kernel<NT, GATE>, wmap, umap, amap, args);
}

template <bool GATE>
cudaError_t launch_wide(const GemmCall& c, cudaStream_t stream) {
  CUtensorMap wmap, umap, amap;
  if (!encode_tiles(&wmap, c.w, c.args.n, c.k, c.ws, 128) || !encode_tiles(&amap, c.a, c.args.m, c.k, c.as, 128))
    return cudaErrorInvalidValue;
  umap = wmap;
  if (GATE && !encode_tiles(&umap, c.u, c.args.n, c.k, c.us, 128)) return cudaErrorInvalidValue;
  const cudaError_t e =
      cudaFuncSetAttribute(fp8_wide_kernel<GATE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kWideSmem);
  if (e != cudaSuccess) return e;
  const int columns = GATE ? 128 : 256;
  const int64_t tiles = static_cast<int64_t>((c.args.m + 255) / 256) * ((c.args.n + columns - 1) / columns);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * static_cast<unsigned>(tiles < 74 ? tiles : 74));
  cfg.blockDim = dim3(kWideThreads);
  cfg.dynamicSmemBytes = kWideSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, fp8_wide_kernel<GATE>, wmap, umap, amap, c.args);
}

template <bool GATE>
cudaError_t launch_gemm_rows(const GemmCall& c, cudaStream_t stream) {
  const GemmArgs& a = c.args;
  const int columns = GATE ? 128 : 256;
  if (a.m >= 256 && static_cast<int64_t>((a.m + 255) / 256) * ((a.n + columns - 1) / columns) >= 37)
    return launch_wide<GATE>(c, stream);
  const int nt = a.m <= 16 ? 16 : a.m <= 32 ? 32 : 64;
  const int64_t tiles = static_cast<int64_t>((a.n + kTileRows - 1) / kTileRows) * ((a.m + nt - 1) / nt);
  int splits = 1;  // as many blocks as one wave of the 148 SMs holds, a column group each at least
  while (splits < 8 && tiles * splits * 2 <= 148 && splits * 2 <= a.groups) splits *= 2;
  switch (nt) {
    case 16: return launch_gemm<16, GATE>(c, splits, stream);
    case 32: return launch_gemm<32, GATE>(c, splits, stream);
    default: return launch_gemm<64, GATE>(c, splits, stream);
  }
}

}  // namespace

cudaError_t launch_fp8_linear(const void* a, const float* sa, const void* w, const float* sw, void* out, int out_f32,
                              int m, int n, int k, int64_t as, int64_t ws, cudaStream_t stream) {
  const int groups = (k + kFp8Group - 1) / kFp8Group;
  return launch_gemm_rows<false>({a, w, nullptr, as, ws, 0, k, {sa, sw, nullptr, out, nullptr, m, n, groups, 1, out_f32}},
                                 stream);
}

cudaError_t launch_fp8_gate_up(const void* a, const float* sa, const void* gate, const float* sg, const void* up,
                               const float* su, void* out, float* out_scale, int m, int n, int k, int64_t as,
                               int64_t gs, int64_t us, cudaStream_t stream) {
  const int groups = (k + kFp8Group - 1) / kFp8Group;
  return launch_gemm_rows<true>({a, gate, up, as, gs, us, k, {sa, sg, su, out, out_scale, m, n, groups, 1, 0}}, stream);
}

}  // namespace dkv
