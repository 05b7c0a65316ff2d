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
// fp8_gemm_kernel (few tokens) puts the weights on the 128 lanes of the accumulator and NT
// tokens on its columns: the weights are what a decoder step has to stream, a tile holds 128 of
// their rows whatever the token count, and 16 to 64 tokens waste little tensor work on padding.
// The column groups of one tile are divided among the S blocks of a cluster when the tiles
// alone would leave SMs idle; their partial sums cross by bulk copies between the SMs' shared
// memories and are added in rank order. Small calls are bound by latency, a chain of the
// previous kernel's end (~1 us), the first copies (~0.5), the products (~0.2), the scaling
// (0.1 to 0.2 a group) and the sums and stores (0.3 to 0.8): 1 x 1600 x 960 2.7 us, 64 x 960 x
// 2560 3.6, 333 x 1001 x 1040 5.2; many weight rows by memory: 25 x 49280 x 960 11.1 us, 4.7 of
// 6.6 TB/s. (Times here: one launch of a replayed graph of 20, unless said.)
//
// fp8_wide_kernel (many tokens) is described below: 4096^3 64.5 us (76 in a long run of calls, under
// the power cap), 2.13 PFLOP/s, 65 % of twice the measured bf16 rate (a plain library product of
// these e4m3 matrices, without block scales: 49.5 us), bound by the round trip of an accumulator
// between the tensor cores and the threads that scale it, and by 3.46 tiles per pair of SMs taking
// the time of 4.
//
// GATE computes two products with the same rows, G and U, and writes silu(g) * u as e4m3
// rows: a tile of 128 intermediate columns is exactly one column group of the next product,
// so its scale is found in the tile.
#include <cuda.h>

#include <type_traits>

#include "fp8.cuh"
#include "tc_ptx.cuh"

namespace dkv {

using namespace ptx;

constexpr long long kGemmWaitCycles = 400000000LL;  // ~0.2 s: a healthy wait is microseconds
constexpr int kGemmThreads = 256;  // warps 0-3: scale and add; 4: copies; 5: MMA issue; all: the final sums
constexpr int kTileRows = 128;     // weight rows of a tile
constexpr int kMaxSplits = 16;
constexpr int kMaxGroups = 16384 / kFp8Group;  // of the widest rows
constexpr int kMaxGemmSmem = 210 * 1024;  // dynamic shared memory of any plan

struct GemmArgs {
  const float* sa;         // [m, groups]
  const float* sw;         // [ceil(n / 128), groups]
  const float* su;         // GATE: the same for the up weights
  void* out;               // [m, n] bf16 / fp32, or e4m3 with GATE
  float* out_scale;        // GATE: [m, ceil(n / 128)]
  int m, n, groups, splits, stages;
  int out_f32;
};

template <int NT, bool GATE>
struct GemmTile {
  static constexpr int kParts = GATE ? 2 : 1;
  static constexpr int kWeightBytes = kTileRows * kFp8Group;  // one operand tile of one group
  static constexpr int kTokenBytes = NT * kFp8Group;
  static constexpr int kStageBytes = kParts * kWeightBytes + kTokenBytes;
  static constexpr int kCols = NT * kParts;  // TMEM columns of one accumulator
  // Column groups in flight at most: operands in shared memory and an accumulator in TMEM each.
  static constexpr int kStages = 4;
  static constexpr int kTmemCols = kCols * 4;
  // blocks per SM: while one starts, loads or sums up, others keep the copies going
  static constexpr int kBlocks = kCols <= 32 ? 3 : 2;
  static_assert(kParts * NT * kTileRows * 4 <= 3 * kStageBytes, "one block's sums fit the smallest operand ring");
  static_assert(1024 + kStages * kStageBytes + kParts * NT * 4 * kMaxGroups <= kMaxGemmSmem, "whole tiles");
  static_assert(1024 + kStages * kStageBytes +
                        kParts * 4 * ((NT + kMaxSplits - 1) * kTileRows + NT * ((kMaxGroups + 1) / 2)) <= kMaxGemmSmem,
                "split tiles: sums of every rank's share, rounded up, and half of the scales at most");
  static_assert(kTmemCols * kBlocks <= 512 && kTmemCols >= 32 && (kTmemCols & (kTmemCols - 1)) == 0, "TMEM allocation");
  // operand ring, partial sums of `splits` blocks (one block's reuse the ring), scale products
  static int mail_bytes(int splits) {
    return splits > 1 ? kParts * splits * ((NT + splits - 1) / splits) * kTileRows * 4 : 0;
  }
  static int smem(int stages, int splits, int groups_per_split) {
    return 1024 + stages * kStageBytes + mail_bytes(splits) + kParts * groups_per_split * NT * 4;
  }
};

// h = silu(g) * u of four values, with e = 2^(-|g| log2 e) <= 1 and d = 1 + e in [1, 2]:
// silu(g) = g / d for g >= 0 and g e / d below, which neither overflows nor loses small results.
// The four quotients share one reciprocal of d0 d1 d2 d3: the special-function unit, a quarter
// of a result per clock and lane group, is what bounds this epilogue (five uses here; a power
// and a reciprocal each took 2048 clocks per 128 x 128 tile, IEEE expf and division more). Off
// by a few fp32 units (the exponent's rounding by |g| of them), far under the 2^-4 of the
// rounding to e4m3 that follows. A NaN spreads within its column group, whose scale is NaN.
__device__ __forceinline__ void silu_times4(const float* g, const float* u, float* h) {
  float num[4], d[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float e = ex2(-1.4426950408889634f * fabsf(g[j]));
    d[j] = 1.0f + e;
    num[j] = (g[j] < 0.f ? g[j] * e : g[j]) * u[j];
  }
  const float d01 = d[0] * d[1], d23 = d[2] * d[3];
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(d01 * d23));
  const float r01 = r * d23, r23 = r * d01;  // 1 / d01, 1 / d23
  h[0] = num[0] * (r01 * d[1]);
  h[1] = num[1] * (r01 * d[0]);
  h[2] = num[2] * (r23 * d[3]);
  h[3] = num[3] * (r23 * d[2]);
}

template <int NT, bool GATE>
__global__ void __launch_bounds__(kGemmThreads, GemmTile<NT, GATE>::kBlocks)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap umap,
                const __grid_constant__ CUtensorMap amap, const GemmArgs a) {
  using T = GemmTile<NT, GATE>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[3 * T::kStages + 1];
  __shared__ uint32_t tmem_slot;
  __shared__ int issued[2];  // groups whose copies and products were issued
  const uint32_t ring = (smem_addr(smem_raw) + 1023u) & ~1023u;
  uint8_t* const ring_ptr = smem_raw + (ring - smem_addr(smem_raw));
  // this block's own partial sums [part][token][weight row], in the ring once it is read
  float* const own = reinterpret_cast<float*>(ring_ptr);
  // ... and every block's for the tokens that it adds up: [rank][part][token][weight row]
  const int local = (NT + a.splits - 1) / a.splits;
  const uint32_t mail = ring + a.stages * T::kStageBytes;
  float* const scales = reinterpret_cast<float*>(
      ring_ptr + a.stages * T::kStageBytes + (a.splits > 1 ? a.splits * T::kParts * local * kTileRows * 4 : 0));
  const uint32_t full = smem_addr(bars);        // a stage's operands are there
  const uint32_t done = full + 8 * T::kStages;  // ... its products are done: accumulator complete, operands read
  const uint32_t freed = done + 8 * T::kStages; // ... and the accumulator is read
  const uint32_t mailed = freed + 8 * T::kStages;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = blockIdx.x % a.splits;
  const int tile = blockIdx.x / a.splits;
  const int token0 = blockIdx.y * NT;
  const int per = (a.groups + a.splits - 1) / a.splits;
  const int group0 = rank * per;
  const int count = max(0, min(per, a.groups - group0));
  const int live = min(NT, a.m - token0);
  const int mine = max(0, min(local, live - rank * local));  // tokens that this block adds up

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * T::kStages; ++i) mbar_init(full + 8 * i, 1);
    for (int i = 0; i < T::kStages; ++i) mbar_init(freed + 8 * i, 4);  // one arrival per warp
    mbar_init(mailed, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 4 && lane == 0) {
    prefetch_tensor_map(&wmap);
    if (GATE) prefetch_tensor_map(&umap);
    prefetch_tensor_map(&amap);
    // The weights of the first stages set out for L2 while the previous kernel finishes.
    for (int i = 0; i < min(count, a.stages); ++i) {
      tile2d_prefetch(&wmap, (group0 + i) * kFp8Group, tile * kTileRows);
      if (GATE) tile2d_prefetch(&umap, (group0 + i) * kFp8Group, tile * kTileRows);
    }
  }
  if (threadIdx.x == 0 && a.splits > 1) mbar_arrive_expect_tx(mailed, a.splits * T::kParts * mine * kTileRows * 4);
  __syncthreads();
  bool ran_out = false;  // a wait for this block's products did
  if (a.splits > 1) cluster_arrive_release();  // this block has started: others may write to it
  pdl_wait();  // operands are the previous kernels' output

  // Copies and products are issued by one thread each, whose every instruction waits for the
  // last: the loops are unrolled over the stages, so that nothing but the waits, the issues
  // and a few additions is left in them (with addresses and descriptors made on the way, the
  // issuing took longer than the products).
  if (warp == 4) {
    const bool issuer = elect_one();
    const auto copy = [&](int s, int i) {
      const uint32_t dst = ring + s * T::kStageBytes;
      const int x = (group0 + i) * kFp8Group;
      mbar_arrive_expect_tx(full + 8 * s, T::kStageBytes);
      tile2d_g2s(dst, &wmap, x, tile * kTileRows, full + 8 * s);
      if (GATE) tile2d_g2s(dst + T::kWeightBytes, &umap, x, tile * kTileRows, full + 8 * s);
      tile2d_g2s(dst + T::kParts * T::kWeightBytes, &amap, x, token0, full + 8 * s);
    };
    if (issuer) {
#pragma unroll
      for (int s = 0; s < T::kStages; ++s) {
        if (s >= count || s == a.stages) break;
        copy(s, s);
      }
    }
    __syncwarp();
    named_bar_sync(4, 64);  // no wait of limited time before this block has its TMEM
    if (issuer) {
      bool ok = true;
      int i = min(count, a.stages);
      for (uint32_t phase = 0; i < count && ok; phase ^= 1) {
#pragma unroll
        for (int s = 0; s < T::kStages; ++s, ++i) {
          if (i >= count || s == a.stages) break;
          ok = mbar_wait(done + 8 * s, phase, kGemmWaitCycles);
          if (!ok) break;
          copy(s, i);
        }
      }
      issued[0] = i;
    }
    __syncwarp();
  } else if (warp == 5) {
    // TMEM is taken after the wait and before the trigger: a waiting block never holds what
    // the grid it waits for still needs, and no dependent starts before every block has it.
    tmem_alloc(smem_addr(&tmem_slot), T::kTmemCols);
    tmem_relinquish();
    pdl_trigger();
    tc_fence_before();
    named_bar_arrive(4, 64);
    named_bar_arrive(2, 160);  // the products need not wait for the scales
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    if (elect_one()) {
      constexpr uint32_t idesc = idesc_e4m3(kTileRows, NT);
      const uint64_t wd0 = sw128_desc(ring, 16, 1024);
      const uint64_t ud0 = wd0 + (T::kWeightBytes >> 4);
      const uint64_t ad0 = wd0 + (T::kParts * T::kWeightBytes >> 4);
      bool ok = true;
      int i = 0;
      for (uint32_t phase = 0; i < count && ok; phase ^= 1) {
#pragma unroll
        for (int s = 0; s < T::kStages; ++s, ++i) {
          if (i >= count || s == a.stages) break;
          ok = mbar_wait(full + 8 * s, phase, kGemmWaitCycles);
          if (ok && i >= a.stages) ok = mbar_wait(freed + 8 * s, phase ^ 1, kGemmWaitCycles);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int j = 0; j < kFp8Group / 32; ++j) {  // 32 columns are 32 bytes: 2 descriptor units
            const uint32_t at = s * (T::kStageBytes >> 4) + 2 * j;
            umma_f8(tmem + s * T::kCols, wd0 + at, ad0 + at, idesc, j > 0);
            if (GATE) umma_f8(tmem + s * T::kCols + NT, ud0 + at, ad0 + at, idesc, j > 0);
          }
          umma_commit(done + 8 * s);
        }
      }
      issued[1] = i;
    }
    __syncwarp();
  } else if (warp < 4) {
    // the scale products of this block's groups: scales[part][group][token]
    for (int i = threadIdx.x; i < count * NT; i += 128) {
      const int token = i / count;
      const int g = i - token * count;
      const float s = token0 + token < a.m ? a.sa[static_cast<int64_t>(token0 + token) * a.groups + group0 + g] : 0.f;
      const int64_t block = static_cast<int64_t>(tile) * a.groups + group0 + g;
      scales[g * NT + token] = s * a.sw[block];
      if (GATE) scales[(count + g) * NT + token] = s * a.su[block];
    }
    tc_fence_before();
    named_bar_sync(2, 160);  // the scales of all four warps, and TMEM's address
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    constexpr int kStep = T::kCols <= 32 ? 16 : 32;
    float acc[T::kCols];
#pragma unroll
    for (int j = 0; j < T::kCols; ++j) acc[j] = 0.f;
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    bool ok = true;
    for (int i = 0, slot = 0, phase = 0; i < count && ok; ++i) {
      ok = __all_sync(0xffffffffu, mbar_wait(done + 8 * slot, phase, kGemmWaitCycles));
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < T::kCols; c += kStep) {
        uint32_t p[kStep];
        if constexpr (kStep == 32) {
          tmem_ld32(tmem + lanes + slot * T::kCols + c, p);
        } else {
          tmem_ld16(tmem + lanes + slot * T::kCols + c, p);
        }
        tmem_wait_ld();
        const float* sc = scales + (c < NT ? i * NT + c : (count + i) * NT + c - NT);
#pragma unroll
        for (int j = 0; j < kStep; j += 4) {
          const float4 f = *reinterpret_cast<const float4*>(sc + j);
          float2* ac = reinterpret_cast<float2*>(acc + c + j);
          ac[0] = fma2(make_float2(__uint_as_float(p[j]), __uint_as_float(p[j + 1])), make_float2(f.x, f.y), ac[0]);
          ac[1] = fma2(make_float2(__uint_as_float(p[j + 2]), __uint_as_float(p[j + 3])), make_float2(f.z, f.w), ac[1]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(freed + 8 * slot);
      if (++slot == a.stages) slot = 0, phase ^= 1;
    }
    // Where a wait ran out, copies may still arrive on these sums: they are not used or sent, and
    // this block's tokens, and those of the blocks that wait for its sums, become NaN below.
#pragma unroll
    for (int j = 0; j < T::kCols; ++j) own[j * kTileRows + threadIdx.x] = acc[j];
    ran_out = !ok;
    if (a.splits > 1) {
      // Rank r adds up tokens [r * local, (r + 1) * local): one bulk copy per rank and part
      // (single stores to another block's shared memory were 5 times slower).
      fence_proxy_async_smem();
      cluster_wait_acquire();
      ran_out = named_bar_or(3, 128, ran_out);
      const int to = threadIdx.x;
      const int n = min(local, live - to * local);
      if (to < a.splits && n > 0 && !ran_out) {
#pragma unroll
        for (int p = 0; p < T::kParts; ++p)
          bulk_s2s(dsmem_addr(mail + (rank * T::kParts + p) * local * kTileRows * 4, to),
                   ring + (p * NT + to * local) * kTileRows * 4, n * kTileRows * 4, dsmem_addr(mailed, to));
      }
    }
  }
  if (a.splits > 1) {
    if (warp >= 4) cluster_wait_acquire();
    cluster_arrive_relaxed();  // this block has its TMEM, and its sums are on their way
  }
  // TMEM goes back before this block waits for another one: what holds TMEM never depends
  // on a block that may still be waiting for some.
  tc_fence_before();
  ran_out = __syncthreads_or(ran_out);
  if (warp == 5) {
    if (ran_out && lane == 0) {  // copies and products that still use this block's memories end first
      for (int j = max(0, issued[0] - a.stages); j < issued[0]; ++j)
        mbar_wait(full + 8 * (j % a.stages), (j / a.stages) & 1, kGemmWaitCycles);
      for (int j = max(0, issued[1] - a.stages); j < issued[1]; ++j)
        mbar_wait(done + 8 * (j % a.stages), (j / a.stages) & 1, kGemmWaitCycles);
    }
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_slot, T::kTmemCols);
  }
  const float* sums = own;
  int parts_apart = NT * kTileRows;
  bool complete = !ran_out;
  if (a.splits > 1) {
    sums = reinterpret_cast<const float*>(ring_ptr + a.stages * T::kStageBytes);
    parts_apart = local * kTileRows;
    // The time counts from when every block had its TMEM, which another stream's kernel may hold for
    // long; where all goes well that is past before the sums are here. A block that ran out sends nothing.
    if (mine > 0) complete = mbar_wait(mailed, 0, kGemmWaitCycles);
    __syncwarp();
    cluster_wait_acquire();
    if (!complete) complete = mbar_wait(mailed, 0, kGemmWaitCycles);
  }

  // A warp per token, 4 weight rows (output columns) per lane: neighbouring ones where a row's
  // start lets them be stored together, else every 32nd, so that neighbouring lanes store
  // neighbouring columns.
  const bool vectors = GATE || (a.n & 3) == 0;
  const int col = tile * kTileRows + (vectors ? lane * 4 : lane);
  const int first = a.splits > 1 ? rank * local : 0;
  const auto take = [&](const float* at) {
    at += vectors ? lane * 4 : lane;
    return vectors ? *reinterpret_cast<const float4*>(at) : make_float4(at[0], at[32], at[64], at[96]);
  };
  for (int i = warp; i < (a.splits > 1 ? mine : live); i += kGemmThreads / 32) {
    const int t = first + i;
    float4 sum[T::kParts];
#pragma unroll
    for (int p = 0; p < T::kParts; ++p) {
      const float* at = sums + p * parts_apart + i * kTileRows;
      sum[p] = take(at);
      for (int r = 1; r < a.splits; ++r) {
        const float4 v = take(at + r * T::kParts * parts_apart);
        sum[p].x += v.x;
        sum[p].y += v.y;
        sum[p].z += v.z;
        sum[p].w += v.w;
      }
      if (!complete) sum[p].x = sum[p].y = sum[p].z = sum[p].w = __int_as_float(0x7fc00000);
    }
    const int64_t row = token0 + t;
    if (GATE) {  // n is a multiple of 16: a lane's 4 columns are all inside or all outside
      float4 h = make_float4(0.f, 0.f, 0.f, 0.f);
      if (col < a.n) silu_times4(&sum[0].x, &sum[T::kParts - 1].x, &h.x);
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
      const float e[4] = {v.x, v.y, v.z, v.w};
      if (a.out_f32) {
        float* o = static_cast<float*>(a.out) + at;
        if (vectors) {
          if (col < a.n) *reinterpret_cast<float4*>(o) = v;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (col + 32 * j < a.n) o[32 * j] = e[j];
        }
      } else {
        __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.out) + at;
        if (vectors) {
          if (col < a.n) *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (col + 32 * j < a.n) o[32 * j] = __float2bfloat16_rn(e[j]);
        }
      }
    }
  }
  if (a.splits > 1) {  // the copies out of this block's memory have arrived; nothing to order:
    cluster_arrive_relaxed();  // a release would wait for this block's stores first
    cluster_wait_acquire();
  }
}

// ---- many tokens -----------------------------------------------------------------
// fp8_wide_kernel keeps the tensor cores busy when there are tokens for it: a pair of
// blocks works on a tile of 256 tokens x 256 weight rows, each block with 128 of the
// tokens on its accumulators' lanes and half of the weight rows in its shared memory (so
// per group and block 32 KB arrive for 128 x 256 x 128 products; blocks of their own would
// need 48, and L2 gives an SM ~65 bytes per clock). Two accumulators of 256 columns fill
// TMEM: while the tensor cores sum one group into one (512 clocks at their rate), the eight
// epilogue warps scale and add the other. An accumulator's round (products, completion,
// reading, release) takes ~1400 clocks, so two of them make a group ~700. In the builds that tried
// them, four accumulators of 128 columns lost (products of 128 columns run at half rate: 96 us for
// 4096^3 against 67), as did sixteen epilogue warps of 64 columns (72.6 against 70.3).
// A thread owns one token and 128 columns; a group costs it a scale product and 64 packed FMAs.
// The grid is persistent (one pair per two SMs): a tile's way out overlaps the next tile's first
// groups. GATE gives the pair's first block the gate rows and the second the up rows of the
// same 128 intermediate columns: each thread then holds matching columns of G and U.
constexpr int kWideThreads = 384;  // warps 0-7: scale and add; 8: copies; 9: MMA issue; 10, 11: scales
constexpr int kWideStages = 4;
constexpr int kWideHalf = 128 * kFp8Group;  // bytes of one block's operand tile of one group
constexpr int kWideStageBytes = 2 * kWideHalf;
constexpr int kWideChunk = 16;  // groups whose scales are staged at a time
constexpr int kWidePairs = 74;  // of blocks, all SMs
constexpr int kWideScales = kWideChunk * 128 + 2 * kWideChunk;  // [group][token], then [group][half] of the weights
constexpr int kTurnBytes = 32 * 128;  // of output: 32 tokens x 128 bytes
constexpr int kWideSmem = 1024 + kWideStages * kWideStageBytes + 8 * 2 * kTurnBytes + 2 * kWideScales * 4;
constexpr int kWideCols = 256;
constexpr int kWideSlots = 2;
constexpr uint32_t kWideTmem = kWideSlots * kWideCols;

// A warp's output leaves through one of its two pieces of shared memory: 32 tokens (one per
// lane) x BYTES (64 or 128), as 16-byte words w, in the swizzled order of a tensor map's box of
// the same shape (word c of row r is exchanged by r % 8, with 64-byte rows by (r / 2) % 4: free
// of bank conflicts), and from there as one tile copy that runs on while the warp goes on
// (stores by the threads, in whole lines or not, held the epilogue up by 1000 clocks per 64
// columns: every byte passes the shared memory and the store path of the SM).
template <int BYTES>
__device__ __forceinline__ void store_tile(const CUtensorMap* map, int x, int y, bool inside, const uint4* w,
                                           uint8_t* piece) {
  const int lane = threadIdx.x & 31;
  if (lane == 0) bulk_wait_read<1>();  // the tile before last has left this piece
  __syncwarp();
#pragma unroll
  for (int c = 0; c < BYTES / 16; ++c) {
    const int at = BYTES == 128 ? c ^ (lane & 7) : c ^ ((lane >> 1) & 3);
    *reinterpret_cast<uint4*>(piece + lane * BYTES + at * 16) = w[c];
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    if (inside) tile2d_s2g(map, x, y, smem_addr(piece));
    bulk_commit();
  }
}

// The same for rows that no tensor map can describe (a row's start not on 16 bytes): a lane
// stores one aligned 4-byte word of a row, the warp a row at a time, eight rows read at once. A
// bf16 row that starts between words is shifted by one element, its ends stored alone. Rows
// from `tokens` on and columns from `columns` on (of the warp's `128 / SIZE`) are left alone;
// `out` is the first row's first column, rows are n elements apart.
template <int SIZE>
__device__ __forceinline__ void store_words(uint8_t* out, int64_t n, bool odd_start, int tokens, int columns,
                                            const uint4* w, uint8_t* piece) {
  const int lane = threadIdx.x & 31;
  __syncwarp();  // the last call's reads
#pragma unroll
  for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(piece + lane * 128 + ((c ^ (lane & 7)) << 4)) = w[c];
  __syncwarp();
  if (columns <= 0) return;
#pragma unroll 1
  for (int r0 = 0; r0 < 32 && r0 < tokens; r0 += 8) {
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = *reinterpret_cast<const uint32_t*>(piece + (r0 + i) * 128 + (((lane >> 2) ^ i) << 4) + (lane & 3) * 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool row = r0 + i < tokens;
      uint8_t* dst = out + (r0 + i) * n * SIZE;
      if constexpr (SIZE == 4) {
        if (row && lane < columns) reinterpret_cast<uint32_t*>(dst)[lane] = v[i];
      } else {
        const uint32_t next = __shfl_down_sync(0xffffffffu, v[i], 1);
        const int c = 2 * lane;
        uint16_t* e = reinterpret_cast<uint16_t*>(dst);
        if (!odd_start == !((r0 + i) & n & 1)) {  // the row starts on a word
          if (row && c + 1 < columns) *reinterpret_cast<uint32_t*>(e + c) = v[i];
          if (row && c + 1 == columns) e[c] = static_cast<uint16_t>(v[i]);
        } else {
          if (row && c + 2 < columns && lane < 31) *reinterpret_cast<uint32_t*>(e + c + 1) = (v[i] >> 16) | (next << 16);
          if (row && c + 1 < columns && (c + 2 == columns || lane == 31)) e[c + 1] = static_cast<uint16_t>(v[i] >> 16);
          if (row && lane == 0) e[0] = static_cast<uint16_t>(v[i]);
        }
      }
    }
  }
}

// How a pair kernel gives out its tiles and stores them: three kernels, because what the other
// two need takes registers and clocks from the loop over the groups (when they were split, one kernel
// for whole and half tiles took 34.8 us for 2048 x 4096 x 4096 against 32.7, and 90 for 4096 x 4097 x
// 4096 with words in it against 84).
// kHalves: of at most three rounds, the last one's tiles (at most half as many as there are pairs)
// are cut into halves of 128 weight rows. Products of 128 columns run at half rate (0.31 us a group
// for 0.40 of a whole tile), but two pairs share a tile: 512 x 4096 x 4096 17.2 -> 15.4 us, after
// two whole rounds (2048 x 5120 x 960) 16.9 -> 16.3. After three whole rounds of 32 groups (4096^3)
// they cost more than they give (70.7 -> 73.2 in a long run); other numbers of groups after three were
// not measured. GATE's tiles stay whole: a column group needs both halves.
// kWords: the output's rows do not start on 16 bytes.
enum class WideForm { kWhole, kHalves, kWords };

WideForm wide_form(const GemmArgs& a, int64_t tiles, bool gate) {
  if (gate) return WideForm::kWhole;
  if (static_cast<int64_t>(a.n) * (a.out_f32 ? 4 : 2) % 16 != 0) return WideForm::kWords;
  const int64_t rest = tiles % kWidePairs;
  return rest > 0 && 2 * rest <= kWidePairs && tiles < 3 * kWidePairs ? WideForm::kHalves : WideForm::kWhole;
}

// The tiles of one pair of blocks, `pairs` apart, first token fastest.
template <bool HALVES>
struct WideWork {
  int pair, pairs, tiles_m, rounds, units;

  __device__ __forceinline__ WideWork(const GemmArgs& a, int columns)
      : pair(blockIdx.x >> 1), pairs(gridDim.x >> 1), tiles_m((a.m + 255) / 256) {
    const int tiles = tiles_m * ((a.n + columns - 1) / columns);
    rounds = tiles / pairs;
    const int rest = tiles - rounds * pairs;
    units = rounds + (pair < (HALVES ? 2 * rest : rest));
  }
  // Unit k: its first token, its tile of weight rows, and which half of it (-1: all).
  __device__ __forceinline__ void unit(int k, int& token0, int& tn, int& half) const {
    const bool cut = HALVES && k == rounds;
    const int tile = k * pairs + (cut ? pair >> 1 : pair);
    half = cut ? pair & 1 : -1;
    token0 = (tile % tiles_m) * 256;
    tn = tile / tiles_m;
  }
};

template <bool GATE, WideForm FORM>
__global__ void __launch_bounds__(kWideThreads, 1)
fp8_wide_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap umap,
                const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap omap, const GemmArgs a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * kWideStages + kWideSlots + 4];
  __shared__ uint32_t tmem_slot;
  __shared__ float amax_part[2][2][128];  // GATE: [tile parity][column part][token]
  const uint32_t ring = (smem_addr(smem_raw) + 1023u) & ~1023u;
  const uint32_t full = smem_addr(bars);         // rank 0's: both blocks' copies of a stage
  // each block's own: a stage's products are done, its accumulator complete and its buffers
  // empty (one commit for both)
  const uint32_t done = full + 8 * kWideStages;
  const uint32_t freed = done + 8 * kWideStages;  // rank 0's: both blocks have read an accumulator
  const uint32_t staged = freed + 8 * kWideSlots;  // each block's own: a chunk of scales is there
  const uint32_t used = staged + 16;               // ... and no longer needed
  uint8_t* const pieces = smem_raw + (ring - smem_addr(smem_raw)) + kWideStages * kWideStageBytes;  // 1024-byte aligned
  float* const scales = reinterpret_cast<float*>(pieces + 8 * 2 * kTurnBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1;
  constexpr bool kHalves = FORM == WideForm::kHalves;
  const WideWork<kHalves> work(a, GATE ? 128 : 256);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * kWideStages; ++i) mbar_init(full + 8 * i, 1);
    for (int i = 0; i < kWideSlots; ++i) mbar_init(freed + 8 * i, 8 + (rank == 0));  // own epilogue warps, and rank 1 as one
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
  const int total = work.units * a.groups;  // groups of all tiles

  // 384 x 168 registers at launch = 128 x (72 + 216 + 216). Each role gets ready, and waits for
  // the previous kernel, whose output the operands are, right before its first access.
  if (warp >= 8) {
    regs_give<72>();
    if (warp == 9) {
      // TMEM is taken after the wait and before the trigger (see fp8_gemm_kernel). The blocks'
      // rendezvous after it is relaxed: a release at cluster scope would take ~0.5 us, and
      // what follows it are tcgen05 operations, fenced on both sides.
      pdl_wait();
      tmem_alloc_pair(smem_addr(&tmem_slot), kWideTmem);
      tmem_relinquish_pair();
      tc_fence_before();
      named_bar_arrive(2, 288);  // the epilogue warps may read TMEM's address
    }
    cluster_arrive_relaxed();
    if (warp == 9) {
      cluster_wait_acquire();
      tc_fence_after();
      pdl_trigger();  // after both blocks' allocation
    }
    // No wait of limited time begins before both blocks have their TMEM, which another stream's
    // kernel may hold for long: each role waits for the rendezvous before its first.
    if (warp == 8) {
      const bool issuer = elect_one();
      const uint32_t full0 = dsmem_addr(full, 0);
      const CUtensorMap* const rows = GATE && rank == 1 ? &umap : &wmap;
      int unit = 0, x = 0, token0, row0;
      const auto next = [&] {  // a half tile's box holds 64 rows more than its products read
        int tn, half;
        work.unit(unit++, token0, tn, half);
        token0 += rank * 128;
        row0 = GATE ? tn * 128 : half < 0 ? tn * 256 + rank * 128 : tn * 256 + half * 128 + rank * 64;
      };
      const auto copy = [&](int s) {
        const uint32_t dst = ring + s * kWideStageBytes;
        if (rank == 0) mbar_arrive_expect_tx(full + 8 * s, 2 * kWideStageBytes);
        tile2d_g2s_pair(dst, &amap, x, token0, full0 + 8 * s);
        tile2d_g2s_pair(dst + kWideHalf, rows, x, row0, full0 + 8 * s);
        x += kFp8Group;
        if (x >= a.groups * kFp8Group) {
          x = 0;
          next();
        }
      };
      next();
      if (issuer) {
        pdl_wait();
#pragma unroll
        for (int s = 0; s < kWideStages; ++s) {
          if (s >= total) break;
          copy(s);
        }
      }
      __syncwarp();
      cluster_wait_acquire();
      if (issuer) {
        bool ok = true;
        int i = min(total, kWideStages);
        for (uint32_t phase = 0; i < total && ok; phase ^= 1) {
#pragma unroll
          for (int s = 0; s < kWideStages; ++s, ++i) {
            if (i >= total) break;
            ok = mbar_wait(done + 8 * s, phase, kGemmWaitCycles);
            if (!ok) break;
            copy(s);
          }
        }
        // Both blocks' last copies arrive before the pair leaves, also where a wait ran out here or
        // in another warp (elsewhere the products have waited for them already).
        if (rank == 0)
          for (int j = max(0, i - kWideStages); j < i; ++j)
            mbar_wait(full + 8 * (j % kWideStages), (j / kWideStages) & 1, kGemmWaitCycles);
      }
    } else if (warp == 9 && rank == 1 && elect_one()) {
      // rank 1's eight warps reach rank 0 as one arrival
      const uint32_t freed0 = dsmem_addr(freed, 0);
      for (int i = 0; i < total; ++i) {
        const int slot = i % kWideSlots;
        if (!mbar_wait(freed + 8 * slot, (i / kWideSlots) & 1, kGemmWaitCycles)) break;
        mbar_arrive_cluster(freed0 + 8 * slot);
      }
    } else if (warp == 9 && rank == 0 && elect_one()) {
      const uint32_t tmem = tmem_slot;
      const int cut = work.rounds * a.groups;  // from here on half tiles
      const uint64_t ad0 = sw128_desc(ring, 16, 1024);
      const uint64_t wd0 = ad0 + (kWideHalf >> 4);
      bool ok = true;
      int i = 0;
      static_assert(kWideStages == 2 * kWideSlots, "a stage uses accumulator s % 2, in its turn s / 2");
      for (uint32_t phase = 0; i < total && ok; phase ^= 1) {
#pragma unroll
        for (int s = 0; s < kWideStages; ++s, ++i) {
          if (i >= total) break;
          const int slot = s % kWideSlots;
          const uint32_t idesc = !kHalves || i < cut ? idesc_e4m3(256, kWideCols) : idesc_e4m3(256, kWideCols / 2);
          ok = mbar_wait(full + 8 * s, phase, kGemmWaitCycles);
          // an accumulator goes round twice while the stages go round once
          if (ok && i >= kWideSlots) ok = mbar_wait(freed + 8 * slot, s < kWideSlots ? 1 : 0, kGemmWaitCycles);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int j = 0; j < kFp8Group / 32; ++j) {
            const uint32_t at = s * (kWideStageBytes >> 4) + 2 * j;
            umma_f8_pair(tmem + slot * kWideCols, ad0 + at, wd0 + at, idesc, j > 0);
          }
          umma_commit_pair(done + 8 * s);
        }
      }
      // The last arrivals from the other block are waited for as all others are: this block must
      // not leave, and its shared memory go to another, while one is on its way. Where a wait ran
      // out, the products in flight end before TMEM is freed.
      for (int j = max(0, i - kWideSlots); j < i; ++j) {
        if (ok)
          mbar_wait(freed + 8 * (j % kWideSlots), (j / kWideSlots) & 1, kGemmWaitCycles);
        else
          mbar_wait(done + 8 * (j % kWideStages), (j / kWideStages) & 1, kGemmWaitCycles);
      }
    }
    if (warp >= 10) {
      pdl_wait();
      // The scales arrive as rows of groups, and each epilogue thread needs one row: read by
      // that thread, every group would be 32 cache lines per warp. Copied flat and turned
      // over in shared memory, it is one conflict-free load.
      const int t = threadIdx.x - 32 * 10;
      int c = 0;
      bool ok = true, met = false;
      for (int unit = 0; unit < work.units && ok; ++unit) {
        int token0, tn, half;
        work.unit(unit, token0, tn, half);
        token0 += rank * 128;
        const int tokens = min(128, a.m - token0);  // may be negative: nothing to read
        const float* sw0 = a.sw + static_cast<int64_t>(GATE ? tn : 2 * tn) * a.groups;
        const float* sw1 = GATE ? a.su + static_cast<int64_t>(tn) * a.groups
                                : a.sw + static_cast<int64_t>(min(2 * tn + 1, (a.n + 127) / 128 - 1)) * a.groups;
        for (int g0 = 0; g0 < a.groups; g0 += kWideChunk, ++c) {
          const int n = min(kWideChunk, a.groups - g0);
          if (c == 2) {
            __syncwarp();
            cluster_wait_acquire();
            met = true;
          }
          if (c >= 2 && !mbar_wait(used + 8 * (c & 1), ((c >> 1) + 1) & 1, kGemmWaitCycles)) {
            ok = false;
            break;
          }
          // asynchronous 4-byte copies: all of them in flight at once, and none in registers
          const uint32_t dst = smem_addr(scales + (c & 1) * kWideScales);
          const int g = t % kWideChunk;
          if (g < n) {
            const float* src = a.sa + (static_cast<int64_t>(token0) + t / kWideChunk) * a.groups + g0 + g;
            for (int token = t / kWideChunk; token < tokens; token += 64 / kWideChunk, src += 64 / kWideChunk * a.groups)
              cp_async4(dst + (g * 128 + token) * 4, src);
          }
          if (t < 2 * n) cp_async4(dst + (kWideChunk * 128 + t) * 4, (t & 1 ? sw1 : sw0) + g0 + (t >> 1));
          cp_async_mbar_arrive(staged + 8 * (c & 1));
        }
      }
      __syncwarp();
      if (!met) cluster_wait_acquire();  // no third chunk
    }
    __syncwarp();
  } else {
    regs_take<216>();
    cluster_arrive_relaxed();
    pdl_wait();
    named_bar_sync(2, 288);
    cluster_wait_acquire();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const int part = warp >> 2;
    const int token_in = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    uint8_t* const turn = pieces + warp * 2 * kTurnBytes;
    int i = 0, chunk = 0;
    bool ok = true;
    const auto next_chunk = [&] {  // this warp is done with a chunk of scales
      __syncwarp();
      if (lane == 0) mbar_arrive(used + 8 * (chunk & 1));
      ++chunk;
    };
    for (int unit = 0, parity = 0; unit < work.units; ++unit, parity ^= 1) {
      int token, tn, half;
      work.unit(unit, token, tn, half);
      token += rank * 128 + token_in;
      const bool whole = !kHalves || half < 0;
      const int second = GATE ? 0 : whole ? part : half;  // which of the tile's weight blocks
      const uint32_t columns = tmem + lanes + part * (GATE || !whole ? 64 : 128);
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
        const float* sw = scales + (chunk & 1) * kWideScales + kWideChunk * 128 + 2 * (g % kWideChunk) + second;
        const float f0 = sa * sw[0], f1 = GATE ? sa * sw[1] : f0;
        const int slot = i % kWideSlots;
        const int s = i % kWideStages;
        ok = ok && __all_sync(0xffffffffu, mbar_wait(done + 8 * s, (i / kWideStages) & 1, kGemmWaitCycles));
        if (!ok) continue;
        tc_fence_after();
        const uint32_t src = columns + slot * kWideCols;
        // 32 columns at a time, the next ones on their way from TMEM while these are added
        const auto add = [&](auto chunks) {
          constexpr int kChunks = decltype(chunks)::value;
          uint32_t p[2][32];
          tmem_ld32(src, p[0]);
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            tmem_wait_ld();
            if (c + 1 < kChunks) {
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
              ac[j] =
                  fma2(make_float2(__uint_as_float(p[c & 1][2 * j]), __uint_as_float(p[c & 1][2 * j + 1])), f, ac[j]);
          }
        };
        if (whole)
          add(std::integral_constant<int, 4>{});
        else
          add(std::integral_constant<int, 2>{});
      }
      next_chunk();
      if (!ok) {  // a wait that ran out leaves NaN, not a stale tile
#pragma unroll
        for (int j = 0; j < 128; ++j) acc[j] = __int_as_float(0x7fc00000);
      }
      if (GATE) {
        const int col0 = tn * 128 + part * 64;
        float amax = 0.f;
        const int inside = a.n - col0;  // a multiple of 16, like the columns below
#pragma unroll
        for (int j = 0; j < 64; j += 16) {
          float m = 0.f;
#pragma unroll
          for (int i = j; i < j + 16; i += 4) {
            silu_times4(acc + i, acc + 64 + i, acc + i);
            m = max_nan(m, max_nan(max_nan(fabsf(acc[i]), fabsf(acc[i + 1])), max_nan(fabsf(acc[i + 2]), fabsf(acc[i + 3]))));
          }
          if (j < inside) amax = max_nan(amax, m);
        }
        amax_part[parity][part][token_in] = amax;
        named_bar_sync(1, 256);
        amax = max_nan(max_nan(amax, amax_part[parity][part ^ 1][token_in]), kFp8Floor);
        const float inverse = __fdiv_rn(kFp8Max, amax);
        uint4 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = codes16(acc + 16 * j, inverse);
        // n is a multiple of 16: a tensor map describes every output
        store_tile<64>(&omap, col0, token - lane, col0 < a.n && token - lane < a.m, w, turn + parity * kTurnBytes);
        if (live && part == 0) a.out_scale[static_cast<int64_t>(token) * blocks + tn] = __fdiv_rn(amax, kFp8Max);
      } else if (a.out_f32) {
#pragma unroll
        for (int j = 0; j < 128; j += 32) {
          if (j == 64 && !whole) break;
          const int col = tn * 256 + (whole ? part * 128 : half * 128 + part * 64) + j;
          const uint4* w = reinterpret_cast<const uint4*>(acc + j);
          if constexpr (FORM != WideForm::kWords)
            store_tile<128>(&omap, col, token - lane, col < a.n && token - lane < a.m, w, turn + (j / 32 & 1) * kTurnBytes);
          else
            store_words<4>(static_cast<uint8_t*>(a.out) + (static_cast<int64_t>(token - lane) * a.n + col) * 4, a.n, false,
                           a.m - (token - lane), a.n - col, w, turn);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 128; j += 64) {
          if (j == 64 && !whole) break;
          const int col = tn * 256 + (whole ? part * 128 : half * 128 + part * 64) + j;
          uint4 w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float* v = acc + j + 8 * i;
            w[i] = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                              pack_bf16x2(v[6], v[7]));
          }
          if constexpr (FORM != WideForm::kWords)
            store_tile<128>(&omap, col, token - lane, col < a.n && token - lane < a.m, w, turn + (j / 64) * kTurnBytes);
          else
            store_words<2>(static_cast<uint8_t*>(a.out) + (static_cast<int64_t>(token - lane) * a.n + col) * 2, a.n,
                           (static_cast<int64_t>(token - lane) * a.n + col) & 1, a.m - (token - lane), a.n - col, w, turn);
        }
      }
    }
    if (lane == 0) bulk_wait_read<0>();  // the pieces are read; the grid ends when all is written
  }
  // the other block's copies, arrivals and products are done with this one (no memory to order:
  // a release would wait for this block's stores)
  tc_fence_before();
  cluster_arrive_relaxed();
  cluster_wait_acquire();
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

// The output's tiles of 32 rows x 128 bytes (e4m3: 64) as store_tile writes them; an output whose
// rows do not start on 16 bytes has none, and its map is not used.
bool encode_output(CUtensorMap* map, const GemmArgs& a, bool gate) {
  const FnEncode fn = encoder();
  if (fn == nullptr) return false;
  const int size = gate ? 1 : a.out_f32 ? 4 : 2;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(a.n), static_cast<cuuint64_t>(a.m)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(a.n) * size};
  if (strides[0] % 16 != 0) return true;
  const cuuint32_t boxes[2] = {static_cast<cuuint32_t>(gate ? 64 : 128 / size), 32};
  const cuuint32_t steps[2] = {1, 1};
  return fn(map,
            gate        ? CU_TENSOR_MAP_DATA_TYPE_UINT8
            : a.out_f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                        : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
            2, a.out, dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
            gate ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct GemmCall {
  const void *a, *w, *u;
  int64_t as, ws, us;  // row strides in bytes
  int k;
  GemmArgs args;
};

// Operand stages of the split kernel: one more where blocks have an SM to themselves; two or three
// share it otherwise.
int gemm_stages(const GemmArgs& a, int tokens, int splits) {
  const int64_t blocks = static_cast<int64_t>((a.n + kTileRows - 1) / kTileRows) * splits * ((a.m + tokens - 1) / tokens);
  return blocks <= 148 ? 4 : 3;
}

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
  const int per = (args.groups + splits - 1) / splits;
  args.stages = gemm_stages(args, NT, splits);
  static_assert(T::kStages == 4, "gemm_stages");
  const int smem = T::smem(args.stages, splits, per);
  // the same limit for every call: threads that launch other shapes at the same time set it too
  cudaError_t e =
      cudaFuncSetAttribute(fp8_gemm_kernel<NT, GATE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxGemmSmem);
  if (e == cudaSuccess && splits > 8)
    e = cudaFuncSetAttribute(fp8_gemm_kernel<NT, GATE>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
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

template <bool GATE, WideForm FORM>
cudaError_t launch_wide(const GemmCall& c, int64_t tiles, cudaStream_t stream) {
  CUtensorMap wmap, umap, amap, omap = {};
  if (!encode_tiles(&wmap, c.w, c.args.n, c.k, c.ws, 128) || !encode_tiles(&amap, c.a, c.args.m, c.k, c.as, 128))
    return cudaErrorInvalidValue;
  umap = wmap;
  if (!encode_output(&omap, c.args, GATE)) return cudaErrorInvalidValue;
  if (GATE && !encode_tiles(&umap, c.u, c.args.n, c.k, c.us, 128)) return cudaErrorInvalidValue;
  const cudaError_t e =
      cudaFuncSetAttribute(fp8_wide_kernel<GATE, FORM>, cudaFuncAttributeMaxDynamicSharedMemorySize, kWideSmem);
  if (e != cudaSuccess) return e;
  const int64_t units = FORM == WideForm::kHalves && tiles < kWidePairs ? 2 * tiles : tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * static_cast<unsigned>(units < kWidePairs ? units : kWidePairs));
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
  return cudaLaunchKernelEx(&cfg, fp8_wide_kernel<GATE, FORM>, wmap, umap, amap, omap, c.args);
}

// Which kernel, how many tokens per tile and how many blocks per tile: the least time by a
// model fitted to a sweep of all of them over 49 shapes (1 to 8192 tokens, 128 to 49280 weight
// rows, 256 to 16384 columns; weights beyond L2; in us on a B200, mostly within 10 %). With c
// the accumulator columns of a token tile (tokens, doubled by GATE):
//   split kernel  start 2.0 + 0.012 c (GATE 0.5 more), 0.9 for every block an SM has to start
//                 beyond its first; per column group 0.12 + 0.003 c, or the time in which all
//                 blocks' operands come from L2 at 13 bytes/ps; summing up a split tile 0.3 + 0.02 c
//   pair kernel   start 3.0; per round of 74 tiles 0.40 per column group and 1.2 (GATE 2.0), a
//                 round of half tiles 0.31 and 1.0
// Measured on either side of its borders: 512 x 960 x 960 4.3 us by 32 tokens a tile (16: 5.6, 64:
// 5.2, pairs 6.0); 64 x 960 x 2560 3.6 by 16 tokens and 4 blocks a tile (one block: 5.6, three 3.9,
// five 5.4; 32 tokens and four blocks 4.2; 64 and five 4.9); 2048 x 1600 x 960 7.9 by pairs (64
// tokens: 12.0); gate/up 25 x 2560 x 960 4.9 by 16 tokens and one block (two blocks 5.1; 32 tokens
// and four 5.2), 512 x 2560 x 960 8.3 by pairs (32 tokens: 15.6). dkv_fp8_plan gives a call's choice.
struct GemmPlan {
  int tokens;  // per tile; 256: the pair kernel
  int splits;
};

int64_t wide_tiles(const GemmArgs& a, bool gate) {
  const int columns = gate ? 128 : 256;
  return static_cast<int64_t>((a.m + 255) / 256) * ((a.n + columns - 1) / columns);
}

GemmPlan make_gemm_plan(const GemmArgs& a, bool gate) {
  const int m = a.m, n = a.n, groups = a.groups;
  const int parts = gate ? 2 : 1;
  const int64_t pair_tiles = wide_tiles(a, gate);
  const bool halves = wide_form(a, pair_tiles, gate) == WideForm::kHalves;
  GemmPlan best{256, 1};
  const float round = groups * 0.40f + (gate ? 2.0f : 1.2f);
  float least = 3.0f + static_cast<float>(pair_tiles / kWidePairs) * round;
  if (pair_tiles % kWidePairs > 0) least += halves ? groups * 0.31f + 1.0f : round;
  for (int nt = 16; nt <= (gate ? 32 : 64); nt *= 2) {
    const int64_t tiles = static_cast<int64_t>((n + kTileRows - 1) / kTileRows) * ((m + nt - 1) / nt);
    if (tiles > INT32_MAX / kMaxSplits || (m + nt - 1) / nt > 65535) continue;
    const float columns = static_cast<float>(nt * parts);
    const float stage = (parts * kTileRows + nt) * kFp8Group * 1e-6f / 13.f;  // us per block at 13 bytes/ps
    for (int s = 1; s <= kMaxSplits && s <= groups; ++s) {
      const int per = (groups + s - 1) / s;
      if ((groups + per - 1) / per != s) continue;  // a block would have nothing to do
      const int64_t blocks = tiles * s;
      // blocks that start at once, one per SM: clusters stay within a GPC, of which there are
      // eight of at least 16 SMs, and sizes that do not divide 16 pack less tightly
      const float room = s == 1 ? 148.f : 16 % s == 0 ? 128.f : 0.9f * 8 * (18 / s) * s;
      float group = 0.12f + 0.003f * columns;
      if (blocks * stage > group) group = blocks * stage;
      float time = 2.0f + 0.012f * columns + (gate ? 0.5f : 0.f) + per * group;
      if (s > 1) time += 0.3f + 0.02f * columns + (blocks > 2 * room ? 0.2f * per * group : 0.f);
      if (blocks > room) time += 0.9f * (blocks > 296 ? blocks / 148.f - 1 : 1.f);
      if (time < least) {
        least = time;
        best = {nt, s};
      }
      if (blocks > 4 * 148) break;  // more blocks only add their own start
    }
  }
  return best;
}

template <bool GATE>
cudaError_t launch_pairs(const GemmCall& c, cudaStream_t stream) {
  const int64_t tiles = wide_tiles(c.args, GATE);
  if constexpr (!GATE) {
    switch (wide_form(c.args, tiles, GATE)) {
      case WideForm::kHalves: return launch_wide<GATE, WideForm::kHalves>(c, tiles, stream);
      case WideForm::kWords: return launch_wide<GATE, WideForm::kWords>(c, tiles, stream);
      default: break;
    }
  }
  return launch_wide<GATE, WideForm::kWhole>(c, tiles, stream);
}

template <bool GATE>
cudaError_t launch_planned(const GemmCall& c, cudaStream_t stream) {
  const GemmPlan p = make_gemm_plan(c.args, GATE);
  switch (p.tokens) {
    case 16: return launch_gemm<16, GATE>(c, p.splits, stream);
    case 32: return launch_gemm<32, GATE>(c, p.splits, stream);
    case 64: return launch_gemm<GATE ? 32 : 64, GATE>(c, p.splits, stream);
    default: return launch_pairs<GATE>(c, stream);
  }
}

}  // namespace

// out_bits 8: gate/up. plan: tokens per tile (256: pairs), blocks per tile, stages, the pair kernel's form.
void fp8_plan(int m, int n, int k, int out_bits, int* plan) {
  const bool gate = out_bits == 8;
  const GemmArgs a{nullptr, nullptr, nullptr, nullptr, nullptr, m, n, (k + kFp8Group - 1) / kFp8Group, 1, 0, out_bits == 32};
  const GemmPlan p = make_gemm_plan(a, gate);
  const bool pairs = p.tokens == 256;
  plan[0] = p.tokens;
  plan[1] = pairs ? 1 : p.splits;
  plan[2] = pairs ? kWideStages : gemm_stages(a, p.tokens, p.splits);
  plan[3] = pairs ? static_cast<int>(wide_form(a, wide_tiles(a, gate), gate)) : 0;
}

cudaError_t launch_fp8_linear(const void* a, const float* sa, const void* w, const float* sw, void* out, int out_f32,
                              int m, int n, int k, int64_t as, int64_t ws, cudaStream_t stream) {
  const int groups = (k + kFp8Group - 1) / kFp8Group;
  return launch_planned<false>({a, w, nullptr, as, ws, 0, k, {sa, sw, nullptr, out, nullptr, m, n, groups, 1, 0, out_f32}},
                                 stream);
}

cudaError_t launch_fp8_gate_up(const void* a, const float* sa, const void* gate, const float* sg, const void* up,
                               const float* su, void* out, float* out_scale, int m, int n, int k, int64_t as,
                               int64_t gs, int64_t us, cudaStream_t stream) {
  const int groups = (k + kFp8Group - 1) / kFp8Group;
  return launch_planned<true>({a, gate, up, as, gs, us, k, {sa, sg, su, out, out_scale, m, n, groups, 1, 0, 0}}, stream);
}

}  // namespace dkv
