// Rows and weights turned to 8 bits (sm_100a): e4m3 codes with fp32 scales (fp8.cuh).
//
// quantize_rows_kernel   <- bf16 rows, one scale per row and 128 columns
// quantize_weight_kernel <- bf16 weights, one scale per 128 x 128 block
// add_rms_norm_fp8_kernel <- the decoder layer's residual add and the next RMSNorm with its
//                    weight (cuda_rms, src/gpu_ops.py:9-12), written as the rows the next
//                    projection reads: x_out = bf16(x + y) and
//                    h = x_out * rsqrt(mean(x_out^2) + eps) * weight, kept in fp32 up to its
//                    one rounding, to e4m3.
//
// All are bound by memory: 2 bytes read and 1 + 4/128 written per element (the norm with a
// residual reads 2 and writes 2 more). Every thread owns 16 consecutive columns: two 16-byte
// loads, one 16-byte store, and a group of 128 columns is 8 neighbouring lanes, so its
// maximum takes three shuffles. Measured: rows 8191 x 2560 10.1 us (6.3 of 6.6 TB/s), norm
// 2048 x 8192 with a residual 18.9 us (6.2 TB/s), 8192 x 960 10.1 (5.5), without one 4097 x 4096
// 10.0 (5.1); a decode step's single row is all latency, 1.5 and 1.9 us. Weights, quantised once
// per model: 16384 x 16384 229 us (3.5 TB/s), 1600 x 960 2.6.
#include "fp8.cuh"

namespace dkv {

constexpr int kQuantThreads = 256;

__device__ __forceinline__ void load16(const uint16_t* p, float* x) {
  const uint4* w = reinterpret_cast<const uint4*>(p);
  unpack16(w[0], w[1], x);
}

// Maximum over the 8 lanes of a column group.
__device__ __forceinline__ float group_max(float m) {
  m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
  return max_nan(m, __shfl_xor_sync(0xffffffffu, m, 4));
}

// Stores a lane's 16 codes of a group (where the row reaches that far) and, from the
// group's first lane, its scale.
__device__ __forceinline__ void store_group(const float* v, float amax, bool inside, bool first, uint8_t* q, float* scale) {
  amax = max_nan(amax, kFp8Floor);
  if (inside) *reinterpret_cast<uint4*>(q) = codes16(v, __fdiv_rn(kFp8Max, amax));
  if (first) *scale = __fdiv_rn(amax, kFp8Max);
}

// x: bf16 [rows, width], rows xs apart; q: [rows, width] and scale [rows, groups], contiguous.
__global__ void __launch_bounds__(kQuantThreads, 1)
quantize_rows_kernel(const uint16_t* __restrict__ x, uint8_t* __restrict__ q, float* __restrict__ scale, int64_t xs,
                     uint32_t width, uint32_t groups, uint32_t units) {
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  const uint32_t unit = blockIdx.x * (kQuantThreads / 8) + threadIdx.x / 8;  // (row, group)
  const uint32_t row = unit / groups;
  const uint32_t group = unit - row * groups;
  const uint32_t part = threadIdx.x & 7;
  const uint32_t col = group * kFp8Group + part * 16;
  const bool inside = unit < units && col < width;
  float v[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] = 0.f;
  if (inside) load16(x + row * xs + col, v);
  const float amax = group_max(amax16(v));
  store_group(v, amax, inside, unit < units && part == 0, q + static_cast<int64_t>(row) * width + col,
              scale + unit);
}

// One block per 128 x 128 weights: 8 threads per row, 32 rows at a time.
// w: bf16 [n, k], rows ws apart; q: [n, k] and scale [ceil(n / 128), ceil(k / 128)], contiguous.
__global__ void __launch_bounds__(kQuantThreads, 1)
quantize_weight_kernel(const uint16_t* __restrict__ w, uint8_t* __restrict__ q, float* __restrict__ scale, int64_t ws,
                       int n, int k, int groups) {
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  const int bn = blockIdx.x / groups;
  const int bk = blockIdx.x - bn * groups;
  const int col = bk * kFp8Group + (threadIdx.x & 7) * 16;
  const int row0 = bn * kFp8Group + (threadIdx.x >> 3);
  float v[4][16];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = row0 + 32 * i;
    if (row < n && col < k) {
      load16(w + row * ws + col, v[i]);
      amax = max_nan(amax, amax16(v[i]));
    }
  }
  __shared__ float part[kQuantThreads / 32];
  amax = group_max(amax);
  amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 8));
  amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 16));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = amax;
  __syncthreads();
  amax = kFp8Floor;
#pragma unroll
  for (int i = 0; i < kQuantThreads / 32; ++i) amax = max_nan(amax, part[i]);
  const float inverse = __fdiv_rn(kFp8Max, amax);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = row0 + 32 * i;
    if (row < n && col < k) *reinterpret_cast<uint4*>(q + static_cast<int64_t>(row) * k + col) = codes16(v[i], inverse);
  }
  if (threadIdx.x == 0) scale[blockIdx.x] = __fdiv_rn(amax, kFp8Max);
}

// One row per WARPS warps at a time, two chunks of 16 columns per thread: width <= 1024 *
// WARPS. Rows of one warp share a block of four. A block works through rows a grid apart: its
// weights stay in registers, and the next row is on its way while this one is summed up, scaled
// and stored (one row per block left the memory idle in between: 4097 x 4096 15.1 us). A row
// is held as the bf16 it is (the residual sum is bf16 by definition), half the registers of
// fp32. The sum of squares runs in fp32 in a fixed order (a thread's columns, a butterfly over
// the warp, the warps in turn).
constexpr int kNormFp8Chunks = 2;
// Blocks per SM: 16 warps (20 without a residual, which needs fewer registers).
template <int WARPS, bool ADD>
constexpr int kNormFp8Blocks = WARPS == 1 ? (ADD ? 4 : 5) : WARPS == 16 ? 1 : (ADD ? 16 : 20) / WARPS;

struct NormRow {
  uint4 x[kNormFp8Chunks][2], y[kNormFp8Chunks][2];
};

template <int WARPS, bool ADD>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : 32 * WARPS, kNormFp8Blocks<WARPS, ADD>)
add_rms_norm_fp8_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ y, uint16_t* __restrict__ x_out,
                        uint8_t* __restrict__ q, float* __restrict__ scale, const uint16_t* __restrict__ weight,
                        int64_t rows, int width, int groups, int64_t xs, int64_t ys, int64_t os, float eps) {
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  int64_t row = WARPS == 1 ? static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5) : blockIdx.x;
  const int64_t step = WARPS == 1 ? static_cast<int64_t>(gridDim.x) * 4 : gridDim.x;
  const int lane = WARPS == 1 ? (threadIdx.x & 31) : threadIdx.x;
  __shared__ float part[2][WARPS];
  const auto load = [&](int64_t r, NormRow& v) {
#pragma unroll
    for (int i = 0; i < kNormFp8Chunks; ++i) {
      const int c = (lane + 32 * WARPS * i) * 16;
      if (c >= width || r >= rows) continue;
      const uint4* a = reinterpret_cast<const uint4*>(x + r * xs + c);
      v.x[i][0] = a[0];
      v.x[i][1] = a[1];
      if (ADD) {
        const uint4* b = reinterpret_cast<const uint4*>(y + r * ys + c);
        v.y[i][0] = b[0];
        v.y[i][1] = b[1];
      }
    }
  };
  uint4 wv[kNormFp8Chunks][2];
  NormRow v;
#pragma unroll
  for (int i = 0; i < kNormFp8Chunks; ++i) {
    const int c = (lane + 32 * WARPS * i) * 16;
    wv[i][0] = wv[i][1] = v.x[i][0] = v.x[i][1] = v.y[i][0] = v.y[i][1] = make_uint4(0, 0, 0, 0);
    if (c < width) {  // columns past the row stay zeros: they add nothing to the sum or the maximum
      wv[i][0] = __ldg(reinterpret_cast<const uint4*>(weight + c));
      wv[i][1] = __ldg(reinterpret_cast<const uint4*>(weight + c) + 1);
    }
  }
  load(row, v);
  for (int turn = 0; row < rows; row += step, turn ^= 1) {  // whole warps, and blocks of more, leave together
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < kNormFp8Chunks; ++i) {
      float f[16];
      unpack16(v.x[i][0], v.x[i][1], f);
      if (ADD) {
        const int c = (lane + 32 * WARPS * i) * 16;
        float b[16];
        unpack16(v.y[i][0], v.y[i][1], b);
        uint32_t s[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] = pack_bf16x2(__fadd_rn(f[2 * j], b[2 * j]), __fadd_rn(f[2 * j + 1], b[2 * j + 1]));
        v.x[i][0] = make_uint4(s[0], s[1], s[2], s[3]);
        v.x[i][1] = make_uint4(s[4], s[5], s[6], s[7]);
        if (c < width) {
          uint4* dst = reinterpret_cast<uint4*>(x_out + row * os + c);
          dst[0] = v.x[i][0];
          dst[1] = v.x[i][1];
        }
        unpack16(v.x[i][0], v.x[i][1], f);
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) ss = __fmaf_rn(f[j], f[j], ss);
    }
    const uint4 now[kNormFp8Chunks][2] = {{v.x[0][0], v.x[0][1]}, {v.x[1][0], v.x[1][1]}};
    load(row + step, v);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    if (WARPS > 1) {  // two sets of partial sums: a warp may be a row ahead of the slowest
      if ((threadIdx.x & 31) == 0) part[turn][threadIdx.x >> 5] = ss;
      __syncthreads();
      ss = part[turn][0];
#pragma unroll
      for (int i = 1; i < WARPS; ++i) ss += part[turn][i];
    }
    const float rstd = rsqrtf(__fdiv_rn(ss, static_cast<float>(width)) + eps);
#pragma unroll
    for (int i = 0; i < kNormFp8Chunks; ++i) {
      const int c = (lane + 32 * WARPS * i) * 16;
      if (32 * WARPS * i * 16 >= width) break;  // the same for every lane
      float h[16], w[16];
      unpack16(now[i][0], now[i][1], h);
      unpack16(wv[i][0], wv[i][1], w);
#pragma unroll
      for (int j = 0; j < 16; ++j) h[j] = __fmul_rn(__fmul_rn(h[j], rstd), w[j]);
      const float amax = group_max(amax16(h));
      store_group(h, amax, c < width, c < width && (lane & 7) == 0, q + row * width + c,
                  scale + row * groups + c / kFp8Group);
    }
  }
}

namespace {

// Programmatic dependents of the launch before them (see decoder_ops.cu): each kernel
// waits before its first access and only then lets its own dependent start.
template <class Kernel, class... Args>
cudaError_t launch_rows(unsigned blocks, int threads, cudaStream_t stream, Kernel kernel, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

struct NormArgs {
  const uint16_t *x, *y;
  uint16_t* x_out;
  uint8_t* q;
  float* scale;
  const uint16_t* weight;
  int64_t rows;
  int width, groups;
  int64_t xs, ys, os;
  float eps;
};

template <int WARPS, bool ADD>
cudaError_t launch_norm(const NormArgs& a, cudaStream_t stream) {
  const int64_t all = WARPS == 1 ? (a.rows + 3) / 4 : a.rows;
  const int64_t wave = 148 * kNormFp8Blocks<WARPS, ADD>;
  const unsigned blocks = static_cast<unsigned>(all < wave ? all : wave);
  return launch_rows(blocks, WARPS == 1 ? 128 : 32 * WARPS, stream, add_rms_norm_fp8_kernel<WARPS, ADD>, a.x, a.y,
                     a.x_out, a.q, a.scale, a.weight, a.rows, a.width, a.groups, a.xs, a.ys, a.os, a.eps);
}

template <bool ADD>
cudaError_t launch_norm_width(const NormArgs& a, cudaStream_t stream) {
  if (a.width <= 1024) return launch_norm<1, ADD>(a, stream);
  if (a.width <= 2048) return launch_norm<2, ADD>(a, stream);
  if (a.width <= 4096) return launch_norm<4, ADD>(a, stream);
  if (a.width <= 8192) return launch_norm<8, ADD>(a, stream);
  return launch_norm<16, ADD>(a, stream);
}

}  // namespace

cudaError_t launch_fp8_quantize(const void* x, void* q, float* scale, int64_t rows, int width, int64_t xs,
                                cudaStream_t stream) {
  const uint32_t groups = (width + kFp8Group - 1) / kFp8Group;
  const uint32_t units = static_cast<uint32_t>(rows) * groups;
  const unsigned blocks = (units + kQuantThreads / 8 - 1) / (kQuantThreads / 8);
  return launch_rows(blocks, kQuantThreads, stream, quantize_rows_kernel, static_cast<const uint16_t*>(x),
                     static_cast<uint8_t*>(q), scale, xs, static_cast<uint32_t>(width), groups, units);
}

cudaError_t launch_fp8_quantize_weight(const void* w, void* q, float* scale, int n, int k, int64_t ws,
                                       cudaStream_t stream) {
  const int groups = (k + kFp8Group - 1) / kFp8Group;
  const unsigned blocks = static_cast<unsigned>((n + kFp8Group - 1) / kFp8Group) * groups;
  return launch_rows(blocks, kQuantThreads, stream, quantize_weight_kernel, static_cast<const uint16_t*>(w),
                     static_cast<uint8_t*>(q), scale, ws, n, k, groups);
}

cudaError_t launch_add_rms_norm_fp8(const void* x, const void* y, void* x_out, void* q, float* scale,
                                    const void* weight, int64_t rows, int width, int64_t xs, int64_t ys, int64_t os,
                                    float eps, cudaStream_t stream) {
  const NormArgs a{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(y), static_cast<uint16_t*>(x_out),
                   static_cast<uint8_t*>(q), scale, static_cast<const uint16_t*>(weight), rows, width,
                   (width + kFp8Group - 1) / kFp8Group, xs, ys, os, eps};
  return y != nullptr ? launch_norm_width<true>(a, stream) : launch_norm_width<false>(a, stream);
}

}  // namespace dkv
