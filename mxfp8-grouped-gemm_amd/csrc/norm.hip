// Layer norm and root-mean-square norm over the rows of a matrix, forward and
// backward.
//
//   xhat = (x - mu) r, mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps)
//   y    = xhat w + b                         (RMS: mu = 0, no b)
//   u    = dy w;  dx = r (u - mean(u) - xhat mean(u xhat))      (RMS: no mean(u))
//   dw   = sum over rows of dy xhat, db = sum over rows of dy
//
// Memory-bound: a row is read once and kept in registers (16-byte chunks, CH a
// thread), so mean and variance are two exact passes over registers; statistics
// and sums are fp32.  Workgroups are persistent and take rows blockIdx, blockIdx
// + grid, ...: w and b stay in registers, the next row's loads go out before the
// current row's reductions, and in the backward pass every workgroup keeps its
// own dw and db, written once at its end and added over workgroups in a fixed
// order by a second kernel (no atomics: the sums are the same on every run).
#include <algorithm>

#include "mx_device.h"
#include "mxgg_internal.h"

namespace mxgg {
namespace {

// 512 threads leave 256 registers each: rows of up to 16384 stay in them in both
// passes; the backward pass of longer ones spills.
constexpr int kNormMaxThreads = 512;

// EPC elements of a 16-byte chunk, read and written at any element alignment.
template <typename T>
struct Elems;
template <>
struct Elems<float> {
  static constexpr int kCount = 4;
  __device__ static float get(const uint4& v, int j) {
    return __uint_as_float(j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w);
  }
  __device__ static uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                      __float_as_uint(f[3]));
  }
  __device__ static float one(const float* p) { return *p; }
  __device__ static void put(float* p, float f) { *p = f; }
};
template <>
struct Elems<uint16_t> {
  static constexpr int kCount = 8;
  __device__ static float get(const uint4& v, int j) {
    const uint32_t w = j < 2 ? v.x : j < 4 ? v.y : j < 6 ? v.z : v.w;
    return (j & 1) ? bf16_hi(w) : bf16_lo(w);
  }
  __device__ static uint4 pack(const float* f) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
  }
  __device__ static float one(const uint16_t* p) { return bf16_bits_to_f32(*p); }
  __device__ static void put(uint16_t* p, float f) { *p = (uint16_t)pack_bf16x2(f, 0.0f); }
};

// n of a chunk's elements (0 past the end of the row).
template <typename T>
__device__ __forceinline__ uint4 load_chunk(const T* p, int n) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (n >= Elems<T>::kCount) {
    __builtin_memcpy(&v, p, 16);
  } else if (n > 0) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < Elems<T>::kCount; ++j)
      if (j < n) {
        if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(p[j]);
        else w[j >> 1] |= (uint32_t)p[j] << (16 * (j & 1));
      }
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}
template <typename T>
__device__ __forceinline__ void store_chunk(T* p, const float* f, int n) {
  if (n >= Elems<T>::kCount) {
    const uint4 v = Elems<T>::pack(f);
    __builtin_memcpy(p, &v, 16);
  } else {
#pragma unroll
    for (int j = 0; j < Elems<T>::kCount; ++j)
      if (j < n) Elems<T>::put(p + j, f[j]);
  }
}

// Weight or bias element c (fp32 or bf16), 0 past the end.
__device__ __forceinline__ float param_at(const void* p, int bf16, int c, int cols) {
  if (c >= cols) return 0.0f;
  return bf16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(p)[c])
              : static_cast<const float*>(p)[c];
}

// Sum over the workgroup; every thread gets it.  `slots` holds one value per wave
// and is free again after the next barrier.
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off);
  return v;
}
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float (*slots)[kNormMaxThreads / 64]) {
  const int waves = (int)(blockDim.x >> 6);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  if (waves == 1) return;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) slots[i][threadIdx.x >> 6] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = 0.0f;
    for (int w = 0; w < waves; ++w) v[i] += slots[i][w];
  }
}

template <typename T, int CH, bool CENTER>
__global__ __launch_bounds__(kNormMaxThreads) void k_norm_fwd(NormArgs a) {
  constexpr int E = Elems<T>::kCount;
  __shared__ float slots[2][2][1][kNormMaxThreads / 64];  // [row parity][sum]
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);
  const int threads = (int)blockDim.x;
  int n[CH];
  float w[CH * E], b[CH * E];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int at = (threadIdx.x + c * threads) * E;
    n[c] = min(max(a.cols - at, 0), E);
#pragma unroll
    for (int j = 0; j < E; ++j) {
      w[c * E + j] = a.w ? param_at(a.w, a.w_bf16, at + j, a.cols) : 1.0f;
      b[c * E + j] = CENTER && a.b ? param_at(a.b, a.b_bf16, at + j, a.cols) : 0.0f;
    }
  }
  const float cols = (float)a.cols;  // sums are divided: a constant row's mean is its value
  uint4 next[CH];
  int64_t row = blockIdx.x;
#pragma unroll
  for (int c = 0; c < CH; ++c)
    next[c] = load_chunk<T>(x + row * a.ldx + (int64_t)(threadIdx.x + c * threads) * E, n[c]);
  for (int parity = 0; row < a.rows; row += gridDim.x, parity ^= 1) {
    float v[CH * E];
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < E; ++j) v[c * E + j] = Elems<T>::get(next[c], j);
    const int64_t after = row + gridDim.x;
    if (after < a.rows) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
        next[c] = load_chunk<T>(x + after * a.ldx + (int64_t)(threadIdx.x + c * threads) * E, n[c]);
    }
    float mu = 0.0f;
    if (CENTER) {
      float s[1] = {0.0f};
#pragma unroll
      for (int i = 0; i < CH * E; ++i) s[0] += v[i];
      block_sum<1>(s, slots[parity][0]);
      mu = s[0] / cols;
    }
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < E; ++j) {
        float& d = v[c * E + j];
        if (CENTER) d = j < n[c] ? d - mu : 0.0f;
        s[0] = __builtin_fmaf(d, d, s[0]);
      }
    block_sum<1>(s, slots[parity][1]);
    const float r = 1.0f / sqrtf(s[0] / cols + a.eps);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float o[E];
#pragma unroll
      for (int j = 0; j < E; ++j)
        o[j] = CENTER ? __builtin_fmaf(v[c * E + j] * r, w[c * E + j], b[c * E + j])
                      : v[c * E + j] * r * w[c * E + j];
      store_chunk<T>(y + row * a.ldy + (int64_t)(threadIdx.x + c * threads) * E, o, n[c]);
    }
    if (a.stats && threadIdx.x == 0) {
      if (CENTER) a.stats[row] = mu;
      a.stats[a.rows + row] = r;
    }
  }
}

template <typename T, int CH, bool CENTER>
__global__ __launch_bounds__(kNormMaxThreads) void k_norm_bwd(NormGradArgs a) {
  constexpr int E = Elems<T>::kCount;
  __shared__ float slots[2][2][kNormMaxThreads / 64];
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(a.dy);
  T* dx = static_cast<T*>(a.dx);
  const int threads = (int)blockDim.x;
  int n[CH];
  float w[CH * E], dw[CH * E], db[CH * E];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int at = (threadIdx.x + c * threads) * E;
    n[c] = min(max(a.cols - at, 0), E);
#pragma unroll
    for (int j = 0; j < E; ++j) {
      w[c * E + j] = a.w ? param_at(a.w, a.w_bf16, at + j, a.cols) : 1.0f;
      dw[c * E + j] = db[c * E + j] = 0.0f;
    }
  }
  const float inv = 1.0f / (float)a.cols;
  uint4 nx[CH], ng[CH];
  int64_t row = blockIdx.x;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int64_t at = (int64_t)(threadIdx.x + c * threads) * E;
    nx[c] = load_chunk<T>(x + row * a.ldx + at, n[c]);
    ng[c] = load_chunk<T>(dy + row * a.lddy + at, n[c]);
  }
  for (int parity = 0; row < a.rows; row += gridDim.x, parity ^= 1) {
    const float mu = CENTER ? a.stats[row] : 0.0f, r = a.stats[a.rows + row];
    float h[CH * E], g[CH * E];
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int i = c * E + j;
        // past the end of the row dy is 0, so xhat's value there does not matter
        h[i] = (Elems<T>::get(nx[c], j) - mu) * r;
        g[i] = Elems<T>::get(ng[c], j);
        dw[i] = __builtin_fmaf(g[i], h[i], dw[i]);
        db[i] += g[i];
        g[i] *= w[i];
        s[0] = __builtin_fmaf(g[i], h[i], s[0]);
        s[1] += g[i];
      }
    const int64_t after = row + gridDim.x;
    if (after < a.rows) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int64_t at = (int64_t)(threadIdx.x + c * threads) * E;
        nx[c] = load_chunk<T>(x + after * a.ldx + at, n[c]);
        ng[c] = load_chunk<T>(dy + after * a.lddy + at, n[c]);
      }
    }
    if (!dx) continue;
    block_sum<2>(s, slots[parity]);
    const float mh = s[0] * inv, mg = CENTER ? s[1] * inv : 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float o[E];
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int i = c * E + j;
        o[j] = r * (g[i] - mg - h[i] * mh);
      }
      store_chunk<T>(dx + row * a.lddx + (int64_t)(threadIdx.x + c * threads) * E, o, n[c]);
    }
  }
  // this workgroup's part of dw and db: fp32 [2][grid][cols]
  if (!a.partial) return;
  float* pw = a.partial + (int64_t)blockIdx.x * a.cols;
  float* pb = pw + (int64_t)gridDim.x * a.cols;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int at = (threadIdx.x + c * threads) * E;
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (j < n[c]) {
        if (a.dw) pw[at + j] = dw[c * E + j];
        if (a.db) pb[at + j] = db[c * E + j];
      }
  }
}

// dw[c] and db[c] (blockIdx.y) from the partials of `parts` workgroups: 64
// columns a workgroup, 4 runs of workgroups side by side, added in order.
constexpr int kNormReduceCols = 64, kNormReduceRuns = 4;
__global__ __launch_bounds__(kNormReduceCols* kNormReduceRuns) void k_norm_reduce(
    const float* __restrict__ partial, int parts, int cols, void* dw, int dw_bf16, void* db,
    int db_bf16) {
  __shared__ float sums[kNormReduceRuns][kNormReduceCols];
  const int lane = threadIdx.x % kNormReduceCols, run = threadIdx.x / kNormReduceCols;
  const int c = blockIdx.x * kNormReduceCols + lane;
  void* out = blockIdx.y ? db : dw;
  if (!out) return;
  const int bf16 = blockIdx.y ? db_bf16 : dw_bf16;
  const float* p = partial + (int64_t)blockIdx.y * parts * cols;
  const int per = (parts + kNormReduceRuns - 1) / kNormReduceRuns;
  float s = 0.0f;
  if (c < cols)
    for (int i = run * per; i < min(parts, (run + 1) * per); ++i) s += p[(int64_t)i * cols + c];
  sums[run][lane] = s;
  __syncthreads();
  if (run != 0 || c >= cols) return;
  for (int i = 1; i < kNormReduceRuns; ++i) s += sums[i][lane];
  if (bf16)
    static_cast<uint16_t*>(out)[c] = (uint16_t)pack_bf16x2(s, 0.0f);
  else
    static_cast<float*>(out)[c] = s;
}

// Threads, and chunks a thread, for a row: as few chunks as kNormMaxThreads allow.
struct NormShape {
  int ch, threads;
};
NormShape norm_shape(int cols, int per_chunk) {
  const int chunks = (cols + per_chunk - 1) / per_chunk;
  int ch = 2;
  while (ch * kNormMaxThreads < chunks) ch *= 2;
  const int threads = (chunks + ch - 1) / ch;
  return {ch, (threads + 63) / 64 * 64};
}

template <typename T, bool CENTER>
hipError_t run_fwd(const NormArgs& a, int grid, const NormShape& s, hipStream_t stream) {
  if (s.ch == 2)
    hipLaunchKernelGGL((k_norm_fwd<T, 2, CENTER>), dim3(grid), dim3(s.threads), 0, stream, a);
  else if (s.ch == 4)
    hipLaunchKernelGGL((k_norm_fwd<T, 4, CENTER>), dim3(grid), dim3(s.threads), 0, stream, a);
  else if (sizeof(T) == 2 || s.ch == 8)  // 32768 is the longest row: 8 chunks of bf16
    hipLaunchKernelGGL((k_norm_fwd<T, 8, CENTER>), dim3(grid), dim3(s.threads), 0, stream, a);
  else if constexpr (sizeof(T) == 4)
    hipLaunchKernelGGL((k_norm_fwd<T, 16, CENTER>), dim3(grid), dim3(s.threads), 0, stream, a);
  return hipGetLastError();
}
template <typename T, bool CENTER>
hipError_t run_bwd(const NormGradArgs& a, int grid, const NormShape& s, hipStream_t stream) {
  if (s.ch == 2)
    hipLaunchKernelGGL((k_norm_bwd<T, 2, CENTER>), dim3(grid), dim3(s.threads), 0, stream, a);
  else if (s.ch == 4)
    hipLaunchKernelGGL((k_norm_bwd<T, 4, CENTER>), dim3(grid), dim3(s.threads), 0, stream, a);
  else if (sizeof(T) == 2 || s.ch == 8)  // 32768 is the longest row: 8 chunks of bf16
    hipLaunchKernelGGL((k_norm_bwd<T, 8, CENTER>), dim3(grid), dim3(s.threads), 0, stream, a);
  else if constexpr (sizeof(T) == 4)
    hipLaunchKernelGGL((k_norm_bwd<T, 16, CENTER>), dim3(grid), dim3(s.threads), 0, stream, a);
  return hipGetLastError();
}

// Waves that a CU holds of these kernels, and the grid that fills the chip.
int norm_grid(int64_t rows, int threads, int waves_cu) {
  const int64_t per_cu = std::max(1, waves_cu / (threads / 64));
  return (int)std::min<int64_t>(rows, std::max(1, device_cu_count()) * per_cu);
}

}  // namespace

hipError_t launch_norm_fwd(const NormArgs& a, hipStream_t stream) {
  if (a.rows == 0) return hipSuccess;
  const NormShape s = norm_shape(a.cols, a.bf16 ? 8 : 4);
  const int grid = norm_grid(a.rows, s.threads, 16);
  if (a.bf16)
    return a.center ? run_fwd<uint16_t, true>(a, grid, s, stream)
                    : run_fwd<uint16_t, false>(a, grid, s, stream);
  return a.center ? run_fwd<float, true>(a, grid, s, stream)
                  : run_fwd<float, false>(a, grid, s, stream);
}

int norm_grad_parts(int64_t rows, int cols, int bf16) {
  return rows == 0 ? 0 : norm_grid(rows, norm_shape(cols, bf16 ? 8 : 4).threads, 14);
}

hipError_t launch_norm_bwd(const NormGradArgs& a, hipStream_t stream) {
  const int parts = norm_grad_parts(a.rows, a.cols, a.bf16);
  hipError_t err = hipSuccess;
  if (parts > 0) {
    const NormShape s = norm_shape(a.cols, a.bf16 ? 8 : 4);
    if (a.bf16)
      err = a.center ? run_bwd<uint16_t, true>(a, parts, s, stream)
                     : run_bwd<uint16_t, false>(a, parts, s, stream);
    else
      err = a.center ? run_bwd<float, true>(a, parts, s, stream)
                     : run_bwd<float, false>(a, parts, s, stream);
  }
  if (err != hipSuccess || (!a.dw && !a.db)) return err;
  const dim3 grid((unsigned)((a.cols + kNormReduceCols - 1) / kNormReduceCols), 2);
  hipLaunchKernelGGL(k_norm_reduce, grid, dim3(kNormReduceCols * kNormReduceRuns), 0, stream,
                     a.partial, parts, a.cols, a.dw, a.w_bf16, a.db, a.b_bf16);
  return hipGetLastError();
}

}  // namespace mxgg
