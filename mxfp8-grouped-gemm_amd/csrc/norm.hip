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
// and sums are fp32.  A short row belongs to one wave (no barriers, the waves of a
// workgroup run apart), a longer one to a workgroup.  Workgroups are persistent:
// w and b stay in registers, the next row's loads go out before the current row's
// reductions, and in the backward pass every workgroup keeps its own dw and db,
// written once at its end and added over workgroups in a fixed order by a second
// kernel (no atomics: the sums are the same on every run).
//
// 16384 x 7168 bf16 layer norm: forward 82 us (5.7 TB/s), backward 142 (5.0), sum over
// workgroups 6.  64 rows: 4.5 us, a launch, one row's loads and two reductions.
#include <algorithm>

#include "mx_device.h"
#include "mxgg_internal.h"

namespace mxgg {
namespace {

// Leaves a thread 256 registers: enough for 16 elements of every operand, not for 32 or
// 64 in the backward pass (see norm_shape).
constexpr int kNormMaxThreads = 512;
constexpr int kWaveRows = 4;          // waves, and rows at a time, of a workgroup of one-wave rows

// The elements of a 16-byte chunk, read and written at any element alignment.
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

// n of a chunk's elements (0 past the end of the row).  Outputs are written past
// the caches, and the backward pass reads past them too (16384 x 7168 bf16: its
// 169 us become 152); the forward pass is faster with ordinary loads (81 us, 95
// past the caches).
template <bool STREAM, typename T>
__device__ __forceinline__ uint4 load_chunk(const T* p, int n) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (n >= Elems<T>::kCount) {
    if (STREAM && (reinterpret_cast<uintptr_t>(p) & 15u) == 0) {
      const u32x4 u = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
      v = make_uint4(u[0], u[1], u[2], u[3]);
    } else {
      __builtin_memcpy(&v, p, 16);
    }
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
    if ((reinterpret_cast<uintptr_t>(p) & 15u) == 0)
      __builtin_nontemporal_store(u32x4{v.x, v.y, v.z, v.w}, reinterpret_cast<u32x4*>(p));
    else
      __builtin_memcpy(p, &v, 16);
  } else {
#pragma unroll
    for (int j = 0; j < Elems<T>::kCount; ++j)
      if (j < n) Elems<T>::put(p + j, f[j]);
  }
}

// E elements of the weight or bias from c on (fp32 or bf16), 0 past the end.
template <int E>
__device__ __forceinline__ void load_params(const void* p, int bf16, int c, int cols, float* v) {
  const float* f = static_cast<const float*>(p) + c;
  const uint16_t* h = static_cast<const uint16_t*>(p) + c;
  if (c + E <= cols) {
    if (bf16) {
      uint16_t u[E];
      __builtin_memcpy(u, h, sizeof(u));
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] = bf16_bits_to_f32(u[j]);
    } else {
      __builtin_memcpy(v, f, 4 * E);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < E; ++j)
    v[j] = c + j >= cols ? 0.0f : bf16 ? bf16_bits_to_f32(h[j]) : f[j];
}

// Sums over the row's threads, in every one of them.  `slots` holds one value per
// wave and is free again after the next barrier; 16 lanes read them together.
template <bool WAVE, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*slots)[kNormMaxThreads / 64]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  const int waves = (int)(blockDim.x >> 6);
  if (WAVE || waves == 1) return;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) slots[i][threadIdx.x >> 6] = v[i];
  }
  __syncthreads();
  const int w = threadIdx.x & 15;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = row16_sum(w < waves ? slots[i][w] : 0.0f);
}

// A thread's place: first row, rows to the next one, and its number among the
// `threads` of its row.
template <bool WAVE>
struct RowPlace {
  int64_t first, step;
  int thread, threads;
  __device__ __forceinline__ RowPlace() {
    if (WAVE) {
      const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
      first = (int64_t)blockIdx.x * kWaveRows + wave;
      step = (int64_t)gridDim.x * kWaveRows;
      thread = threadIdx.x & 63;
      threads = 64;
    } else {
      first = blockIdx.x;
      step = gridDim.x;
      thread = threadIdx.x;
      threads = blockDim.x;
    }
  }
};

template <typename T, int CH, bool CENTER, bool WAVE>
__global__ __launch_bounds__(WAVE ? 64 * kWaveRows : kNormMaxThreads) void k_norm_fwd(NormArgs a) {
  constexpr int E = Elems<T>::kCount;
  __shared__ float slots[2][2][1][kNormMaxThreads / 64];  // [row parity][sum]
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);
  const RowPlace<WAVE> at_row;
  int n[CH];
  float w[CH * E], b[CH * E];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int at = (at_row.thread + c * at_row.threads) * E;
    n[c] = min(max(a.cols - at, 0), E);
#pragma unroll
    for (int j = 0; j < E; ++j) {
      w[c * E + j] = 1.0f;
      b[c * E + j] = 0.0f;
    }
    if (a.w) load_params<E>(a.w, a.w_bf16, at, a.cols, w + c * E);
    if (CENTER && a.b) load_params<E>(a.b, a.b_bf16, at, a.cols, b + c * E);
  }
  const float cols = (float)a.cols;  // sums are divided: a constant row's mean is its value
  uint4 next[CH];
  int64_t row = at_row.first;
  if (row < a.rows)
#pragma unroll
    for (int c = 0; c < CH; ++c)
      next[c] = load_chunk<false>(x + row * a.ldx + (int64_t)(at_row.thread + c * at_row.threads) * E, n[c]);
  for (int parity = 0; row < a.rows; row += at_row.step, parity ^= 1) {
    float v[CH * E];
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < E; ++j) v[c * E + j] = Elems<T>::get(next[c], j);
    const int64_t after = row + at_row.step;
    if (after < a.rows) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
        next[c] = load_chunk<false>(x + after * a.ldx + (int64_t)(at_row.thread + c * at_row.threads) * E, n[c]);
    }
    float mu = 0.0f;
    if (CENTER) {
      float s[1] = {0.0f};
#pragma unroll
      for (int i = 0; i < CH * E; ++i) s[0] += v[i];
      row_sum<WAVE, 1>(s, slots[parity][0]);
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
    row_sum<WAVE, 1>(s, slots[parity][1]);
    const float r = 1.0f / sqrtf(s[0] / cols + a.eps);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float o[E];
#pragma unroll
      for (int j = 0; j < E; ++j)
        o[j] = CENTER ? __builtin_fmaf(v[c * E + j] * r, w[c * E + j], b[c * E + j])
                      : v[c * E + j] * r * w[c * E + j];
      store_chunk<T>(y + row * a.ldy + (int64_t)(at_row.thread + c * at_row.threads) * E, o, n[c]);
    }
    if (a.stats && at_row.thread == 0) {
      if (CENTER) a.stats[row] = mu;
      a.stats[a.rows + row] = r;
    }
  }
}

// Outputs of the norm with the residual's addition.
enum { kOutSame, kOutMx, kOutBlock };
constexpr int kScaleRun = 16;  // rows whose scales leave together

// Largest |o| bit pattern of the lanes that hold one block of 32 (MX) or 128 elements.
template <int OUT, int E>
__device__ __forceinline__ uint32_t block_amax(uint32_t m) {
  m = quad_max(m);
  if (OUT == kOutMx && E == 8) return m;
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x141, 0xF, 0xF, false));  // 8 lanes
  if (OUT == kOutMx) return m;
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x140, 0xF, 0xF, false));  // 16
  if (E == 8) return m;
  const auto p = __builtin_amdgcn_permlane16_swap(m, m, false, false);             // 32
  return max((uint32_t)p[0], (uint32_t)p[1]);
}

// E8M0 byte of a block of fp32 values from the bit pattern of the largest, by the
// rules of the bf16 casts (e8m0_from_amax16).
__device__ __forceinline__ uint32_t e8m0_from_amax32(uint32_t amax, int mode) {
  const int ex = (int)(amax >> 23);
  const uint32_t mant = amax & 0x7FFFFFu;
  const int b = ex - 8 + (mode == kModeRceil && mant > 0x600000u ? 1 : 0);
  if (ex == 255) return mant ? 255u : (mode == kModeRceil ? 254u : 247u);
  return (uint32_t)(b < 0 ? 0 : b);
}

// E payload bytes of o under the block's E8M0 byte.
template <int E>
__device__ __forceinline__ void mx_payload(const float* o, uint32_t b, int mode, uint32_t* w) {
#pragma unroll
  for (int k = 0; k < E / 4; ++k) {
    const float *f = o + 4 * k;
    if (mode == kModeRceil)
      w[k] = __any(b >= 254u) ? encode4_any<kModeRceil, false>(f[0], f[1], f[2], f[3], b)
                              : encode4_finite<kModeRceil, false>(f[0], f[1], f[2], f[3], b);
    else
      w[k] = __any(b == 255u) ? encode4_any<kModeFloor, false>(f[0], f[1], f[2], f[3], b)
                              : encode4_finite<kModeFloor, false>(f[0], f[1], f[2], f[3], b);
  }
}

// Root-mean-square norm of h = x + residual (ADD; rounded to T, as it is kept) or of x.
//   kOutSame  : y in T, rows dealt out as in k_norm_fwd
//   kOutMx    : e4m3 and an E8M0 byte for each 32, rounded once from fp32
//   kOutBlock : e4m3 and an fp32 scale for each 128 (block_scale)
// Scales are laid out block by block, rows next to each other, so the 8-bit outputs
// are computed for `run` consecutive rows a workgroup, their scales gathered in LDS
// and written as one run for each block (a byte at a time they would be a memory
// transaction each: 224 a row of 7168); runs of one row write theirs at once.
// Memory-bound, 16384 x 7168 bf16: both sums and the norm 168-177 us (5.5 TB/s of two
// streams in and two out), its backward pass with the residual stream's gradient 166
// (5.7); 8-bit results 167-169 us.
template <typename T, int CH, bool WAVE, int OUT, bool ADD>
__global__ __launch_bounds__(WAVE ? 64 * kWaveRows : kNormMaxThreads) void k_add_norm(AddNormArgs a) {
  constexpr int E = Elems<T>::kCount;
  constexpr bool kQuant = OUT != kOutSame;
  constexpr int kMaxBlocks = (WAVE ? 1024 : 32768) / (OUT == kOutMx ? 32 : 128);
  constexpr int kScaleBytes = kQuant ? kMaxBlocks * kScaleRun * (OUT == kOutMx ? 1 : 4) : 16;
  __shared__ float slots[2][1][kNormMaxThreads / 64];
  __shared__ __attribute__((aligned(16))) uint8_t held[kScaleBytes];
  const T* x = static_cast<const T*>(a.x);
  const T* res = static_cast<const T*>(a.res);
  T* h = static_cast<T*>(a.h);
  T* y = static_cast<T*>(a.y);
  const RowPlace<WAVE> at_row;
  const int lane_row = WAVE ? (int)(threadIdx.x >> 6) : 0, rows_at_once = WAVE ? kWaveRows : 1;
  int n[CH];
  float w[CH * E];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int at = (at_row.thread + c * at_row.threads) * E;
    n[c] = min(max(a.cols - at, 0), E);
#pragma unroll
    for (int j = 0; j < E; ++j) w[c * E + j] = 1.0f;
    if (a.w) load_params<E>(a.w, a.w_bf16, at, a.cols, w + c * E);
  }
  const float cols = (float)a.cols;
  uint4 nx[CH], nr[CH];
  const auto fetch = [&](int64_t row) __attribute__((always_inline)) {
    if (row >= a.rows) return;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int64_t at = (int64_t)(at_row.thread + c * at_row.threads) * E;
      nx[c] = load_chunk<false>(x + row * a.ldx + at, n[c]);
      if (ADD) nr[c] = load_chunk<false>(res + row * a.ldres + at, n[c]);
    }
  };
  const int run = kQuant ? a.run : rows_at_once;
  int parity = 0;
  fetch((int64_t)blockIdx.x * run + lane_row);
  for (int64_t base = (int64_t)blockIdx.x * run; base < a.rows; base += (int64_t)gridDim.x * run) {
    for (int i = lane_row; i < run; i += rows_at_once) {
      const int64_t row = base + i;
      if (row >= a.rows) break;
      float v[CH * E];
#pragma unroll
      for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int j = 0; j < E; ++j) {
          v[c * E + j] = Elems<T>::get(nx[c], j);
          if (ADD) v[c * E + j] += Elems<T>::get(nr[c], j);
        }
        if (ADD) {
          const uint4 kept = Elems<T>::pack(v + c * E);
          store_chunk<T>(h + row * a.ldh + (int64_t)(at_row.thread + c * at_row.threads) * E,
                         v + c * E, n[c]);
#pragma unroll
          for (int j = 0; j < E; ++j) v[c * E + j] = Elems<T>::get(kept, j);
        }
      }
      fetch(i + rows_at_once < run ? row + rows_at_once
                                   : base + (int64_t)gridDim.x * run + lane_row);
      float s[1] = {0.0f};
#pragma unroll
      for (int k = 0; k < CH * E; ++k) s[0] = __builtin_fmaf(v[k], v[k], s[0]);
      row_sum<WAVE, 1>(s, slots[parity]);
      parity ^= 1;
      const float r = 1.0f / sqrtf(s[0] / cols + a.eps);
      if (a.stats && at_row.thread == 0) a.stats[a.rows + row] = r;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int chunk = at_row.thread + c * at_row.threads;
        float o[E];
#pragma unroll
        for (int j = 0; j < E; ++j) o[j] = v[c * E + j] * r * w[c * E + j];
        if constexpr (!kQuant) {
          store_chunk<T>(y + row * a.ldy + (int64_t)chunk * E, o, n[c]);
        } else {
          uint32_t m = 0;
#pragma unroll
          for (int j = 0; j < E; ++j)
            m = max(m, j < n[c] ? __float_as_uint(o[j]) & 0x7FFFFFFFu : 0u);
          m = block_amax<OUT, E>(m);
          uint32_t p[E / 4];
          constexpr int kLanes = (OUT == kOutMx ? 32 : 128) / E;
          const bool first = chunk % kLanes == 0 && n[c] > 0;
          if constexpr (OUT == kOutMx) {
            const uint32_t b = e8m0_from_amax32(m, a.mode);
            mx_payload<E>(o, b, a.mode, p);
            if (first && run == 1) static_cast<uint8_t*>(a.scales)[chunk / kLanes * a.lds + row] = (uint8_t)b;
            else if (first) held[chunk / kLanes * kScaleRun + i] = (uint8_t)b;
          } else {
            const float sc = block_scale(__uint_as_float(m));
            const BlockDivisor d(sc);
#pragma unroll
            for (int k = 0; k < E / 4; ++k) {
              p[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(d(o[4 * k]), d(o[4 * k + 1]), 0, false);
              p[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(d(o[4 * k + 2]), d(o[4 * k + 3]),
                                                               (int)p[k], true);
            }
            if (first && run == 1) static_cast<float*>(a.scales)[chunk / kLanes * a.lds + row] = sc;
            else if (first) reinterpret_cast<float*>(held)[chunk / kLanes * kScaleRun + i] = sc;
          }
          if (n[c] > 0) {  // whole chunks: the width is a multiple of 16
            uint8_t* q = a.q + row * a.ldq + (int64_t)chunk * E;
            if constexpr (E == 8) store_stream(q, make_uint2(p[0], p[1]));
            else __builtin_nontemporal_store(p[0], reinterpret_cast<uint32_t*>(q));
          }
        }
      }
    }
    if (kQuant && run > 1) {
      __syncthreads();
      constexpr int kWidth = OUT == kOutMx ? 32 : 128, kSize = OUT == kOutMx ? 1 : 4;
      const int blocks = (a.cols + kWidth - 1) / kWidth;
      const int rows = (int)min((int64_t)run, a.rows - base);
      uint8_t* out = static_cast<uint8_t*>(a.scales) + base * kSize;
      if (rows == kScaleRun) {
        constexpr int kParts = kScaleRun * kSize / 16;  // 16-byte pieces of a block's scales
        for (int k = threadIdx.x; k < blocks * kParts; k += blockDim.x) {
          const uint4 v = *reinterpret_cast<const uint4*>(held + 16 * k);
          __builtin_memcpy(out + (int64_t)(k / kParts) * a.lds * kSize + 16 * (k % kParts), &v, 16);
        }
      } else {
        for (int k = threadIdx.x; k < blocks * kScaleRun; k += blockDim.x) {
          const int b = k / kScaleRun, i = k % kScaleRun;
          if (i >= rows) continue;
          if constexpr (OUT == kOutMx)
            out[(int64_t)b * a.lds + i] = held[k];
          else
            reinterpret_cast<float*>(out)[(int64_t)b * a.lds + i] = reinterpret_cast<float*>(held)[k];
        }
      }
      __syncthreads();
    }
  }
}

// ADD (root-mean-square norm, no bias): a.add is added to dx.
template <typename T, int CH, bool CENTER, bool WAVE, bool ADD>
__global__ __launch_bounds__(WAVE ? 64 * kWaveRows : kNormMaxThreads) void k_norm_bwd(NormGradArgs a) {
  constexpr int E = Elems<T>::kCount;
  __shared__ float slots[2][2][kNormMaxThreads / 64];
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(a.dy);
  T* dx = static_cast<T*>(a.dx);
  const T* add = static_cast<const T*>(a.add);
  const RowPlace<WAVE> at_row;
  int n[CH];
  float w[CH * E], dw[CH * E], db[CH * E];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int at = (at_row.thread + c * at_row.threads) * E;
    n[c] = min(max(a.cols - at, 0), E);
#pragma unroll
    for (int j = 0; j < E; ++j) {
      w[c * E + j] = 1.0f;
      dw[c * E + j] = db[c * E + j] = 0.0f;
    }
    if (a.w) load_params<E>(a.w, a.w_bf16, at, a.cols, w + c * E);
  }
  const float cols = (float)a.cols;
  uint4 nx[CH], ng[CH];
  int64_t row = at_row.first;
  if (row < a.rows)
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int64_t at = (int64_t)(at_row.thread + c * at_row.threads) * E;
      nx[c] = load_chunk<true>(x + row * a.ldx + at, n[c]);
      ng[c] = load_chunk<true>(dy + row * a.lddy + at, n[c]);
    }
  for (int parity = 0; row < a.rows; row += at_row.step, parity ^= 1) {
    const float mu = CENTER ? a.stats[row] : 0.0f, r = a.stats[a.rows + row];
    // the chunks stay packed; xhat and dy w are formed again after the sums
    uint4 cx[CH], cg[CH], ca[CH];
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      cx[c] = nx[c];
      cg[c] = ng[c];
      // of this row, not ahead as the others: there are no registers for both
      if (ADD) ca[c] = load_chunk<true>(
          add + row * a.ldadd + (int64_t)(at_row.thread + c * at_row.threads) * E, n[c]);
    }
    const int64_t after = row + at_row.step;
    if (after < a.rows) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int64_t at = (int64_t)(at_row.thread + c * at_row.threads) * E;
        nx[c] = load_chunk<true>(x + after * a.ldx + at, n[c]);
        ng[c] = load_chunk<true>(dy + after * a.lddy + at, n[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int i = c * E + j;
        // past the end of the row dy is 0, so xhat's value there does not matter
        const float h = (Elems<T>::get(cx[c], j) - mu) * r, g = Elems<T>::get(cg[c], j);
        dw[i] = __builtin_fmaf(g, h, dw[i]);
        if (!ADD) db[i] += g;
        const float u = g * w[i];
        s[0] = __builtin_fmaf(u, h, s[0]);
        s[1] += u;
      }
    if (!dx) continue;
    row_sum<WAVE, 2>(s, slots[parity]);
    const float mh = s[0] / cols, mg = CENTER ? s[1] / cols : 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float o[E];
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float h = (Elems<T>::get(cx[c], j) - mu) * r;
        o[j] = r * (Elems<T>::get(cg[c], j) * w[c * E + j] - mg - h * mh);
        if (ADD) o[j] += Elems<T>::get(ca[c], j);
      }
      store_chunk<T>(dx + row * a.lddx + (int64_t)(at_row.thread + c * at_row.threads) * E, o, n[c]);
    }
  }
  // this workgroup's part of dw and db: fp32 [2][grid][cols]
  if (!a.partial) return;
  float* pw = a.partial + (int64_t)blockIdx.x * a.cols;
  float* pb = pw + (int64_t)gridDim.x * a.cols;
  if constexpr (WAVE) {  // the waves' sums first, in wave order
    __shared__ float part[kWaveRows][64 * CH * E];
    for (int k = 0; k < 2; ++k) {
      if (k ? ADD || !a.db : !a.dw) continue;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < CH * E; ++i)
        part[threadIdx.x >> 6][i * 64 + at_row.thread] = k ? db[i] : dw[i];
      __syncthreads();
      for (int e = threadIdx.x; e < 64 * CH * E; e += 64 * kWaveRows) {
        const int i = e >> 6, col = ((e & 63) + i / E * 64) * E + i % E;
        float v = 0.0f;
        for (int u = 0; u < kWaveRows; ++u) v += part[u][e];
        if (col < a.cols) (k ? pb : pw)[col] = v;
      }
    }
    return;
  }
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int at = (at_row.thread + c * at_row.threads) * E;
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (j < n[c]) {
        if (a.dw) pw[at + j] = dw[c * E + j];
        if (!ADD && a.db) pb[at + j] = db[c * E + j];
      }
  }
}

// dw[c] and db[c] (blockIdx.y) from the partials of `parts` workgroups: 64
// columns a workgroup, 16 runs of partials side by side, joined in order.
constexpr int kNormReduceCols = 64, kNormReduceRuns = 16;
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
  float s = 0.0f;
  if (c < cols) {
    constexpr int kAhead = 8;  // loads in flight
    for (int i0 = run; i0 < parts; i0 += kNormReduceRuns * kAhead) {
      float v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = i0 + u * kNormReduceRuns;
        v[u] = i < parts ? p[(int64_t)i * cols + c] : 0.0f;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) s += v[u];
    }
  }
  sums[run][lane] = s;
  __syncthreads();
  if (run != 0 || c >= cols) return;
  for (int i = 1; i < kNormReduceRuns; ++i) s += sums[i][lane];
  if (bf16)
    static_cast<uint16_t*>(out)[c] = (uint16_t)pack_bf16x2(s, 0.0f);
  else
    static_cast<float*>(out)[c] = s;
}

// How a row of `cols` is shared out: rows of at most 1024 elements go to one wave,
// longer ones to a workgroup with four chunks a thread, or more where 512 threads
// ask for it.  Four chunks against one a thread (7168 bf16: 256 threads against
// 896), forward 81 us against 88, with the backward pass 250 against 263: fewer
// waves share a row's reductions.  One wave against a workgroup, forward / backward us:
// 65536 x 512 bf16 21 / 53 and 41 / 83, 65536 x 1024 bf16 41 / 75 and 45 / 99, fp32
// 80 / 141 and 79 / 156.
// Rows that take 8 or 16 chunks a thread (fp32 above 8192, bf16 above 16384) keep w, dw,
// db and two streams of 32 or 64 elements, which do not fit 256 registers: the backward
// kernel spills 164 of them (fp32 to 16384), 1474 (fp32 above) or 1006 (bf16 above
// 16384), the forward one up to 548.  Layer norm, forward / backward TB/s of the bytes in
// and out: fp32 4096 x 8192 (4 chunks) 5.8 / 5.2, 4096 x 16384 (8) 5.1 / 3.8, 2048 x 32768
// (16) 2.8 / 0.7; bf16 4096 x 16384 (4) 5.5 / 3.9, 2048 x 32768 (8) 3.8 / 0.6.
struct NormShape {
  int ch, threads;
  bool wave;
};
NormShape norm_shape(int cols, int per_chunk) {
  const int chunks = (cols + per_chunk - 1) / per_chunk;
  if (cols <= 1024) {
    int ch = 1;
    while (64 * ch < chunks) ch *= 2;
    return {ch, 64 * kWaveRows, true};
  }
  int ch = 4;
  while (kNormMaxThreads * ch < chunks) ch *= 2;
  return {ch, ((chunks + ch - 1) / ch + 63) / 64 * 64, false};
}

template <typename T, bool CENTER, int CH, bool WAVE>
void run_norm(const NormArgs& a, int grid, int threads, hipStream_t stream) {
  hipLaunchKernelGGL((k_norm_fwd<T, CH, CENTER, WAVE>), dim3(grid), dim3(threads), 0, stream, a);
}
template <typename T, bool CENTER, int CH, bool WAVE>
void run_norm(const NormGradArgs& a, int grid, int threads, hipStream_t stream) {
  if (!CENTER && a.add)
    hipLaunchKernelGGL((k_norm_bwd<T, CH, false, WAVE, true>), dim3(grid), dim3(threads), 0, stream, a);
  else
    hipLaunchKernelGGL((k_norm_bwd<T, CH, CENTER, WAVE, false>), dim3(grid), dim3(threads), 0, stream, a);
}
// Chunks reached: one wave 1, 2 (bf16: 1024 = 2 * 64 * 8) and 4 (fp32); workgroups
// 4, 8 (bf16: 32768 = 8 * 512 * 8) and 16 (fp32).
template <typename T, bool CENTER, typename Args>
hipError_t run_shape(const Args& a, int grid, const NormShape& s, hipStream_t stream) {
  constexpr bool kF32 = sizeof(T) == 4;
  if (s.wave) {
    if (s.ch == 1) run_norm<T, CENTER, 1, true>(a, grid, s.threads, stream);
    else if (!kF32 || s.ch == 2) run_norm<T, CENTER, 2, true>(a, grid, s.threads, stream);
    else if constexpr (kF32) run_norm<T, CENTER, 4, true>(a, grid, s.threads, stream);
  } else {
    if (s.ch == 4) run_norm<T, CENTER, 4, false>(a, grid, s.threads, stream);
    else if (!kF32 || s.ch == 8) run_norm<T, CENTER, 8, false>(a, grid, s.threads, stream);
    else if constexpr (kF32) run_norm<T, CENTER, 16, false>(a, grid, s.threads, stream);
  }
  return hipGetLastError();
}
template <typename Args>
hipError_t run_types(const Args& a, int grid, const NormShape& s, hipStream_t stream) {
  if (a.bf16)
    return a.center ? run_shape<uint16_t, true>(a, grid, s, stream)
                    : run_shape<uint16_t, false>(a, grid, s, stream);
  return a.center ? run_shape<float, true>(a, grid, s, stream)
                  : run_shape<float, false>(a, grid, s, stream);
}

// Workgroups: 32 chunks a lane on every compute unit (32 KB of a row's loads in
// flight each).  7168 bf16, waves a unit, forward us: 4 112, 8 81, 12 89, 16 93;
// with the backward pass 4 294, 8 250, 12 310 (its registers hold 8).
int norm_grid(int64_t rows, const NormShape& s) {
  const int waves = std::max(1, 32 / s.ch);
  const int64_t per_cu = std::max(1, waves / (s.threads / 64));
  const int64_t own = s.wave ? (rows + kWaveRows - 1) / kWaveRows : rows;
  return (int)std::min<int64_t>(own, std::max(1, device_cu_count()) * per_cu);
}

// The norm with the residual's addition has more work an element than k_norm_fwd, and rows of
// a workgroup take two chunks a thread where they fit, as long as the sum and the norm leave
// as they are only up to 2^26 elements.  7168 bf16, two chunks against four, us, sum and norm
// / E8M0 / fp32 scales: 64 rows 3.5 / 4.6 / 4.4 and 4.7 / 7.5 / 6.2, 1024 8.0 / 11.0 / 9.8 and
// 9.0 / 12.9 / 11.3, 4096 35.2 / 36.8 / 35.0 and 36.7 / 40.2 / 37.9, 16384 174 / 169 / 167
// and 169 / 173 / 170.
NormShape add_norm_shape(const AddNormArgs& a) {
  const int per_chunk = a.bf16 ? 8 : 4, chunks = (a.cols + per_chunk - 1) / per_chunk;
  const NormShape s = norm_shape(a.cols, per_chunk);
  if (s.wave || chunks > 2 * kNormMaxThreads || (!a.q && a.rows * a.cols > INT64_C(1) << 26)) return s;
  return {2, ((chunks + 1) / 2 + 63) / 64 * 64, false};
}

template <typename T, int CH, bool WAVE>
void run_add_norm(const AddNormArgs& a, int grid, int threads, hipStream_t stream) {
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), 0, stream, a);
  };
  if (!a.q) go(k_add_norm<T, CH, WAVE, kOutSame, true>);
  else if (a.mx) a.res ? go(k_add_norm<T, CH, WAVE, kOutMx, true>) : go(k_add_norm<T, CH, WAVE, kOutMx, false>);
  else a.res ? go(k_add_norm<T, CH, WAVE, kOutBlock, true>) : go(k_add_norm<T, CH, WAVE, kOutBlock, false>);
}
template <typename T>
void run_add_shape(const AddNormArgs& a, int grid, const NormShape& s, hipStream_t stream) {
  constexpr bool kF32 = sizeof(T) == 4;
  if (s.wave) {
    if (s.ch == 1) run_add_norm<T, 1, true>(a, grid, s.threads, stream);
    else if (!kF32 || s.ch == 2) run_add_norm<T, 2, true>(a, grid, s.threads, stream);
    else if constexpr (kF32) run_add_norm<T, 4, true>(a, grid, s.threads, stream);
  } else {
    if (s.ch == 2) run_add_norm<T, 2, false>(a, grid, s.threads, stream);
    else if (s.ch == 4) run_add_norm<T, 4, false>(a, grid, s.threads, stream);
    else if (!kF32 || s.ch == 8) run_add_norm<T, 8, false>(a, grid, s.threads, stream);
    else if constexpr (kF32) run_add_norm<T, 16, false>(a, grid, s.threads, stream);
  }
}

}  // namespace

hipError_t launch_add_norm(AddNormArgs a, hipStream_t stream) {
  if (a.rows == 0) return hipSuccess;
  const NormShape s = add_norm_shape(a);
  int grid = norm_grid(a.rows, s);
  if (a.q) {  // runs of up to 16 rows, as long as every workgroup has one
    const int64_t unit = s.wave ? kWaveRows : 1, own = (a.rows + unit * grid - 1) / (unit * grid);
    a.run = (int32_t)(unit * std::min<int64_t>(own, kScaleRun / unit));
    grid = (int)std::min<int64_t>(grid, (a.rows + a.run - 1) / a.run);
  }
  if (a.bf16) run_add_shape<uint16_t>(a, grid, s, stream);
  else run_add_shape<float>(a, grid, s, stream);
  return hipGetLastError();
}

hipError_t launch_norm_fwd(const NormArgs& a, hipStream_t stream) {
  if (a.rows == 0) return hipSuccess;
  const NormShape s = norm_shape(a.cols, a.bf16 ? 8 : 4);
  return run_types(a, norm_grid(a.rows, s), s, stream);
}

int norm_grad_parts(int64_t rows, int cols, int bf16) {
  const NormShape s = norm_shape(cols, bf16 ? 8 : 4);
  return rows == 0 ? 0 : norm_grid(rows, s);
}

hipError_t launch_norm_bwd(const NormGradArgs& a, hipStream_t stream) {
  const int parts = norm_grad_parts(a.rows, a.cols, a.bf16);
  hipError_t err = hipSuccess;
  if (parts > 0) err = run_types(a, parts, norm_shape(a.cols, a.bf16 ? 8 : 4), stream);
  if (err != hipSuccess || (!a.dw && !a.db)) return err;
  const dim3 grid((unsigned)((a.cols + kNormReduceCols - 1) / kNormReduceCols), 2);
  hipLaunchKernelGGL(k_norm_reduce, grid, dim3(kNormReduceCols * kNormReduceRuns), 0, stream,
                     a.partial, parts, a.cols, a.dw, a.w_bf16, a.db, a.b_bf16);
  return hipGetLastError();
}

}  // namespace mxgg
