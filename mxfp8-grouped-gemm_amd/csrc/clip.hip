// Global norm of many gradients, and clipping in place.
//
//   norm = sqrt(sum over all tensors of g^2),  g <- g min(1, max_norm / (norm + eps))
//
// Two passes.  The first leaves one sum of squares a workgroup; squares and sums are
// fp64, which the vector units do many times faster than memory delivers: a square of an
// fp32 or bf16 value is exact (48 bits; no overflow at 1e19, nothing lost below 1e-23), and
// each addition rounds to 2^-53, so the norm is the fp32 rounding of the true one but next
// to a border between two.  In the second
// every workgroup adds all of the partial sums in the same order, so the factor is the
// same in each and from run to run, and ends without touching its gradients where
// nothing is clipped.
//
// Memory-bound: each gradient is read twice and written once.  The second pass goes
// through the tensors backwards and finds what the first read last in the cache.  235 M
// bf16 gradients: 85-101 us (4.7-5.5 TB/s) and 146 (6.4, part of it from the cache); fp32
// 163-165 us (5.8) for the norm.
#include <algorithm>

#include "mx_device.h"
#include "mxgg_internal.h"

namespace mxgg {
namespace {

constexpr int kClipThreads = 256;
constexpr int kClipVec = 8;                    // consecutive elements of a thread
constexpr int kClipRuns = 8;                   // runs of kClipThreads * kClipVec in flight
constexpr int64_t kClipStep = (int64_t)kClipThreads * kClipVec * kClipRuns;
constexpr int kClipTensors = 190;              // of a launch: the 4 KB of kernel arguments
constexpr int64_t kClipParts = 2048;           // workgroups of a large call: 8 a compute unit

struct ClipTensor {
  void* p;
  int64_t n : 62;
  uint64_t bf16 : 1;
};
struct ClipTable {
  ClipTensor t[kClipTensors];
  int32_t first[kClipTensors + 1];  // first workgroup of each tensor
  int32_t count;
  int32_t part0;                    // partial sum of this launch's first workgroup
  int32_t parts;                    // of all launches
  int64_t chunk;                    // elements of a workgroup
  double* part;
  float* norm;
  double max_norm, eps;
};
static_assert(sizeof(ClipTable) <= 4096, "kernel arguments");

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

// Eight elements as they are stored: two 16-byte words of fp32, one of bf16.
template <bool BF16>
struct Run {
  u32x4 w[BF16 ? 1 : 2];
};
template <bool BF16>
__device__ __forceinline__ void load_run(Run<BF16>& r, const void* p, int64_t i, int n) {
  if (n >= kClipVec) {
#pragma unroll
    for (int k = 0; k < (BF16 ? 1 : 2); ++k)
      r.w[k] = *reinterpret_cast<const u32x4_any*>(static_cast<const uint8_t*>(p) +
                                                   i * (BF16 ? 2 : 4) + 16 * k);
    return;
  }
#pragma unroll
  for (int j = 0; j < kClipVec; ++j) {
    uint32_t v = 0;
    if (j < n) v = BF16 ? static_cast<const uint16_t*>(p)[i + j] : static_cast<const uint32_t*>(p)[i + j];
    if constexpr (BF16) r.w[0][j / 2] = (j & 1) ? r.w[0][j / 2] | v << 16 : v;
    else r.w[j / 4][j % 4] = v;
  }
}
template <bool BF16>
__device__ __forceinline__ float element(const Run<BF16>& r, int j) {
  if constexpr (BF16) return (j & 1) ? bf16_hi(r.w[0][j / 2]) : bf16_lo(r.w[0][j / 2]);
  else return __uint_as_float(r.w[j / 4][j % 4]);
}
template <bool BF16>
__device__ __forceinline__ void store_scaled(void* p, int64_t i, int n, const Run<BF16>& r, float f) {
  Run<BF16> o;
#pragma unroll
  for (int j = 0; j < kClipVec; j += 2) {
    const float a = element(r, j) * f, b = element(r, j + 1) * f;
    if constexpr (BF16) {
      o.w[0][j / 2] = pack_bf16x2(a, b);
    } else {
      o.w[j / 4][j % 4] = __float_as_uint(a);
      o.w[j / 4][j % 4 + 1] = __float_as_uint(b);
    }
  }
  if (n >= kClipVec) {
#pragma unroll
    for (int k = 0; k < (BF16 ? 1 : 2); ++k)
      *reinterpret_cast<u32x4_any*>(static_cast<uint8_t*>(p) + i * (BF16 ? 2 : 4) + 16 * k) = o.w[k];
    return;
  }
#pragma unroll
  for (int j = 0; j < kClipVec; ++j)
    if (j < n) {
      if constexpr (BF16) static_cast<uint16_t*>(p)[i + j] = (uint16_t)(o.w[0][j / 2] >> (16 * (j & 1)));
      else static_cast<uint32_t*>(p)[i + j] = o.w[j / 4][j % 4];
    }
}

// Sum over the workgroup, in every thread; the same order on every run.
__device__ __forceinline__ double group_sum(double v, double* slots) {
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int w = 0; w < kClipThreads / 64; ++w) v += slots[w];
  return v;
}

// The part of tensor t that workgroup `block` of its own holds, one run of eight at a
// time: f(run, first element, elements).
template <bool BF16, class F>
__device__ __forceinline__ void for_runs(const ClipTensor& t, int64_t block, int64_t chunk, F f) {
  const int64_t end = min((int64_t)t.n, (block + 1) * chunk);
  for (int64_t base = block * chunk; base < end; base += kClipStep) {
    Run<BF16> r[kClipRuns];
    const int64_t i0 = base + (int64_t)threadIdx.x * kClipVec;
    if (base + kClipStep <= end) {
#pragma unroll
      for (int u = 0; u < kClipRuns; ++u)
        load_run<BF16>(r[u], t.p, i0 + u * kClipThreads * kClipVec, kClipVec);
#pragma unroll
      for (int u = 0; u < kClipRuns; ++u) f(r[u], i0 + u * kClipThreads * kClipVec, kClipVec);
    } else {
#pragma unroll
      for (int u = 0; u < kClipRuns; ++u) {
        const int64_t i = i0 + u * kClipThreads * kClipVec, left = end - i;
        const int n = left >= kClipVec ? kClipVec : left > 0 ? (int)left : 0;
        load_run<BF16>(r[u], t.p, i, n);
        if (n > 0) f(r[u], i, n);
      }
    }
  }
}

__device__ __forceinline__ int tensor_of(const ClipTable& a, int block) {
  int lo = 0, hi = a.count;  // last tensor that starts at or before this workgroup
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.first[mid] <= block) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ __launch_bounds__(kClipThreads) void k_clip_sums(ClipTable a) {
  __shared__ double slots[kClipThreads / 64];
  const int at = tensor_of(a, blockIdx.x);
  const ClipTensor t = a.t[at];
  const int64_t block = (int)blockIdx.x - a.first[at];
  double s = 0.0;
  const auto add = [&](const auto& r, int64_t, int) {
#pragma unroll
    for (int j = 0; j < kClipVec; ++j) {
      const double g = element(r, j);
      s = __builtin_fma(g, g, s);
    }
  };
  if (t.bf16) for_runs<true>(t, block, a.chunk, add);
  else for_runs<false>(t, block, a.chunk, add);
  s = group_sum(s, slots);
  if (threadIdx.x == 0) a.part[a.part0 + blockIdx.x] = s;
}

__global__ __launch_bounds__(kClipThreads) void k_clip_scale(ClipTable a, int clip) {
  __shared__ double slots[kClipThreads / 64];
  double s = 0.0;
  for (int i = threadIdx.x; i < a.parts; i += kClipThreads) s += a.part[i];
  const double norm = sqrt(group_sum(s, slots));
  if (a.norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = (float)norm;
  if (!clip || a.count == 0) return;
  // no factor where there is nothing to clip: an infinite bound (inf / inf), or zeros under a
  // bound of zero (0 / 0)
  if (norm == norm && (a.max_norm == __builtin_inf() || norm + a.eps == 0.0)) return;
  const float f = (float)(a.max_norm / (norm + a.eps));
  if (f >= 1.0f) return;  // a NaN goes on: its gradients become NaN
  const int b = (int)(gridDim.x - 1 - blockIdx.x), at = tensor_of(a, b);
  const ClipTensor t = a.t[at];
  const int64_t block = b - a.first[at];
  if (t.bf16)
    for_runs<true>(t, block, a.chunk, [&](const auto& r, int64_t i, int n) {
      store_scaled<true>(t.p, i, n, r, f);
    });
  else
    for_runs<false>(t, block, a.chunk, [&](const auto& r, int64_t i, int n) {
      store_scaled<false>(t.p, i, n, r, f);
    });
}

// Elements of a workgroup: whole steps, so many that a large call has kClipParts.
int64_t clip_chunk(int64_t total) {
  const int64_t per = (total + kClipParts - 1) / kClipParts;
  return std::max<int64_t>(1, (per + kClipStep - 1) / kClipStep) * kClipStep;
}

}  // namespace

int64_t clip_parts(const mxgg_grad_tensor* tensors, int64_t count) {
  int64_t total = 0, parts = 0;
  for (int64_t i = 0; i < count; ++i) total += tensors[i].n;
  const int64_t chunk = clip_chunk(total);
  for (int64_t i = 0; i < count; ++i) parts += (tensors[i].n + chunk - 1) / chunk;
  return parts;
}

hipError_t launch_clip(const mxgg_grad_tensor* tensors, int64_t count,
                       const mxgg_clip_options* options, double* part, float* norm,
                       hipStream_t stream) {
  const bool clip = options != nullptr;
  ClipTable a;
  int64_t total = 0;
  for (int64_t i = 0; i < count; ++i) total += tensors[i].n;
  a.chunk = clip_chunk(total);
  a.parts = (int32_t)clip_parts(tensors, count);
  a.part = part;
  a.max_norm = clip ? options->max_norm : 0.0;
  a.eps = clip ? options->eps : 0.0;
  for (int pass = 0; pass < 2; ++pass) {
    int64_t done = 0, i = 0;
    a.norm = norm;
    do {
      a.count = 0;
      a.part0 = (int32_t)done;
      int64_t blocks = 0;
      for (; i < count && a.count < kClipTensors; ++i) {
        const int64_t own = (tensors[i].n + a.chunk - 1) / a.chunk;
        if (own == 0) continue;
        a.t[a.count] = {tensors[i].data, tensors[i].n, tensors[i].dtype == MXGG_OUT_BF16};
        a.first[a.count++] = (int32_t)blocks;
        blocks += own;
      }
      a.first[a.count] = (int32_t)blocks;
      done += blocks;
      if (pass == 0) {
        if (blocks > 0)
          hipLaunchKernelGGL(k_clip_sums, dim3((unsigned)blocks), dim3(kClipThreads), 0, stream, a);
      } else if (a.norm || (clip && blocks > 0)) {  // the norm alone takes one workgroup
        const unsigned grid = clip && blocks > 0 ? (unsigned)blocks : 1u;
        hipLaunchKernelGGL(k_clip_scale, dim3(grid), dim3(kClipThreads), 0, stream, a, clip ? 1 : 0);
        a.norm = nullptr;
      }
      const hipError_t err = hipGetLastError();
      if (err != hipSuccess) return err;
    } while (i < count);
  }
  return hipSuccess;
}

}  // namespace mxgg
