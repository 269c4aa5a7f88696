// One AdamW step over many tensors in one launch per kAdamTensors of them.
//
//   p <- p (1 - lr wd)
//   m <- b1 m + (1 - b1) g        v <- b2 v + (1 - b2) g^2
//   p <- p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Everything is computed in fp32 from fp32 or bf16 weights and gradients; with
// a master copy (fp32) the step is taken there and the weight is its rounding.
// The tensors' addresses travel in the kernel's arguments (no table to copy to
// the device); a workgroup finds its tensor by a search over the prefix of
// chunk counts.
//
// 8-bit states are MXFP8: e4m3 payloads with one E8M0 byte for every 32
// consecutive elements, 1.03 bytes a value.  The second moment is kept as its
// root, whose range is half as many powers of two: e4m3 spans 2^18 below a
// block's largest value, so 2^36 of v.  Both are read, updated in fp32, used
// unrounded for the step and rounded to nearest only when stored.
//
// Memory-bound: 22 bytes an element for bf16 weights and gradients with fp32
// states, 10.1 with 8-bit ones.  A thread takes 8 consecutive elements (16-byte
// accesses); four lanes hold one block of 32.
#include "mx_device.h"
#include "mxgg_internal.h"

namespace mxgg {
namespace {

constexpr int kAdamThreads = 256;
constexpr int kAdamVec = 8;
// Elements of a workgroup, 8 a thread.  235 M bf16 weights with fp32 states and
// master copy: 1231 us (5.3 TB/s); twice as many elements in two trips 1249, runs
// of 4 whose lanes follow each other without gaps 1253.  8-bit states: 420 to 435 us.
constexpr int64_t kAdamChunk = kAdamThreads * kAdamVec;
constexpr int kAdamTensors = 48;      // of a launch: 3.3 of the 4 KB of kernel arguments

struct AdamTable {
  AdamTensor t[kAdamTensors];
  int32_t first[kAdamTensors + 1];  // first workgroup of each tensor
  int32_t count;
  AdamScalars s;
};
static_assert(sizeof(AdamTable) <= 4096, "kernel arguments");

// Words at any element alignment, as one access each.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));

// Eight consecutive fp32 or bf16 values at p + i; FULL: all of them lie inside the
// tensor, else `n` of them do and the rest read as 0.
template <bool FULL>
__device__ __forceinline__ void load8(const void* p, bool bf16, int64_t i, int n, float (&v)[8]) {
  if (bf16) {
    const uint16_t* q = static_cast<const uint16_t*>(p) + i;
    u32x4 w;
    if constexpr (FULL) {
      w = *reinterpret_cast<const u32x4_any*>(q);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j += 2)
        w[j / 2] = (j < n ? q[j] : 0u) | (j + 1 < n ? (uint32_t)q[j + 1] : 0u) << 16;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (j & 1) ? bf16_hi(w[j >> 1]) : bf16_lo(w[j >> 1]);
    return;
  }
  const float* q = static_cast<const float*>(p) + i;
#pragma unroll
  for (int k = 0; k < 8; k += 4) {
    if constexpr (FULL) {
      const u32x4 w = *reinterpret_cast<const u32x4_any*>(q + k);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[k + j] = __uint_as_float(w[j]);
    } else {
#pragma unroll
      for (int j = k; j < k + 4; ++j) v[j] = j < n ? q[j] : 0.0f;
    }
  }
}
template <bool FULL>
__device__ __forceinline__ void store8(void* p, bool bf16, int64_t i, int n, const float (&v)[8]) {
  if (bf16) {
    uint16_t* q = static_cast<uint16_t*>(p) + i;
    const u32x4 w{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                  pack_bf16x2(v[6], v[7])};
    if constexpr (FULL) {
      *reinterpret_cast<u32x4_any*>(q) = w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) q[j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
    }
    return;
  }
  float* q = static_cast<float*>(p) + i;
#pragma unroll
  for (int k = 0; k < 8; k += 4) {
    if constexpr (FULL) {
      *reinterpret_cast<u32x4_any*>(q + k) =
          u32x4{__float_as_uint(v[k]), __float_as_uint(v[k + 1]), __float_as_uint(v[k + 2]),
                __float_as_uint(v[k + 3])};
    } else {
#pragma unroll
      for (int j = k; j < k + 4; ++j)
        if (j < n) q[j] = v[j];
    }
  }
}

// Eight values of an 8-bit state: payload bytes at q + i, block byte b.  Byte
// 255 stands for a block of NaN (its payload bytes are NaN codes).
template <bool FULL>
__device__ __forceinline__ void unpack8(const uint8_t* q, const uint8_t* s, int64_t i, int n,
                                        float (&v)[8]) {
  uint32_t w[2] = {0, 0};
  if constexpr (FULL) {
    const u32x2 u = *reinterpret_cast<const u32x2_any*>(q + i);
    w[0] = u[0];
    w[1] = u[1];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) w[j >> 2] |= (uint32_t)q[i + j] << (8 * (j & 3));
  }
  const uint32_t b = n > 0 ? s[i >> 5] : 1u;
  const float scale = __uint_as_float(b == 0u ? 0x00400000u : b << 23);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[k], false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[k], true);
    v[4 * k] = lo[0] * scale;
    v[4 * k + 1] = lo[1] * scale;
    v[4 * k + 2] = hi[0] * scale;
    v[4 * k + 3] = hi[1] * scale;
  }
}

// Rounds eight values to an 8-bit state under the scale of their block of 32,
// which the four lanes of a quad hold together: every lane of the wave calls it.
// b = ceil(log2(amax / 448)) + 127, at least 1 (normal scales); 255 if the block
// holds an infinity or a NaN.
template <bool FULL>
__device__ __forceinline__ void pack8(uint8_t* q, uint8_t* s, int64_t i, int n,
                                      const float (&v)[8]) {
  uint32_t amax = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(v[j]) & 0x7FFFFFFFu);
  amax = quad_max(n > 0 ? amax : 0u);
  const int ex = (int)(amax >> 23);
  int b = ex - 8 + ((amax & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  b = ex == 255 ? 255 : max(1, min(b, 254));
  uint32_t w[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = __builtin_ldexpf(v[4 * k + j], 127 - b);
    const uint32_t u = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    w[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], (int)u, true);
    if (b == 255) w[k] = 0x7F7F7F7Fu;
  }
  if constexpr (FULL) {
    *reinterpret_cast<u32x2_any*>(q + i) = u32x2{w[0], w[1]};
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) q[i + j] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
  }
  if (n > 0 && (i & 31) == 0) s[i >> 5] = (uint8_t)b;
}

// Eight consecutive elements from i on; every lane of the wave calls it.
template <bool SMALL, bool FULL>
__device__ __forceinline__ void step(const AdamTensor& t, const AdamScalars& s, int64_t i) {
  // every product and sum rounds by itself: a fused multiply-add would make the
  // states depend on how the compiler pairs them
#pragma clang fp contract(off)
  const int64_t left = t.n - i;
  const int n = FULL || left >= 8 ? 8 : left > 0 ? (int)left : 0;
  void* weights = t.master ? static_cast<void*>(t.master) : t.param;
  const bool w_bf16 = !t.master && t.param_bf16;
  float p[8], g[8], m[8], v[8];
  load8<FULL>(weights, w_bf16, i, n, p);
  load8<FULL>(t.grad, t.grad_bf16, i, n, g);
  if constexpr (SMALL) {
    unpack8<FULL>(static_cast<const uint8_t*>(t.m), t.m_scales, i, n, m);
    unpack8<FULL>(static_cast<const uint8_t*>(t.v), t.v_scales, i, n, v);
  } else {
    load8<FULL>(t.m, false, i, n, m);
    load8<FULL>(t.v, false, i, n, v);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    m[j] = m[j] * s.beta1 + g[j] * s.one_beta1;
    const float old = SMALL ? v[j] * v[j] : v[j];
    const float now = old * s.beta2 + (g[j] * g[j]) * s.one_beta2;
    const float root = sqrtf(now);
    v[j] = SMALL ? root : now;
    p[j] = p[j] * s.decay - s.step_size * (m[j] / (root * s.inv_root_bias2 + s.eps));
  }
  if constexpr (SMALL) {
    pack8<FULL>(static_cast<uint8_t*>(t.m), t.m_scales, i, n, m);
    pack8<FULL>(static_cast<uint8_t*>(t.v), t.v_scales, i, n, v);
  } else {
    store8<FULL>(t.m, false, i, n, m);
    store8<FULL>(t.v, false, i, n, v);
  }
  store8<FULL>(weights, w_bf16, i, n, p);
  if (t.master) store8<FULL>(t.param, t.param_bf16, i, n, p);
}

template <bool SMALL>
__global__ __launch_bounds__(kAdamThreads) void k_adamw(AdamTable a) {
  int lo = 0, hi = a.count;  // last tensor that starts at or before this workgroup
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.first[mid] <= (int)blockIdx.x) lo = mid; else hi = mid;
  }
  const AdamTensor t = a.t[lo];
  const int64_t base = (int64_t)((int)blockIdx.x - a.first[lo]) * kAdamChunk;
  const bool full = base + kAdamChunk <= t.n;  // the tensor's last workgroup may not be
  const int64_t i = base + (int64_t)threadIdx.x * kAdamVec;
  if (full)
    step<SMALL, true>(t, a.s, i);
  else
    step<SMALL, false>(t, a.s, i);
}

}  // namespace

hipError_t launch_adamw(const AdamTensor* tensors, int64_t count, int state_bits,
                        const AdamScalars& scalars, hipStream_t stream) {
  // workgroups of a launch, below the grid's 2^32 work-items
  constexpr int64_t kMaxBlocks = INT64_C(1) << 23;
  for (int64_t i = 0; i < count;) {
    AdamTable a;
    a.s = scalars;
    a.count = 0;
    int64_t blocks = 0;
    for (; i < count && a.count < kAdamTensors; ++i) {
      const int64_t own = (tensors[i].n + kAdamChunk - 1) / kAdamChunk;
      if (own == 0) continue;
      if (blocks > 0 && blocks + own > kMaxBlocks) break;
      a.t[a.count] = tensors[i];
      a.first[a.count++] = (int32_t)blocks;
      blocks += own;
    }
    if (blocks == 0) continue;
    a.first[a.count] = (int32_t)blocks;
    if (state_bits == 8)
      hipLaunchKernelGGL((k_adamw<true>), dim3((unsigned)blocks), dim3(kAdamThreads), 0, stream, a);
    else
      hipLaunchKernelGGL((k_adamw<false>), dim3((unsigned)blocks), dim3(kAdamThreads), 0, stream,
                         a);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

int64_t adamw_max_elements() { return (INT64_C(1) << 23) * kAdamChunk; }

}  // namespace mxgg
