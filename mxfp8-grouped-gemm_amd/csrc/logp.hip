// Log probabilities of given tokens from logits, with the entropy of the distribution
// and its top alternatives, and their gradient.
//
//   p = softmax(z / T),  lp = (z_t - m) / T - log S,  S = sum exp((z - m) / T), m = max z
//   H = log S - sum p (z - m) / T                 (a sum of terms of one sign)
//   dz = (sum of the gradients g_e at the chosen tokens e
//         - p (sum g_e + g_H ((z - m) / T - log S + H))) / T
//
// Memory-bound: the logits are read once.  A thread keeps a running maximum, the sum of
// exponentials below it and the sum of exponentials times exponents, all fp32 in units
// of log 2, rescaled when a run of its elements has a larger maximum.  (m, log S) are
// kept apart, so nothing is lost where the logits share a large offset.
//
// The k best: the pass leaves the maximum of every 64 consecutive logits in LDS.  The
// k-th largest of 64 interleaved groups' maxima (of 256 where k is large) bounds the k-th
// best from below; the few runs of 64 that reach it are read again and what reaches it is
// collected, a few more than k values, among which k are picked by value, then lowest index.
// Where fewer than k runs hold a logit above -inf (a row, or what its mask leaves of it, of
// fewer than 64 k logits) there is no bound and all of them are candidates; so are thousands
// of equal logits.  Up to 512 are ranked at once; more are searched by one wave for each of
// the k, and more than the list holds by reading the row again for each.
//
// Few rows are split over workgroups, whose results a second kernel joins in order.
//
// Measured: 4096 x 131072 bf16 191-200 us (5.4-5.6 TB/s), with 8 alternatives 205, their
// gradient 379 (5.7 TB/s read and written); 1000 x 50021 fp32 34 us (6.0), with 20
// alternatives 41; 16 x 131072 with 8 alternatives 11.7 us (with 64 23.8), 16 x 32000 8.2,
// where the chain of dependent steps counts, not the 4 MB.  Without a bound, 16 rows of bf16:
// 500 logits with 20 alternatives 17 us, 1000 with 20 48 (with 16, bounded, 8.5), 2000 with 64
// 246 (with 20 7.3), 3000 with 64 113; 1000 x 3000 fp32 with 64 237.
#include <algorithm>

#include "mx_device.h"
#include "mxgg_internal.h"

namespace mxgg {
namespace {

constexpr int kLogpThreads = 512;
constexpr int kLogpWaves = kLogpThreads / 64;
constexpr int kAhead = 4;                  // 16-byte loads of a thread in flight
constexpr int kSeg = 64;                   // consecutive logits under one maximum
constexpr int kMaxSegs = 4096;
constexpr int64_t kMaxPart = (int64_t)kSeg * kMaxSegs;
constexpr int64_t kMinPart = 8192;         // elements of a workgroup, at least
constexpr int64_t kWholeBytes = 128 << 10; // rows of up to this many stay whole
constexpr int kMaxParts = 64;              // of a row
constexpr int kList = 2048;                // candidates
constexpr int kMaxTop = 64;
// Alternatives up to which 64 groups bound well: 64 of 64 leave 300 candidates and more,
// 16 x 131072 with 64 alternatives 107 us (23.8 with 256 groups), with 20 13.7.
constexpr int kCoarse = 32;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kLowest = -3.402823466e+38f;
constexpr float kFar = -1e6f;              // an exponent whose power of two is 0
constexpr float kInf = __builtin_inff();

template <typename T>
struct Logits;
template <>
struct Logits<float> {
  static constexpr int kCount = 4;
  __device__ static float get(const uint4& v, int j) {
    return __uint_as_float(j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w);
  }
  __device__ static float one(const float* p) { return *p; }
};
template <>
struct Logits<uint16_t> {
  static constexpr int kCount = 8;
  __device__ static float get(const uint4& v, int j) {
    const uint32_t w = j < 2 ? v.x : j < 4 ? v.y : j < 6 ? v.z : v.w;
    return (j & 1) ? bf16_hi(w) : bf16_lo(w);
  }
  __device__ static float one(const uint16_t* p) { return bf16_bits_to_f32(*p); }
};
// A chunk of n logits from p on; what lies past them reads as -inf.
template <typename T>
__device__ __forceinline__ uint4 load_logits(const T* p, int n) {
  constexpr int E = Logits<T>::kCount;
  uint4 v;
  if (n >= E) {
    __builtin_memcpy(&v, p, 16);
    return v;
  }
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = E == 4 ? 0xFF800000u : 0xFF80FF80u;
#pragma unroll
  for (int j = 0; j < E; ++j)
    if (j < n) {
      if constexpr (E == 4) w[j] = __float_as_uint(p[j]);
      else w[j >> 1] = (j & 1) ? (w[j >> 1] & 0xFFFFu) | (uint32_t)p[j] << 16
                               : (w[j >> 1] & 0xFFFF0000u) | p[j];
    }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Sums relative to a maximum, in units of log 2: s = sum 2^d, w = sum 2^d d.
struct Sums {
  float m, s, w;
};
__device__ __forceinline__ void rescale(Sums& a, float m, float c) {
  // an empty side has no sums: the exponent is clamped so that it stays a number
  const float d = __builtin_fmaxf((a.m - __builtin_fmaxf(m, kLowest)) * c, kFar);
  const float f = __builtin_amdgcn_exp2f(d);
  a.w = f * __builtin_fmaf(d, a.s, a.w);
  a.s *= f;
  a.m = m;
}
__device__ __forceinline__ float wave_max(float x) {
  x = __builtin_fmaxf(x, dpp_mov<0xB1>(x));
  x = __builtin_fmaxf(x, dpp_mov<0x4E>(x));
  x = __builtin_fmaxf(x, dpp_mov<0x141>(x));
  x = __builtin_fmaxf(x, dpp_mov<0x140>(x));
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __builtin_fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
  const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __builtin_fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
// Over the wave, in every lane, in an order that does not change.
__device__ __forceinline__ Sums wave_join(Sums a, float c) {
  rescale(a, wave_max(a.m), c);
  return {a.m, wave_sum(a.s), wave_sum(a.w)};
}
// The same over N parts in LDS, one after the other.
template <int N>
__device__ __forceinline__ Sums join_all(const Sums* p, float c) {
  float m = p[0].m;
#pragma unroll
  for (int i = 1; i < N; ++i) m = __builtin_fmaxf(m, p[i].m);
  Sums t{m, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    Sums a = p[i];
    rescale(a, m, c);
    t.s += a.s;
    t.w += a.w;
  }
  return t;
}
// A candidate as an integer that orders by value, then by lowest index: the value's bits
// made monotone (-0 as 0) above the inverted index.  0 is none.
__device__ __forceinline__ uint64_t key_of(float v, int64_t index) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  const uint32_t o = u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
  return (uint64_t)o << 32 | (0xFFFFFFFFu - (uint32_t)index);
}
struct Pick {
  float v;
  int32_t i;  // -1: none
};
__device__ __forceinline__ Pick pick_of(uint64_t key) {
  if (key == 0) return {-kInf, -1};
  const uint32_t o = (uint32_t)(key >> 32);
  return {__uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xFFFFFFFFu)),
          (int32_t)(0xFFFFFFFFu - (uint32_t)key)};
}
__device__ __forceinline__ uint64_t wave_max_key(uint64_t x) {
  for (int d = 1; d < 64; d <<= 1) x = max(x, (uint64_t)__shfl_xor((unsigned long long)x, d));
  return x;
}

// The k-th largest of 64 lanes' values (-inf where fewer are above it): the smallest of those
// that fewer than k others are above.
__device__ __forceinline__ float kth_of_lanes(float x, int k) {
  int above = 0;
#pragma unroll
  for (int j = 0; j < 64; ++j)
    above += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), j)) > x ? 1 : 0;
  return -wave_max(above < k ? -x : -kInf);
}
// The same of the first 256 threads' values, for the workgroup; held: 256 values, low: 4.
__device__ __forceinline__ float kth_of_group(float x, int k, float* held, float* low) {
  const int tid = threadIdx.x;
  if (tid < 256) held[tid] = x;
  __syncthreads();
  if (tid < 256) {
    int above = 0;
#pragma unroll 8
    for (int j = 0; j < 256; j += 4) {
      const float4 o = *reinterpret_cast<const float4*>(held + j);
      above += (o.x > x ? 1 : 0) + (o.y > x ? 1 : 0) + (o.z > x ? 1 : 0) + (o.w > x ? 1 : 0);
    }
    const float m = -wave_max(above < k ? -x : -kInf);
    if ((tid & 63) == 0) low[tid >> 6] = m;
  }
  __syncthreads();
  return __builtin_fminf(__builtin_fminf(low[0], low[1]), __builtin_fminf(low[2], low[3]));
}

// The k best of n different keys in LDS (0 is none), in falling order, by every thread of
// the workgroup: f(rank, key), called by whichever thread has it.  Up to kRanked are
// ranked against each other at once; more are searched by the first wave for each of
// the k.
constexpr int kRanked = 512;
template <class F>
__device__ __forceinline__ void pick_best(uint64_t* list, int n, int k, F f) {
  if (n <= kRanked) {
    for (int i = threadIdx.x; i < max(n, k); i += blockDim.x) {
      const uint64_t own = i < n ? list[i] : 0;
      int rank = 0, valid = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) {
        const uint64_t o = list[j];
        rank += o > own ? 1 : 0;
        valid += o != 0 ? 1 : 0;
      }
      if (own != 0 && rank < k) f(rank, own);
      if (i < k && i >= valid) f(i, 0);
    }
    return;
  }
  if (threadIdx.x >= 64) return;
  const int lane = threadIdx.x;
  const auto best_of_lane = [&] {
    uint64_t b = 0;
    for (int j = lane; j < n; j += 64) b = max(b, list[j]);
    return b;
  };
  uint64_t mine = best_of_lane();
  for (int r = 0; r < k; ++r) {
    const uint64_t top = wave_max_key(mine);
    if (lane == 0) f(r, top);
    if (mine == top && top != 0) {
      for (int j = lane; j < n; j += 64)
        if (list[j] == top) list[j] = 0;
      mine = best_of_lane();
    }
  }
}

__device__ __forceinline__ int64_t target_of(const LogpArgs& a, int64_t row) {
  return a.target64 ? static_cast<const int64_t*>(a.target)[row]
                    : static_cast<const int32_t*>(a.target)[row];
}

// The target's logit, where log probabilities are wanted; read long before it is used.
template <typename T>
__device__ __forceinline__ float target_logit(const LogpArgs& a, int64_t row, int64_t at) {
  if (!a.log_probs || at < 0 || at >= a.V) return 0.0f;
  return Logits<T>::one(static_cast<const T*>(a.z) + row * a.ldz + at);
}
// A row's results from its sums; rows of nothing but -inf: no alternatives, no entropy.
// at, z: the target and its logit.
__device__ __forceinline__ void write_row(const LogpArgs& a, int64_t row, const Sums& t, float log_s,
                                          int64_t at, float z) {
  const bool dead = t.m == -kInf && t.s == 0.0f;
  const float ent = dead ? 0.0f : log_s - kLn2 * (t.w / t.s);
  if (a.entropy) a.entropy[row] = ent;
  if (a.log_probs) {
    const bool in = at >= 0 && at < a.V;
    a.log_probs[row] = !in ? __uint_as_float(0x7FC00000u) : dead ? -kInf : (z - t.m) * a.inv_t - log_s;
  }
  if (a.stats) {  // log S = inf: p is 0 everywhere
    a.stats[row] = dead ? 0.0f : t.m;
    a.stats[a.T + row] = dead ? kInf : log_s;
    a.stats[2 * a.T + row] = ent;
  }
}
__device__ __forceinline__ void write_pick(const LogpArgs& a, int64_t row, int r, uint64_t key,
                                           const Sums& t, float log_s) {
  const Pick p = pick_of(key);
  const bool bad = !(t.s == t.s);  // a NaN or an infinity among the logits
  a.top_ids[row * a.k + r] = bad ? -1 : p.i;
  a.top_lp[row * a.k + r] =
      bad ? __uint_as_float(0x7FC00000u) : p.i < 0 ? -kInf : (p.v - t.m) * a.inv_t - log_s;
}
__device__ __forceinline__ void write_ignored(const LogpArgs& a, int64_t row, int thread, int threads) {
  if (thread == 0) {
    if (a.entropy) a.entropy[row] = 0.0f;
    if (a.log_probs) a.log_probs[row] = 0.0f;
    if (a.stats) {
      a.stats[row] = a.stats[2 * a.T + row] = 0.0f;
      a.stats[a.T + row] = kInf;
    }
  }
  for (int r = thread; r < a.k; r += threads) {
    a.top_ids[row * a.k + r] = -1;
    a.top_lp[row * a.k + r] = -kInf;
  }
}

// One part of a row (all of it where a.parts is 1).
template <typename T, bool TOP>
__global__ __launch_bounds__(kLogpThreads) void k_logp(LogpArgs a) {
  constexpr int E = Logits<T>::kCount;
  constexpr int kSegLanes = kSeg / E;
  __shared__ Sums parts[kLogpWaves];
  __shared__ float seg_max[TOP ? kMaxSegs : 1];
  __shared__ __attribute__((aligned(16))) uint64_t list[TOP ? kList : 1];
  __shared__ uint16_t segs[TOP ? kMaxSegs : 1];
  __shared__ int counts[2];
  __shared__ float bound, low[4];
  const int64_t row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t target = a.target ? target_of(a, row) : -1;
  if (a.target && target == a.ignore) {
    if (a.parts == 1) write_ignored(a, row, tid, kLogpThreads);
    return;
  }
  const float z_target = a.parts == 1 && tid == 0 ? target_logit<T>(a, row, target) : 0.0f;
  const int64_t first = part * a.part_len;
  const int len = (int)max((int64_t)0, min(a.part_len, a.V - first));
  const T* z = static_cast<const T*>(a.z) + row * a.ldz + first;
  if (TOP && tid < 2) counts[tid] = 0;
  Sums t{-kInf, 0.0f, 0.0f};
  constexpr int kStep = kLogpThreads * E;  // elements of one load of the workgroup
  for (int base = 0; base < len; base += kStep * kAhead) {
    uint4 v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = base + u * kStep + tid * E;
      v[u] = load_logits<T>(z + i, len - i);
    }
    float top = -kInf;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      float m = Logits<T>::get(v[u], 0);
#pragma unroll
      for (int j = 1; j < E; ++j) m = __builtin_fmaxf(m, Logits<T>::get(v[u], j));
      top = __builtin_fmaxf(top, m);
      if (TOP) {
        m = __builtin_fmaxf(m, dpp_mov<0xB1>(m));
        m = __builtin_fmaxf(m, dpp_mov<0x4E>(m));
        m = __builtin_fmaxf(m, dpp_mov<0x141>(m));
        if (kSegLanes == 16) m = __builtin_fmaxf(m, dpp_mov<0x140>(m));
        const int s = (base + u * kStep + tid * E) / kSeg;
        if (lane % kSegLanes == 0 && s * kSeg < len) seg_max[s] = m;
      }
    }
    if (top > t.m) rescale(t, top, a.c);
    const float m = __builtin_fmaxf(t.m, kLowest);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float d = (Logits<T>::get(v[u], j) - m) * a.c;
        const float e = __builtin_amdgcn_exp2f(d);
        t.s += e;
        t.w = __builtin_fmaf(e, __builtin_fmaxf(d, kFar), t.w);
      }
  }
  t = wave_join(t, a.c);
  if (lane == 0) parts[wave] = t;
  __syncthreads();
  t = join_all<kLogpWaves>(parts, a.c);
  const float log_s = logf(t.s);
  uint64_t* out = a.part_top + (row * a.parts + part) * a.k;
  if (tid == 0) {
    if (a.parts == 1) write_row(a, row, t, log_s, target, z_target);
    else a.part_sums[row * a.parts + part] = make_float4(t.m, t.s, t.w, 0.0f);
  }
  if constexpr (TOP) {
    const int nseg = (len + kSeg - 1) / kSeg;
    const auto best_of = [&](int from, int step) {
      float best = -kInf;
      for (int s = from; s < nseg; s += step) best = __builtin_fmaxf(best, seg_max[s]);
      return best;
    };
    float b;
    if (a.k <= kCoarse) {
      if (wave == 0) {
        b = kth_of_lanes(best_of(lane, 64), a.k);
        if (lane == 0) bound = b;
      }
      __syncthreads();
      b = bound;
    } else {
      b = kth_of_group(tid < 256 ? best_of(tid, 256) : -kInf, a.k, reinterpret_cast<float*>(list), low);
    }
    for (int s = tid; s < nseg; s += kLogpThreads)
      if (seg_max[s] >= b && seg_max[s] > -kInf) segs[atomicAdd(&counts[0], 1)] = (uint16_t)s;
    __syncthreads();
    const int n = counts[0];
    constexpr int kSegsAhead = 4;
    for (int q0 = wave; q0 < n; q0 += kLogpWaves * kSegsAhead) {
      float v[kSegsAhead];
      int at[kSegsAhead];
#pragma unroll
      for (int u = 0; u < kSegsAhead; ++u) {
        const int q = q0 + u * kLogpWaves;
        at[u] = q < n ? segs[q] * kSeg + lane : len;
        v[u] = at[u] < len ? Logits<T>::one(z + at[u]) : -kInf;
      }
#pragma unroll
      for (int u = 0; u < kSegsAhead; ++u) {
        const bool in = v[u] >= b && v[u] > -kInf;
        const uint64_t who = __ballot(in);
        if (who == 0) continue;
        int to = 0;
        if (lane == 0) to = atomicAdd(&counts[1], __popcll(who));
        to = __shfl(to, 0) + __popcll(who & ((1ull << lane) - 1));
        if (in && to < kList) list[to] = key_of(v[u], first + at[u]);
      }
    }
    __syncthreads();
    const int found = counts[1];
    const auto give = [&](int r, uint64_t key) {
      if (a.parts == 1) write_pick(a, row, r, key, t, log_s);
      else out[r] = key;
    };
    if (found <= kList) {
      pick_best(list, found, a.k, give);
      return;
    }
    // too many reach the bound: one pass over the part for each of the k
    uint64_t last = ~0ull;
    for (int r = 0; r < a.k; ++r) {
      uint64_t mine = 0;
      for (int i = tid; i < len; i += kLogpThreads) {
        const float v = Logits<T>::one(z + i);
        const uint64_t key = v > -kInf ? key_of(v, first + i) : 0;
        if (key < last) mine = max(mine, key);
      }
      mine = wave_max_key(mine);
      if (lane == 0) list[wave] = mine;
      __syncthreads();
      last = 0;
      for (int w = 0; w < kLogpWaves; ++w) last = max(last, list[w]);
      if (tid == 0) give(r, last);
      __syncthreads();
      if (last == 0) {  // none left
        for (int q = r + 1 + tid; q < a.k; q += kLogpThreads) give(q, 0);
        return;
      }
    }
  }
}

// Joins the parts of a row.
template <typename T>
__global__ __launch_bounds__(256) void k_logp_join(LogpArgs a) {
  __shared__ __attribute__((aligned(16))) uint64_t list[kMaxParts * kMaxTop];
  __shared__ Sums sums;
  __shared__ float bound, low[4];
  __shared__ int count;
  const int64_t row = blockIdx.x;
  const int64_t target = a.target ? target_of(a, row) : -1;
  if (a.target && target == a.ignore) {
    write_ignored(a, row, threadIdx.x, blockDim.x);
    return;
  }
  const float z_target = threadIdx.x == 0 ? target_logit<T>(a, row, target) : 0.0f;
  const int n = (int)a.parts * a.k;
  const uint64_t* from = a.part_top + row * a.parts * a.k;
  constexpr int kOwn = kMaxParts * kMaxTop / 256;
  uint64_t own[kOwn];
#pragma unroll
  for (int u = 0; u < kOwn; ++u) {
    own[u] = 0;
    if (u * 256 < n && u * 256 + (int)threadIdx.x < n) own[u] = from[u * 256 + threadIdx.x];
  }
  // the first candidates of every part (they are in falling order), as many as threads hold
  const int p = (int)(threadIdx.x % (uint32_t)a.parts), r = (int)(threadIdx.x / (uint32_t)a.parts);
  const float best = r < a.k ? pick_of(from[p * a.k + r]).v : -kInf;
  if (threadIdx.x < 64) {  // a lane for each part, at most kMaxParts
    Sums t{-kInf, 0.0f, 0.0f};
    if (threadIdx.x < a.parts) {
      const float4 v = a.part_sums[row * a.parts + threadIdx.x];
      t = Sums{v.x, v.y, v.z};
    }
    t = wave_join(t, a.c);
    const float b = n > 0 && a.k <= kCoarse ? kth_of_lanes(best, a.k) : 0.0f;
    if (threadIdx.x == 0) {
      sums = t;
      bound = b;
      count = 0;
    }
  }
  __syncthreads();
  const Sums t = sums;
  const float log_s = logf(t.s);
  if (threadIdx.x == 0) write_row(a, row, t, log_s, target, z_target);
  if (n == 0) return;
  const float b = a.k <= kCoarse ? bound
                                 : kth_of_group(best, a.k, reinterpret_cast<float*>(list), low);
#pragma unroll
  for (int u = 0; u < kOwn; ++u)  // in any order: the keys order themselves
    if (own[u] != 0 && pick_of(own[u]).v >= b) list[atomicAdd(&count, 1)] = own[u];
  __syncthreads();
  pick_best(list, count, a.k, [&](int r, uint64_t key) { write_pick(a, row, r, key, t, log_s); });
}

// dz of one part of a row.  The elements that were chosen (target, alternatives) are
// written again at the end, after this workgroup's other stores.
constexpr int kGradThreads = 256;
template <typename T>
__global__ __launch_bounds__(kGradThreads) void k_logp_grad(LogpGradArgs a) {
  constexpr int E = Logits<T>::kCount;
  __shared__ int32_t ids[kMaxTop + 1];
  __shared__ float gs[kMaxTop + 1];
  const int64_t row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const int tid = threadIdx.x;
  const int64_t first = part * a.part_len;
  const int len = (int)max((int64_t)0, min(a.part_len, a.V - first));
  const T* z = static_cast<const T*>(a.z) + row * a.ldz + first;
  T* dz = static_cast<T*>(a.dz) + row * a.V + first;
  const int64_t at = !a.target ? -1
                     : a.target64 ? static_cast<const int64_t*>(a.target)[row]
                                  : static_cast<const int32_t*>(a.target)[row];
  const bool ignored = a.target && at == a.ignore;
  const float m = a.stats[row], log_s = a.stats[a.T + row], ent = a.stats[2 * a.T + row];
  const bool none = ignored || log_s == kInf;  // nothing depends on these logits
  // the gradients at chosen tokens
  const int k = a.g_top ? a.k : 0;
  for (int e = tid; e <= k; e += kGradThreads) {
    float g = 0.0f;
    int32_t id = -1;
    if (e == k) {
      if (a.g_lp) {
        g = a.g_lp[row];
        if (at >= 0 && at < a.V) id = (int32_t)at;
        else g = __uint_as_float(0x7FC00000u);  // its log probability is NaN
      }
    } else {
      id = a.top_ids[row * a.k + e];
      g = id >= 0 ? a.g_top[row * a.k + e] : 0.0f;
    }
    ids[e] = id;
    gs[e] = g;
  }
  __syncthreads();
  float sum = 0.0f;
  for (int e = 0; e <= k; ++e) sum += gs[e];
  const float gh = a.g_ent ? a.g_ent[row] : 0.0f;
  // p = 2^((z - m) c - log2 S); -p / T (sum + gh (log p + H)) = p (q + r d), d = (z - m) c - log2 S
  const float shift = log_s * kLog2e;
  const float q = -(sum + gh * ent) * a.inv_t, r = -gh * kLn2 * a.inv_t;
  const auto grad = [&](float x) __attribute__((always_inline)) {
    const float d = __builtin_fmaf(x - m, a.c, -shift);
    return __builtin_amdgcn_exp2f(d) * __builtin_fmaf(r, __builtin_fmaxf(d, kFar), q);
  };
  constexpr int kStep = kGradThreads * E;
  for (int base = 0; base < len; base += kStep * kAhead) {
    uint4 v[kAhead];
    if (!none) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = base + u * kStep + tid * E;
        v[u] = load_logits<T>(z + i, len - i);
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = base + u * kStep + tid * E;
      if (i >= len) continue;
      uint32_t w[4] = {0, 0, 0, 0};
      if (!none) {
#pragma unroll
        for (int j = 0; j < E; j += 2) {
          const float x = grad(Logits<T>::get(v[u], j)), y = grad(Logits<T>::get(v[u], j + 1));
          if constexpr (E == 4) {
            w[j] = __float_as_uint(x);
            w[j + 1] = __float_as_uint(y);
          } else {
            w[j / 2] = pack_bf16x2(x, y);
          }
        }
      }
      T* p = dz + i;
      if (len - i >= E) {
        if ((reinterpret_cast<uintptr_t>(p) & 15u) == 0)
          __builtin_nontemporal_store(u32x4{w[0], w[1], w[2], w[3]}, reinterpret_cast<u32x4*>(p));
        else
          __builtin_memcpy(p, w, 16);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (i + j < len) {
            if constexpr (E == 4) p[j] = __uint_as_float(w[j]);
            else p[j] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
          }
      }
    }
  }
  if (none) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the row's stores, before those of other waves
  __syncthreads();
  for (int e = tid; e <= k; e += kGradThreads) {
    const int64_t i = ids[e] - first;
    if (ids[e] < 0 || i < 0 || i >= len) continue;
    float g = 0.0f;  // the same token may be chosen more than once
    for (int o = 0; o <= k; ++o) g += ids[o] == ids[e] ? gs[o] : 0.0f;
    const float x = __builtin_fmaf(g, a.inv_t, grad(Logits<T>::one(z + i)));
    if constexpr (E == 4) dz[i] = x;
    else dz[i] = (uint16_t)pack_bf16x2(x, 0.0f);
  }
}

// Parts of a row: one where there is a row for each compute unit or rows are short, else as
// many as fill the chip twice over, of kMinPart elements at least; at most kMaxPart (the
// maxima held in LDS) each.  Whole against split, us, without and with 8 alternatives: 256 x
// 131072 bf16 14.9 / 21.8 and 17.5 / 26.1, 128 rows of it 12.8 / 19.9 and 11.4 / 19.4; 16 x
// 65536 7.3 / 12.1 and 7.2 / 13.3, 16 x 32000 4.9 / 8.8 and 7.2 / 13.7; fp32 with 8, 16 x
// 65536 13.6 and 12.4, 16 x 32000 9.3 and 12.6.  Parts of 4096, 8192 and 16384 (16 x 131072
// bf16 with 8): 14.1, 12.2, 12.4.
int64_t logp_part_len(const LogpArgs& a) {
  const int64_t cus = std::max(1, device_cu_count());
  const bool whole = a.T >= cus || a.V * (a.bf16 ? 2 : 4) <= kWholeBytes;
  int64_t parts = whole ? 1 : (2 * cus + a.T - 1) / std::max<int64_t>(a.T, 1);
  parts = std::min(parts, (a.V + kMinPart - 1) / kMinPart);
  parts = std::min<int64_t>(parts, kMaxParts);
  parts = std::max(parts, (a.V + kMaxPart - 1) / kMaxPart);
  // whole runs of 64, and 16-byte aligned parts where the rows are
  const int64_t len = (a.V + parts - 1) / parts;
  return (len + kSeg - 1) / kSeg * kSeg;
}

}  // namespace

int64_t logp_workspace_bytes(const LogpArgs& args) {
  const int64_t len = logp_part_len(args), parts = (args.V + len - 1) / len;
  return parts == 1 ? 0 : args.T * parts * (16 + 8 * (int64_t)args.k);
}

hipError_t launch_logp(LogpArgs a, uint8_t* ws, hipStream_t stream) {
  a.part_len = logp_part_len(a);
  a.parts = (a.V + a.part_len - 1) / a.part_len;
  if (a.parts > 1) {
    a.part_sums = reinterpret_cast<float4*>(ws);
    a.part_top = reinterpret_cast<uint64_t*>(ws + 16 * a.T * a.parts);
  }
  const dim3 grid((unsigned)(a.T * a.parts));
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kLogpThreads), 0, stream, a);
  };
  if (a.bf16) a.k ? go(k_logp<uint16_t, true>) : go(k_logp<uint16_t, false>);
  else a.k ? go(k_logp<float, true>) : go(k_logp<float, false>);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess || a.parts == 1) return err;
  if (a.bf16) hipLaunchKernelGGL(k_logp_join<uint16_t>, dim3((unsigned)a.T), dim3(256), 0, stream, a);
  else hipLaunchKernelGGL(k_logp_join<float>, dim3((unsigned)a.T), dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_logp_grad(LogpGradArgs a, hipStream_t stream) {
  a.part_len = 16384;
  a.parts = (a.V + a.part_len - 1) / a.part_len;
  const dim3 grid((unsigned)(a.T * a.parts));
  if (a.bf16) hipLaunchKernelGGL(k_logp_grad<uint16_t>, grid, dim3(kGradThreads), 0, stream, a);
  else hipLaunchKernelGGL(k_logp_grad<float>, grid, dim3(kGradThreads), 0, stream, a);
  return hipGetLastError();
}

bool logp_fits(int64_t tokens, int64_t vocab) {
  LogpArgs a{};
  a.T = tokens;
  a.V = vocab;
  if (vocab > kMaxPart * kMaxParts || tokens >= INT64_C(1) << 23) return false;
  const int64_t len = logp_part_len(a), parts = (vocab + len - 1) / len;
  return tokens * parts < INT64_C(1) << 23 && tokens * ((vocab + 16383) / 16384) < INT64_C(1) << 24;
}

}  // namespace mxgg
