// Routing decision of a MoE layer: which experts every token goes to, with
// which weights, and the gradient of the weights with respect to the logits.
//
//   s = 1 / (1 + exp(-x))  or  softmax(x) over the token's experts (fp32)
//   c = s + bias; without a bias c = x, which orders experts as s does
//   groups of experts/groups consecutive experts: a group's worth is its best c,
//   or the sum of its two best s (+ bias); the top_groups best groups stay
//   the topk experts of largest c in them, largest first, ties (also between
//   groups) to the lowest index; a NaN c ranks above every number
//   weights: scale * s, or scale * s / (sum of the selected s); for softmax the
//   latter is the softmax over the selected logits alone (the row's sum cancels)
// An expert with c = -inf (or x = -inf) is out of the choice; a slot that no
// expert is left for gets id -1 and weight 0.
//
// Selection: c becomes a double with the expert's index in the mantissa bits that an
// fp32 value leaves zero: one v_max_f64 then compares value and index together, at
// the full rate of the vector unit, and no two keys are equal.  A token is held by 2^k lanes of VPL experts each; every
// lane sorts its keys in registers down to the L largest and log2(lanes)
// butterfly steps merge the sorted lists (L max and a bitonic clean each).
//
// 131072 tokens, 256 fp32 experts in 8 groups, sigmoid and bias: 52 us, 134 MB read at
// 2.6 TB/s; bound by the vector unit, busy for 45 of them: sigmoids, keys and sorting
// networks take about as much each.  One
// token: 5.2 us, a launch and its chain of dependent steps.  The gradient writes every
// logit's and reads the chosen ones: 27 us, 5 TB/s.
#include <algorithm>

#include "mx_device.h"
#include "mxgg_internal.h"

namespace mxgg {
namespace {

constexpr int kTopkThreads = 256;
constexpr int kTopkWaves = kTopkThreads / 64;
constexpr int kGradTile = 2048;  // gradients of a wave's tile, at most
constexpr int kGradSlots = 128;  // and slots

// LDS index with one word of padding every 32: lanes that walk rows of 32 words
// in step fall on different banks.
__host__ __device__ constexpr int pad32(int i) { return i + (i >> 5); }

// LDS writes of this wave's lanes before, reads of other lanes' words after.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

constexpr float kNegInf = -__builtin_inff();

__device__ __forceinline__ double join_f64(uint32_t lo, uint32_t hi) {
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ uint32_t low_word(double v) {
  return (uint32_t)__builtin_bit_cast(uint64_t, v);
}
__device__ __forceinline__ uint32_t high_word(double v) {
  return (uint32_t)(__builtin_bit_cast(uint64_t, v) >> 32);
}
// A key: an fp32 value as a double, with the index in the ten lowest mantissa bits,
// which are zero in every such double; turned over so that the lower index is the
// larger of two equal values, above and below zero.  Infinities and NaN become the
// numbers +-2^1022 and 2^1023, so that keys are ordered and none is a NaN; an absent
// one is -2^1023, below every key whatever its low word holds.
constexpr uint32_t kIndexMask = 1023u;
static_assert(kMaxGroups <= (int)kIndexMask + 1, "an expert index takes ten bits");
constexpr uint32_t kNanHigh = 0x7FE00000u, kAbsentHigh = 0xFFE00000u;
__device__ __forceinline__ uint32_t turned(uint32_t idx, uint32_t high) {
  return ((kIndexMask - idx) ^ (uint32_t)((int32_t)high >> 31)) & kIndexMask;
}
__device__ __forceinline__ double finite_key(float v, uint32_t idx) {
  const double d = v;
  return join_f64(low_word(d) | turned(idx, high_word(d)), high_word(d));
}
__device__ __forceinline__ double any_key(float v, uint32_t idx) {
  const double d = v;
  uint32_t high = high_word(d);
  high = __builtin_fabsf(v) == __builtin_inff() ? high - 0x00200000u : high;
  high = v != v ? kNanHigh : high;
  return join_f64((v != v ? 0u : low_word(d)) | turned(idx, high), high);
}
__device__ __forceinline__ double with_index(double key, uint32_t idx) {
  return join_f64((low_word(key) & ~kIndexMask) | turned(idx, high_word(key)), high_word(key));
}
__device__ __forceinline__ float value_of(double key) {
  const float v = (float)join_f64(low_word(key) & ~kIndexMask, high_word(key));
  return high_word(key) == kNanHigh ? __builtin_nanf("") : v;
}
__device__ __forceinline__ int index_of(double key) {
  return (int)turned(low_word(key) & kIndexMask, high_word(key));
}
__device__ __forceinline__ bool absent(double key) { return high_word(key) == kAbsentHigh; }
__device__ __forceinline__ double absent_if(bool out, double key) {
  return join_f64(low_word(key), out ? kAbsentHigh : high_word(key));
}

// Plain v_max_f64 / v_min_f64: the keys are ordinary numbers, so the
// canonicalising steps that fmax would add are left out.
__device__ __forceinline__ double dmax(double a, double b) {
  double r;
  asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ double dmin(double a, double b) {
  double r;
  asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ void exchange(double& hi, double& lo) {
  const double a = dmax(hi, lo);
  lo = dmin(hi, lo);
  hi = a;
}

// Batcher's odd-even merge sort of a[LO .. LO + N), descending: N = 8 takes 19
// exchanges, 16 63, 32 191.
template <int LO, int N, int R, int TOTAL>
__device__ __forceinline__ void merge_net(double (&a)[TOTAL]) {
  if constexpr (2 * R < N) {
    merge_net<LO, N, 2 * R>(a);
    merge_net<LO + R, N, 2 * R>(a);
#pragma unroll
    for (int i = LO + R; i + R < LO + N; i += 2 * R) exchange(a[i], a[i + R]);
  } else {
    exchange(a[LO], a[LO + R]);
  }
}
template <int LO, int N, int TOTAL>
__device__ __forceinline__ void sort_net(double (&a)[TOTAL]) {
  if constexpr (N > 1) {
    sort_net<LO, N / 2>(a);
    sort_net<LO + N / 2, N / 2>(a);
    merge_net<LO, N, 1>(a);
  }
}
// The L largest of two descending lists, descending.
template <int L>
__device__ __forceinline__ void merge_top(double (&a)[L], const double (&b)[L]) {
#pragma unroll
  for (int i = 0; i < L; ++i) a[i] = dmax(a[i], b[L - 1 - i]);
#pragma unroll
  for (int k = L / 2; k >= 1; k >>= 1)
#pragma unroll
    for (int i = 0; i < L; ++i)
      if ((i & k) == 0) exchange(a[i], a[i + k]);
}

__device__ __forceinline__ double shfl_xor_f64(double v, int off) {
  return join_f64((uint32_t)__shfl_xor((int)low_word(v), off),
                  (uint32_t)__shfl_xor((int)high_word(v), off));
}
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  return join_f64((uint32_t)__builtin_amdgcn_mov_dpp((int)low_word(v), CTRL, 0xF, 0xF, false),
                  (uint32_t)__builtin_amdgcn_mov_dpp((int)high_word(v), CTRL, 0xF, 0xF, false));
}

// The list of the L largest over this lane's run of `off` lanes, which all hold the
// run's list, and the run beside it.  Any lane of the other run will do as the
// partner: within 16 lanes a DPP mirror (VALU only) reaches one.
template <int L>
__device__ __forceinline__ void merge_lanes(double (&a)[L], int off) {
  double b[L];
  if (off == 1) {
#pragma unroll
    for (int i = 0; i < L; ++i) b[i] = dpp_f64<0xB1>(a[i]);   // quad_perm [1,0,3,2]
  } else if (off == 2) {
#pragma unroll
    for (int i = 0; i < L; ++i) b[i] = dpp_f64<0x4E>(a[i]);   // quad_perm [2,3,0,1]
  } else if (off == 4) {
#pragma unroll
    for (int i = 0; i < L; ++i) b[i] = dpp_f64<0x141>(a[i]);  // row_half_mirror
  } else if (off == 8) {
#pragma unroll
    for (int i = 0; i < L; ++i) b[i] = dpp_f64<0x140>(a[i]);  // row_mirror
  } else {
#pragma unroll
    for (int i = 0; i < L; ++i) b[i] = shfl_xor_f64(a[i], off);
  }
  merge_top<L>(a, b);
}

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }
constexpr float kSigmoidZero = -88.72284f;  // expf(-x) overflows below: the result is 0

// The same bits for |x| <= 87: no range tests in the exponential, and one Newton
// step on v_rcp_f32 for the quotient, which returns the correctly rounded 1 / d for
// every mantissa of d (compared with the division once for all 2^23 of them, and at other
// exponents; tests/test_gpu_route_precision.py ranks four million logits, neighbours of
// each other, by both sequences).
constexpr float kModerate = 87.0f;
__device__ __forceinline__ float reciprocal(float d) {
  const float r = __builtin_amdgcn_rcpf(d);
  return __builtin_fmaf(__builtin_fmaf(-r, d, 1.0f), r, r);
}
__device__ __forceinline__ float sigmoid_moderate(float x) {
  return reciprocal(1.0f + exp_moderate(-x));
}

__device__ __forceinline__ float load_one(const float* p) { return *p; }
__device__ __forceinline__ float load_one(const uint16_t* p) { return bf16_bits_to_f32(*p); }
__device__ __forceinline__ void store_one(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_one(uint16_t* p, float v) {
  *p = (uint16_t)pack_bf16x2(v, 0.0f);
}

// Four consecutive values, at any alignment of an element.
struct RawF32 {
  float v[4];
  __device__ __forceinline__ void load(const float* p) { __builtin_memcpy(v, p, 16); }
  __device__ __forceinline__ float get(int i) const { return v[i]; }
};
struct RawBf16 {
  uint32_t v[2];
  __device__ __forceinline__ void load(const uint16_t* p) { __builtin_memcpy(v, p, 8); }
  __device__ __forceinline__ float get(int i) const {
    return (i & 1) ? bf16_hi(v[i >> 1]) : bf16_lo(v[i >> 1]);
  }
};
__device__ __forceinline__ RawF32 raw4(const float*) { return RawF32{}; }
__device__ __forceinline__ RawBf16 raw4(const uint16_t*) { return RawBf16{}; }
__device__ __forceinline__ void store4(float* p, const float4& q) { __builtin_memcpy(p, &q, 16); }
__device__ __forceinline__ void store4(uint16_t* p, const float4& q) {
  const uint32_t w[2] = {pack_bf16x2(q.x, q.y), pack_bf16x2(q.z, q.w)};
  __builtin_memcpy(p, w, 8);
}

// n <= MAX consecutive logits into a wave's padded LDS tile: all loads first.
template <int MAX, typename T>
__device__ __forceinline__ void load_tile(const T* __restrict__ x, int n, float* tile) {
  const int lane = threadIdx.x & 63;
  constexpr int kLoads = (MAX + 255) / 256;
  decltype(raw4(x)) c[kLoads];
#pragma unroll
  for (int j = 0; j < kLoads; ++j) {
    const int i = 4 * (lane + 64 * j);
    if (i + 4 <= n) c[j].load(x + i);
  }
#pragma unroll
  for (int j = 0; j < kLoads; ++j) {
    const int i = 4 * (lane + 64 * j);
    if (i + 4 <= n) {
#pragma unroll
      for (int u = 0; u < 4; ++u) tile[pad32(i) + u] = c[j].get(u);  // within one run of 32
    } else {
      for (int u = i; u < n; ++u) tile[pad32(u)] = load_one(x + u);
    }
  }
}

// p / K for p < 2048 and K <= 32, from recip = ceil(2^20 / K).
__device__ __forceinline__ int div_k(int p, uint32_t recip) {
  return (int)(((uint32_t)p * recip) >> 20);
}

// A wave's share of the workgroup's LDS, in words.
struct TopkLds {
  int ids, values, stats, words;
  __host__ __device__ TopkLds(int E, int K, int tokens) {
    ids = pad32(tokens * E);
    values = ids + tokens * K;
    stats = (values + tokens * K + 1) & ~1;
    words = stats + 2 * tokens;
  }
};

template <int VPL, int L, typename T>
__global__ __launch_bounds__(kTopkThreads) void k_route_topk(RouteTopkArgs a) {
  static_assert(VPL >= L, "a lane's list is cut from its own experts");
  extern __shared__ float lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int per_wave = 64 / a.lanes;
  const int64_t t0 = ((int64_t)blockIdx.x * kTopkWaves + wave) * per_wave;
  const int nt = (int)std::min<int64_t>(per_wave, std::max<int64_t>(0, a.tokens - t0));
  // of every wave: its logits, then the slots' ids and values and (max, sum) of a
  // token's softmax; the bias behind the waves
  const TopkLds at(a.E, a.K, per_wave);
  float* tile = lds + wave * at.words;
  int32_t* pk = reinterpret_cast<int32_t*>(tile + at.ids);
  float* val = tile + at.values;
  float2* stats = reinterpret_cast<float2*>(tile + at.stats);
  float* bias_s = lds + kTopkWaves * at.words;
  load_tile<64 * VPL, T>(static_cast<const T*>(a.logits) + t0 * a.E, nt * a.E, tile);
  __shared__ uint32_t odd_s[kTopkWaves];  // whether a wave's part of the bias is infinite or NaN
  if (a.bias != nullptr) {
    uint32_t most = 0;
    for (int e = tid; e < a.E; e += kTopkThreads) {
      const float b = a.bias[e];
      most = max(most, __float_as_uint(b) & 0x7FFFFFFFu);
      bias_s[pad32(e)] = b;
    }
    const bool odd = __any(most >= 0x7F800000u);
    if (lane == 0) odd_s[wave] = odd;
  }
  __syncthreads();
  if (nt == 0) return;

  // this lane's experts: VPL of group g, from offset o in it
  const int tok = lane / a.lanes, sub = lane & (a.lanes - 1);
  const int per = a.E / a.groups;
  const int g = sub / a.lanes_group, o = (sub & (a.lanes_group - 1)) * VPL;
  const int count = tok < nt && g < a.groups ? min(max(per - o, 0), VPL) : 0;
  const int e0 = g * per + o;
  // Where every lane has VPL experts or none, on the padding's grid, their words
  // follow each other: no address or test per expert (131072 x 256: 66 -> 55 us).
  const bool whole = per % VPL == 0 && a.E % 32 == 0;
  const int word0 = count > 0 ? pad32(tok * a.E + e0) : 0;
  float x[VPL];
  if (whole) {
#pragma unroll
    for (int v = 0; v < VPL; ++v) x[v] = tile[word0 + v];
    if (count == 0) {
#pragma unroll
      for (int v = 0; v < VPL; ++v) x[v] = kNegInf;
    }
  } else {
#pragma unroll
    for (int v = 0; v < VPL; ++v) x[v] = v < count ? tile[pad32(tok * a.E + e0 + v)] : kNegInf;
  }

  // softmax statistics of the whole row, where the choice or the weights need them
  float top = 0.0f, total = 1.0f;
  const bool sums = a.groups > 1 && a.group_best == 2;
  if (a.softmax && (a.bias != nullptr || !a.renorm || sums)) {
    top = kNegInf;
#pragma unroll
    for (int v = 0; v < VPL; ++v) top = __builtin_fmaxf(top, x[v]);
    for (int off = 1; off < a.lanes; off <<= 1) top = __builtin_fmaxf(top, __shfl_xor(top, off));
    if (top == kNegInf) top = 0.0f;
    // in runs of 8 and then by pairs, as lanes of 8 experts each add them: a token's
    // scores, and so a choice that goes by them, do not depend on the experts a lane
    static_assert(VPL == 8 || VPL == 32, "a power of two of runs");
    float run[VPL / 8];
#pragma unroll
    for (int r = 0; r < VPL / 8; ++r) {
      run[r] = 0.0f;
#pragma unroll
      for (int v = 8 * r; v < 8 * r + 8; ++v) run[r] += expf(x[v] - top);
    }
#pragma unroll
    for (int w = 1; w < VPL / 8; w *= 2)
#pragma unroll
      for (int r = 0; r < VPL / 8; r += 2 * w) run[r] += run[r + w];
    total = run[0];
    for (int off = 1; off < a.lanes; off <<= 1) total += __shfl_xor(total, off);
    if (total == 0.0f) total = 1.0f;  // every expert is out
    if (sub == 0 && tok < nt) stats[tok] = make_float2(top, total);
  }

  // choice keys, and the L largest of the lane
  double list[L];
  {
    // Most waves hold no infinity or NaN (nor, where a sigmoid is taken, a logit past
    // 87): the largest bit patterns, signed and not, say so for 32 experts in 32
    // operations, and such keys take 5 operations instead of 12 (131072 x 256: 55 -> 52
    // us).  A lane without experts is put right after the sort.
    int32_t high = 0;
    uint32_t low = 0;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      high = max(high, (int32_t)__float_as_uint(x[v]));
      low = max(low, __float_as_uint(x[v]));
    }
    const bool sigmoids = a.bias != nullptr && !a.softmax;
    const uint32_t bound = sigmoids ? __float_as_uint(kModerate) : 0x7F7FFFFFu;
    bool usual = __all(count == 0 || ((uint32_t)high <= bound && low <= (bound | 0x80000000u)));
    if (a.bias != nullptr)
#pragma unroll
      for (int w = 0; w < kTopkWaves; ++w) usual &= odd_s[w] == 0u;
    float c[VPL];
#pragma unroll
    for (int v = 0; v < VPL; ++v) c[v] = x[v];
    if (a.bias != nullptr) {
      if (a.softmax) {
#pragma unroll
        for (int v = 0; v < VPL; ++v) c[v] = expf(x[v] - top) / total;
      } else if (usual) {
#pragma unroll
        for (int v = 0; v < VPL; ++v) c[v] = sigmoid_moderate(x[v]);
      } else {
#pragma unroll
        for (int v = 0; v < VPL; ++v) c[v] = sigmoid(x[v]);
      }
      if (whole) {
        const float* bias = bias_s + (count > 0 ? pad32(e0) : 0);
#pragma unroll
        for (int v = 0; v < VPL; ++v) c[v] += bias[v];
      } else {
#pragma unroll
        for (int v = 0; v < VPL; ++v) c[v] += bias_s[pad32(min(e0 + v, a.E - 1))];
      }
    }
    double key[VPL];
    if (usual) {
#pragma unroll
      for (int v = 0; v < VPL; ++v) key[v] = finite_key(c[v] + 0.0f, (uint32_t)(e0 + v));
    } else {
#pragma unroll
      for (int v = 0; v < VPL; ++v)
        key[v] = absent_if(x[v] == kNegInf || c[v] == kNegInf,
                           any_key(c[v] + 0.0f, (uint32_t)(e0 + v)));
    }
#pragma unroll
    for (int i = 0; i < L; ++i) list[i] = key[i];
    sort_net<0, L>(list);
#pragma unroll
    for (int v0 = L; v0 < VPL; v0 += L) {
      double more[L];
#pragma unroll
      for (int i = 0; i < L; ++i) more[i] = key[v0 + i];
      sort_net<0, L>(more);
      merge_top<L>(list, more);
    }
#pragma unroll
    for (int i = 0; i < L; ++i) list[i] = absent_if(count == 0, list[i]);
  }
  for (int off = 1; off < a.lanes_group; off <<= 1) merge_lanes<L>(list, off);

  // groups: the list now holds the group's best; rank its worth among the token's
  if (a.groups > 1) {
    double mine = with_index(list[0], (uint32_t)g);
    if (sums) {
      float w[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        w[i] = value_of(list[i]);
        if (a.bias == nullptr) w[i] = a.softmax ? expf(w[i] - top) / total : sigmoid(w[i]);
        if (absent(list[i])) w[i] = 0.0f;
      }
      mine = any_key(w[0] + w[1] + 0.0f, (uint32_t)g);
    }
    mine = absent_if(absent(list[0]), mine);
    int above = 0;
    for (int off = a.lanes_group; off < a.lanes; off += a.lanes_group)
      above += shfl_xor_f64(mine, off) > mine ? 1 : 0;
    if (above >= a.top_groups) {
#pragma unroll
      for (int i = 0; i < L; ++i) list[i] = absent_if(true, list[i]);
    }
    for (int off = a.lanes_group; off < a.lanes; off <<= 1) merge_lanes<L>(list, off);
  }

  // weights: one (token, slot) a lane, sums over a token's slots in slot order
  if (sub == 0 && tok < nt) {
#pragma unroll
    for (int i = 0; i < L; ++i)
      if (i < a.K) pk[tok * a.K + i] = absent(list[i]) ? -1 : index_of(list[i]);
  }
  wave_sync();
  const int slots = nt * a.K;
  for (int p = lane; p < slots; p += 64) {
    const int t = div_k(p, a.k_recip), e = pk[p];
    const float* row_x = tile;
    float s = 0.0f, xe = 0.0f;
    if (e >= 0) {
      xe = row_x[pad32(t * a.E + e)];
      if (!a.softmax) {
        s = sigmoid(xe);
      } else if (!a.renorm) {
        s = expf(xe - stats[t].x) / stats[t].y;
      } else {
        // relative to the largest selected logit: the first slot's without a bias
        float m = row_x[pad32(t * a.E + pk[t * a.K])];
        if (a.bias != nullptr)
          for (int j = 1; j < a.K; ++j) {
            const int ej = pk[t * a.K + j];
            if (ej >= 0) m = __builtin_fmaxf(m, row_x[pad32(t * a.E + ej)]);
          }
        s = expf(xe - m);
      }
    }
    val[p] = s;
    // for the gradient the logit: a score that is 1 to the last bit has lost its slope
    if (a.sel != nullptr && !a.softmax) a.sel[t0 * a.K + p] = xe;
  }
  wave_sync();
  for (int p = lane; p < slots; p += 64) {
    const int t = div_k(p, a.k_recip);
    float w = val[p], s = w;
    if (a.renorm) {
      float sum = 0.0f;
      for (int j = 0; j < a.K; ++j) sum += val[t * a.K + j];
      w = sum == 0.0f ? 0.0f : w / sum;
      if (a.softmax) s = w;
    }
    const int64_t at = t0 * a.K + p;
    a.idx[at] = pk[p];
    a.weights[at] = a.scale * w;
    if (a.sel != nullptr && a.softmax) a.sel[at] = s;
  }
}

// Gradient of the weights: dw [tokens][K] -> d logits [tokens][E].
//   sigmoid        : dx = ds sigma(x) sigma(-x), zero for experts not selected
//   softmax, renorm: dx = p (dp - sum p dp) over the selected, zero elsewhere
//   softmax alone  : dx = p (dp - sum p dp) over the whole row (p from the logits)
// with ds = scale dw, or scale (dw - sum dw s / S) / S where s is divided by its
// sum S over the slots.  A wave takes NT whole tokens: the rows are put together
// in LDS from the slots and leave as one run of memory.
template <typename T>
__global__ __launch_bounds__(kTopkThreads) void k_route_topk_grad(RouteTopkGradArgs a) {
  __shared__ float grad_s[kTopkWaves][kGradTile];
  __shared__ float2 slot_s[kTopkWaves][kGradSlots];  // (s, s dw) of a slot
  __shared__ float slope_s[kTopkWaves][kGradSlots];  // ds / dx of a sigmoid
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t t0 = ((int64_t)blockIdx.x * kTopkWaves + wave) * a.tokens_wave;
  const int nt = (int)std::min<int64_t>(a.tokens_wave, std::max<int64_t>(0, a.tokens - t0));
  if (nt == 0) return;
  float* grad = grad_s[wave];
  float2* slot = slot_s[wave];
  float* slope = slope_s[wave];
  const int n = nt * a.E, slots = nt * a.K;
  const int32_t* idx = a.idx + t0 * a.K;
  const float* sel = a.sel + t0 * a.K;
  const float* dw = a.dweights + t0 * a.K;
  for (int p = lane; p < slots; p += 64) {  // slots without an expert add nothing
    const bool live = (uint32_t)idx[p] < (uint32_t)a.E;
    float s = live ? sel[p] : 0.0f;
    if (!a.softmax) {  // from the logit, without 1 - s
      const float e = expf(-__builtin_fabsf(s)), r = reciprocal(1.0f + e);
      slope[p] = e * r * r;
      s = !live || s < kSigmoidZero ? 0.0f : s < 0.0f ? e * r : r;
    }
    slot[p] = make_float2(s, live ? s * dw[p] : 0.0f);
  }
  for (int i = 4 * lane; i < n; i += 256)
    *reinterpret_cast<float4*>(grad + i) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  wave_sync();
  for (int p = lane; p < slots; p += 64) {
    const int t = div_k(p, a.k_recip), e = idx[p];
    if ((uint32_t)e >= (uint32_t)a.E) continue;
    float dot = 0.0f, sum = 0.0f;
    if (a.renorm)
      for (int j = 0; j < a.K; ++j) {
        sum += slot[t * a.K + j].x;
        dot += slot[t * a.K + j].y;
      }
    const float s = slot[p].x, d = dw[p];
    float g;
    if (a.softmax)
      g = a.scale * (a.renorm ? s * (d - dot) : d);
    else if (a.renorm)
      g = sum == 0.0f ? 0.0f : a.scale * (d - dot / sum) / sum * slope[p];
    else
      g = a.scale * d * slope[p];
    grad[t * a.E + e] = g;
  }
  wave_sync();
  if (a.softmax && !a.renorm) {
    const int lanes = 64 / a.tokens_wave, t = lane / lanes, sub = lane & (lanes - 1);
    const T* x = static_cast<const T*>(a.logits) + (t0 + t) * a.E;
    if (t < nt) {
      float top = kNegInf, total = 0.0f, dot = 0.0f;
      for (int e = sub; e < a.E; e += lanes) top = __builtin_fmaxf(top, load_one(x + e));
      for (int off = 1; off < lanes; off <<= 1) top = __builtin_fmaxf(top, __shfl_xor(top, off));
      if (top == kNegInf) top = 0.0f;
      for (int e = sub; e < a.E; e += lanes) total += expf(load_one(x + e) - top);
      for (int off = 1; off < lanes; off <<= 1) total += __shfl_xor(total, off);
      if (total == 0.0f) total = 1.0f;
      for (int j = 0; j < a.K; ++j) dot += a.scale * slot[t * a.K + j].y;
      for (int e = sub; e < a.E; e += lanes) {
        const float p = expf(load_one(x + e) - top) / total;
        grad[t * a.E + e] = p * (grad[t * a.E + e] - dot);
      }
    }
    wave_sync();
  }
  T* out = static_cast<T*>(a.dlogits) + t0 * a.E;
  for (int i = 4 * lane; i < n; i += 256) {
    if (i + 4 <= n)
      store4(out + i, *reinterpret_cast<const float4*>(grad + i));
    else
      for (int u = i; u < n; ++u) store_one(out + u, grad[u]);
  }
}

int next_pow2(int v) {
  int p = 1;
  while (p < v) p <<= 1;
  return p;
}

// Lanes of a group and of a token.  Longer lists take more lanes, so fewer tokens
// and slots a wave: the LDS of a workgroup stays below 64 KB.
template <int VPL, int L>
void set_lanes(RouteTopkArgs& a) {
  const int per = a.E / a.groups, groups = next_pow2(a.groups);
  a.lanes_group = std::max(next_pow2((per + VPL - 1) / VPL), L / 8 / groups);
  a.lanes = a.lanes_group * groups;
}

template <int VPL, int L, typename T>
hipError_t run_topk(RouteTopkArgs a, hipStream_t stream) {
  set_lanes<VPL, L>(a);
  const int64_t tokens = (int64_t)kTopkWaves * (64 / a.lanes);
  const int words = kTopkWaves * TopkLds(a.E, a.K, 64 / a.lanes).words + (a.bias ? pad32(a.E) : 0);
  hipLaunchKernelGGL((k_route_topk<VPL, L, T>), dim3((unsigned)((a.tokens + tokens - 1) / tokens)),
                     dim3(kTopkThreads), 4 * words, stream, a);
  return hipGetLastError();
}

// Lists of the smallest length that holds topk, cut from 32 experts a lane (32
// lanes hold 1024).  Few tokens take 8 experts a lane where 64 lanes hold them: more
// waves of less work, as long as 32 a lane leave a SIMD without a wave.  256 experts
// in 8 groups, 32 / 8 a lane, us: 1 token 6.8 / 5.2, 4096 7.7 / 7.3, 8192 (a wave a
// SIMD) 7.9 / 9.6, 131072 52 / 86; 32 experts: 32768 tokens 8.5 / 5.7, 65536 (a wave a
// SIMD) 8.8 / 7.4, 131072 10.8 / 11.4.
template <typename T>
hipError_t run_topk_list(RouteTopkArgs a, hipStream_t stream) {
  if (a.K <= 8) {
    set_lanes<32, 8>(a);
    const int64_t waves = (a.tokens * a.lanes + 63) / 64;
    set_lanes<8, 8>(a);
    if (a.lanes <= 64 && waves < 4 * std::max(1, device_cu_count()))
      return run_topk<8, 8, T>(a, stream);
    return run_topk<32, 8, T>(a, stream);
  }
  if (a.K <= 16) return run_topk<32, 16, T>(a, stream);
  return run_topk<32, 32, T>(a, stream);
}

}  // namespace

hipError_t launch_route_topk(RouteTopkArgs a, hipStream_t stream) {
  if (a.tokens == 0) return hipSuccess;
  a.k_recip = (uint32_t)(((1u << 20) + a.K - 1) / a.K);
  return a.bf16 ? run_topk_list<uint16_t>(a, stream) : run_topk_list<float>(a, stream);
}

hipError_t launch_route_topk_grad(RouteTopkGradArgs a, hipStream_t stream) {
  if (a.tokens == 0) return hipSuccess;
  a.k_recip = (uint32_t)(((1u << 20) + a.K - 1) / a.K);
  // whole tokens a wave, a power of two: as many as its LDS tile holds, and about a
  // slot for every lane (16384 x 32, top-8: 64 tokens a wave 17.0 us, 8 tokens 3.7)
  a.tokens_wave = next_pow2((64 + a.K - 1) / a.K);
  while (a.tokens_wave * a.E > kGradTile) a.tokens_wave >>= 1;
  const int64_t tokens = (int64_t)kTopkWaves * a.tokens_wave;
  const dim3 grid((unsigned)((a.tokens + tokens - 1) / tokens));
  if (a.bf16)
    hipLaunchKernelGGL((k_route_topk_grad<uint16_t>), grid, dim3(kTopkThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((k_route_topk_grad<float>), grid, dim3(kTopkThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace mxgg
