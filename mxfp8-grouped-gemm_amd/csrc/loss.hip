// Softmax cross entropy of a linear layer, z = x W^T (bf16 operands), without the
// logits z [tokens, vocab] ever being kept.
//
//   loss[t] = lse[t] - z[t][target[t]],   lse[t] = log sum_v exp(z[t][v])
//   d[t][v] = (exp(z[t][v] - lse[t]) - [v = target[t]]) g[t]
//   dx = d W,   dW = d^T x        (g: the loss's gradient per token, 0 where ignored)
//
// Forward: 256 (vocabulary) x 256 (token) tiles of z on the matrix cores; every
// tile leaves one maximum and one sum of exponentials a token, joined over the
// tiles by a second kernel.
// Backward: pieces of the vocabulary.  The tiles of a piece are computed again
// (8 T H V operations in all, 6 with kept logits) and leave d rounded to bf16,
// as d [T][piece] and as d^T [piece][T]; with W^T of the piece and x^T (plain
// transposes) both products then run with operands that are contiguous along
// their contraction.  Rounding d is one bf16 rounding per term of sums whose
// result is rounded to bf16 anyway.  dx is carried over pieces in fp32.
// Few output tiles are split along the contraction, and the fp32 partials added
// in order.
#include <algorithm>

#include "gemm_tile.h"

namespace mxgg {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kTile = 256;

struct __align__(16) LossSmem {
  uint8_t ring[2][kStageBytes];
};

// Rows row0 .. of a bf16 matrix as a tile operand, `cols` of them contiguous.
__device__ __forceinline__ Operand tile_rows(const uint16_t* p, int64_t ld, int64_t row0,
                                             int64_t rows, int64_t cols) {
  const int64_t n = std::min<int64_t>(kTile, rows - row0);
  Operand o;
  o.data = make_desc(p + row0 * ld, (uint32_t)(((n - 1) * ld + cols) * 2));
  o.scale = o.data;  // not read
  o.ld = (uint32_t)(ld * 2);
  o.lds = 0;
  o.row0 = 0;
  o.hi = 128;
  return o;
}

// Tile of a workgroup.  Workgroups go round-robin to the 8 XCDs: each XCD takes a
// contiguous run of tiles in an order of bands of 8 token tiles, so the 32 tiles
// it works on at a time share 8 + 4 operand panels in its L2.
__device__ __forceinline__ void tile_of(int np, int nq, int& p, int& q) {
  const int total = np * nq, per = total / 8, rest = total % 8;
  const int xcd = (int)blockIdx.x % 8, slot = (int)blockIdx.x / 8;
  const int n = xcd * per + min(xcd, rest) + slot;
  const int band = n / (8 * np), in = n - band * 8 * np;
  const int width = min(8, nq - band * 8);
  p = in / width;
  q = band * 8 + in % width;
}

// This lane's place in a wave's 128 x 128 part of a tile: accumulator
// 8 (4G + i) + 4H + j, register r, is P index 128 wp + 64 G + 16 g + 4 r + i and
// Q index 128 wq + 64 H + 4 c + j.
struct Place {
  int wp, wq, g, c;
  __device__ __forceinline__ Place() {
    const int lane = threadIdx.x & 63, wave = (int)wave_id();
    wp = wave & 1;
    wq = wave >> 1;
    g = lane >> 4;
    c = lane & 15;
  }
  __device__ __forceinline__ int p(int G, int r, int i) const {
    return 128 * wp + 64 * G + 16 * g + 4 * r + i;
  }
  __device__ __forceinline__ int q(int H, int j) const { return 128 * wq + 64 * H + 4 * c + j; }
};

// Target of token t: its word, -1 = ignored, -2 = outside the vocabulary.
__device__ __forceinline__ int64_t target_of(const LossArgs& a, int64_t t) {
  const int64_t v = a.target64 ? static_cast<const int64_t*>(a.target)[t]
                               : (int64_t) static_cast<const int32_t*>(a.target)[t];
  return v == a.ignore_index ? -1 : v >= 0 && v < a.V ? v : -2;
}

// Statistics of a tile: part[p tile][t] = (max, sum of exp(z - max)) over the
// tile's words, and the target's logit.
__global__ __launch_bounds__(kThreads, 1) void k_loss_fwd(LossArgs a) {
  __shared__ LossSmem sm;
  const int np = (int)((a.V + kTile - 1) / kTile), nq = (int)((a.T + kTile - 1) / kTile);
  int pt, qt;
  tile_of(np, nq, pt, qt);
  const int64_t p0 = (int64_t)pt * kTile, q0 = (int64_t)qt * kTile;
  const Operand P = tile_rows(a.w, a.ldw, p0, a.V, a.H);
  const Operand Q = tile_rows(a.x, a.ldx, q0, a.T, a.H);
  v4f acc[64];
  mainloop<false, false, false, true>(sm, P, Q, 0u, (uint32_t)(2 * a.H), acc);

  const Place at;
  const int words = (int)std::min<int64_t>(kTile, a.V - p0);
  if (words < kTile) {  // past the vocabulary: no word
#pragma unroll
    for (int k = 0; k < 64; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (at.p(k >> 5, r, (k >> 3) & 3) >= words) acc[k][r] = -__builtin_inff();
  }
  float2* joined = reinterpret_cast<float2*>(&sm.ring[0][0]);  // [wp][token]
#pragma unroll
  for (int H = 0; H < 2; ++H)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float m = -__builtin_inff();
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) m = __builtin_fmaxf(m, acc[8 * k + 4 * H + j][r]);
      m = __builtin_fmaxf(m, __shfl_xor(m, 16));
      m = __builtin_fmaxf(m, __shfl_xor(m, 32));
      const float shift = m == -__builtin_inff() ? 0.0f : -m * kLog2e;
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          s += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[8 * k + 4 * H + j][r], kLog2e, shift));
      s += __shfl_xor(s, 16);
      s += __shfl_xor(s, 32);
      if (at.g == 0) joined[256 * at.wp + at.q(H, j)] = make_float2(m, s);
      // the target's logit, where it is one of this wave's words
      const int64_t t = q0 + at.q(H, j);
      const int64_t word = t < a.T ? target_of(a, t) - p0 - 128 * at.wp : -1;
      if (__any(word >= 0 && word < 128)) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (word == at.p(k >> 2, r, k & 3) - 128 * at.wp)
              a.target_logit[t] = acc[8 * k + 4 * H + j][r];
      }
    }
  __syncthreads();
  const int64_t t = q0 + threadIdx.x;
  if (t >= a.T) return;
  const float2 u = joined[threadIdx.x], v = joined[256 + threadIdx.x];
  const float m = __builtin_fmaxf(u.x, v.x);
  const float base = m == -__builtin_inff() ? 0.0f : m;
  a.part[(int64_t)pt * a.T + t] =
      make_float2(m, u.y * __builtin_amdgcn_exp2f((u.x - base) * kLog2e) +
                         v.y * __builtin_amdgcn_exp2f((v.x - base) * kLog2e));
}

// lse and loss of every token from its tiles' statistics: 16 tokens a workgroup,
// 16 runs of tiles each.
constexpr int kJoinTokens = 16, kJoinRuns = 16;
__global__ __launch_bounds__(kJoinTokens* kJoinRuns) void k_loss_join(LossArgs a, int tiles) {
  __shared__ float2 run_s[kJoinRuns][kJoinTokens];
  const int k = threadIdx.x % kJoinTokens, run = threadIdx.x / kJoinTokens;
  const int64_t t = (int64_t)blockIdx.x * kJoinTokens + k;
  float m = -__builtin_inff(), s = 0.0f;
  const auto join = [&](float2 v) {
    const float top = __builtin_fmaxf(m, v.x);
    const float base = top == -__builtin_inff() ? 0.0f : top;
    s = s * __builtin_amdgcn_exp2f((m - base) * kLog2e) +
        v.y * __builtin_amdgcn_exp2f((v.x - base) * kLog2e);
    m = top;
  };
  if (t < a.T)
    for (int i = run; i < tiles; i += kJoinRuns) join(a.part[(int64_t)i * a.T + t]);
  run_s[run][k] = make_float2(m, s);
  __syncthreads();
  if (run != 0 || t >= a.T) return;
  for (int i = 1; i < kJoinRuns; ++i) join(run_s[i][k]);
  const float lse = m + __builtin_amdgcn_logf(s) * kLn2;
  const int64_t target = target_of(a, t);
  const float nan = __builtin_nanf("");
  a.stats[t] = target == -2 ? nan : lse;
  a.token_loss[t] = target == -1 ? 0.0f : target == -2 ? nan : lse - a.target_logit[t];
}

// Sum (or mean over the tokens that count) of the token losses, in a fixed
// order, and the reciprocal count behind the tokens' lse.
constexpr int kReduceThreads = 1024;
__global__ __launch_bounds__(kReduceThreads) void k_loss_reduce(LossArgs a) {
  __shared__ float sums[kReduceThreads];
  __shared__ int64_t counts[kReduceThreads];
  float s = 0.0f;
  int64_t n = 0;
  for (int64_t t = threadIdx.x; t < a.T; t += kReduceThreads) {
    s += a.token_loss[t];
    n += target_of(a, t) != -1;
  }
  sums[threadIdx.x] = s;
  counts[threadIdx.x] = n;
  for (int off = kReduceThreads / 2; off >= 1; off >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < off) {
      sums[threadIdx.x] += sums[threadIdx.x + off];
      counts[threadIdx.x] += counts[threadIdx.x + off];
    }
  }
  if (threadIdx.x == 0) {
    a.loss[0] = a.mean ? sums[0] / (float)counts[0] : sums[0];
    a.stats[a.T] = a.mean ? 1.0f / (float)counts[0] : 1.0f;
  }
}

// d of words v0 .. v0 + width of the vocabulary (width: the piece's words rounded
// up to 256; words past the vocabulary, and tokens past the last, get zeros).
__global__ __launch_bounds__(kThreads, 1) void k_loss_grad_tile(LossArgs a, int64_t v0, int width) {
  __shared__ LossSmem sm;
  const int np = width / kTile, nq = (int)((a.T + kTile - 1) / kTile);
  int pt, qt;
  tile_of(np, nq, pt, qt);
  const int64_t p0 = v0 + (int64_t)pt * kTile, q0 = (int64_t)qt * kTile;
  const Place at;
  v4f acc[64];
  const Operand P = tile_rows(a.w, a.ldw, p0, a.V, a.H);
  const Operand Q = tile_rows(a.x, a.ldx, q0, a.T, a.H);
  mainloop<false, false, false, true>(sm, P, Q, 0u, (uint32_t)(2 * a.H), acc);
  const int words = (int)std::min<int64_t>(kTile, a.V - p0);
#pragma unroll
  for (int H = 0; H < 2; ++H)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t t = q0 + at.q(H, j);
      float shift = 0.0f, g = 0.0f;
      int64_t word = -1;
      if (t < a.T) {
        word = target_of(a, t);
        if (word != -1) {
          shift = -a.stats[t] * kLog2e;
          g = a.per_token ? a.grad_loss[t] : a.grad_loss[0] * a.stats[a.T];
        }
        word -= p0;
      }
      const bool none = g == 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int p = at.p(k >> 2, r, k & 3);
          const float z = acc[8 * k + 4 * H + j][r];
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(z, kLog2e, shift));
          acc[8 * k + 4 * H + j][r] =
              none || p >= words ? 0.0f : (e - (word == p ? 1.0f : 0.0f)) * g;
        }
    }
  if (a.d != nullptr) {  // rows of tokens: 16 consecutive words a lane
    const int64_t ldd = width;
#pragma unroll
    for (int H = 0; H < 2; ++H)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t t = q0 + at.q(H, j);
        if (t >= a.T) continue;
#pragma unroll
        for (int G = 0; G < 2; ++G) {
          uint32_t w[8];
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int u = 0; u < 2; ++u)
              w[2 * r + u] = pack_bf16x2(acc[8 * (4 * G + 2 * u) + 4 * H + j][r],
                                         acc[8 * (4 * G + 2 * u + 1) + 4 * H + j][r]);
          uint4* o = reinterpret_cast<uint4*>(a.d + t * ldd + (int64_t)pt * kTile + at.p(G, 0, 0));
          o[0] = make_uint4(w[0], w[1], w[2], w[3]);
          o[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
      }
  }
  if (a.dt != nullptr) {  // rows of words: 4 consecutive tokens a lane, 64 a row
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int H = 0; H < 2; ++H) {
          const int64_t row = (int64_t)pt * kTile + at.p(k >> 2, r, k & 3);
          *reinterpret_cast<uint2*>(a.dt + row * a.ldt + q0 + at.q(H, 0)) =
              make_uint2(pack_bf16x2(acc[8 * k + 4 * H][r], acc[8 * k + 4 * H + 1][r]),
                         pack_bf16x2(acc[8 * k + 4 * H + 2][r], acc[8 * k + 4 * H + 3][r]));
        }
  }
}

// out[c][r] = in[r][c], rows of `out` filled with zeros from r = rows to ldo.
__global__ __launch_bounds__(256) void k_transpose(const uint16_t* __restrict__ in, int64_t ldi,
                                                   int64_t rows, int64_t cols,
                                                   uint16_t* __restrict__ out, int64_t ldo) {
  __shared__ uint16_t tile[64][66];
  const int64_t r0 = (int64_t)blockIdx.y * 64, c0 = (int64_t)blockIdx.x * 64;
  for (int i = threadIdx.x; i < 64 * 8; i += 256) {
    const int r = i >> 3, c = 8 * (i & 7);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r0 + r < rows && c0 + c < cols)
      v = *reinterpret_cast<const uint4*>(in + (r0 + r) * ldi + c0 + c);
    uint32_t* d = reinterpret_cast<uint32_t*>(&tile[r][c]);
    d[0] = v.x; d[1] = v.y; d[2] = v.z; d[3] = v.w;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 64 * 8; i += 256) {
    const int c = i >> 3, r = 8 * (i & 7);
    if (c0 + c >= cols || r0 + r >= ldo) continue;
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      w[k] = tile[r + 2 * k][c] | (uint32_t)tile[r + 2 * k + 1][c] << 16;
    *reinterpret_cast<uint4*>(out + (c0 + c) * ldo + r0 + r) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// out[q][p] = sum_k Q[q][k] P[p][k] (+ out's fp32 value so far), written as bf16,
// or as fp32 (partials of the ranges of k along blockIdx.y, nq * np apart).
struct ProductArgs {
  const uint16_t* P;
  const uint16_t* Q;
  const float* before;  // fp32 [nq][np] to add, or nullptr
  uint16_t* out;        // bf16 [nq][np], or nullptr
  float* out32;         // fp32 [ranges][nq][np]
  int64_t ldp, ldq, np, nq, k;  // elements
  int64_t range;                // k of a range, a multiple of 64
};
__global__ __launch_bounds__(kThreads, 1) void k_product(ProductArgs a) {
  __shared__ LossSmem sm;
  const int pts = (int)((a.np + kTile - 1) / kTile), qts = (int)((a.nq + kTile - 1) / kTile);
  int pt, qt;
  tile_of(pts, qts, pt, qt);
  const int64_t p0 = (int64_t)pt * kTile, q0 = (int64_t)qt * kTile;
  const int64_t k0 = (int64_t)blockIdx.y * a.range, k1 = std::min<int64_t>(a.k, k0 + a.range);
  const Operand P = tile_rows(a.P + k0, a.ldp, p0, a.np, k1 - k0);
  const Operand Q = tile_rows(a.Q + k0, a.ldq, q0, a.nq, k1 - k0);
  v4f acc[64];
  mainloop<false, false, false, true>(sm, P, Q, 0u, (uint32_t)(2 * (k1 - k0)), acc);
  const Place at;
  float* out32 = a.out32 + (int64_t)blockIdx.y * a.nq * a.np;
#pragma unroll
  for (int H = 0; H < 2; ++H)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t q = q0 + at.q(H, j);
      if (q >= a.nq) continue;
#pragma unroll
      for (int G = 0; G < 2; ++G)
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // 8 consecutive columns
          const int64_t p = p0 + at.p(G, 2 * h, 0);
          if (p >= a.np) continue;
          float v[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) v[u] = acc[8 * (4 * G + (u & 3)) + 4 * H + j][2 * h + (u >> 2)];
          const int64_t o = q * a.np + p;
          if (a.before != nullptr) {
            const float4 b0 = *reinterpret_cast<const float4*>(a.before + o);
            const float4 b1 = *reinterpret_cast<const float4*>(a.before + o + 4);
            v[0] += b0.x; v[1] += b0.y; v[2] += b0.z; v[3] += b0.w;
            v[4] += b1.x; v[5] += b1.y; v[6] += b1.z; v[7] += b1.w;
          }
          if (a.out != nullptr) {
            *reinterpret_cast<uint4*>(a.out + o) =
                make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                           pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
          } else {
            *reinterpret_cast<float4*>(out32 + o) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(out32 + o + 4) = make_float4(v[4], v[5], v[6], v[7]);
          }
        }
    }
}

// Sum of the partials of the ranges in order (after `before`), as bf16 or fp32.
__global__ __launch_bounds__(256) void k_product_join(const float* __restrict__ part, int ranges,
                                                      int64_t n, const float* before,
                                                      uint16_t* out, float* out32) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  float4 s = before ? *reinterpret_cast<const float4*>(before + i) : make_float4(0, 0, 0, 0);
  for (int k = 0; k < ranges; ++k) {
    const float4 v = *reinterpret_cast<const float4*>(part + k * n + i);
    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  }
  if (out)
    *reinterpret_cast<uint2*>(out + i) = make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
  else
    *reinterpret_cast<float4*>(out32 + i) = s;
}

int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
int64_t tiles(int64_t n) { return (n + kTile - 1) / kTile; }

// Ranges of k that a product is cut into: as many as give every compute unit a
// tile, of at least 512 elements each.
int product_ranges(int64_t np, int64_t nq, int64_t k) {
  const int64_t n = tiles(np) * tiles(nq), cus = std::max(1, device_cu_count());
  return (int)std::max<int64_t>(1, std::min<int64_t>(cus / n, k / 512));
}

hipError_t run_product(ProductArgs a, float* partials, float* acc, hipStream_t stream) {
  const int ranges = product_ranges(a.np, a.nq, a.k);
  a.range = up((a.k + ranges - 1) / ranges, 64);
  const int used = (int)((a.k + a.range - 1) / a.range);
  const dim3 grid((unsigned)(tiles(a.np) * tiles(a.nq)), (unsigned)used);
  if (used == 1) {
    a.out32 = acc;
    hipLaunchKernelGGL(k_product, grid, dim3(kThreads), 0, stream, a);
    return hipGetLastError();
  }
  const float* before = a.before;
  uint16_t* out = a.out;
  a.before = nullptr;
  a.out = nullptr;
  a.out32 = partials;
  hipLaunchKernelGGL(k_product, grid, dim3(kThreads), 0, stream, a);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  const int64_t n = a.np * a.nq;
  hipLaunchKernelGGL(k_product_join, dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, stream,
                     partials, used, n, before, out, acc);
  return hipGetLastError();
}

hipError_t transpose(const uint16_t* in, int64_t ldi, int64_t rows, int64_t cols, uint16_t* out,
                     int64_t ldo, hipStream_t stream) {
  const dim3 grid((unsigned)((cols + 63) / 64), (unsigned)((ldo + 63) / 64));
  hipLaunchKernelGGL(k_transpose, grid, dim3(256), 0, stream, in, ldi, rows, cols, out, ldo);
  return hipGetLastError();
}

// Words of a piece: d, d^T and W^T of it stay within kPieceBytes, the pieces of
// one vocabulary are alike.
constexpr int64_t kPieceBytes = INT64_C(1) << 30;
int64_t piece_words(const LossArgs& a) {
  const int64_t most = std::max<int64_t>(kTile, kPieceBytes / (4 * up(a.T, kTile) + 2 * a.H) / kTile * kTile);
  const int64_t pieces = (a.V + most - 1) / most;
  return up((a.V + pieces - 1) / pieces, kTile);
}

// Offsets of the gradient's workspace.
struct GradSpace {
  int64_t piece, d, dt, wt, xt, acc, part, bytes;
};
GradSpace grad_space(const LossArgs& a, bool need_x, bool need_w) {
  GradSpace s{};
  s.piece = piece_words(a);
  const int64_t ldt = up(a.T, kTile);
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += up(bytes, 256);
    return o;
  };
  int64_t part = 0;
  if (need_x) {
    s.d = take(a.T * s.piece * 2);
    s.wt = take(a.H * s.piece * 2);
    if (s.piece < a.V) s.acc = take(a.T * a.H * 4);
    const int ranges = product_ranges(a.H, a.T, s.piece);
    if (ranges > 1) part = ranges * a.T * a.H * 4;
  }
  if (need_w) {
    s.dt = take(s.piece * ldt * 2);
    s.xt = take(a.H * ldt * 2);
    const int64_t rows = std::min(s.piece, a.V);
    for (int64_t n : {rows, a.V - (a.V - 1) / s.piece * s.piece}) {  // a piece, and the last one
      const int ranges = product_ranges(a.H, n, ldt);
      if (ranges > 1) part = std::max<int64_t>(part, ranges * n * a.H * 4);
    }
  }
  s.part = take(part);
  s.bytes = at;
  return s;
}

}  // namespace

int64_t loss_workspace_bytes(const LossArgs& a) {
  return up(tiles(a.V) * a.T * 8, 256) + up(a.T * 4, 256) * 2;
}

hipError_t launch_loss(LossArgs a, uint8_t* ws, hipStream_t stream) {
  if (a.T > 0) {
    a.part = reinterpret_cast<float2*>(ws);
    a.target_logit = reinterpret_cast<float*>(ws + up(tiles(a.V) * a.T * 8, 256));
    if (!a.token_loss) a.token_loss = a.target_logit + up(a.T * 4, 256) / 4;
    hipLaunchKernelGGL(k_loss_fwd, dim3((unsigned)(tiles(a.V) * tiles(a.T))), dim3(kThreads), 0,
                       stream, a);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    hipLaunchKernelGGL(k_loss_join, dim3((unsigned)((a.T + kJoinTokens - 1) / kJoinTokens)),
                       dim3(kJoinTokens * kJoinRuns), 0, stream, a, (int)tiles(a.V));
    err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  if (!a.loss) return hipSuccess;
  hipLaunchKernelGGL(k_loss_reduce, dim3(1), dim3(kReduceThreads), 0, stream, a);
  return hipGetLastError();
}

int64_t loss_grad_workspace_bytes(const LossArgs& a, bool need_x, bool need_w) {
  return a.T == 0 ? 0 : grad_space(a, need_x, need_w).bytes;
}

hipError_t launch_loss_grad(LossArgs a, uint16_t* dx, uint16_t* dw, uint8_t* ws,
                            hipStream_t stream) {
  const GradSpace s = grad_space(a, dx != nullptr, dw != nullptr);
  a.ldt = up(a.T, kTile);
  a.d = dx ? reinterpret_cast<uint16_t*>(ws + s.d) : nullptr;
  a.dt = dw ? reinterpret_cast<uint16_t*>(ws + s.dt) : nullptr;
  uint16_t* wt = reinterpret_cast<uint16_t*>(ws + s.wt);
  uint16_t* xt = reinterpret_cast<uint16_t*>(ws + s.xt);
  float* acc = reinterpret_cast<float*>(ws + s.acc);
  float* part = reinterpret_cast<float*>(ws + s.part);
  hipError_t err;
  if (dw && (err = transpose(a.x, a.ldx, a.T, a.H, xt, a.ldt, stream)) != hipSuccess) return err;
  for (int64_t v0 = 0; v0 < a.V; v0 += s.piece) {
    const int64_t words = std::min<int64_t>(s.piece, a.V - v0);
    const int64_t width = up(words, kTile);
    hipLaunchKernelGGL(k_loss_grad_tile, dim3((unsigned)(width / kTile * tiles(a.T))),
                       dim3(kThreads), 0, stream, a, v0, (int)width);
    if ((err = hipGetLastError()) != hipSuccess) return err;
    if (dx) {
      err = transpose(a.w + v0 * a.ldw, a.ldw, words, a.H, wt, width, stream);
      if (err != hipSuccess) return err;
      ProductArgs p{};
      p.P = wt;
      p.ldp = width;
      p.np = a.H;
      p.Q = a.d;
      p.ldq = width;
      p.nq = a.T;
      p.k = width;
      p.before = v0 > 0 ? acc : nullptr;
      p.out = v0 + words == a.V ? dx : nullptr;
      if ((err = run_product(p, part, acc, stream)) != hipSuccess) return err;
    }
    if (dw) {
      ProductArgs p{};
      p.P = xt;
      p.ldp = a.ldt;
      p.np = a.H;
      p.Q = a.dt;
      p.ldq = a.ldt;
      p.nq = words;
      p.k = up(a.T, 8);
      p.out = dw + v0 * a.H;
      if ((err = run_product(p, part, nullptr, stream)) != hipSuccess) return err;
    }
  }
  return hipSuccess;
}

}  // namespace mxgg
