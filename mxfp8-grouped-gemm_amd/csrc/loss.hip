// Softmax cross entropy of a linear layer, z = x W^T (bf16 operands), without the
// logits z [tokens, vocab] ever being kept.
//
//   loss[t] = lse[t] - z[t][target[t]],   lse[t] = log sum_v exp(z[t][v])
//   d[t][v] = (exp(z[t][v] - lse[t]) - [v = target[t]]) g[t]
//   dx = d W,   dW = d^T x        (g: the loss's gradient per token, 0 where ignored)
//
// Forward: 256 (vocabulary) x 256 (token) tiles of z on the matrix cores; every
// tile leaves one maximum m and one sum s of exp(z - m) a token, joined over the tiles
// by a second kernel.  Few tokens stream W past the tiles.
// lse = m + log(s) is never formed: a token that is sure of its target has a loss and
// a p - 1 far below the spacing of fp32 numbers at lse.  The loss is (m - z) + log(s),
// and m and 1 / s are kept for p = exp(z - m) / s.
// Backward: pieces of the vocabulary.  The tiles of a piece are computed again
// (8 T H V operations in all, 6 with kept logits) and leave d / g rounded to bf16,
// [T][piece].  Both products read it, W and x as they lie: an operand that is not
// contiguous along its contraction is transposed on the way from LDS to registers.
// Where g is one number for all tokens it multiplies the products' sums in fp32,
// so what is rounded is p - 1 or p itself: one bf16 rounding per term of sums whose
// result is rounded to bf16 anyway.  dx is carried over pieces in fp32.
// A product with few tiles is split along the contraction, and the fp32 partials
// added in order.
//
// 4096 tokens, 131072 words, hidden 7168, on two cards: forward 5.0 and 5.3 ms (1.54 and
// 1.44 PFLOP/s), tiles of d 5.2 and 5.5, products 10.9 and 11.6 (1.41 and 1.32); a large
// product of the library runs 1.51 to 1.52 on the first.
// Bound by the matrix cores at the clock that the power limit leaves.  128 x 32000 x
// 1024, forward: 16.4 us, the 66 MB of W at 4 TB/s in one round of small tiles.
#include <algorithm>

#include "gemm_tile.h"

namespace mxgg {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();
constexpr int kTile = 256;
constexpr int kSmallTile = 128;

// What a tile's tokens bring to its epilogue, loaded by one thread each with the first
// stages of the main loop.
struct TokenInfo {
  int32_t word;  // target's place among the tile's words, kNoWord or kIgnored
  float most, scale, g;  // scale = g / s
};
constexpr int32_t kNoWord = -1, kIgnored = -2;
struct __align__(16) LossSmem {
  uint8_t ring[2][kStageBytes];
  TokenInfo token[kTile];
};

// Tiles of 128 x 128 for calls that large ones would leave most of the chip idle:
// four waves of 64 x 64, four ring stages of 64 contraction elements (three in
// flight), one barrier a stage.  A row is 128 bytes, its 16-byte chunk c at
// c ^ swz(row), so a half-wave's fragment read touches every bank twice.
constexpr uint32_t kSmallOp = 128u * kStageK;  // one operand of a stage: 16 KB
constexpr int kSmallLoads = 8;                 // of a wave for a stage
struct __align__(16) SmallSmem {
  uint8_t ring[4][2 * kSmallOp];
};
union TileSmem {
  LossSmem large;
  SmallSmem small;
};

// Rows row0 .. of a bf16 matrix as a tile operand, `cols` elements of each.
__device__ __forceinline__ Operand tile_rows(const uint16_t* p, int64_t ld, int64_t row0,
                                             int64_t rows, int64_t cols, int tile = kTile) {
  const int64_t n = std::min<int64_t>(tile, rows - row0);
  Operand o;
  o.data = make_desc(p + row0 * ld, (uint32_t)(((n - 1) * ld + cols) * 2));
  o.scale = o.data;  // not read
  o.ld = (uint32_t)(ld * 2);
  o.lds = 0;
  o.row0 = 0;
  o.hi = 128;
  return o;
}

// Columns col0 .. of a bf16 matrix of k rows as a K-major tile operand.
__device__ __forceinline__ Operand tile_columns(const uint16_t* p, int64_t ld, int64_t k,
                                                int64_t col0, int64_t cols) {
  Operand o;
  o.data = o.scale = desc_t{0, 0, 0, 0};  // not read
  o.base = reinterpret_cast<const uint8_t*>(p + col0);
  o.bytes = ((k - 1) * ld + cols - col0) * 2;
  o.ld = (uint32_t)(ld * 2);
  o.lds = 0;
  o.row0 = 0;
  o.hi = 128;
  return o;
}

// Tile `block` of np x nq.  Workgroups go round-robin to the 8 XCDs: each XCD takes a
// contiguous run of tiles in an order of bands of 8 token tiles, so the 32 tiles
// it works on at a time share 8 + 4 operand panels in its L2.
__device__ __forceinline__ void tile_of(int block, int np, int nq, int& p, int& q) {
  const int total = np * nq, per = total / 8, rest = total % 8;
  const int xcd = block % 8, slot = block / 8;
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

// Accumulators of a wave's 64 x 64 part of a small tile: acc[4F + J], register r of
// lane c + 16g, is P index 64 wp + 16 F + 4 g + r and Q index 64 wq + 16 J + c.
__device__ __forceinline__ void small_loop(SmallSmem& sm, const Operand& P, const Operand& Q,
                                           uint32_t kend, v4f (&acc)[16]) {
  const uint32_t lane = threadIdx.x & 63u, wave = wave_id();
  const uint32_t wp = wave & 1u, wq = wave >> 1, m = lane & 15u, g = lane >> 4;
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  const uint32_t nst = (kend + kStageK - 1) / kStageK;
  // Load i of wave w fills rows 32i + 8w .. + 7 of an operand, eight lanes a row.
  const uint32_t row = 8u * wave + (lane >> 3);
  const uint32_t kcol = 16u * ((lane & 7u) ^ swz(row));
  const uint32_t vp = row * P.ld + kcol, vq = row * Q.ld + kcol;
  const auto load = [&](uint32_t s) __attribute__((always_inline)) {
    const uint32_t k0 = s * kStageK, dst = lds_offset(sm.ring[s & 3u]) + 1024u * wave;
    const bool ok = k0 + kcol < kend;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      dma_x4(P.data, dst + 4096u * i, ok ? vp + k0 : kOobOffset, 32u * i * P.ld);
      dma_x4(Q.data, dst + kSmallOp + 4096u * i, ok ? vq + k0 : kOobOffset, 32u * i * Q.ld);
    }
  };
  const uint32_t lo = ((g ^ swz(m)) << 4), hi = (((g + 4u) ^ swz(m)) << 4);
  const uint32_t rp = (64u * wp + m) * kStageK, rq = kSmallOp + (64u * wq + m) * kStageK;
  load(0);
  if (nst > 1) load(1);
  if (nst > 2) load(2);
  for (uint32_t s = 0; s < nst; ++s) {
    // stage s has landed for every wave, and every wave has read stage s - 1, whose
    // slot the next load takes
    if (s + 2 < nst) wait_barrier<2 * kSmallLoads>();
    else if (s + 1 < nst) wait_barrier<kSmallLoads>();
    else wait_barrier<0>();
    __builtin_amdgcn_sched_barrier(0);
    if (s + 3 < nst) load(s + 3);
    const uint8_t* st = sm.ring[s & 3u];
    Frags f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f.a[i] = lds_v8i(st + rp + lo + 2048 * i, st + rp + hi + 2048 * i);
      f.b[i] = lds_v8i(st + rq + lo + 2048 * i, st + rq + hi + 2048 * i);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[4 * i + j] = mfma_bf16_stage(f.a[i], f.b[j], acc[4 * i + j]);
  }
  release_barrier();
}

// Target of token t: its word, -1 = ignored, -2 = outside the vocabulary.
__device__ __forceinline__ int64_t target_of(const LossArgs& a, int64_t t) {
  const int64_t v = a.target64 ? static_cast<const int64_t*>(a.target)[t]
                               : (int64_t) static_cast<const int32_t*>(a.target)[t];
  return v == a.ignore_index ? -1 : v >= 0 && v < a.V ? v : -2;
}

// The logits of a large tile, and what its tokens (from q0) bring in sm.token; `first` is
// the tile's first word.
template <bool GRAD>
__device__ __forceinline__ void logits(LossSmem& sm, const LossArgs& a, int64_t first, int64_t q0,
                                       v4f (&acc)[64]) {
  const Operand P = tile_rows(a.w, a.ldw, first, a.V, a.H);
  const Operand Q = tile_rows(a.x, a.ldx, q0, a.T, a.H);
  const uint32_t kend = (uint32_t)(2 * a.H);
  const int64_t t = q0 + threadIdx.x;
  int64_t target = -1;
  float most = 0.0f, over_sum = 0.0f, g = 1.0f;
  if (t < a.T) {
    target = target_of(a, t);
    if (GRAD) {
      most = a.stats[t];
      over_sum = a.stats[a.T + t];
    }
    if (GRAD && a.per_token) g = a.grad_loss[t];
  }
  Stream<false> st;
  st.init(P, Q, 0u, kend);
  st.prologue(sm.ring[0], sm.ring[1], P, Q, 0u, (kend + kStageK - 1) / kStageK);
  const int64_t word = target - first;
  sm.token[threadIdx.x] = {target == -1                 ? kIgnored
                           : word >= 0 && word < kTile ? (int32_t)word
                                                        : kNoWord,
                           most, over_sum * g, g};
  mainloop<false, false, true, true, false, false, 0>(sm, P, Q, 0u, kend, acc);
}

// exp(z - m).
__device__ __forceinline__ float exp_over(float z, float m) {
  return __builtin_amdgcn_exp2f((z - m) * kLog2e);
}
// What to subtract where m is the largest of some words, or of none (-infinity).
__device__ __forceinline__ float or_zero(float m) { return m == kNegInf ? 0.0f : m; }

// (max, sum of exp(z - max)) of two sets of words.
__device__ __forceinline__ float2 join_halves(float2 u, float2 v) {
  const float m = __builtin_fmaxf(u.x, v.x), sub = or_zero(m);
  return make_float2(m, u.y * exp_over(u.x, sub) + v.y * exp_over(v.x, sub));
}

// Statistics of a tile: part[part row][t] = (max, sum of exp(z - max)) over the
// tile's words, and the target's logit.
__device__ __forceinline__ void fwd_tile(LossSmem& sm, const LossArgs& a, int64_t p0, int64_t q0,
                                         int64_t part_row) {
  v4f acc[64];
  logits<false>(sm, a, p0, q0, acc);

  const Place at;
  const int words = (int)std::min<int64_t>(kTile, a.V - p0);
  if (words < kTile) {  // past the vocabulary: no word
#pragma unroll
    for (int k = 0; k < 64; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (at.p(k >> 5, r, (k >> 3) & 3) >= words) acc[k][r] = kNegInf;
  }
  float2* joined = reinterpret_cast<float2*>(&sm.ring[0][0]);  // [wp][token]
#pragma unroll
  for (int H = 0; H < 2; ++H)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float m = kNegInf;
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) m = __builtin_fmaxf(m, acc[8 * k + 4 * H + j][r]);
      m = __builtin_fmaxf(m, __shfl_xor(m, 16));
      m = __builtin_fmaxf(m, __shfl_xor(m, 32));
      const float sub = or_zero(m);
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) s += exp_over(acc[8 * k + 4 * H + j][r], sub);
      s += __shfl_xor(s, 16);
      s += __shfl_xor(s, 32);
      if (at.g == 0) joined[256 * at.wp + at.q(H, j)] = make_float2(m, s);
      // the target's logit, where it is one of this wave's words
      const int64_t t = q0 + at.q(H, j);
      const int word = sm.token[at.q(H, j)].word - 128 * at.wp;
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
  a.part[part_row * a.T + t] = join_halves(joined[threadIdx.x], joined[256 + threadIdx.x]);
}

// The same for a small tile.
__device__ __forceinline__ void fwd_tile_small(SmallSmem& sm, const LossArgs& a, int64_t p0,
                                               int64_t q0, int64_t part_row) {
  const Operand P = tile_rows(a.w, a.ldw, p0, a.V, a.H, kSmallTile);
  const Operand Q = tile_rows(a.x, a.ldx, q0, a.T, a.H, kSmallTile);
  v4f acc[16];
  small_loop(sm, P, Q, (uint32_t)(2 * a.H), acc);

  const Place at;
  const int words = (int)std::min<int64_t>(kSmallTile, a.V - p0);
  const int first = 64 * at.wp + 4 * at.g;  // + 16 F + r
  float2* joined = reinterpret_cast<float2*>(&sm.ring[0][0]);  // [wp][token]
#pragma unroll
  for (int J = 0; J < 4; ++J) {
    const int q = 64 * at.wq + 16 * J + at.c;
    float z[16], m = kNegInf;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      z[i] = first + 16 * (i >> 2) + (i & 3) < words ? acc[4 * (i >> 2) + J][i & 3]
                                                     : kNegInf;
      m = __builtin_fmaxf(m, z[i]);
    }
    m = __builtin_fmaxf(m, __shfl_xor(m, 16));
    m = __builtin_fmaxf(m, __shfl_xor(m, 32));
    const float sub = or_zero(m);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += exp_over(z[i], sub);
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if (at.g == 0) joined[kSmallTile * at.wp + q] = make_float2(m, s);
    const int64_t t = q0 + q, word = t < a.T ? target_of(a, t) - p0 - first : -1;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (word == 16 * (i >> 2) + (i & 3)) a.target_logit[t] = z[i];
  }
  __syncthreads();
  const int64_t t = q0 + threadIdx.x;
  if (threadIdx.x >= kSmallTile || t >= a.T) return;
  a.part[part_row * a.T + t] = join_halves(joined[threadIdx.x], joined[kSmallTile + threadIdx.x]);
}

// Large tiles for the first large_words words, small ones for the rest.
__global__ __launch_bounds__(kThreads, 1) void k_loss_fwd(LossArgs a, int64_t large_words) {
  __shared__ TileSmem sm;
  const int np = (int)((large_words + kTile - 1) / kTile), nq = (int)((a.T + kTile - 1) / kTile);
  const int large = np * nq, block = (int)blockIdx.x;
  int pt, qt;
  if (block < large) {
    tile_of(block, np, nq, pt, qt);
    fwd_tile(sm.large, a, (int64_t)pt * kTile, (int64_t)qt * kTile, pt);
  } else {
    const int ns = (int)((a.V - large_words + kSmallTile - 1) / kSmallTile);
    tile_of(block - large, ns, (int)((a.T + kSmallTile - 1) / kSmallTile), pt, qt);
    fwd_tile_small(sm.small, a, large_words + (int64_t)pt * kSmallTile, (int64_t)qt * kSmallTile,
                   np + pt);
  }
}

// The forward pass of few tokens, which reads W once and has little else to do: 64
// words a tile (16 / 32 / 64 of them, 32 tokens, 70016 x 2048: 117 / 91 / 79 us, since x
// is read for every tile), the four waves of a workgroup a quarter of the contraction
// each (stages of 64 in turn), operands straight from memory to registers.  A workgroup
// keeps the statistics of its tiles and leaves one a token.
constexpr int kFewFrags = 4, kFewWords = 16 * kFewFrags;
template <int NB>  // tokens / 16
struct FewStage {
  v8i w[kFewFrags], x[NB];
};
template <int NB>
__global__ __launch_bounds__(kThreads) void k_loss_few(LossArgs a, int tiles) {
  // partial sums of the waves: [tile parity][wave][word block][token block][lane]
  __shared__ v4f part_s[2][4][kFewFrags][NB][64];
  const uint32_t lane = threadIdx.x & 63u, wave = wave_id(), m = lane & 15u, g = lane >> 4;
  const uint32_t kend = (uint32_t)(2 * a.H), nst = (kend + kStageK - 1) / kStageK;
  const auto rows_of = [](const uint16_t* p, int64_t ld, int64_t rows, int64_t cols)
                           __attribute__((always_inline)) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(p), (short)0,
                                             (int)(((rows - 1) * ld + cols) * 2), 0x00020000);
  };
  const auto xs = rows_of(a.x, a.ldx, a.T, a.H);
  const uint32_t ldw = (uint32_t)(2 * a.ldw), ldx = (uint32_t)(2 * a.ldx);
  // the statistics of tokens 16 j + m, j % 4 = this wave, and their targets
  float most[(NB + 3) / 4], sum[(NB + 3) / 4];
  int64_t target[(NB + 3) / 4];
#pragma unroll
  for (int i = 0; i < (NB + 3) / 4; ++i) {
    const int64_t t = 16 * (4 * i + (int64_t)wave) + m;
    most[i] = kNegInf;
    sum[i] = 0.0f;
    target[i] = t < a.T ? target_of(a, t) : -1;
  }
  int parity = 0;
  for (int tile = (int)blockIdx.x; tile < tiles; tile += (int)gridDim.x, parity ^= 1) {
    const int64_t p0 = (int64_t)tile * kFewWords;
    const int64_t words = std::min<int64_t>(kFewWords, a.V - p0);
    const auto ws = rows_of(a.w + p0 * a.ldw, a.ldw, words, a.H);
    v4f acc[kFewFrags][NB];
#pragma unroll
    for (int F = 0; F < kFewFrags; ++F)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[F][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const auto load = [&](FewStage<NB>& st, uint32_t s) __attribute__((always_inline)) {
      const uint32_t k = s * kStageK + 16u * g;  // chunk g, and g + 4
      const auto chunk = [&](auto rsrc, uint32_t row, uint32_t ld) __attribute__((always_inline)) {
        const u32x4 lo = __builtin_amdgcn_raw_buffer_load_b128(
            rsrc, k < kend ? row * ld + k : kOobOffset, 0, 0);
        const u32x4 hi = __builtin_amdgcn_raw_buffer_load_b128(
            rsrc, k + 64u < kend ? row * ld + k + 64u : kOobOffset, 0, 0);
        return v8i{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3],
                   (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
      };
#pragma unroll
      for (uint32_t F = 0; F < kFewFrags; ++F) st.w[F] = chunk(ws, 16u * F + m, ldw);
#pragma unroll
      for (uint32_t j = 0; j < NB; ++j) st.x[j] = chunk(xs, 16u * j + m, ldx);
    };
    const auto multiply = [&](const FewStage<NB>& st) __attribute__((always_inline)) {
#pragma unroll
      for (int F = 0; F < kFewFrags; ++F)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[F][j] = mfma_bf16_stage(st.w[F], st.x[j], acc[F][j]);
    };
    // two stages in flight (loads past the last one are zeros)
    FewStage<NB> st[2];
    load(st[0], wave);
    load(st[1], wave + 4u);
    for (uint32_t s = wave; s < nst; s += 8u) {
      multiply(st[0]);
      load(st[0], s + 8u);
      multiply(st[1]);
      load(st[1], s + 12u);
    }
#pragma unroll
    for (int F = 0; F < kFewFrags; ++F)
#pragma unroll
      for (int j = 0; j < NB; ++j) part_s[parity][wave][F][j][lane] = acc[F][j];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < (NB + 3) / 4; ++i) {
      const int j = 4 * i + (int)wave;
      if (j >= NB) break;
      // words 16 F + 4 g + r of token 16 j + m
      float z[4 * kFewFrags], best = most[i];
#pragma unroll
      for (int F = 0; F < kFewFrags; ++F) {
        v4f v = part_s[parity][0][F][j][lane];
#pragma unroll
        for (int w = 1; w < 4; ++w) v += part_s[parity][w][F][j][lane];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          z[4 * F + r] = 16 * F + 4 * (int)g + r < words ? v[r] : kNegInf;
          best = __builtin_fmaxf(best, z[4 * F + r]);
        }
      }
      best = __builtin_fmaxf(best, __shfl_xor(best, 16));
      best = __builtin_fmaxf(best, __shfl_xor(best, 32));
      const float sub = or_zero(best);
      sum[i] *= exp_over(most[i], sub);  // this lane's words
      most[i] = best;
#pragma unroll
      for (int u = 0; u < 4 * kFewFrags; ++u) sum[i] += exp_over(z[u], sub);
      const int64_t word = target[i] - p0 - 4 * (int64_t)g;
#pragma unroll
      for (int u = 0; u < 4 * kFewFrags; ++u)
        if (word == 16 * (u >> 2) + (u & 3)) a.target_logit[16 * j + m] = z[u];
    }
  }
#pragma unroll
  for (int i = 0; i < (NB + 3) / 4; ++i) {
    const int64_t t = 16 * (4 * i + (int64_t)wave) + m;
    float s = sum[i];
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if (g == 0 && t < a.T) a.part[(int64_t)blockIdx.x * a.T + t] = make_float2(most[i], s);
  }
}

// Statistics and loss of every token from its tiles': 16 tokens a workgroup,
// 16 runs of tiles each.
constexpr int kJoinTokens = 16, kJoinRuns = 16;
__global__ __launch_bounds__(kJoinTokens* kJoinRuns) void k_loss_join(LossArgs a, int tiles) {
  __shared__ float2 run_s[kJoinRuns][kJoinTokens];
  const int k = threadIdx.x % kJoinTokens, run = threadIdx.x / kJoinTokens;
  const int64_t t = (int64_t)blockIdx.x * kJoinTokens + k;
  float2 sum = make_float2(kNegInf, 0.0f);
  constexpr int kAhead = 8;  // loads in flight
  if (t < a.T)
    for (int i0 = run; i0 < tiles; i0 += kJoinRuns * kAhead) {
      float2 v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = i0 + u * kJoinRuns;
        v[u] = i < tiles ? a.part[(int64_t)i * a.T + t] : make_float2(kNegInf, 0.0f);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) sum = join_halves(sum, v[u]);
    }
  run_s[run][k] = sum;
  __syncthreads();
  if (run != 0 || t >= a.T) return;
  for (int i = 1; i < kJoinRuns; ++i) sum = join_halves(sum, run_s[i][k]);
  const int64_t target = target_of(a, t);
  const float nan = __builtin_nanf("");
  a.stats[t] = sum.x;
  a.stats[a.T + t] = target == -1 ? 0.0f : target == -2 ? nan : 1.0f / sum.y;
  if (target < 0) {
    a.token_loss[t] = target == -1 ? 0.0f : nan;
    return;
  }
  a.token_loss[t] = (sum.x - a.target_logit[t]) + logf(sum.y);
}

// Sum (or mean over the tokens that count) of the token losses, in a fixed
// order, and the factor of their gradients behind the tokens' statistics: the reciprocal
// count of the mean, 0 where no token counts (its mean is 0 / 0, but nothing has a
// gradient).
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
    a.stats[2 * a.T] = counts[0] == 0 ? 0.0f : a.mean ? 1.0f / (float)counts[0] : 1.0f;
  }
}

// d of the tile of words v0 + p0 .. and tokens q0 ..; row t of d at a.d + t * width.
// Words past the vocabulary get zeros.
__device__ __forceinline__ void grad_tile(LossSmem& sm, const LossArgs& a, int64_t v0, int64_t p0,
                                          int64_t q0, int64_t width) {
  const Place at;
  v4f acc[64];
  logits<true>(sm, a, v0 + p0, q0, acc);
  const int words = (int)std::min<int64_t>(kTile, a.V - v0 - p0);
#pragma unroll
  for (int H = 0; H < 2; ++H)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const TokenInfo own = sm.token[at.q(H, j)];
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int p = at.p(k >> 2, r, k & 3);
          const float e = exp_over(acc[8 * k + 4 * H + j][r], own.most);
          acc[8 * k + 4 * H + j][r] =
              own.word == kIgnored || p >= words
                  ? 0.0f
                  : __builtin_fmaf(e, own.scale, own.word == p ? -own.g : 0.0f);
        }
    }
  // rows of tokens: 16 consecutive words a lane
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
        uint4* o = reinterpret_cast<uint4*>(a.d + t * width + p0 + at.p(G, 0, 0));
        o[0] = make_uint4(w[0], w[1], w[2], w[3]);
        o[1] = make_uint4(w[4], w[5], w[6], w[7]);
      }
    }
}

// The same for a small tile (without words where the width ends in one).
__device__ __forceinline__ void grad_tile_small(SmallSmem& sm, const LossArgs& a, int64_t v0,
                                                int64_t p0, int64_t q0, int64_t width) {
  v4f acc[16];
  if (v0 + p0 < a.V) {
    const Operand P = tile_rows(a.w, a.ldw, v0 + p0, a.V, a.H, kSmallTile);
    const Operand Q = tile_rows(a.x, a.ldx, q0, a.T, a.H, kSmallTile);
    small_loop(sm, P, Q, (uint32_t)(2 * a.H), acc);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const Place at;
  const int words = (int)std::min<int64_t>(kSmallTile, a.V - v0 - p0);
  const int first = 64 * at.wp + 4 * at.g;
#pragma unroll
  for (int J = 0; J < 4; ++J) {
    const int64_t t = q0 + 64 * at.wq + 16 * J + at.c;
    if (t >= a.T) continue;
    const int64_t target = target_of(a, t);
    const float g = target != -1 && a.per_token ? a.grad_loss[t] : 1.0f;
    const float most = a.stats[t], scale = a.stats[a.T + t] * g;
    const int64_t word = target - v0 - p0 - first;
#pragma unroll
    for (int F = 0; F < 4; ++F) {
      float v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = exp_over(acc[4 * F + J][r], most);
        v[r] = target == -1 || first + 16 * F + r >= words
                   ? 0.0f
                   : __builtin_fmaf(e, scale, word == 16 * F + r ? -g : 0.0f);
      }
      *reinterpret_cast<uint2*>(a.d + t * width + p0 + first + 16 * F) =
          make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    }
  }
}

// d of words v0 .. v0 + width (width: the piece's words rounded up to 256): large
// tiles for the first large_words of them, small ones for the rest.
__global__ __launch_bounds__(kThreads, 1) void k_loss_grad_tile(LossArgs a, int64_t v0, int width,
                                                                int large_words) {
  __shared__ TileSmem sm;
  const int np = (large_words + kTile - 1) / kTile, nq = (int)((a.T + kTile - 1) / kTile);
  const int large = np * nq, block = (int)blockIdx.x;
  int pt, qt;
  if (block < large) {
    tile_of(block, np, nq, pt, qt);
    grad_tile(sm.large, a, v0, (int64_t)pt * kTile, (int64_t)qt * kTile, width);
  } else {
    tile_of(block - large, (width - np * kTile) / kSmallTile,
            (int)((a.T + kSmallTile - 1) / kSmallTile), pt, qt);
    grad_tile_small(sm.small, a, v0, np * kTile + (int64_t)pt * kSmallTile,
                    (int64_t)qt * kSmallTile, width);
  }
}

// out[q][p] = scale * sum_k Q[q][k] P[k][p] (+ out's fp32 value so far), written as
// bf16, or as fp32 (a partial of every range of k, nq * np apart).  P is K-major; Q
// is [nq][k], or K-major ([k][nq]) with QK.  Q's rows go on to a multiple of 8, with
// zeros: a 16-byte load is cut at the end of its buffer by whole dwords.
struct Product {
  const uint16_t* P;
  const uint16_t* Q;
  const float* before;  // fp32 [nq][np] to add, or nullptr
  uint16_t* out;        // bf16 [nq][np], or nullptr
  float* out32;         // fp32 [ranges][nq][np]
  const float* scale;   // two factors, at scale[0] and scale2[0], or nullptr; a zero at
  const float* scale2;  // scale2 makes the output 0 whatever is at scale
  const float* live;    // not QK: [nq], 0 for rows that are 0 whatever the scale
  int64_t ldp, ldq, np, nq, k;  // elements
  int64_t range;                // k of a range, a multiple of 64
  int32_t blocks;               // workgroups: tiles times ranges
};

template <bool QK>
__device__ __forceinline__ void product_tile(LossSmem& sm, const Product& a, int block) {
  const int pts = (int)((a.np + kTile - 1) / kTile), qts = (int)((a.nq + kTile - 1) / kTile);
  const int range = block / (pts * qts);
  int pt, qt;
  tile_of(block - range * pts * qts, pts, qts, pt, qt);
  const int64_t p0 = (int64_t)pt * kTile, q0 = (int64_t)qt * kTile;
  const int64_t k0 = (int64_t)range * a.range, k = std::min<int64_t>(a.k - k0, a.range);
  const Operand P = tile_columns(a.P + k0 * a.ldp, a.ldp, k, p0, a.np);
  const Operand Q = QK ? tile_columns(a.Q + k0 * a.ldq, a.ldq, k, q0, (a.nq + 7) / 8 * 8)
                       : tile_rows(a.Q + k0, a.ldq, q0, a.nq, (k + 7) / 8 * 8);
  // loaded ahead of the main loop: behind it they cost a tile 0.2 us
  const float grad = a.scale ? a.scale[0] : 1.0f, factor = a.scale ? a.scale2[0] : 1.0f;
  const float scale = factor == 0.0f ? 0.0f : grad * factor;
  const bool odd_scale = !QK && !(__builtin_fabsf(scale) < __builtin_inff());
  v4f acc[64];
  mainloop<false, false, false, true, true, QK>(sm, P, Q, 0u, (uint32_t)(2 * k), acc);
  const Place at;
  float* out32 = a.out32 + (int64_t)range * a.nq * a.np;
  // Accumulator 8F + J, register r: P index 128 wp + 16 F + 4 g + r, and Q index
  // 128 wq + 16 J + c (K-major), or that of Place::q.
#pragma unroll
  for (int J = 0; J < 8; ++J) {
    const int64_t q = q0 + (QK ? 128 * at.wq + 16 * J + at.c : at.q(J >> 2, J & 3));
    const bool row = q < a.nq;
    // a row of zeros stays one under a factor that is not finite
    const float times = odd_scale && row && a.live[q] == 0.0f ? 0.0f : scale;
#pragma unroll
    for (int F = 0; F < 8; F += 2) {
      float v[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int64_t p = p0 + 128 * at.wp + 16 * (F + u) + 4 * at.g, o = q * a.np + p;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[u][r] = acc[8 * (F + u) + J][r] * times;
        if (!row || p >= a.np) continue;
        if (a.before != nullptr) {
          const float4 b = *reinterpret_cast<const float4*>(a.before + o);
          v[u][0] += b.x; v[u][1] += b.y; v[u][2] += b.z; v[u][3] += b.w;
        }
        if (a.out == nullptr)
          *reinterpret_cast<float4*>(out32 + o) = make_float4(v[u][0], v[u][1], v[u][2], v[u][3]);
      }
      if (a.out == nullptr) continue;
      // Lanes of rows g and g + 1 (g even) change quads, so that one holds 8
      // consecutive columns of fragment F and the other of fragment F + 1.
      u32x2 w[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
        w[u] = u32x2{pack_bf16x2(v[u][0], v[u][1]), pack_bf16x2(v[u][2], v[u][3])};
      const auto lo = __builtin_amdgcn_permlane16_swap(w[0][0], w[1][0], false, false);
      const auto hi = __builtin_amdgcn_permlane16_swap(w[0][1], w[1][1], false, false);
      const int64_t p = p0 + 128 * at.wp + 16 * (F + (at.g & 1)) + 8 * (at.g >> 1);
      if (row && p < a.np)
        *reinterpret_cast<uint4*>(a.out + q * a.np + p) = make_uint4(lo[0], hi[0], lo[1], hi[1]);
    }
  }
}

// Both products of a piece in one launch, the one with the longer tiles first: the
// short tiles of the other fill the compute units that its last round leaves idle.
// Bound by the matrix cores at the clock that the power limit leaves: 4096 tokens,
// 131072 words, hidden 7168 1.32 to 1.41 PFLOP/s, and with 1024 tokens (short tiles of dW) the
// main loop runs at 1.6 GHz, with 64 tokens at 2.3.  Loading the next tile's stages
// before the stores, fewer instructions in the epilogue, streaming stores and half the
// workgroups in reverse order each left the launch as long as it was: a shorter
// epilogue lowers the main loop's clock.
__global__ __launch_bounds__(kThreads, 1) void k_products(Product dx, Product dw, int dx_first) {
  __shared__ LossSmem sm;
  const int first = dx_first ? dx.blocks : dw.blocks, block = (int)blockIdx.x;
  if ((block < first) == (dx_first != 0))
    product_tile<false>(sm, dx, dx_first ? block : block - first);
  else
    product_tile<true>(sm, dw, dx_first ? block - first : block);
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
int64_t small_tiles(int64_t n) { return (n + kSmallTile - 1) / kSmallTile; }

// How many of `words` words of logits go by large tiles: all of them, or whole
// rounds of the chip where the rest is one round of small tiles (none of them, where
// everything is).  A round of small tiles takes about half as long as one of large
// ones.  Hidden size 1024, all small / all large, us: 128 tokens, 32000 words (250
// small tiles) 25.8 / 33.8; 128 x 64000 (500) 46.2 / 38.9; 256 x 32000 (500) 40.9 /
// 33.6.  1000 x 50021 x 2048, three rounds and 56 small tiles / four: 175 / 197.
int64_t large_words(const LossArgs& a, int64_t words) {
  const int64_t cus = std::max(1, device_cu_count()), nq = std::max<int64_t>(1, tiles(a.T));
  const int64_t whole = tiles(words) * nq / cus * cus / nq * kTile;
  const int64_t left = words - whole;
  return left > 0 && small_tiles(left) * small_tiles(a.T) <= cus ? whole : words;
}
// Forward passes of at most 64 tokens that k_loss_few takes.  Up to 8 tokens: all of
// more than one round of small tiles.  Else those whose tiles would leave so much of
// the chip's last round empty that rereading x for every 64 words, which grows with the
// tokens, costs less.  Words x hidden (small tiles), us, against the tiles: 8 tokens,
// 65536 x 4096 (512) 121 and 136, 131072 x 4096 (1024) 223 and 211, 32000 x 4096 (250)
// 62 and 47; 16 / 32 / 64 tokens, 16384 x 4096 (128) 27 / 31 / 38 and 42 / 43 / 44,
// 35328 x 2136 (276) 41 / 43 / 59 and 50 / 50 / 50, 70016 x 2048 (547) 69 / 79 / 109 and
// 72 / 73 / 74, 131072 x 4096 234 / 251 / 333 and 209 / 211 / 216.
bool few_tokens(const LossArgs& a) {
  const int64_t n = small_tiles(a.V), cus = std::max(1, device_cu_count());
  const int64_t room = (n + cus - 1) / cus * cus;  // small tiles in as many rounds
  if (a.T < 1 || a.T > 64) return false;
  return (a.T <= 8 && n > cus) || 5 * room >= (6 + (a.T + 15) / 16) * n;
}
int64_t few_blocks(const LossArgs& a) {
  return std::min<int64_t>((a.V + kFewWords - 1) / kFewWords,
                           4 * std::max(1, device_cu_count()));
}
// Rows of statistics, and workgroups, of such a launch.
int64_t part_rows(int64_t words, int64_t large) {
  return tiles(large) + (words > large ? small_tiles(words - large) : 0);
}
int64_t tile_blocks(const LossArgs& a, int64_t words, int64_t large) {
  return tiles(large) * tiles(a.T) +
         (words > large ? small_tiles(words - large) * small_tiles(a.T) : 0);
}

// Ranges of k for a product: none takes more stages than about two thirds of what a
// compute unit gets of the launch's work (so that the longest tiles do not outlast
// the rest), none less than 512 of k; the partials stay below two tiles a unit.
// A tile's start and end cost about as much as kTileStages stages.  A share of a
// quarter / half / two thirds / all of it, us: 1000 tokens, 50021 words, hidden 2048
// 779 / 762 / 752 / 748; 64 x 131072 x 7168 1656 / 1687 / 1685 / 1740.
constexpr int64_t kTileStages = 8;
int64_t stages(int64_t k) { return (k + 63) / 64; }
int product_ranges(int64_t np, int64_t nq, int64_t k, int64_t work) {
  const int64_t n = tiles(np) * tiles(nq), cus = std::max(1, device_cu_count());
  const int64_t share = std::max<int64_t>(1, work * 2 / (3 * cus));
  return (int)std::max<int64_t>(
      1, std::min({(stages(k) + share - 1) / share, k / 512, 2 * cus / n}));
}
int64_t product_work(int64_t np, int64_t nq, int64_t k) {
  return tiles(np) * tiles(nq) * (stages(k) + kTileStages);
}

// Words of a piece: its d stays within kPieceBytes, and the pieces of one vocabulary
// are alike.  64 MiB / 256 MiB / 1 GiB / 4 GiB of d, ms: 4096 tokens, 131072 words,
// hidden 7168 22.3 / 22.0 / 21.6 / 21.7; 16384 x 32000 x 1024 4.35 / 3.76 / 3.60 / 3.60:
// what a piece costs beside its products (dx in fp32, the ends of its launches).
constexpr int64_t kPieceBytes = INT64_C(1) << 30;
int64_t piece_words(const LossArgs& a) {
  const int64_t most = std::min<int64_t>(
      std::max<int64_t>(kTile, kPieceBytes / (2 * a.T) / kTile * kTile), INT64_C(1) << 21);
  const int64_t pieces = (a.V + most - 1) / most;
  return up((a.V + pieces - 1) / pieces, kTile);
}

// Ranges of the two products of a piece of `words` words; the same where only one
// gradient is wanted, which then has the same bits.
struct PieceRanges {
  int dx, dw;
};
PieceRanges piece_ranges(const LossArgs& a, int64_t words) {
  const int64_t work = product_work(a.H, a.T, words) + product_work(a.H, words, a.T);
  return {product_ranges(a.H, a.T, words, work), product_ranges(a.H, words, a.T, work)};
}

// Offsets of the gradient's workspace.
struct GradSpace {
  int64_t piece, d, acc, part_x, part_w, bytes;
};
GradSpace grad_space(const LossArgs& a, bool need_x, bool need_w) {
  GradSpace s{};
  s.piece = piece_words(a);
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += up(bytes, 256);
    return o;
  };
  s.d = take(a.T * s.piece * 2);
  if (need_x && s.piece < a.V) s.acc = take(a.T * a.H * 4);
  int64_t part_x = 0, part_w = 0;
  const int64_t last = a.V - (a.V - 1) / s.piece * s.piece;
  for (const int64_t words : {std::min(s.piece, a.V), last}) {
    const PieceRanges r = piece_ranges(a, words);
    if (need_x && r.dx > 1) part_x = std::max(part_x, r.dx * a.T * a.H * 4);
    if (need_w && r.dw > 1) part_w = std::max(part_w, r.dw * words * a.H * 4);
  }
  s.part_x = take(part_x);
  s.part_w = take(part_w);
  s.bytes = at;
  return s;
}

// Cuts a product into `ranges` of k (fewer where they come out empty) and gives its
// number of workgroups; with more than one they write partials.
Product cut(Product p, int ranges, float* partials, float* acc) {
  p.range = up((p.k + ranges - 1) / ranges, 64);
  const int used = (int)((p.k + p.range - 1) / p.range);
  p.blocks = (int32_t)(tiles(p.np) * tiles(p.nq) * used);
  p.out32 = acc;
  if (used > 1) {
    p.out = nullptr;
    p.before = nullptr;
    p.out32 = partials;
  }
  return p;
}
hipError_t join(const Product& p, int ranges, float* partials, float* acc, hipStream_t stream) {
  const int64_t range = up((p.k + ranges - 1) / ranges, 64), n = p.np * p.nq;
  const int used = (int)((p.k + range - 1) / range);
  if (used <= 1) return hipSuccess;
  hipLaunchKernelGGL(k_product_join, dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, stream,
                     partials, used, n, p.before, p.out, acc);
  return hipGetLastError();
}

}  // namespace

// Rows of statistics of the forward pass.
static int64_t forward_rows(const LossArgs& a) {
  return few_tokens(a) ? few_blocks(a) : part_rows(a.V, large_words(a, a.V));
}

int64_t loss_workspace_bytes(const LossArgs& a) {
  return up(forward_rows(a) * a.T * 8, 256) + up(a.T * 4, 256) * 2;
}

hipError_t launch_loss(LossArgs a, uint8_t* ws, hipStream_t stream) {
  if (a.T > 0) {
    const int64_t rows = forward_rows(a);
    a.part = reinterpret_cast<float2*>(ws);
    a.target_logit = reinterpret_cast<float*>(ws + up(rows * a.T * 8, 256));
    if (!a.token_loss) a.token_loss = a.target_logit + up(a.T * 4, 256) / 4;
    if (few_tokens(a)) {
      const int n = (int)((a.V + kFewWords - 1) / kFewWords);
      const dim3 grid((unsigned)rows);
      if (a.T <= 16)
        hipLaunchKernelGGL((k_loss_few<1>), grid, dim3(kThreads), 0, stream, a, n);
      else if (a.T <= 32)
        hipLaunchKernelGGL((k_loss_few<2>), grid, dim3(kThreads), 0, stream, a, n);
      else
        hipLaunchKernelGGL((k_loss_few<4>), grid, dim3(kThreads), 0, stream, a, n);
    } else {
      const int64_t large = large_words(a, a.V);
      hipLaunchKernelGGL(k_loss_fwd, dim3((unsigned)tile_blocks(a, a.V, large)), dim3(kThreads), 0,
                         stream, a, large);
    }
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    hipLaunchKernelGGL(k_loss_join, dim3((unsigned)((a.T + kJoinTokens - 1) / kJoinTokens)),
                       dim3(kJoinTokens * kJoinRuns), 0, stream, a, (int)rows);
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
  a.d = reinterpret_cast<uint16_t*>(ws + s.d);
  float* acc = reinterpret_cast<float*>(ws + s.acc);
  float* part_x = reinterpret_cast<float*>(ws + s.part_x);
  float* part_w = reinterpret_cast<float*>(ws + s.part_w);
  for (int64_t v0 = 0; v0 < a.V; v0 += s.piece) {
    const int64_t words = std::min<int64_t>(s.piece, a.V - v0), width = up(words, kTile);
    int64_t large = large_words(a, words);
    if (large == words) large = width;
    hipLaunchKernelGGL(k_loss_grad_tile, dim3((unsigned)tile_blocks(a, width, large)),
                       dim3(kThreads), 0, stream, a, v0, (int)width, (int)large);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    const PieceRanges r = piece_ranges(a, words);
    Product px{}, pw{};
    if (!a.per_token) {
      px.scale = pw.scale = a.grad_loss;
      px.scale2 = pw.scale2 = a.stats + 2 * a.T;
    }
    px.np = pw.np = a.H;
    if (dx) {  // dx[t][h] = sum over words of d[t][v] W[v][h]
      px.P = a.w + v0 * a.ldw;
      px.ldp = a.ldw;
      px.Q = a.d;
      px.ldq = width;
      px.nq = a.T;
      px.k = words;
      px.before = v0 > 0 ? acc : nullptr;
      px.live = a.stats + a.T;
      px.out = v0 + words == a.V ? dx : nullptr;
    }
    if (dw) {  // dW[v][h] = sum over tokens of d[t][v] x[t][h]
      pw.P = a.x;
      pw.ldp = a.ldx;
      pw.Q = a.d;
      pw.ldq = width;
      pw.nq = words;
      pw.k = a.T;
      pw.out = dw + v0 * a.H;
    }
    const Product cx = dx ? cut(px, r.dx, part_x, acc) : px;
    const Product cw = dw ? cut(pw, r.dw, part_w, nullptr) : pw;
    const bool dx_first = dx && (!dw || cx.range >= cw.range);
    hipLaunchKernelGGL(k_products, dim3((unsigned)(cx.blocks + cw.blocks)), dim3(kThreads), 0,
                       stream, cx, cw, (int)dx_first);
    if ((err = hipGetLastError()) != hipSuccess) return err;
    if (dx && (err = join(px, r.dx, part_x, acc, stream)) != hipSuccess) return err;
    if (dw && (err = join(pw, r.dw, part_w, nullptr, stream)) != hipSuccess) return err;
  }
  return hipSuccess;
}

}  // namespace mxgg
