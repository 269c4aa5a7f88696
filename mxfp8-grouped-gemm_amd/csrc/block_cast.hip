// bf16 -> e4m3 with one fp32 scale for each block of 128.
//
//   s = max(amax (1 / 448), 2^-126),  q = e4m3(x / s)         (fp32; nearest even)
//
// A block is 1 x 128 along the row (activations), 128 x 1 along the tokens
// (operands of the weight gradient, written transposed, restarting at every
// group) or a 128 x 128 tile (weights).  amax is taken over the bit patterns of
// |x|, so a NaN makes its block's scale and payload NaN; an infinity makes the
// scale infinite.  1 / s is one division a block; a quotient is a product and its
// correction (BlockDivisor).
//
// Memory-bound: 2 bytes read and 1.03 written an element and output.  16384 x 7168 by rows
// or transposed 55 us (6.5 TB/s), both 77 (6.2); 32 weights of 4096 x 7168 507 (5.5), with
// the transposed copy 687.
#include "mx_device.h"
#include "mxgg_internal.h"

namespace mxgg {
namespace {

constexpr int kBlk = 128;

// Largest value of the 16 lanes of a row, in every one of them.
__device__ __forceinline__ uint32_t row16_max(uint32_t x) {
  x = quad_max(x);
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xF, 0xF, false));  // half mirror
  return max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x140, 0xF, 0xF, false));
}

__device__ __forceinline__ uint32_t cvt4(float a, float b, float c, float d) {
  const uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, (int)w, true);
}
__device__ __forceinline__ uint2 cvt_chunk(const uint4& v, const BlockDivisor& d) {
  return make_uint2(cvt4(d(bf16_lo(v.x)), d(bf16_hi(v.x)), d(bf16_lo(v.y)), d(bf16_hi(v.y))),
                    cvt4(d(bf16_lo(v.z)), d(bf16_hi(v.z)), d(bf16_lo(v.w)), d(bf16_hi(v.w))));
}

// Rows in blocks of 1 x 128: a wave takes one block column of 32 rows, eight loads of
// four rows (16 lanes, 256 bytes, a row), and writes the 32 scales as one run.
constexpr int kRowsWave = 32;
__global__ __launch_bounds__(256) void k_block_rows(const uint16_t* __restrict__ x, int64_t rows,
                                                    int64_t cols, int64_t ldx, uint8_t* q,
                                                    int64_t ldq, float* s, int64_t lds) {
  const int lane = threadIdx.x & 63, g = lane >> 4;
  const uint32_t wide = (uint32_t)((cols + 4 * kBlk - 1) / (4 * kBlk));
  const int64_t kb = (int64_t)(blockIdx.x % wide) * 4 + (threadIdx.x >> 6);
  const int64_t col = kb * kBlk + 8 * (lane & 15);
  const int64_t row0 = (int64_t)(blockIdx.x / wide) * kRowsWave;
  if (kb * kBlk >= cols) return;
  const bool in = col < cols;
  uint4 v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = row0 + 4 * i + g;
    v[i] = make_uint4(0, 0, 0, 0);
    if (in && row < rows) v[i] = *reinterpret_cast<const uint4*>(x + row * ldx + col);
  }
  float own = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = row0 + 4 * i + g;
    const float sc = block_scale(bf16_bits_to_f32(row16_max(amax16_of_chunk(v[i]))));
    if ((lane & 15) == i) own = sc;
    const uint2 w = cvt_chunk(v[i], BlockDivisor(sc));
    if (in && row < rows) store_stream(q + row * ldq + col, w);
  }
  const int64_t row = row0 + 4 * (lane & 15) + g;
  if ((lane & 15) < 8 && row < rows) s[kb * lds + row] = own;
}

struct CastTile {
  const uint16_t* x;     // [batch][rows][ldx]
  const int32_t* ends;   // or nullptr: one group of all rows
  const int32_t* pend;
  uint8_t* q;            // by rows: [batch][rows][ldq], or nullptr
  float* s;              // ROW: [cols / 128][lds]; TILE: [batch][rows / 128][cols / 128]
  uint8_t* qt;           // transposed: [batch][cols][ldqt], or nullptr
  float* st;             // ROW: [tokens / 128][ldst]; TILE: [batch][cols / 128][rows / 128]
  int64_t rows, cols, ldx, ldq, lds, ldqt, ldst, cap;
  int32_t E;
};

// A 128 x 128 tile of a workgroup: thread (tr, c) holds rows 8 tr .. + 7 of the
// eight columns from 8 c on.  The transposed payload goes through LDS, column by
// column (128 bytes each, 8-byte slots XORed with the column's chunk), and leaves in
// whole lines.  TILE: one scale for the tile, in both outputs.
template <bool TILE, bool ROW, bool COL>
__global__ __launch_bounds__(256) void k_block_tile(CastTile a) {
  __shared__ uint64_t bytes[kBlk * 16];
  __shared__ uint4 part[4][16];
  __shared__ int32_t ends_s[kMaxGroups], pend_s[kMaxGroups];
  const int t = threadIdx.x, tr = t >> 4, c = t & 15, lane = t & 63, wave = t >> 6;
  const int64_t P = (int64_t)blockIdx.y * kBlk, col = (int64_t)blockIdx.x * kBlk + 8 * c;
  const int64_t batch = blockIdx.z;
  const uint16_t* x = a.x + batch * a.rows * a.ldx;
  int64_t tok0 = P;
  int ntok = (int)min((int64_t)kBlk, a.rows - P);
  if (!TILE && a.ends) {
    stage_group_tables(a.ends, a.pend, a.E, a.rows, ends_s, pend_s);
    __syncthreads();
    padded_run_tokens(P, kBlk, ends_s, pend_s, a.E, tok0, ntok);
  }
  ntok = max(ntok, 0);
  const bool in = col < a.cols;
  uint4 v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = make_uint4(0, 0, 0, 0);
    if (in && 8 * tr + i < ntok)
      v[i] = *reinterpret_cast<const uint4*>(x + (tok0 + 8 * tr + i) * a.ldx + col);
  }
  // largest |x| of every column over the thread's rows, then over the tile
  uint4 m = make_uint4(0, 0, 0, 0);
  if (COL || TILE) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m.x = pk_max_u16(m.x, abs_bf16x2(v[i].x));
      m.y = pk_max_u16(m.y, abs_bf16x2(v[i].y));
      m.z = pk_max_u16(m.z, abs_bf16x2(v[i].z));
      m.w = pk_max_u16(m.w, abs_bf16x2(v[i].w));
    }
    for (int d = 16; d < 64; d <<= 1) {
      m.x = pk_max_u16(m.x, __shfl_xor(m.x, d));
      m.y = pk_max_u16(m.y, __shfl_xor(m.y, d));
      m.z = pk_max_u16(m.z, __shfl_xor(m.z, d));
      m.w = pk_max_u16(m.w, __shfl_xor(m.w, d));
    }
    if (lane < 16) part[wave][lane] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint4 o = part[w][c];
      m.x = pk_max_u16(m.x, o.x);
      m.y = pk_max_u16(m.y, o.y);
      m.z = pk_max_u16(m.z, o.z);
      m.w = pk_max_u16(m.w, o.w);
    }
  }
  float tile = 1.0f;
  if (TILE) {
    tile = block_scale(bf16_bits_to_f32(row16_max(amax16_of_chunk(m))));
    if (t == 0) {
      const int64_t nb = (a.rows + kBlk - 1) / kBlk, kb = (a.cols + kBlk - 1) / kBlk;
      a.s[(batch * nb + blockIdx.y) * kb + blockIdx.x] = tile;
      if (COL) a.st[(batch * kb + blockIdx.x) * nb + blockIdx.y] = tile;
    }
  }
  const BlockDivisor of_tile(tile);
  if (ROW) {
    float own = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float sc = tile;
      if (!TILE) {
        sc = block_scale(bf16_bits_to_f32(row16_max(amax16_of_chunk(v[i]))));
        if (c == i) own = sc;
      }
      const uint2 w = cvt_chunk(v[i], TILE ? of_tile : BlockDivisor(sc));
      if (in && 8 * tr + i < ntok)
        store_stream(a.q + (batch * a.rows + tok0 + 8 * tr + i) * a.ldq + col, w);
    }
    if (!TILE && c < 8 && 8 * tr + c < ntok) a.s[blockIdx.x * a.lds + tok0 + 8 * tr + c] = own;
  }
  if (COL) {
    const uint32_t words[4] = {m.x, m.y, m.z, m.w};
    float sc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t top = (j & 1) ? words[j >> 1] >> 16 : words[j >> 1] & 0xFFFFu;
      sc[j] = TILE ? tile : block_scale(bf16_bits_to_f32(top));
      const BlockDivisor d = TILE ? of_tile : BlockDivisor(sc[j]);
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t w = j < 2 ? v[i].x : j < 4 ? v[i].y : j < 6 ? v[i].z : v[i].w;
        f[i] = d((j & 1) ? bf16_hi(w) : bf16_lo(w));
      }
      const uint32_t lo = cvt4(f[0], f[1], f[2], f[3]), hi = cvt4(f[4], f[5], f[6], f[7]);
      bytes[(8 * c + j) * 16 + (tr ^ c)] = (uint64_t)hi << 32 | lo;
    }
    if (!TILE && tr == 0 && in) {
#pragma unroll
      for (int j = 0; j < 8; ++j) a.st[blockIdx.y * a.ldst + col + j] = sc[j];
    }
    __syncthreads();
    // 16 bytes a thread, eight threads a column
#pragma unroll
    for (int pass = 0; pass < 4; ++pass) {
      const int oc = 32 * pass + (t >> 3), u = 2 * (t & 7), k = oc >> 3;
      const int64_t ocol = (int64_t)blockIdx.x * kBlk + oc;
      const uint64_t lo = bytes[oc * 16 + (u ^ k)], hi = bytes[oc * 16 + ((u + 1) ^ k)];
      const int64_t at = P + 8 * u;
      if (ocol >= a.cols || at >= a.cap) continue;
      uint8_t* p = a.qt + (batch * a.cols + ocol) * a.ldqt + at;
      if (at + 16 <= a.cap && (reinterpret_cast<uintptr_t>(p) & 15u) == 0) {
        __builtin_nontemporal_store(
            u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)},
            reinterpret_cast<u32x4*>(p));
      } else {
        for (int b = 0; b < 16; ++b)
          if (at + b < a.cap) p[b] = (uint8_t)((b < 8 ? lo >> (8 * b) : hi >> (8 * (b - 8))));
      }
    }
  }
}

// Padded cumulative ends: every group rounded up to whole blocks of 128 tokens.
__global__ __launch_bounds__(256) void k_block_pad_ends(const int32_t* ends, int E, int64_t rows,
                                                        int32_t* pend) {
  __shared__ int32_t m[kMaxGroups];
  monotone_ends_to_lds(ends, E, rows, m);
  if (threadIdx.x != 0) return;
  int32_t at = 0;
  for (int g = 0; g < E; ++g) {
    const int32_t n = m[g] - (g ? m[g - 1] : 0);
    at += (n + kBlk - 1) / kBlk * kBlk;
    pend[g] = at;
  }
}

template <bool TILE, bool ROW, bool COL>
hipError_t run_tile(const CastTile& a, int64_t batch, hipStream_t stream) {
  const dim3 grid((unsigned)((a.cols + kBlk - 1) / kBlk),
                  (unsigned)(((TILE ? a.rows : a.cap) + kBlk - 1) / kBlk), (unsigned)batch);
  hipLaunchKernelGGL((k_block_tile<TILE, ROW, COL>), grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_block_rows(const uint16_t* x, int64_t rows, int64_t cols, int64_t ldx,
                             uint8_t* q, int64_t ldq, float* s, int64_t lds, hipStream_t stream) {
  const dim3 grid((unsigned)((cols + 4 * kBlk - 1) / (4 * kBlk) *
                             ((rows + kRowsWave - 1) / kRowsWave)));
  hipLaunchKernelGGL(k_block_rows, grid, dim3(256), 0, stream, x, rows, cols, ldx, q, ldq, s, lds);
  return hipGetLastError();
}

hipError_t launch_block_tokens(const uint16_t* x, int64_t rows, int64_t cols, int64_t ldx,
                               const int32_t* ends, int64_t E, int64_t cap, uint8_t* q,
                               int64_t ldq, float* s, int64_t lds, uint8_t* qt, float* st,
                               int64_t ldst, int32_t* pend, hipStream_t stream) {
  if (ends) {
    hipLaunchKernelGGL(k_block_pad_ends, dim3(1), dim3(256), 0, stream, ends, (int)E, rows, pend);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  if (cap == 0 || cols == 0) return hipSuccess;
  CastTile a{};
  a.x = x;
  a.ends = ends;
  a.pend = pend;
  a.q = q;
  a.s = s;
  a.qt = qt;
  a.st = st;
  a.rows = rows;
  a.cols = cols;
  a.ldx = ldx;
  a.ldq = ldq;
  a.lds = lds;
  a.ldqt = a.cap = cap;
  a.ldst = ldst;
  a.E = (int32_t)E;
  return q ? run_tile<false, true, true>(a, 1, stream) : run_tile<false, false, true>(a, 1, stream);
}

hipError_t launch_block_weight(const uint16_t* w, int64_t E, int64_t N, int64_t K, uint8_t* q,
                               float* s, uint8_t* qt, float* st, hipStream_t stream) {
  CastTile a{};
  a.x = w;
  a.q = q;
  a.s = s;
  a.qt = qt;
  a.st = st;
  a.rows = a.cap = a.ldqt = N;
  a.cols = a.ldx = a.ldq = K;
  return qt ? run_tile<true, true, true>(a, E, stream) : run_tile<true, true, false>(a, E, stream);
}

}  // namespace mxgg
