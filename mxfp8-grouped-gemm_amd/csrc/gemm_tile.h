// Main loop of the 256 x 256 GEMM tiles: operands streamed through LDS by DMA,
// matrix instructions over registers that are refilled as they free up.  One
// tile is D[p][q] = sum_k P[p][k] Q[q][k] for row-major operands contiguous along
// k; operands, stages and k ranges are counted in BYTES, so the same loop runs
//   e4m3 : v_mfma_scale_f32_16x16x128_f8f6f4, a 128-byte stage is one k step
//   bf16 : v_mfma_f32_16x16x32_bf16, a stage is two k steps: the two 16-byte
//          chunks (g and g + 4) that lane m + 16g holds of row m are its operands
//          of the first and of the second one
// Both instructions return D[4g + r][c] in register r of lane c + 16g.
// A bf16 operand may also be K-MAJOR: rows of the contraction, contiguous along p
// (or q).  A stage is then 64 rows of 256 columns, 512 bytes each, and the
// fragments are read with the transposing ds_read_b64_tr_b16.
#pragma once

#include <type_traits>

#include "mx_device.h"
#include "mxgg_internal.h"

namespace mxgg {
namespace {

constexpr int kTileP = 256;
constexpr int kTileQ = 256;
constexpr int kStageK = 128;    // contraction elements (bytes) per stage
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr uint32_t kOpBytes = 256u * kStageK;          // one operand of one stage: 32 KB
constexpr uint32_t kScaleOff = 2u * kOpBytes;          // scale rows after P and Q data
// Scale block b of a stage at kScaleOff + b * kScaleBlk: [P, Q][256] bytes and
// 64 bytes of padding, so that the lanes of blocks 0 and 1 (one half-wave of
// a scale read) fall on different banks.
constexpr uint32_t kScaleBlk = 576;
constexpr uint32_t kStageBytes = kScaleOff + 4u * kScaleBlk;
constexpr uint32_t kOobOffset = 0x80000000u;           // beyond every num_records we create
// Store instructions of one wave for a tile that lies inside dW, in the weight
// gradient whose stores overlap the next tile: store_bf16_direct's loops, two
// rows of chunks per P half and Q fragment.
constexpr uint32_t kDirectFrags = 8, kDirectHalves = 2, kDirectRows = 2;
constexpr int kAheadStores = kDirectFrags * kDirectHalves * kDirectRows;
// Loads of one wave for one stage: 16 of data, then 2 of scales.
constexpr int kStageLoads = 16, kScaleLoads = 2;
static_assert(kStageLoads + kScaleLoads + kAheadStores <= 63, "vmcnt counts to 63");

// Raw 128-bit buffer descriptor (gfx9 layout: base, stride 0, num_records,
// dst_sel/format word).  Offsets at or past num_records read as zero.
typedef int32_t desc_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ desc_t make_desc(const void* base, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  desc_t d;
  d[0] = (int32_t)(uint32_t)a;
  d[1] = (int32_t)((uint32_t)(a >> 32) & 0xFFFFu);
  d[2] = (int32_t)bytes;
  d[3] = 0x00020000;
  return d;
}

// Readable bytes of a block-major scale array with `nblk` block-rows of
// stride `ld` holding `rows` rows: the scale DMA reads whole 4-row dwords.
__device__ __forceinline__ uint32_t scale_extent(int64_t nblk, int64_t ld, int64_t rows) {
  return (uint32_t)((nblk - 1) * ld + ((rows + 3) & ~(int64_t)3));
}

// One operand of a tile.  Rows at or past `rows` are not clamped: their byte
// offsets lie beyond the descriptor's num_records ((rows-1)*ld + K) and read
// as zero.  The C ABI bounds (rows + 256) * ld below 2^32 so these offsets do
// not wrap.
struct Operand {
  desc_t data;    // [rows][ld] e4m3
  desc_t scale;   // [k-blocks][lds] E8M0, block-major
  uint32_t ld;    // bytes per data row
  uint32_t lds;   // bytes per scale block-row (multiple of 4)
  uint32_t row0;  // first operand row of this tile (multiple of 4)
  // Operand row of tile row 128, minus row0: 128 for a plain tile of 256
  // consecutive rows; F for the gate+up tile of the fused SwiGLU forward
  // (tile rows 0..127 = gate rows, 128..255 = the matching up rows F later).
  uint32_t hi;
  // K-major: first row of the contraction, at the tile's first column; ld as above.
  // Offsets stay within a stage (the stage's rows are the base), so `bytes`, from
  // base to the end of the last row, may pass 32 bits; rows past it read as zero.
  const uint8_t* base;
  int64_t bytes;
};

// Cache-policy operand of the buffer store builtins: the nontemporal bit.
constexpr int kCacheNT = 2;

typedef __attribute__((address_space(3))) void lds_void_t;

__device__ __forceinline__ uint32_t wave_id() {
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
}

// Byte offset of a __shared__ object inside the workgroup's LDS allocation.
__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return (uint32_t)(uintptr_t)((const lds_void_t*)p);
}

// 16-byte chunk swizzle inside a 128-byte LDS slot.  gfx950 serves a
// ds_read_b128 one half-wave (32 lanes, 512 B) at a time over 64 four-byte
// banks; it runs at full rate when every bank holds at most two of the
// half-wave's dwords.  A half-wave reads one chunk from each of 32 consecutive
// slots; the bank quad of (slot s, chunk c) is 8*(s mod 2) + (c ^ swz(s)), and
// with swz(s) = (s/2) mod 8 the 16 quads are each hit exactly twice.
__device__ __forceinline__ uint32_t swz(uint32_t s) { return (s >> 1) & 7u; }

// Wait for this wave's DMA except the youngest `N` instructions and for all
// of its LDS reads, then the workgroup barrier.  Written as assembly so the
// compiler's waitcnt pass can neither relax nor move it (it does not see the
// DMA, and would drop the lgkmcnt part for reads whose results are only used
// after the barrier).
template <int N>
__device__ __forceinline__ void wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// LDS-DMA issued from inline assembly: M0 holds the wave's LDS destination,
// each lane its byte offset into the buffer.  The compiler does not track
// these loads, so it inserts no wait for them in front of LDS reads of the
// other stage; every consumer waits explicitly in wait_barrier().
// M0 is reserved by the compiler, which warns about the clobber; on gfx950 it
// only uses M0 for LDS-DMA, GWS and message instructions, none of which it
// emits in these kernels (the generated code writes M0 only here).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// soff: a wave-uniform byte offset added in the instruction's scalar offset
// field.  The buffer range check covers voff + soff (measured on gfx950: a
// scalar offset alone past num_records reads zero), so a per-load row step
// can ride there instead of costing a vector add per load.
__device__ __forceinline__ void dma_x4(const desc_t& d, uint32_t lds_addr, uint32_t voff,
                                       uint32_t soff = 0) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "buffer_load_dwordx4 %1, %2, %3 offen lds"
      :
      : "s"(lds_addr), "v"(voff), "s"(d), "s"(soff)
      : "memory", "m0");
}
__device__ __forceinline__ void dma_x1(const desc_t& d, uint32_t lds_addr, uint32_t voff,
                                       uint32_t soff = 0) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "buffer_load_dword %1, %2, %3 offen lds"
      :
      : "s"(lds_addr), "v"(voff), "s"(d), "s"(soff)
      : "memory", "m0");
}
#pragma clang diagnostic pop

// Per-thread state of the global -> LDS stream for one tile.
//  Data: wave w's i-th load (i = 0..7) fills LDS bytes [4096i + 1024w, +1024)
//  of an operand, lane l writing 16 B at +16l: slot s = 32i + 8w + l/8 at
//  physical chunk l%8, so the lane fetches logical chunk (l%8) ^ swz(s) of
//  tile row 128(i/4) + 4(8w + l/8) + i%4 (slots 128a + 32b + c hold rows
//  128a + 4c + b).  Eight lanes cover one
//  128-byte line.  swz(s) = (4w + l/16) mod 8 does not depend on i, and the
//  row moves by a lane-independent amount from load to load, so the lane keeps
//  one base offset per operand and adds a uniform step.  Chunks outside
//  [klo, kend) are fetched from an out-of-range offset and land as zeros.
//  Scales: wave w copies block k0/32 + w of both operands: 256 rows = 64 lanes
//  x 4 bytes in row order.  A block outside [klo, kend) lands as zeros (scale
//  2^-127 on zero payload).
//  K-major data (PK, QK): the LDS bytes are the same, row k = 8i + 2w + l/32 of the
//  stage at byte 512 k, and the lane fetches logical chunk (l%32) ^ 2 kswz(k) of that
//  row.  kswz(k) = (k mod 4) + 4 ((k/8) mod 2) changes with i by its last bit only:
//  one base offset for even and one for odd loads.
__device__ __forceinline__ uint32_t kswz(uint32_t k) { return (k & 3u) | ((k >> 3) & 1u) << 2; }

template <bool SCALED, bool MASK = false, bool PK = false, bool QK = false>
struct Stream {
  uint32_t vp, vq;   // lane offset of load 0 without k0
  uint32_t op, oq;   // K-major: lane offset of load 1, less its rows' step
  desc_t dp, dq;     // K-major: the stage's rows
  uint32_t kcol;     // lane's chunk column within a stage (bytes)
  uint32_t sp, sq;   // lane offset of its scale dword within a block-row
  uint32_t klo, kend;

  __device__ __forceinline__ void init(const Operand& P, const Operand& Q, uint32_t lo,
                                       uint32_t hi) {
    klo = lo;
    kend = hi;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = wave_id();
    kcol = 16u * ((lane & 7u) ^ ((4u * wave + (lane >> 4)) & 7u));
    const uint32_t r = 4u * (8u * wave + (lane >> 3));
    vp = (P.row0 + r) * P.ld + kcol;
    vq = (Q.row0 + r) * Q.ld + kcol;
    if constexpr (PK || QK) {
      const uint32_t k = 2u * wave + (lane >> 5);
      const uint32_t even = 16u * ((lane & 31u) ^ (kswz(k) << 1));
      if (PK) {
        vp = k * P.ld + even;
        op = k * P.ld + (even ^ 128u);
      }
      if (QK) {
        vq = k * Q.ld + even;
        oq = k * Q.ld + (even ^ 128u);
      }
    }
    if (SCALED) {
      sp = P.row0 + 4u * lane + (lane >= 32u ? P.hi - 128u : 0u);
      sq = Q.row0 + 4u * lane + (lane >= 32u ? Q.hi - 128u : 0u);
    }
  }

  // Lane offsets of stage k0 (an out-of-range base when the chunk is outside
  // [klo, kend); adding a step to it stays out of range).
  // MASK: a chunk that overlaps [klo, kend) at all is loaded (the bytes outside
  // are zeroed in registers after the fragment reads, mask_frags()).
  __device__ __forceinline__ void stage_base(const Operand& P, const Operand& Q, uint32_t k0,
                                             uint32_t& bp, uint32_t& bq) {
    const uint32_t k = k0 + kcol;
    const bool ok = (MASK ? k + 16u > klo : k >= klo) && k < kend;
    bp = ok ? vp + k0 : kOobOffset;
    bq = ok ? vq + k0 : kOobOffset;
    if (PK) dp = stage_rows(P, k0);
    if (QK) dq = stage_rows(Q, k0);
  }
  __device__ __forceinline__ static desc_t stage_rows(const Operand& X, uint32_t k0) {
    const int64_t off = (int64_t)(k0 >> 1) * X.ld, left = X.bytes - off;
    return make_desc(X.base + off, (uint32_t)(left < 0 ? 0 : left > 0x7FFFFFF0 ? 0x7FFFFFF0 : left));
  }

  __device__ __forceinline__ static uint32_t step(uint32_t i, const Operand& X) {
    return ((i >> 2) * X.hi + (i & 3u)) * X.ld;
  }

  __device__ __forceinline__ void load_p(uint8_t* stage, const Operand& P, uint32_t bp,
                                         uint32_t i) const {
    const uint32_t dst = lds_offset(stage) + 4096u * i + 1024u * wave_id();
    if constexpr (PK)
      dma_x4(dp, dst, (i & 1u) ? op : vp, 8u * i * P.ld);
    else
      dma_x4(P.data, dst, bp, step(i, P));
  }
  __device__ __forceinline__ void load_q(uint8_t* stage, const Operand& Q, uint32_t bq,
                                         uint32_t i) const {
    const uint32_t dst = lds_offset(stage) + kOpBytes + 4096u * i + 1024u * wave_id();
    if constexpr (QK)
      dma_x4(dq, dst, (i & 1u) ? oq : vq, 8u * i * Q.ld);
    else
      dma_x4(Q.data, dst, bq, step(i, Q));
  }
  // Scale rows of k-block k0/32 + wave; operand X = P (OP 0) or Q (OP 1).
  template <int OP>
  __device__ __forceinline__ void load_scale(uint8_t* stage, const Operand& X, uint32_t k0) const {
    if (!SCALED) return;
    const uint32_t wave = wave_id();
    const uint32_t blk = (k0 >> 5) + wave;
    const bool ok = blk >= (klo >> 5) && blk < (kend >> 5);
    // the block's row offset is wave-uniform: it rides in the scalar offset,
    // and an out-of-range block moves the whole load past num_records
    dma_x1(X.scale, lds_offset(stage) + kScaleOff + kScaleBlk * wave + 256u * OP, OP ? sq : sp,
           ok ? blk * X.lds : kOobOffset);
  }

  // The loads of a tile's first two stages (18 each with scales), stage 0 first.
  __device__ __forceinline__ void prologue(uint8_t* s0, uint8_t* s1, const Operand& P,
                                           const Operand& Q, uint32_t kbeg, uint32_t nst) {
    load_scale<0>(s0, P, kbeg);
    load_scale<1>(s0, Q, kbeg);
    issue_data(s0, P, Q, kbeg);
    if (nst > 1) {
      issue_data(s1, P, Q, kbeg + kStageK);
      load_scale<0>(s1, P, kbeg + kStageK);
      load_scale<1>(s1, Q, kbeg + kStageK);
    }
  }

  // The 16 data loads of one stage, back to back (prologue only).
  __device__ __forceinline__ void issue_data(uint8_t* stage, const Operand& P, const Operand& Q,
                                             uint32_t k0) {
    uint32_t bp, bq;
    stage_base(P, Q, k0, bp, bq);
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) load_p(stage, P, bp, i);
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) load_q(stage, Q, bq, i);
  }
};

// Operands of one stage in registers: 8 P fragments and 8 Q fragments of 16
// rows x 128 contraction bytes, and the scale dwords of the lane's 32-block
// for the P rows of fragment halves G = 0, 1 (sa[G]) and the Q rows of
// halves H = 0, 1 (sb[H]).
struct Frags {
  v8i a[8], b[8];
  uint32_t sa[2], sb[2];
};

// Per-lane LDS byte offsets (relative to a stage).
//   v_mfma_scale_f32_16x16x128_f8f6f4 (fp8) operand layout: lane m + 16g
//   serves row m of a fragment with contraction chunks g (bytes 0..15) and
//   g + 4 (bytes 16..31) of the 128-deep stage, the scale of 32-block b of
//   row m comes from lane m + 16b, and D[4g + r][c] sits in register r of
//   lane c + 16g.  Fragment f = 4G + i of wave row-half w holds tile rows
//   128w + 64G + 4m + i (m = 0..15): LDS slots 128w + 32i + 16G + m of the
//   DMA's slot layout.  Its scale byte is byte i of the dword of rows
//   128w + 64G + 4m .. +3 of the lane's block.
// K-major operands: fragment f of a wave half w is its columns 128w + 16f .. + 15.
// ds_read_b64_tr_b16 takes a 4 x 16 block from 16 lanes, lane i the four elements
// 4 (i%4) .. + 3 of row i/4, and returns column i: so lane i of group g reads row
// k = 8g + i/4 (+ 4 for the upper half of its eight, + 32 for the second k step), and
// its 16-byte chunk 2f + (i/2)%2 is XORed with 2 kswz(k), which is the same for
// those rows.  A read's 64 lanes then touch every bank twice.
struct FragAddr {
  uint32_t plo, phi, qlo, qhi, ps, qs;
  uint32_t kp, kq;  // K-major: fragment 0; fragment f at kp ^ 32 f

  __device__ __forceinline__ void init() {
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = threadIdx.x >> 6;
    const uint32_t wp = wave & 1u, wq = wave >> 1;
    const uint32_t m = lane & 15u, g = lane >> 4;
    // swz(128w + 32i + 16G + m) = swz(m) for every w, i, G
    const uint32_t sw = swz(m);
    const uint32_t rp = (wp * 128u + m) * kStageK, rq = kOpBytes + (wq * 128u + m) * kStageK;
    plo = rp + ((g ^ sw) << 4);
    phi = rp + (((g + 4u) ^ sw) << 4);
    qlo = rq + ((g ^ sw) << 4);
    qhi = rq + (((g + 4u) ^ sw) << 4);
    ps = kScaleOff + g * kScaleBlk + wp * 128u + 4u * m;
    qs = kScaleOff + 256u + g * kScaleBlk + wq * 128u + 4u * m;
  }

  __device__ __forceinline__ void init_k_major() {
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = threadIdx.x >> 6;
    const uint32_t wp = wave & 1u, wq = wave >> 1;
    const uint32_t m = lane & 15u, g = lane >> 4;
    const uint32_t k = 8u * g + (m >> 2);
    const uint32_t kb = 512u * k + (kswz(k) << 5) + 16u * ((m >> 1) & 1u) + 8u * (m & 1u);
    kp = kb + 256u * wp;
    kq = kOpBytes + kb + 256u * wq;
  }
};

// Byte offset of fragment f = 4G + i from fragment 0: 16G + 32i slots.
constexpr uint32_t frag_off(int f) {
  return 2048u * (uint32_t)(f >> 2) + 4096u * (uint32_t)(f & 3);
}

__device__ __forceinline__ v8i lds_v8i(const uint8_t* lo, const uint8_t* hi) {
  const uint4 a = *reinterpret_cast<const uint4*>(lo);
  const uint4 b = *reinterpret_cast<const uint4*>(hi);
  v8i f;
  f[0] = (int)a.x; f[1] = (int)a.y; f[2] = (int)a.z; f[3] = (int)a.w;
  f[4] = (int)b.x; f[5] = (int)b.y; f[6] = (int)b.z; f[7] = (int)b.w;
  return f;
}

// A K-major fragment from its lane address: eight contraction elements of each k step.
__device__ __forceinline__ v8i lds_k_major(const uint8_t* p) {
  typedef short v4s __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) v4s lds_v4s;
  v8i f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const u32x2 w = __builtin_bit_cast(
        u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                   (lds_v4s*)(p + 2048 * (k & 1) + 16384 * (k >> 1))));
    f[2 * k] = (int)w[0];
    f[2 * k + 1] = (int)w[1];
  }
  return f;
}

template <bool KM, int F>
__device__ __forceinline__ void read_a(const uint8_t* stage, const FragAddr& fa, Frags& f) {
  if constexpr (KM)
    f.a[F] = lds_k_major(stage + (fa.kp ^ (32u * F)));
  else
    f.a[F] = lds_v8i(stage + fa.plo + frag_off(F), stage + fa.phi + frag_off(F));
}
template <bool KM, int F>
__device__ __forceinline__ void read_b(const uint8_t* stage, const FragAddr& fa, Frags& f) {
  if constexpr (KM)
    f.b[F] = lds_k_major(stage + (fa.kq ^ (32u * F)));
  else
    f.b[F] = lds_v8i(stage + fa.qlo + frag_off(F), stage + fa.qhi + frag_off(F));
}
// Unscaled kernels use scale byte 127 (2^0) in every position.
template <bool SCALED, int G>
__device__ __forceinline__ void read_sa(const uint8_t* stage, const FragAddr& fa, Frags& f) {
  f.sa[G] = SCALED ? *reinterpret_cast<const uint32_t*>(stage + fa.ps + 64u * G) : 0x7F7F7F7Fu;
}
template <bool SCALED, int H>
__device__ __forceinline__ void read_sb(const uint8_t* stage, const FragAddr& fa, Frags& f) {
  f.sb[H] = SCALED ? *reinterpret_cast<const uint32_t*>(stage + fa.qs + 64u * H) : 0x7F7F7F7Fu;
}

// Both k steps of a bf16 stage: the low halves of two fragments, then the high ones.
__device__ __forceinline__ v4f mfma_bf16_stage(const v8i& a, const v8i& b, v4f c) {
  typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
  typedef int v4i __attribute__((ext_vector_type(4)));
  const auto lo = [](const v8i& x) { return __builtin_bit_cast(v8bf, (v4i){x[0], x[1], x[2], x[3]}); };
  const auto hi = [](const v8i& x) { return __builtin_bit_cast(v8bf, (v4i){x[4], x[5], x[6], x[7]}); };
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo(a), lo(b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi(a), hi(b), c, 0, 0, 0);
}

// One MFMA: P fragment PI against Q fragment QJ into accumulator 8 PI + QJ;
// op_sel picks byte PI % 4 of the P scale dword of half PI / 4 and byte
// QJ % 4 of the Q dword of half QJ / 4.
// BF16: both k steps of the stage, no scales.
template <bool BF16, int PI, int QJ>
__device__ __forceinline__ void mma(const Frags& f, v4f (&acc)[64]) {
  if constexpr (BF16) {
    acc[8 * PI + QJ] = mfma_bf16_stage(f.a[PI], f.b[QJ], acc[8 * PI + QJ]);
    return;
  }
  acc[8 * PI + QJ] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
      f.a[PI], f.b[QJ], acc[8 * PI + QJ], 0, 0, PI & 3, (int)f.sa[PI >> 2], QJ & 3,
      (int)f.sb[QJ >> 2]);
}

// Bytes of the 4-byte word at contraction position c that lie in [klo, kend),
// as a byte mask (0xFF per byte inside).
__device__ __forceinline__ uint32_t bytes_below(int n) {
  return n <= 0 ? 0u : (n >= 4 ? 0xFFFFFFFFu : (1u << (8 * n)) - 1u);
}
__device__ __forceinline__ uint32_t word_window(uint32_t c, uint32_t klo, uint32_t kend) {
  return bytes_below((int)kend - (int)c) & ~bytes_below((int)klo - (int)c);
}

// Byte masks of the lane's eight fragment dwords for the stage starting at
// k0: dwords 0..3 hold contraction chunk g (bytes k0 + 16g ..), dwords 4..7
// chunk g + 4.  Every fragment of the stage shares them.
struct KMask {
  uint32_t m[8];
};
__device__ __forceinline__ void k_mask(KMask& km, uint32_t k0, uint32_t klo, uint32_t kend) {
  const uint32_t g = (threadIdx.x & 63u) >> 4;
  const uint32_t clo = k0 + 16u * g, chi = clo + 64u;
#pragma unroll
  for (uint32_t d = 0; d < 4; ++d) {
    km.m[d] = word_window(clo + 4u * d, klo, kend);
    km.m[4 + d] = word_window(chi + 4u * d, klo, kend);
  }
}
// Zero the bytes of a fragment outside [klo, kend) (in both operands: a zero on
// one side alone would still turn a NaN code on the other into NaN).
__device__ __forceinline__ void apply_mask(v8i& x, const KMask& km) {
#pragma unroll
  for (int d = 0; d < 8; ++d) x[d] &= (int)km.m[d];
}

#define MXGG_FENCE() __builtin_amdgcn_sched_barrier(0)

// Workgroup barrier after this wave's LDS reads have returned (no wait on
// the DMA), as assembly for the same reason as wait_barrier().
__device__ __forceinline__ void release_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Accumulate D over k in [klo, kend) (both multiples of 32).  The stages start
// at klo rounded down to 128 so that every stage reads whole cache lines of
// rows whose stride is a multiple of 128; chunks below klo load as zeros.
//
// Stage s lives in slot s%2.  Its 64 MFMAs run P fragments 0..7 against Q
// fragments 0..3 (MFMA n = 4p + q), then against Q fragments 4..7 (n = 32 +
// 4p + q - 4).  Fragment registers are refilled as they free up, so one set of
// 128 VGPRs holds two stages at once and every read has MFMAs to land in:
//     0-8  the rest of stage s from slot s%2: P 4..7 (first used at 16..28),
//          the P scales of half 1 (first used at 16), Q 4..7 and the Q
//          scales of half 1 (first used at 32)
//      12  release barrier: every wave has read all of slot s%2 -> the 18
//          loads of stage s+2 into that slot, one per about three MFMAs up to
//          MFMA 62
//      32  publish barrier: everything older than the 7 loads issued since
//          the release, i.e. all of stage s+1, has landed
//   33-58  the first part of stage s+1 from the other slot: Q 0..3 (free since
//          MFMA 31) and P 0..3, each after its last use in stage s (MFMA
//          35 + 4p), and the scales of halves 0
// A load has at least 34 MFMAs (about 1100 cycles) to land before its
// publish.  Releasing later (MFMA 16 to 24) or placing the loads and reads on
// MFMA pairs measured slower.  The wait counts do not depend on whether
// scales are loaded: the scale loads of a stage come after its data loads,
// and the publish wait leaves exactly the 7 newest (data) loads in flight.
// MASK (unscaled only): [klo, kend) may have any bounds; chunks that straddle
// them are loaded whole and the bytes outside are zeroed in registers right
// after each fragment read.  Only experts whose token range is not a multiple
// of 16 take this path.
// AHEAD (scaled, bf16): the caller issued the loads of the first two stages
// itself (Stream::prologue), then exactly LEFT stores of the tile before,
// or waited for all of it.  vmcnt retires in issue order, so the first waits
// leave those stores in flight: they drain behind this tile's first two stages.
// With fewer stores the counts would reach into the loads; more vector-memory
// instructions (a spill) only make them stricter.
template <bool SCALED, bool MASK = false, bool AHEAD = false, bool BF16 = false, bool PK = false,
          bool QK = false, int LEFT = kAheadStores, class SM>
__device__ __forceinline__ void mainloop(SM& sm, const Operand& P, const Operand& Q,
                                         uint32_t klo, uint32_t kend, v4f (&acc)[64]) {
  static_assert(!(SCALED && MASK), "a scale block cannot be split by a token mask");
  static_assert(BF16 || !(PK || QK), "K-major operands are bf16");
  static_assert(!BF16 || !(SCALED || MASK), "bf16 operands have neither scales nor a byte mask");
  static_assert(SCALED || BF16 || !AHEAD, "the wait counts of AHEAD include the scale loads");
#pragma unroll
  for (int i = 0; i < 64; ++i) acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  if (kend <= klo) return;
  const uint32_t kbeg = klo & ~(uint32_t)(kStageK - 1);
  const uint32_t nst = (kend - kbeg + kStageK - 1) / kStageK;
  Stream<SCALED, MASK, PK, QK> st;
  st.init(P, Q, klo, kend);
  FragAddr fa;
  fa.init();
  if constexpr (PK || QK) fa.init_k_major();
  // Prologue: all of stage 0 and, if there is one, of stage 1 (issued here or by
  // the caller), then publish stage 0 and read the part of it that the loop
  // reads one stage ahead.
  if constexpr (!AHEAD) st.prologue(sm.ring[0], sm.ring[1], P, Q, kbeg, nst);
  constexpr int kLeft = AHEAD ? LEFT : 0;
  if (nst > 1)
    wait_barrier<kStageLoads + (SCALED ? kScaleLoads : 0) + kLeft>();
  else
    wait_barrier<kLeft>();
  MXGG_FENCE();
  Frags f;
  KMask km;
  if constexpr (MASK) k_mask(km, kbeg, klo, kend);
#define MASKA(F) \
  if constexpr (MASK) apply_mask(f.a[F], km)
#define MASKB(F) \
  if constexpr (MASK) apply_mask(f.b[F], km)
  {
    const uint8_t* r0 = sm.ring[0];
    read_b<QK, 0>(r0, fa, f); MASKB(0);
    read_b<QK, 1>(r0, fa, f); MASKB(1);
    read_b<QK, 2>(r0, fa, f); MASKB(2);
    read_b<QK, 3>(r0, fa, f); MASKB(3);
    read_a<PK, 0>(r0, fa, f); MASKA(0);
    read_a<PK, 1>(r0, fa, f); MASKA(1);
    read_a<PK, 2>(r0, fa, f); MASKA(2);
    read_a<PK, 3>(r0, fa, f); MASKA(3);
    read_sa<SCALED, 0>(r0, fa, f);
    read_sb<SCALED, 0>(r0, fa, f);
  }
  // The final reads fetch a stale slot and are never used, so the stage body has
  // no branches.  Two loops over it: the stages whose slot takes a later stage,
  // then the last two (or fewer) without loads.  Loads past the end would fetch
  // zeros, but each holds its wave's issue like any other: a weight gradient
  // over 256 tokens is two stages, and 36 of its 72 loads were such (bf16 dW,
  // 32 experts, N 7168, K 2048, 128 / 256 / 512 tokens each: 232 -> 216,
  // 260 -> 250, 339 -> 321 us; contractions of 16 stages and more level).
  uint32_t s = 0;
  auto stage = [&](auto loads) __attribute__((always_inline)) {
    constexpr bool LOADS = decltype(loads)::value;
    uint8_t* cur = sm.ring[s & 1u];
    uint8_t* nxt = sm.ring[(s & 1u) ^ 1u];
    uint32_t bp = 0, bq = 0;
    if constexpr (LOADS) st.stage_base(P, Q, kbeg + (s + 2) * kStageK, bp, bq);
      mma<BF16, 0, 0>(f, acc); read_a<PK, 4>(cur, fa, f); MASKA(4); MXGG_FENCE();
      mma<BF16, 0, 1>(f, acc); read_sa<SCALED, 1>(cur, fa, f); MXGG_FENCE();
      mma<BF16, 0, 2>(f, acc); read_a<PK, 5>(cur, fa, f); MASKA(5); MXGG_FENCE();
      mma<BF16, 0, 3>(f, acc); read_b<QK, 4>(cur, fa, f); MASKB(4); MXGG_FENCE();
      mma<BF16, 1, 0>(f, acc); read_a<PK, 6>(cur, fa, f); MASKA(6); MXGG_FENCE();
      mma<BF16, 1, 1>(f, acc); read_b<QK, 5>(cur, fa, f); MASKB(5); MXGG_FENCE();
      mma<BF16, 1, 2>(f, acc); read_a<PK, 7>(cur, fa, f); MASKA(7); MXGG_FENCE();
      mma<BF16, 1, 3>(f, acc); read_b<QK, 6>(cur, fa, f); MASKB(6); MXGG_FENCE();
      mma<BF16, 2, 0>(f, acc); read_sb<SCALED, 1>(cur, fa, f); read_b<QK, 7>(cur, fa, f); MASKB(7); MXGG_FENCE();
      mma<BF16, 2, 1>(f, acc); MXGG_FENCE();
      mma<BF16, 2, 2>(f, acc); MXGG_FENCE();
      mma<BF16, 2, 3>(f, acc); MXGG_FENCE();
      release_barrier();
      MXGG_FENCE();
      mma<BF16, 3, 0>(f, acc); if constexpr (LOADS) st.load_p(cur, P, bp, 0); MXGG_FENCE();
      mma<BF16, 3, 1>(f, acc); MXGG_FENCE();
      mma<BF16, 3, 2>(f, acc); MXGG_FENCE();
      mma<BF16, 3, 3>(f, acc); if constexpr (LOADS) st.load_p(cur, P, bp, 1); MXGG_FENCE();
      mma<BF16, 4, 0>(f, acc); MXGG_FENCE();
      mma<BF16, 4, 1>(f, acc); MXGG_FENCE();
      mma<BF16, 4, 2>(f, acc); if constexpr (LOADS) st.load_p(cur, P, bp, 2); MXGG_FENCE();
      mma<BF16, 4, 3>(f, acc); MXGG_FENCE();
      mma<BF16, 5, 0>(f, acc); MXGG_FENCE();
      mma<BF16, 5, 1>(f, acc); if constexpr (LOADS) st.load_p(cur, P, bp, 3); MXGG_FENCE();
      mma<BF16, 5, 2>(f, acc); MXGG_FENCE();
      mma<BF16, 5, 3>(f, acc); MXGG_FENCE();
      mma<BF16, 6, 0>(f, acc); if constexpr (LOADS) st.load_p(cur, P, bp, 4); MXGG_FENCE();
      mma<BF16, 6, 1>(f, acc); MXGG_FENCE();
      mma<BF16, 6, 2>(f, acc); MXGG_FENCE();
      mma<BF16, 6, 3>(f, acc); if constexpr (LOADS) st.load_p(cur, P, bp, 5); MXGG_FENCE();
      mma<BF16, 7, 0>(f, acc); MXGG_FENCE();
      mma<BF16, 7, 1>(f, acc); MXGG_FENCE();
      mma<BF16, 7, 2>(f, acc); if constexpr (LOADS) st.load_p(cur, P, bp, 6); MXGG_FENCE();
      mma<BF16, 7, 3>(f, acc); MXGG_FENCE();
      if (AHEAD && (LOADS ? s == 0 : nst <= 2))
        wait_barrier<(LOADS ? 7 : 0) + kLeft>();
      else
        wait_barrier<LOADS ? 7 : 0>();
      MXGG_FENCE();
      if constexpr (MASK) k_mask(km, kbeg + (s + 1) * kStageK, klo, kend);
      mma<BF16, 0, 4>(f, acc); MXGG_FENCE();
      mma<BF16, 0, 5>(f, acc); read_b<QK, 0>(nxt, fa, f); MASKB(0); MXGG_FENCE();
      mma<BF16, 0, 6>(f, acc); if constexpr (LOADS) st.load_p(cur, P, bp, 7); MXGG_FENCE();
      mma<BF16, 0, 7>(f, acc); MXGG_FENCE();
      mma<BF16, 1, 4>(f, acc); read_a<PK, 0>(nxt, fa, f); MASKA(0); MXGG_FENCE();
      mma<BF16, 1, 5>(f, acc); if constexpr (LOADS) st.load_q(cur, Q, bq, 0); MXGG_FENCE();
      mma<BF16, 1, 6>(f, acc); MXGG_FENCE();
      mma<BF16, 1, 7>(f, acc); read_b<QK, 1>(nxt, fa, f); MASKB(1); MXGG_FENCE();
      mma<BF16, 2, 4>(f, acc); if constexpr (LOADS) st.load_q(cur, Q, bq, 1); MXGG_FENCE();
      mma<BF16, 2, 5>(f, acc); read_a<PK, 1>(nxt, fa, f); MASKA(1); MXGG_FENCE();
      mma<BF16, 2, 6>(f, acc); MXGG_FENCE();
      mma<BF16, 2, 7>(f, acc); if constexpr (LOADS) st.load_q(cur, Q, bq, 2); MXGG_FENCE();
      mma<BF16, 3, 4>(f, acc); MXGG_FENCE();
      mma<BF16, 3, 5>(f, acc); read_b<QK, 2>(nxt, fa, f); MASKB(2); if constexpr (LOADS) st.load_q(cur, Q, bq, 3); MXGG_FENCE();
      mma<BF16, 3, 6>(f, acc); read_a<PK, 2>(nxt, fa, f); MASKA(2); MXGG_FENCE();
      mma<BF16, 3, 7>(f, acc); MXGG_FENCE();
      mma<BF16, 4, 4>(f, acc); if constexpr (LOADS) st.load_q(cur, Q, bq, 4); MXGG_FENCE();
      mma<BF16, 4, 5>(f, acc); MXGG_FENCE();
      mma<BF16, 4, 6>(f, acc); read_a<PK, 3>(nxt, fa, f); MASKA(3); MXGG_FENCE();
      mma<BF16, 4, 7>(f, acc); if constexpr (LOADS) st.load_q(cur, Q, bq, 5); MXGG_FENCE();
      mma<BF16, 5, 4>(f, acc); read_b<QK, 3>(nxt, fa, f); MASKB(3); MXGG_FENCE();
      mma<BF16, 5, 5>(f, acc); MXGG_FENCE();
      mma<BF16, 5, 6>(f, acc); if constexpr (LOADS) st.load_q(cur, Q, bq, 6); MXGG_FENCE();
      mma<BF16, 5, 7>(f, acc); read_sb<SCALED, 0>(nxt, fa, f); MXGG_FENCE();
      mma<BF16, 6, 4>(f, acc); if constexpr (LOADS) st.load_q(cur, Q, bq, 7); MXGG_FENCE();
      mma<BF16, 6, 5>(f, acc); MXGG_FENCE();
      mma<BF16, 6, 6>(f, acc); read_sa<SCALED, 0>(nxt, fa, f); MXGG_FENCE();
      mma<BF16, 6, 7>(f, acc); if constexpr (LOADS) st.template load_scale<0>(cur, P, kbeg + (s + 2) * kStageK); MXGG_FENCE();
      mma<BF16, 7, 4>(f, acc); MXGG_FENCE();
      mma<BF16, 7, 5>(f, acc); MXGG_FENCE();
      mma<BF16, 7, 6>(f, acc); if constexpr (LOADS) st.template load_scale<1>(cur, Q, kbeg + (s + 2) * kStageK); MXGG_FENCE();
      mma<BF16, 7, 7>(f, acc); MXGG_FENCE();
  };
  if constexpr (MASK) {
    // One loop, loads past the end included: the masks of both loops' fragments
    // outnumber the scalar registers (1024 x 1056 fp32 dW of 8 experts, 256
    // unscaled tokens off the 16-token grid: 20.2 -> 18.8 us).
    do stage(std::true_type{});
    while (++s < nst);
    wait_barrier<0>();
  } else {
    for (; s + 2 < nst; ++s) stage(std::true_type{});
    do stage(std::false_type{});
    while (++s < nst);
  }
#undef MASKA
#undef MASKB
  // Every wave has read its last fragments, and its loads have landed (the last
  // publish wait), before the next tile's loads reuse the slots.
  release_barrier();
}

#undef MXGG_FENCE

// Value of the neighbouring lane (lane ^ 1) through a DPP quad permutation
// [1, 0, 3, 2]: a VALU move, no LDS round trip (unlike a shuffle).
__device__ __forceinline__ uint32_t swap_lane_pair(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xF, 0xF, false);
}

}  // namespace
}  // namespace mxgg
