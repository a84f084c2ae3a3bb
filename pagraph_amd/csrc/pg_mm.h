// Tiles of matrix products on the matrix cores (gfx950), for operands of 16-bit parts whose reduction range is padded to whole
// tiles of 64: acc[BM x BN] += sum over parts and k of A(m, k) B(n, k), fp32 accumulation.
//
// Tiles travel from memory into LDS without passing through registers (16 bytes a lane), one tile ahead of the one being
// multiplied, two buffers, one barrier a step. An operand is stored either way round:
//   ROWS: p[row][k], k contiguous     -> LDS tile [rows][64], fragments are plain 16-byte reads
//   COLS: p[k][row], row contiguous   -> LDS tile [64][rows], fragments come from the transposing LDS reads (4 x 16 blocks)
// so that no operand is ever transposed in memory. LDS-direct loads write 64 lanes x 16 bytes contiguously, so the bank swizzle is
// applied to the address each lane fetches: the 16-byte chunk at position p of a tile row is chunk p ^ swizzle(row).
#pragma once
#include "pg_elem.h"

namespace pg {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x16 mma(bf16_t, s16x8 a, s16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(f16_t, s16x8 a, s16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

enum { ROWS = 0, COLS = 1 };
constexpr int kDepth = 64;                     // reduction depth of a tile

typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void glb_void;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// 64 lanes x 16 bytes: lane l's bytes land at lds + 16 l (lds wave-uniform)
__device__ __forceinline__ void dma16(const void* g, void* lds) {
  __builtin_amdgcn_global_load_lds((glb_void*)g, (lds_void*)lds, 16, 0, 0);
}

// one operand of a tile: R rows of the product from r0 on
struct Operand {
  const void* p;
  int64_t ld, part;      // elements between rows, between parts
  int64_t r0;            // first row of the tile (ROWS) / first column (COLS)
  int64_t rows;          // memory rows that exist: beyond them the last one is read again (its products are dropped or meet zeros)
  int64_t width;         // COLS: columns that exist (a multiple of 8)
};

template <int KIND, int R, int WAVES>
struct TileLoad {
  static constexpr int T = R * kDepth * 2 / 1024 / WAVES;       // 1 KB pieces per wave
  uint32_t row[T], col[T];
  const char* base;
  uint32_t ld2;
  int64_t limit;
  __device__ __forceinline__ void init(const Operand& o, int wave, int lane) {
    ld2 = (uint32_t)o.ld * 2;
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const int piece = wave * T + t;
      if constexpr (KIND == ROWS) {
        const int r = piece * 8 + lane / 8, chunk = (lane & 7) ^ ((r >> 1) & 7);
        const int64_t last = o.rows - 1 - o.r0;
        row[t] = (uint32_t)(r < last ? r : last) * ld2 + chunk * 16;
      } else {
        constexpr int CH = R / 8, PER = 64 / CH;                 // chunks of a tile row, tile rows of a piece
        const int k = piece * PER + lane / CH, chunk = (lane % CH) ^ swz(k);
        const int64_t last = o.width - 8 - o.r0, c = chunk * 8 < last ? chunk * 8 : last;
        row[t] = k;
        col[t] = (uint32_t)(c * 2);
      }
    }
    base = (const char*)o.p + (KIND == ROWS ? o.r0 * o.ld : o.r0) * 2;
    limit = o.rows - 1;
  }
  static __device__ __forceinline__ int swz(int k) { return (((k & 3) | ((k >> 1) & 4)) << 1) & (R / 8 - 1); }
  __device__ __forceinline__ void issue(int64_t part, int64_t k0, short* lds, int wave) const {
    if constexpr (KIND == ROWS) {
      const char* b = base + (part + k0) * 2;
#pragma unroll
      for (int t = 0; t < T; ++t) dma16(b + row[t], lds + (wave * T + t) * 512);
    } else {
      const char* b = base + part * 2 + k0 * ld2;
      const int64_t left = limit - k0;
      const uint32_t last = left < kDepth ? (uint32_t)left : kDepth;
#pragma unroll
      for (int t = 0; t < T; ++t) dma16(b + ((row[t] < last ? row[t] : last) * ld2 + col[t]), lds + (wave * T + t) * 512);
    }
  }
};

// the MFMA operand of rows [rb, rb + 32) at depth 16 kk: lane l holds row rb + l % 32, k = 16 kk + 8 (l / 32) + 0..7
template <int KIND, int R>
__device__ __forceinline__ s16x8 fragment(const short* lds, int rb, int kk, int lane) {
  if constexpr (KIND == ROWS) {
    const int r = rb + (lane & 31), chunk = kk * 2 + (lane >> 5);
    return *reinterpret_cast<const s16x8*>(lds + r * kDepth + ((chunk ^ ((r >> 1) & 7)) << 3));
  } else {
    const int i = lane & 15, g = lane >> 4;
    const int k = kk * 16 + (g >> 1) * 8 + (i >> 2), chunk = (rb >> 3) + (g & 1) * 2 + ((i & 3) >> 1);
    const short* s = lds + k * R + ((chunk ^ TileLoad<COLS, R, 1>::swz(k)) << 3) + (i & 1) * 4;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)s);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(s + 4 * R));        // k + 4: the same swizzle
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// Tile shape: BM x BN by WR x WC waves. NP parts per value: 1, or 3 (fp32 as three bf16 parts, six products, smallest first)
template <typename E_, int NP_, int BM_, int BN_, int WR_, int WC_>
struct Shape {
  typedef E_ E;
  static constexpr int NP = NP_, BM = BM_, BN = BN_, WR = WR_, WC = WC_, WAVES = WR * WC, THREADS = WAVES * 64;
  static constexpr int FI = BM / WR / 32, FJ = BN / WC / 32;    // 32 x 32 blocks of a wave
  static constexpr int TILE = (BM + BN) * kDepth;               // elements of one buffer
};

template <typename S, int KA, int KB>
__device__ __forceinline__ void mm_step(const short* __restrict__ cur, short* __restrict__ next, bool more, const TileLoad<KA, S::BM, S::WAVES>& la,
                                        const TileLoad<KB, S::BN, S::WAVES>& lb, int64_t pa, int64_t pb, int64_t k_next, int wave, int lane,
                                        f32x16 (&acc)[S::FI][S::FJ]) {
  if (more) {
    la.issue(pa, k_next, next, wave);
    lb.issue(pb, k_next, next + S::BM * kDepth, wave);
  }
  const int wm = wave / S::WC, wn = wave % S::WC;
#pragma unroll
  for (int kk = 0; kk < kDepth / 16; ++kk) {
    s16x8 a[S::FI], b[S::FJ];
#pragma unroll
    for (int i = 0; i < S::FI; ++i) a[i] = fragment<KA, S::BM>(cur, wm * (S::BM / S::WR) + i * 32, kk, lane);
#pragma unroll
    for (int j = 0; j < S::FJ; ++j) b[j] = fragment<KB, S::BN>(cur + S::BM * kDepth, wn * (S::BN / S::WC) + j * 32, kk, lane);
#pragma unroll
    for (int i = 0; i < S::FI; ++i)
#pragma unroll
      for (int j = 0; j < S::FJ; ++j) acc[i][j] = mma(typename S::E(), a[i], b[j], acc[i][j]);
  }
}

// acc += the product over [k_lo, k_hi), whole tiles. buf0, buf1: S::TILE elements of LDS each; on return every wave may still be
// reading one of them (synchronise before reusing them).
template <typename S, int KA, int KB>
__device__ __forceinline__ void mm_product(const Operand& oa, const Operand& ob, int64_t k_lo, int64_t k_hi, short* buf0, short* buf1,
                                           f32x16 (&acc)[S::FI][S::FJ]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  TileLoad<KA, S::BM, S::WAVES> la;
  TileLoad<KB, S::BN, S::WAVES> lb;
  la.init(oa, wave, lane);
  lb.init(ob, wave, lane);
  const int64_t steps1 = (k_hi - k_lo) / kDepth;
  const int64_t steps = S::NP == 3 ? 6 * steps1 : steps1;
  if (steps <= 0) return;
  // parts of the step's operands: (2,0) (1,1) (0,2) (1,0) (0,1) (0,0)
  int seg = 0;
  int64_t k = k_lo;
  auto part_a = [&]() -> int64_t { return S::NP == 3 ? (seg == 0 ? 2 : seg == 1 || seg == 3 ? 1 : 0) * oa.part : 0; };
  auto part_b = [&]() -> int64_t { return S::NP == 3 ? (seg == 2 ? 2 : seg == 1 || seg == 4 ? 1 : 0) * ob.part : 0; };
  auto advance = [&] {
    k += kDepth;
    if (S::NP == 3 && k >= k_hi) {
      k = k_lo;
      ++seg;
    }
  };
  la.issue(part_a(), k, buf0, wave);
  lb.issue(part_b(), k, buf0 + S::BM * kDepth, wave);
  for (int64_t s = 0; s < steps; s += 2) {
    advance();
    __syncthreads();                                   // this step's tile has landed, the other buffer's readers are done
    mm_step<S, KA, KB>(buf0, buf1, s + 1 < steps, la, lb, part_a(), part_b(), k, wave, lane, acc);
    if (s + 1 < steps) {
      advance();
      __syncthreads();
      mm_step<S, KA, KB>(buf1, buf0, s + 2 < steps, la, lb, part_a(), part_b(), k, wave, lane, acc);
    }
  }
}

// Workgroups go round the 8 XCDs in turn: give each XCD a contiguous run of tiles, so that its own L2 sees a tile's neighbours
__device__ __forceinline__ int64_t xcd_run(int64_t b, int64_t total) {
  const int64_t per = total / 8, rest = total % 8, x = b % 8, i = b / 8;
  return x * per + (x < rest ? x : rest) + i;
}

}  // namespace pg
