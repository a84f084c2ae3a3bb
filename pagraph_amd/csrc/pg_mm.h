// Tiles of matrix products on the matrix cores (gfx950), for operands of 16-bit parts whose reduction range is padded to whole
// multiples of 64: acc[BM x BN] += sum over parts and k of A(m, k) B(n, k), fp32 accumulation.
//
// Tiles of depth 32 travel from memory into LDS without passing through registers (16 bytes a lane), into NB buffers, NB - 1 tiles
// ahead of the one being multiplied, one barrier a step: a step of a 256 x 256 tile is about 1000 cycles of matrix work, a load
// that misses the XCD's L2 takes two to three times that. An operand is stored either way round:
//   ROWS: p[row][k], k contiguous     -> LDS tile [rows][32], fragments are plain 16-byte reads
//   COLS: p[k][row], row contiguous   -> LDS tile [32][rows], fragments come from the transposing LDS reads (4 x 16 blocks)
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
constexpr int kDepth = 32;                     // reduction depth of a tile
constexpr int kPad = 64;                       // what rows of parts are padded to

typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void glb_void;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// 64 lanes x 16 bytes: lane l's bytes land at lds + 16 l (lds wave-uniform)
__device__ __forceinline__ void dma16(const void* g, void* lds) {
  __builtin_amdgcn_global_load_lds((glb_void*)g, (lds_void*)lds, 16, 0, 0);
}

// a value that is the same for all lanes, where the compiler cannot know it (what came out of a division, say): in scalar registers
// from here on, so that addresses made from it are scalar too
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)v) | (int64_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32;
}

// one operand of a tile: R rows of the product from r0 on. Memory holds whole tiles of the reduction range
struct Operand {
  const void* p;
  int64_t ld, part;      // elements between rows, between parts
  int64_t r0;            // first row of the tile (ROWS) / first column (COLS)
  int64_t rows;          // ROWS: rows that exist; beyond them the last one is read again (its products are dropped)
  int64_t width;         // COLS: columns that exist (a multiple of 8); likewise
};

template <int KIND, int R, int WAVES>
struct TileLoad {
  static constexpr int T = R * kDepth * 2 / 1024 / WAVES;       // 1 KB pieces per wave
  uint32_t offset[T];                                           // the lane's, from the tile's first element
  const char *base, *at;                                        // the tile's at depth 0, the next one to load
  int64_t step, part;
  __device__ __forceinline__ void init(const Operand& o, int64_t k_lo, int wave, int lane) {
    const uint32_t ld2 = (uint32_t)o.ld * 2;
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const int piece = wave * T + t;
      if constexpr (KIND == ROWS) {
        const int r = piece * 16 + lane / 4, chunk = (lane & 3) ^ ((r >> 2) & 3);
        const int64_t last = o.rows - 1 - o.r0;
        offset[t] = (uint32_t)(r < last ? r : last) * ld2 + chunk * 16;
      } else {
        constexpr int CH = R / 8, PER = 64 / CH;                 // chunks of a tile row, tile rows of a piece
        const int k = piece * PER + lane / CH, chunk = (lane % CH) ^ swz(k);
        const int64_t last = o.width - 8 - o.r0, c = chunk * 8 < last ? chunk * 8 : last;
        offset[t] = k * ld2 + (uint32_t)(c * 2);
      }
    }
    step = KIND == ROWS ? kDepth * 2 : kDepth * o.ld * 2;
    part = o.part * 2;
    base = (const char*)o.p + (KIND == ROWS ? (o.r0 * o.ld + k_lo) : (o.r0 + k_lo * o.ld)) * 2;
  }
  __device__ __forceinline__ void start(int p) { at = base + p * part; }
  __device__ __forceinline__ void issue(short* lds, int wave) {
#pragma unroll
    for (int t = 0; t < T; ++t) dma16(at + offset[t], lds + (wave * T + t) * 512);
    at += step;
  }
  // COLS: 16 lanes of a transposing read take 32 bytes of four tile rows, their neighbours the next 32 bytes of the same rows: the
  // four (with the other half-wave's: eight) rows are moved 64 bytes apart in the 256 bytes of banks
  static __device__ __forceinline__ int swz(int k) {
    return R >= 256 ? ((k & 3) | ((k >> 1) & 4)) << 2 : R == 128 ? (k & 3) << 2 : ((k >> 1) & 1) << 2;
  }
};

// the MFMA operand of rows [rb, rb + 32) at depth 16 kk: lane l holds row rb + l % 32, k = 16 kk + 8 (l / 32) + 0..7
// (restrict: with alias information on every read the compiler leaves the waits for loads into LDS to wait_loads; without, it
// waits for all of them before a transposing read)
template <int KIND, int R>
__device__ __forceinline__ s16x8 fragment(const short* __restrict__ lds, int rb, int kk, int lane) {
  if constexpr (KIND == ROWS) {
    const int r = rb + (lane & 31), chunk = kk * 2 + (lane >> 5);
    return *reinterpret_cast<const s16x8*>(lds + r * kDepth + ((chunk ^ ((r >> 2) & 3)) << 3));
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
template <typename E_, int NP_, int BM_, int BN_, int WR_, int WC_, int NB_>
struct Shape {
  typedef E_ E;
  static constexpr int NP = NP_, BM = BM_, BN = BN_, WR = WR_, WC = WC_, NB = NB_, WAVES = WR * WC, THREADS = WAVES * 64;
  static constexpr int FI = BM / WR / 32, FJ = BN / WC / 32;    // 32 x 32 blocks of a wave
  static constexpr int TILE = (BM + BN) * kDepth;               // elements of one buffer
};

// LDS of a kernel: ONE array of NB tile buffers and `extra` shorts behind them (several variables would carry alias
// information of their own, see fragment)
#define PG_MM_LDS(S, name, extra) __shared__ __align__(16) short name[S::NB * S::TILE + (extra)]

template <int VM>
__device__ __forceinline__ void wait_loads() {          // at most VM loads of this wave still under way
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((VM & 15) | 7 << 4 | 15 << 8 | (VM >> 4) << 14);
}
__device__ __forceinline__ void wait_reads() { __builtin_amdgcn_s_waitcnt(15 | 7 << 4 | 0 << 8 | 3 << 14); }      // none of its LDS reads

template <typename S, int KA, int KB>
struct Product {
  static constexpr int LOADS = TileLoad<KA, S::BM, S::WAVES>::T + TileLoad<KB, S::BN, S::WAVES>::T;     // of a wave, per tile
  TileLoad<KA, S::BM, S::WAVES> la;
  TileLoad<KB, S::BN, S::WAVES> lb;
  int seg, seg_steps, seg_left, wave, lane;

  // parts of the operands in turn: (2,0) (1,1) (0,2) (1,0) (0,1) (0,0)
  __device__ __forceinline__ void start() {
    la.start(S::NP == 3 ? (seg == 0 ? 2 : seg == 1 || seg == 3 ? 1 : 0) : 0);
    lb.start(S::NP == 3 ? (seg == 2 ? 2 : seg == 1 || seg == 4 ? 1 : 0) : 0);
  }
  __device__ __forceinline__ void issue(short* buf) {
    la.issue(buf, wave);
    lb.issue(buf + S::BM * kDepth, wave);
    if (S::NP == 3 && --seg_left == 0) {
      seg_left = seg_steps;
      ++seg;
      start();
    }
  }
  struct Fragments {
    s16x8 a[S::FI], b[S::FJ];
  };
  __device__ __forceinline__ void read(const short* tile, int kk, Fragments& f) const {
    const int wm = wave / S::WC, wn = wave % S::WC;
#pragma unroll
    for (int i = 0; i < S::FI; ++i) f.a[i] = fragment<KA, S::BM>(tile, wm * (S::BM / S::WR) + i * 32, kk, lane);
#pragma unroll
    for (int j = 0; j < S::FJ; ++j) f.b[j] = fragment<KB, S::BN>(tile + S::BM * kDepth, wn * (S::BN / S::WC) + j * 32, kk, lane);
  }
  static __device__ __forceinline__ void multiply(const Fragments& f, f32x16 (&acc)[S::FI][S::FJ]) {
#pragma unroll
    for (int i = 0; i < S::FI; ++i)
#pragma unroll
      for (int j = 0; j < S::FJ; ++j) acc[i][j] = mma(typename S::E(), f.a[i], f.b[j], acc[i][j]);
  }
  // One step. f: the tile's fragments of depth 0, read half a step ago; leaves with the next tile's (LAST: there is none). Reads run
  // behind the matrix instructions of the half tile before. At the barrier every wave's loads of the next tile have landed (full:
  // those of the NB - 2 tiles behind it may still be under way) and every wave has its second half of this tile in registers: its
  // buffer is the one that is filled again, with the tile NB further on.
  template <bool LAST>
  __device__ __forceinline__ void step(short* cur, const short* next, bool full, bool more, Fragments& f, f32x16 (&acc)[S::FI][S::FJ]) {
    // in this order, whatever the scheduler thinks of the registers; the reads waited for were issued half a tile ago
    Fragments g;
    wait_reads();
    read(cur, 1, g);
    __builtin_amdgcn_sched_barrier(0);
    multiply(f, acc);
    __builtin_amdgcn_sched_barrier(0);
    wait_reads();
    if constexpr (!LAST) {
      if (full) wait_loads<(S::NB - 2) * LOADS>(); else wait_loads<0>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      read(next, 0, f);
      if (more) issue(cur);
    }
    __builtin_amdgcn_sched_barrier(0);
    multiply(g, acc);
    __builtin_amdgcn_sched_barrier(0);
  }
};

// What bounds it: the waves of a workgroup come to the barrier of each step together, so the two of a SIMD read, wait and multiply at the
// same time. 256 x 256 tiles of K = 1024: matrix units busy in 56 to 59 % of the cycles, LDS in 22 % without bank conflicts, waves
// waiting 26 to 30 % of theirs: 1.0 to 1.15 PF in bf16 where the library's 16384^3 product reaches 1.47 on the same card.
template <typename S, int KA, int KB>
__device__ __forceinline__ void mm_run(Product<S, KA, KB>& p, int steps, short* buf, f32x16 (&acc)[S::FI][S::FJ]) {
  // steps is even: reduction ranges are multiples of kPad
  constexpr int N = Product<S, KA, KB>::LOADS, NB = S::NB;
  static_assert(kDepth == 32, "two fragments a tile");
  typename Product<S, KA, KB>::Fragments f;
  const int first = steps < NB ? steps : NB;
  for (int i = 0; i < first; ++i) p.issue(buf + i * S::TILE);
  if (first == NB) wait_loads<(NB - 1) * N>(); else wait_loads<N>();          // (two or more tiles)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  p.read(buf, 0, f);
  int left = steps;
  for (; left >= 2 * NB; left -= NB) {
#pragma unroll
    for (int i = 0; i < NB; ++i) p.template step<false>(buf + i * S::TILE, buf + (i + 1) % NB * S::TILE, true, true, f, acc);
  }
  int at = 0;
#pragma unroll 1
  for (; left > 1; --left) {
    const int next = at + 1 == NB ? 0 : at + 1;
    p.template step<false>(buf + at * S::TILE, buf + next * S::TILE, left >= NB, left > NB, f, acc);
    at = next;
  }
  p.template step<true>(buf + at * S::TILE, buf, false, false, f, acc);
}

// acc += the product over [k_lo, k_hi), whole tiles. On return every wave may still be reading the buffers (synchronise before
// reusing them).
template <typename S, int KA, int KB>
__device__ __forceinline__ void mm_product(const Operand& oa, const Operand& ob, int64_t k_lo, int64_t k_hi, short* buf,
                                           f32x16 (&acc)[S::FI][S::FJ]) {
  Product<S, KA, KB> p;
  p.lane = threadIdx.x & 63;
  p.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  p.la.init(oa, k_lo, p.wave, p.lane);
  p.lb.init(ob, k_lo, p.wave, p.lane);
  p.seg = 0;
  p.seg_steps = p.seg_left = uniform((int)((k_hi - k_lo) / kDepth));
  p.start();
  const int steps = (S::NP == 3 ? 6 : 1) * p.seg_steps;
  if (steps <= 0) return;
  mm_run<S, KA, KB>(p, steps, buf, acc);
}

// Workgroups go round the 8 XCDs in turn: give each XCD a contiguous run of tiles, so that its own L2 sees a tile's neighbours
__device__ __forceinline__ uint32_t xcd_run(uint32_t b, uint32_t total) {
  const uint32_t per = total / 8, rest = total % 8, x = b % 8, i = b / 8;
  return x * per + (x < rest ? x : rest) + i;
}

}  // namespace pg
