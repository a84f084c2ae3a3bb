// The class head's three passes for narrow rows (K padded to 64s: 16-bit rows up to 256, for gradients 192, fp32 rows up to 128):
// nothing of size [n, C] leaves the registers.
//
// One kernel, three roles. A wave keeps 32 XB "x" rows in registers as matrix operands and walks the other side's rows "y", whose
// tiles all four waves share in LDS:
//   STATS  x = rows of h, y = classes: running maximum and sum of exponentials of every row (per split of the classes)
//   DH     x = rows of h, y = classes: dh^T += W^T G^T
//   DW     x = classes,   y = rows:    dW^T += h^T G, db += sum G
// z^T[y][x] leaves the first product with a lane holding one x and, of 32 y, the 16 that 8 (e / 4) + 4 (lane / 32) + e % 4 names. G
// is computed in place and IS the second product's operand: that product sums over y, in whatever order, so the other operand is
// read from the same LDS tile in the order the lanes hold (the transposing LDS reads pick any four consecutive y). No exchange
// between lanes, no trip through LDS.
// 10 n K C operations (2 + 4 + 4) and no G traffic, against 8 n K C and 6 bytes (fp32: 18) per element of [n, C] of the wide form:
// as long as a wave's registers hold its operand rows and its sums, the traffic costs more than the repeated product.
// Measured: fp32 6000 x 64 -> 50000 STATS 213, DH 411, DW 439 us (180, 187, 175 TF of fp32 products, 1.0 to 1.1 PF of bf16 ones;
// the fp32 matrix instructions reach 154 TF), matrix units busy in 60, 63, 53 % of the cycles; bf16 4096 x 256 -> 32000 STATS 79 us =
// 0.85 PF, 38 %. A wave's products, then its exponentials and the splitting of G, then products again: other waves' products only
// partly cover what is between.
// Exponents are kept in base 2: z log2(e) + b log2(e) is one fused multiply-add, and fp16's scale of G, 2^14, rides in the exponent.
#pragma once
#include "pg_mm.h"

namespace pg {

enum { NX_STATS = 0, NX_DH = 1, NX_DW = 2 };

struct NxArgs {
  const void *x, *y;               // parts of rows of KP elements
  int64_t x_ld, x_part, x_rows, y_ld, y_part, y_rows;
  int64_t nx, ny, K;               // rows that count
  const float *side0, *side1, *side2, *side3;      // per y: STATS, DH: bias (base 2); DW: largest logits, labels, row factors, inverse
                                   // sums. Padded past ny
  const float *xa, *xi, *xb;       // per x: DH: largest logit, inverse sum, row factor; DW: bias (base 2)
  const int32_t* xlab;             // per x: STATS, DH: labels (-1: none)
  float2* part;                    // STATS: [x][splits]
  float* zlab;
  float *acc, *accb;               // partial sums [splits][nx][K], [splits][nx]
  void *out, *outb;                // direct outputs (one split)
  const float *f1, *f2;
  int64_t range;                   // y per split
  int32_t splits, scaled;          // scaled: rows carry factors other than 0 and 1
};

template <typename T> struct Mul;      // pg_xent_linear.hip

// 2^v of a logit less its row's largest one. A row without a gradient (ignored, or behind the last one) has the inverse sum 0 and
// must not reach dW with the NaN that an infinite weight makes of its zeros: the smaller of NaN and 0 is 0. In rows that count, the
// inverse sum itself is NaN then
__device__ __forceinline__ float lx_exp(float v) { return __builtin_amdgcn_exp2f(fminf(v, 0.f)); }

// 32-row blocks a wave keeps: two where the registers allow, each read of the other side's tile then feeds two products. Not in
// fp32: its six products a read keep the matrix units busy, and two blocks leave two waves of three (6000 x 64 -> 50000 with
// gradients 1244 against 1080 us)
constexpr int narrow_xb(int parts, int kp, int mode) { return parts == 3 ? 1 : mode == NX_STATS ? 2 : kp <= 64 ? 2 : 1; }

template <typename T, int KP, int XB_>
struct Narrow {
  static constexpr int NP = Mul<T>::NP, XB = XB_, KK = KP / 16, KB = KP / 32, WAVES = 4, XT = WAVES * 32 * XB;
  static constexpr int YB = NP * KP <= 256 ? 2 : 1, YT = 32 * YB;
  static constexpr int PART = YT * KP, TILE = NP * PART, PIECES = TILE * 2 / 1024, PER = PIECES / WAVES, CH = KP / 8;
  static_assert(PIECES % WAVES == 0, "whole pieces a wave");
};

// 16-byte chunk c of tile row y sits at position c ^ nx_swz(y): the 16 rows of a quarter-wave's row reads meet 16 different
// 16-byte banks, and of the 8 rows x 64 bytes of a transposing read no bank gets more than two
template <int KP>
__device__ __forceinline__ int nx_swz(int y) {
  return KP % 128 == 0 ? (y & 3) << 2 | ((y >> 2) & 3) : ((y >> 1) & 1) << 2 | ((y >> 2) & 1) << 1 | ((y >> 3) & 1);
}

template <typename N, int KP>
__device__ __forceinline__ s16x8 nx_rows(const short* __restrict__ part, int yb, int kk, int lane) {
  const int y = yb * 32 + (lane & 31), chunk = kk * 2 + (lane >> 5);
  return *reinterpret_cast<const s16x8*>(part + y * KP + ((chunk ^ nx_swz<KP>(y)) << 3));
}
// columns [32 mb, +32) of the tile, reduction over the 16 y that a lane's G values 8 s .. 8 s + 7 stand for
template <typename N, int KP>
__device__ __forceinline__ s16x8 nx_cols(const short* __restrict__ part, int yb, int s, int mb, int lane) {
  const int i = lane & 15, g = lane >> 4, h = g >> 1;
  const int chunk = mb * 4 + (g & 1) * 2 + ((i & 3) >> 1), y = yb * 32 + s * 16 + 4 * h + (i >> 2);
  const short* p = part + y * KP + (i & 1) * 4;
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + ((chunk ^ nx_swz<KP>(y)) << 3)));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 8 * KP + ((chunk ^ nx_swz<KP>(y + 8)) << 3)));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

template <typename T, int NP>
__device__ __forceinline__ f32x16 nx_mma(const s16x8 (&a)[NP], const s16x8 (&b)[NP], f32x16 c) {
  typedef typename Mul<T>::E E;
  if constexpr (NP == 3) {                 // smallest first
    c = mma(E(), a[2], b[0], c);
    c = mma(E(), a[1], b[1], c);
    c = mma(E(), a[0], b[2], c);
    c = mma(E(), a[1], b[0], c);
    c = mma(E(), a[0], b[1], c);
  }
  return mma(E(), a[0], b[0], c);
}

template <typename T, int KP, int XB, int MODE>
struct NarrowState {
  typedef Narrow<T, KP, XB> N;
  s16x8 xf[XB][N::KK][N::NP];
  f32x16 out[MODE == NX_STATS ? 1 : N::KB][XB];
  float m[XB], s[XB];                      // STATS: running maximum, sum; DW: s = column sum of G
  float xa[XB], xi[XB];
  int xl[XB];                              // STATS, DH: the lane's label; DW: the lane's class
  float zl[XB];
};

template <typename T, int KP, int XB, int MODE>
__device__ __forceinline__ void nx_step(const short* __restrict__ cur, const float* __restrict__ side, short* __restrict__ next,
                                        float* __restrict__ side_next, bool more, const NxArgs& a, int64_t y0, int64_t y_next, int wave, int lane,
                                        NarrowState<T, KP, XB, MODE>& st) {
  typedef Narrow<T, KP, XB> N;
  typedef typename Mul<T>::E E;
  constexpr float L2E = 1.44269504088896340736f;
  if (more) {
    const char* base = (const char*)a.y + y_next * a.y_ld * 2;
    const int64_t left = a.y_rows - 1 - y_next;
    const int last = left < N::YT ? (int)left : N::YT;
    const uint32_t ld2 = (uint32_t)a.y_ld * 2;
#pragma unroll
    for (int t = 0; t < N::PER; ++t) {
      const int piece = wave * N::PER + t, part = piece / (N::PIECES / N::NP);
      const int lin = (piece % (N::PIECES / N::NP)) * 64 + lane, row = lin / N::CH, chunk = (lin % N::CH) ^ nx_swz<KP>(row);
      dma16(base + part * a.y_part * 2 + ((uint32_t)(row < last ? row : last) * ld2 + chunk * 16), next + piece * 512);
    }
    if (wave == 0) {
      __builtin_amdgcn_global_load_lds((glb_void*)(a.side0 + y_next + lane), (lds_void*)side_next, 4, 0, 0);
      if constexpr (MODE == NX_DW) {
        __builtin_amdgcn_global_load_lds((glb_void*)(a.side1 + y_next + lane), (lds_void*)(side_next + 64), 4, 0, 0);
        __builtin_amdgcn_global_load_lds((glb_void*)(a.side3 + y_next + lane), (lds_void*)(side_next + 128), 4, 0, 0);
        if (a.scaled) __builtin_amdgcn_global_load_lds((glb_void*)(a.side2 + y_next + lane), (lds_void*)(side_next + 192), 4, 0, 0);
      }
    }
  }
  const int h4 = 4 * (lane >> 5);
#pragma unroll 1
  for (int yb = 0; yb < N::YB; ++yb) {
    f32x16 z[XB] = {};
#pragma unroll
    for (int kk = 0; kk < N::KK; ++kk) {
      s16x8 yf[N::NP];
#pragma unroll
      for (int p = 0; p < N::NP; ++p) yf[p] = nx_rows<N, KP>(cur + p * N::PART, yb, kk, lane);
#pragma unroll
      for (int b = 0; b < XB; ++b) z[b] = nx_mma<T, N::NP>(yf, st.xf[b][kk], z[b]);
    }
    float sv[16];
#pragma unroll
    for (int q = 0; q < 4 && MODE != NX_DW; ++q) {
      const float4 v = *reinterpret_cast<const float4*>(side + yb * 32 + 8 * q + h4);
      sv[4 * q] = v.x; sv[4 * q + 1] = v.y; sv[4 * q + 2] = v.z; sv[4 * q + 3] = v.w;
    }
#pragma unroll
    for (int b = 0; b < XB; ++b) {
      if constexpr (MODE == NX_STATS) {
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          z[b][e] = fmaf(z[b][e], L2E, sv[e]);
          top = fmaxf(top, z[b][e]);
        }
        const int at = st.xl[b] - (int)(y0 + yb * 32) - h4;
        if (__any((unsigned)at < 32u)) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (at == 8 * (e / 4) + e % 4) st.zl[b] = z[b][e];
        }
        const float m = fmaxf(st.m[b], top), base = m == -INFINITY ? 0.f : m;      // nothing but -inf so far: every term is 0
        float s = st.s[b] * __builtin_amdgcn_exp2f(st.m[b] - base);
#pragma unroll
        for (int e = 0; e < 16; ++e) s += __builtin_amdgcn_exp2f(z[b][e] - base);
        st.m[b] = m;
        st.s[b] = s;
      } else {
        if constexpr (MODE == NX_DH) {
#pragma unroll
          for (int e = 0; e < 16; ++e) z[b][e] = __builtin_amdgcn_exp2f(fmaf(z[b][e], L2E, sv[e]) - st.xa[b]) * st.xi[b];
          const int at = st.xl[b] - (int)(y0 + yb * 32) - h4;
          if (__any((unsigned)at < 32u)) {
#pragma unroll
            for (int e = 0; e < 16; ++e) z[b][e] -= at == 8 * (e / 4) + e % 4 ? Mul<T>::G : 0.f;
          }
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) {            // (four rows' values at a time: the registers are full)
            const float4 t4 = *reinterpret_cast<const float4*>(side + yb * 32 + 8 * q + h4);
            const float4 i4 = *reinterpret_cast<const float4*>(side + 128 + yb * 32 + 8 * q + h4);
            const float top[4] = {t4.x, t4.y, t4.z, t4.w}, inv[4] = {i4.x, i4.y, i4.z, i4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              z[b][4 * q + e] = lx_exp(fmaf(z[b][4 * q + e], L2E, st.xa[b]) - top[e]) * inv[e];
            __builtin_amdgcn_sched_barrier(0);
          }
          // the wave's classes are 32 in a row: does any of the block's rows have one of them as its label?
          const int* lab = reinterpret_cast<const int*>(side + 64) + yb * 32;
          if (__any((unsigned)(lab[lane & 31] - (st.xl[b] - (lane & 31))) < 32u)) {
#pragma unroll
            for (int e = 0; e < 16; ++e) z[b][e] -= lab[8 * (e / 4) + h4 + e % 4] == st.xl[b] ? Mul<T>::G : 0.f;
          }
          if (a.scaled) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float f = side[192 + yb * 32 + 8 * (e / 4) + h4 + e % 4];
              z[b][e] = f == 0.f ? 0.f : z[b][e] * f;
            }
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) st.s[b] += z[b][e];
        }
        s16x8 gf[2][N::NP];
#pragma unroll
        for (int p = 0; p < N::NP; ++p)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const E o = (E)z[b][e];
            gf[e / 8][p][e % 8] = __builtin_bit_cast(short, o);
            if (p + 1 < N::NP) z[b][e] -= (float)o;
          }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int mb = 0; mb < N::KB; ++mb) {
            s16x8 cf[N::NP];
#pragma unroll
            for (int p = 0; p < N::NP; ++p) cf[p] = nx_cols<N, KP>(cur + p * N::PART, yb, s, mb, lane);
            st.out[mb][b] = nx_mma<T, N::NP>(cf, gf[s], st.out[mb][b]);
          }
      }
    }
  }
}

// every wave's share of the next tile has landed and none still reads the buffer that is filled next. A barrier alone promises only
// the second: a wave's loads into LDS are its own to wait for
__device__ __forceinline__ void next_tile() {
  wait_loads<0>();
  __syncthreads();
}

// (fp32 of 64 columns: within the registers of a third workgroup on the CU)
template <typename T, int KP, int XB, int MODE>
__global__ __launch_bounds__(256, Mul<T>::NP == 3 && KP == 64 ? 3 : 2) void k_lx_narrow(NxArgs a) {
  typedef Narrow<T, KP, XB> N;
  __shared__ __align__(16) short buf[2 * N::TILE];
  __shared__ __align__(16) float side[2 * 256];
  const uint32_t x_tiles = (uint32_t)ceil_div<int64_t>(a.nx, N::XT), t = xcd_run(blockIdx.x, gridDim.x);
  const int64_t xt = uniform((int)(t % x_tiles));
  const int sp = uniform((int)(t / x_tiles));              // an XCD's workgroups walk the same y at the same time
  const int64_t y_lo = sp * a.range, y_hi = y_lo + a.range < a.ny ? y_lo + a.range : a.ny;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  NarrowState<T, KP, XB, MODE> st;
  int64_t x[XB];
#pragma unroll
  for (int b = 0; b < XB; ++b) {
    x[b] = xt * N::XT + wave * 32 * XB + b * 32 + (lane & 31);
    const int64_t xr = x[b] < a.x_rows ? x[b] : a.x_rows - 1;
    const bool in = x[b] < a.nx;
#pragma unroll
    for (int kk = 0; kk < N::KK; ++kk)
#pragma unroll
      for (int p = 0; p < N::NP; ++p)
        st.xf[b][kk][p] = *reinterpret_cast<const s16x8*>((const short*)a.x + p * a.x_part + xr * a.x_ld + kk * 16 + 8 * (lane >> 5));
    st.m[b] = -INFINITY;
    st.s[b] = 0.f;
    st.zl[b] = -INFINITY;
    if constexpr (MODE == NX_STATS) {
      st.xl[b] = in ? a.xlab[x[b]] : -1;
    } else if constexpr (MODE == NX_DH) {
      const bool counts = in && a.xb[x[b]] != 0.f;
      st.xa[b] = counts ? a.xa[x[b]] : INFINITY;           // rows that do not count: every exponential is 0
      st.xi[b] = counts ? a.xi[x[b]] : 0.f;
      st.xl[b] = counts ? a.xlab[x[b]] : -1;
    } else {
      st.xa[b] = a.xa[x[b]];                               // (padded past the last class)
      st.xl[b] = (int)x[b];
    }
  }
  if constexpr (MODE != NX_STATS) {
#pragma unroll
    for (int i = 0; i < N::KB; ++i)
#pragma unroll
      for (int b = 0; b < XB; ++b) st.out[i][b] = f32x16{};
  }
  if (y_lo < y_hi) {
    // (the first tile through the same code: a step that only loads)
    const char* base = (const char*)a.y + y_lo * a.y_ld * 2;
    const int64_t left = a.y_rows - 1 - y_lo;
    const int last = left < N::YT ? (int)left : N::YT;
#pragma unroll
    for (int t2 = 0; t2 < N::PER; ++t2) {
      const int piece = wave * N::PER + t2, part = piece / (N::PIECES / N::NP);
      const int lin = (piece % (N::PIECES / N::NP)) * 64 + lane, row = lin / N::CH, chunk = (lin % N::CH) ^ nx_swz<KP>(row);
      dma16(base + part * a.y_part * 2 + ((uint32_t)(row < last ? row : last) * (uint32_t)a.y_ld * 2 + chunk * 16), buf + piece * 512);
    }
    if (wave == 0) {
      __builtin_amdgcn_global_load_lds((glb_void*)(a.side0 + y_lo + lane), (lds_void*)side, 4, 0, 0);
      if constexpr (MODE == NX_DW) {
        __builtin_amdgcn_global_load_lds((glb_void*)(a.side1 + y_lo + lane), (lds_void*)(side + 64), 4, 0, 0);
        __builtin_amdgcn_global_load_lds((glb_void*)(a.side3 + y_lo + lane), (lds_void*)(side + 128), 4, 0, 0);
        if (a.scaled) __builtin_amdgcn_global_load_lds((glb_void*)(a.side2 + y_lo + lane), (lds_void*)(side + 192), 4, 0, 0);
      }
    }
    for (int64_t y = y_lo; y < y_hi; y += 2 * N::YT) {
      next_tile();
      nx_step<T, KP, XB, MODE>(buf, side, buf + N::TILE, side + 256, y + N::YT < y_hi, a, y, y + N::YT, wave, lane, st);
      if (y + N::YT < y_hi) {
        next_tile();
        nx_step<T, KP, XB, MODE>(buf + N::TILE, side + 256, buf, side, y + 2 * N::YT < y_hi, a, y + N::YT, y + 2 * N::YT, wave, lane, st);
      }
    }
  }
  const int h4 = 4 * (lane >> 5);
#pragma unroll
  for (int b = 0; b < XB; ++b) {
    if constexpr (MODE == NX_STATS) {
      const float om = __shfl_xor(st.m[b], 32, kWave), os = __shfl_xor(st.s[b], 32, kWave);
      const float m = fmaxf(st.m[b], om), base = m == -INFINITY ? 0.f : m;
      const float s = st.s[b] * __builtin_amdgcn_exp2f(st.m[b] - base) + os * __builtin_amdgcn_exp2f(om - base);
      if (x[b] < a.nx) {
        if (lane < 32) a.part[x[b] * a.splits + sp] = make_float2(m, s);
        const int64_t at = (int64_t)st.xl[b];
        // the label's logit: from the half of the wave that met it
        if (at >= y_lo && at < y_hi && ((at - y_lo) & 4) == h4) a.zlab[x[b]] = st.zl[b];
      }
    } else {
      const bool in = x[b] < a.nx;
      const float f = (a.f1 ? *a.f1 : 1.f) * (a.f2 ? *a.f2 : 1.f) / Mul<T>::G;
      float rf = 1.f;
      if constexpr (MODE == NX_DH) rf = in ? a.xb[x[b]] : 0.f;
      if (in) {
#pragma unroll
        for (int mb = 0; mb < N::KB; ++mb)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int64_t k = mb * 32 + 8 * q + h4;
            if (k >= a.K) continue;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = rf == 0.f ? 0.f : st.out[mb][b][4 * q + e] * rf;
            if (a.splits > 1) {
              store4_tail(a.acc + (sp * a.nx + x[b]) * a.K + k, a.K - k, v);
            } else if (a.out) {          // (db alone may be wanted)
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] *= f;
              store4_tail((T*)a.out + x[b] * a.K + k, a.K - k, v);
            }
          }
      }
      if constexpr (MODE == NX_DW) {
        const float s = st.s[b] + __shfl_xor(st.s[b], 32, kWave);
        if (in && lane < 32) {
          if (a.splits > 1)
            a.accb[sp * a.nx + x[b]] = s;
          else if (a.outb)
            ((T*)a.outb)[x[b]] = (T)(s * f);
        }
      }
    }
  }
}

}  // namespace pg
