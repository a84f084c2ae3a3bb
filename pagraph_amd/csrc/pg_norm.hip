// Dropout as an operator of its own, and layer norm with the residual sum and the dropout in front of it.
//
// Dropout: y = keep * x * 65536 / (65536 - threshold) with the keep mask of pg_dropout_t (include/pagraph_hip.h): the mask is a
// function of (row, column, seed, tag, step), is never stored, and is the one the fused aggregations draw for the same row — the
// backward pass draws it again. One Philox4x32-10 call makes eight 16-bit words: the columns 4p..4p+3 and 4p+256..4p+259 of one
// row, so a thread owns those eight columns ("a pair of pieces") and no word is drawn twice. Ten rounds of two 32x32 products are
// what the ALU pays; the bound is HBM (each element read once, written once): 16384 x 2048 bf16 26.6 us = 5.0 TB/s, 6000 x 602 fp32
// 7.3 us = 4.0 TB/s (rows of no whole 16-byte pieces; six inputs in turn, 8.2 us under a profiler).
//
// Layer norm: s = dropout(x) + residual, y = (s - mean) * rstd * w + b, biased variance. A row lives in the registers of G lanes
// (S pairs of pieces each), so mean and variance are two exact passes over registers and the row is read once. Backward:
//   gh = gy * w, xh = (s - mean) * rstd, ds = rstd * (gh - mean(gh) - xh * mean(gh * xh)) + gs
// in one pass over (gy, s, gs); dw = sum_r gy * xh and db = sum_r gy accumulate in registers over the rows a group walks, are
// added up inside the workgroup and leave as one partial row per workgroup, which a second launch sums in a fixed order
// (deterministic: no atomics). Bound: HBM: 16384 x 2048 bf16 with dropout and residual forward 58 us = 4.6 TB/s, backward 68 to 73 us
// = 4.6 to 4.9 TB/s; 6000 x 602 fp32 with residual 14 us = 4.1 TB/s, and 19.5 us = 3.0 TB/s with 4.8 more for the partial rows: the
// fp32 backward pass reads no row ahead, and its 87 units stand on 128 places of two a lane. Rows above 8192 columns spill there.
#include "pg_elem.h"

namespace pg {

// pairs of pieces of a row of d columns (the counter's second word runs over [0, pairs))
__host__ __device__ inline int row_pairs(int64_t d) {
  const int64_t rem = d % 512, last = (rem + 3) / 4;
  return (int)(d / 512 * 64 + (last > 64 ? 64 : last));
}

// A unit of work is V neighbouring pairs: 4 V columns from unit_col on and 4 V columns 256 further. V = 2 for 16-bit rows of whole
// 16-byte pieces (d % 8 == 0), else 1. RAGGED: d is no multiple of 4 V, a row's last piece is moved element by element.
template <int V>
__device__ __forceinline__ int unit_col(int u) {
  const int q = u * V;
  return (q >> 6) * 512 + (q & 63) * 4;
}
template <typename T, int V, bool RAGGED>
__device__ __forceinline__ void load_piece(const T* __restrict__ row, int c, int d, float (&v)[4 * V]) {
  if (c + 4 * V <= d) {
    T t[4 * V];
    __builtin_memcpy(t, row + c, sizeof(t));
#pragma unroll
    for (int i = 0; i < 4 * V; ++i) v[i] = (float)t[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4 * V; ++i) v[i] = RAGGED && c + i < d ? (float)row[c + i] : 0.f;
  }
}
template <typename T, int V, bool RAGGED>
__device__ __forceinline__ void store_piece(T* __restrict__ row, int c, int d, const float (&v)[4 * V]) {
  if (c + 4 * V <= d) {
    T t[4 * V];
#pragma unroll
    for (int i = 0; i < 4 * V; ++i) t[i] = (T)v[i];
    __builtin_memcpy(row + c, t, sizeof(t));
  } else if (RAGGED) {
#pragma unroll
    for (int i = 0; i < 4 * V; ++i)
      if (c + i < d) row[c + i] = (T)v[i];
  }
}

// the same piece as it stands in memory: half the registers where a 16-bit row has to be kept, and no wait before its use
template <typename T, int V>
struct Raw {
  uint32_t w[V * sizeof(T)];
};
template <typename T, int V, bool RAGGED>
__device__ __forceinline__ void load_raw(const T* __restrict__ row, int c, int d, Raw<T, V>& raw) {
  if (c + 4 * V <= d) {
    __builtin_memcpy(&raw, row + c, sizeof(raw));
  } else {
    T t[4 * V];
#pragma unroll
    for (int i = 0; i < 4 * V; ++i) t[i] = RAGGED && c + i < d ? row[c + i] : (T)0.f;
    __builtin_memcpy(&raw, t, sizeof(raw));
  }
}
template <typename T, int V>
__device__ __forceinline__ void unpack(const Raw<T, V>& raw, float (&v)[4 * V]) {
  T t[4 * V];
  __builtin_memcpy(t, &raw, sizeof(t));
#pragma unroll
  for (int i = 0; i < 4 * V; ++i) v[i] = (float)t[i];
}

// the compiler forgets what it has unpacked, instead of keeping it in twice the registers
template <typename T, int V>
__device__ __forceinline__ void keep_packed(Raw<T, V>& raw) {
#pragma unroll
  for (uint32_t& w : raw.w) asm volatile("" : "+v"(w));
}

struct UnitMask {
  uint32_t w[4];
};
template <int V>
__device__ __forceinline__ void draw_unit(const DropArgs& dr, uint32_t step, uint32_t r, int u, UnitMask (&m)[V]) {
#pragma unroll
  for (int k = 0; k < V; ++k) Philox::gen(r, (uint32_t)(u * V + k), dr.tag, step, dr.k0, dr.k1, m[k].w);
}
// half 0: the unit's first 4 V columns, half 1: those 256 further
template <int V>
__device__ __forceinline__ void drop_piece(float (&v)[4 * V], const UnitMask (&m)[V], int half, uint32_t thr, float scale) {
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const uint32_t w0 = m[k].w[2 * half], w1 = m[k].w[2 * half + 1];
    v[4 * k] = (w0 & 0xffffu) >= thr ? v[4 * k] * scale : 0.f;
    v[4 * k + 1] = (w0 >> 16) >= thr ? v[4 * k + 1] * scale : 0.f;
    v[4 * k + 2] = (w1 & 0xffffu) >= thr ? v[4 * k + 2] * scale : 0.f;
    v[4 * k + 3] = (w1 >> 16) >= thr ? v[4 * k + 3] * scale : 0.f;
  }
}

// (y may be x: a thread has read its unit before it writes it)
template <typename T, int V, bool RAGGED>
__global__ __launch_bounds__(256) void k_dropout(const T* x, int64_t xs, T* y, int64_t ys, int64_t n, int d,
                                                 int units, int rows_per_block, float inv_units, DropArgs dr, uint64_t* step_used) {
  const uint32_t step = drop_step_of(dr);
  if (step_used && blockIdx.x == 0 && threadIdx.x == 0) *step_used = step;
  for (int64_t r0 = (int64_t)blockIdx.x * rows_per_block; r0 < n; r0 += (int64_t)gridDim.x * rows_per_block) {
    const int rows = n - r0 < rows_per_block ? (int)(n - r0) : rows_per_block;
    const int total = rows * units;
    for (int i = threadIdx.x; i < total; i += 256) {
      // (several rows per block only while rows * units <= 512: the quotient in floating point is then exact)
      const int lr = rows_per_block > 1 ? (int)(((float)i + 0.5f) * inv_units) : 0;
      const int u = i - lr * units, c0 = unit_col<V>(u), c1 = c0 + 256;
      const int64_t r = r0 + lr;
      const T* src = x + r * xs;
      T* dst = y + r * ys;
      float a[4 * V], b[4 * V];
      load_piece<T, V, RAGGED>(src, c0, d, a);
      load_piece<T, V, RAGGED>(src, c1, d, b);
      UnitMask m[V];
      draw_unit<V>(dr, step, (uint32_t)r, u, m);
      drop_piece<V>(a, m, 0, dr.thr, dr.scale);
      drop_piece<V>(b, m, 1, dr.thr, dr.scale);
      store_piece<T, V, RAGGED>(dst, c0, d, a);
      store_piece<T, V, RAGGED>(dst, c1, d, b);
    }
  }
}

struct NormArgs {
  const void *x, *res, *w, *b, *gy, *gs;
  void *sum, *y, *dx, *dres;
  float *mean, *rstd, *part;
  uint64_t* step_used;
  int64_t n, xs, rs, ss, ys, gys, gss, dxs, drs;
  int d;
  float eps;
  int32_t w_f32, drop;
  DropArgs dr;
};

// sums over the G lanes of a row's group, K at a time; above one wave through LDS (two slots in turn: a call may start while slow
// waves still read the previous one's). Every lane of the workgroup calls it.
template <int G, int K>
__device__ __forceinline__ void group_sum(float (&v)[K], float* lds, int& turn) {
#pragma unroll
  for (int o = (G < kWave ? G : kWave) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor(v[k], o, kWave);
  if constexpr (G > kWave) {
    constexpr int W = G / kWave, ALL = (G > 256 ? G : 256) / kWave;
    float* s = lds + turn * 2 * ALL;
    turn ^= 1;
    const int wave = threadIdx.x / kWave;
    if ((threadIdx.x & (kWave - 1)) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) s[k * ALL + wave] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) v[k] += s[k * ALL + wave / W * W + i];
    }
  }
}

// which of the workgroup's rows a lane works on: one value a wave from 64 lanes a row on, so that row addresses are scalar
template <int G>
__device__ __forceinline__ int row_of_lane() {
  const int r = threadIdx.x / G;
  return G >= kWave ? __builtin_amdgcn_readfirstlane(r) : r;
}
// A row's number, and in the widest workgroups (128 registers a lane) a lane's, opaque: addresses are made from them where they are
// used, from a scalar base and a 32-bit offset. The compiler would carry one pointer per operand and piece from row to row in
// vector registers: forward of 16384 x 256 bf16 14.3 against 12.1 us, backward of 2048 x 16384 151 against 92. fp32 rows have
// registers for it, or lose more to the order of the loads (6000 x 602 forward 12.7 against 14.9 us).
template <typename T, int G>
__device__ __forceinline__ int64_t fresh_row(int64_t r) {
  if constexpr (sizeof(T) == 4) return r;
  if constexpr (G >= kWave) asm volatile("" : "+s"(r));
  else asm volatile("" : "+v"(r));
  return r;
}
template <int G>
__device__ __forceinline__ int fresh_lane() {
  int l = threadIdx.x;
  if constexpr (G == 1024) asm volatile("" : "+v"(l));
  return l & (G - 1);
}

template <typename T, int V, bool RAGGED>
__device__ __forceinline__ void load_param(const void* p, int f32, int c, int d, float fill, float (&v)[4 * V]) {
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < 4 * V; ++i) v[i] = fill;
  } else if (f32) {
    load_piece<float, V, RAGGED>((const float*)p, c, d, v);
  } else {
    load_piece<T, V, RAGGED>((const T*)p, c, d, v);
  }
}

// G lanes per row, S units per lane: rows of up to 8 V G S columns (half of it below 256 columns)
template <typename T, int V, bool RAGGED, int G, int S>
__global__ __launch_bounds__(G > 256 ? G : 256) void k_norm_fwd(NormArgs a) {
  constexpr int B = G > 256 ? G : 256, RPB = B / G, P = 4 * V;
  __shared__ float lds[G > kWave ? 4 * (B / kWave) : 1];
  int turn = 0;
  const int own = row_of_lane<G>(), d = a.d;
  const float cols = (float)d;
  const uint32_t step = a.drop ? drop_step_of(a.dr) : 0u;
  if (a.drop && a.step_used && blockIdx.x == 0 && threadIdx.x == 0) *a.step_used = step;
  for (int64_t rb = (int64_t)blockIdx.x * RPB; rb < a.n; rb += (int64_t)gridDim.x * RPB) {
    const bool on = rb + own < a.n;
    const int64_t r = fresh_row<T, G>(on ? rb + own : a.n - 1);
    const int lane = fresh_lane<G>();
    const T* x = (const T*)a.x + r * a.xs;
    float v[2 * S][P];
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) load_piece<T, V, RAGGED>(x, unit_col<V>(lane + s * G) + 256 * h, d, v[2 * s + h]);
    if (a.res) {
      const T* res = (const T*)a.res + r * a.rs;
      float t[2 * S][P];
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) load_piece<T, V, RAGGED>(res, unit_col<V>(lane + s * G) + 256 * h, d, t[2 * s + h]);
      if (a.drop) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
          UnitMask m[V];
          draw_unit<V>(a.dr, step, (uint32_t)r, lane + s * G, m);
          drop_piece<V>(v[2 * s], m, 0, a.dr.thr, a.dr.scale);
          drop_piece<V>(v[2 * s + 1], m, 1, a.dr.thr, a.dr.scale);
        }
      }
#pragma unroll
      for (int k = 0; k < 2 * S; ++k) {
        // the sum is handed on in T: what is normalised is that rounded row, which the backward pass reads back
#pragma unroll
        for (int i = 0; i < P; ++i) v[k][i] = (float)(T)(v[k][i] + t[k][i]);
        if (on) store_piece<T, V, RAGGED>((T*)a.sum + r * a.ss, unit_col<V>(lane + k / 2 * G) + 256 * (k & 1), d, v[k]);
      }
    }
    float mean[1] = {0.f}, var[1] = {0.f};
#pragma unroll
    for (int k = 0; k < 2 * S; ++k)
#pragma unroll
      for (int i = 0; i < P; ++i) mean[0] += v[k][i];
    group_sum<G, 1>(mean, lds, turn);
    mean[0] /= cols;
#pragma unroll
    for (int k = 0; k < 2 * S; ++k) {
      const int c = unit_col<V>(lane + k / 2 * G) + 256 * (k & 1);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        v[k][i] -= mean[0];
        if (RAGGED ? c + i < d : c < d) var[0] += v[k][i] * v[k][i];
      }
    }
    group_sum<G, 1>(var, lds, turn);
    const float rstd = 1.f / sqrtf(var[0] / cols + a.eps);
    if (!on) continue;
#pragma unroll
    for (int k = 0; k < 2 * S; ++k) {
      const int c = unit_col<V>(lane + k / 2 * G) + 256 * (k & 1);
      if (c >= d) continue;
      float w[P], b[P];
      load_param<T, V, RAGGED>(a.w, a.w_f32, c, d, 1.f, w);
      load_param<T, V, RAGGED>(a.b, a.w_f32, c, d, 0.f, b);
#pragma unroll
      for (int i = 0; i < P; ++i) v[k][i] = v[k][i] * rstd * w[i] + b[i];
      store_piece<T, V, RAGGED>((T*)a.y + r * a.ys, c, d, v[k]);
    }
    if (a.mean && lane == 0) {
      a.mean[r] = mean[0];
      a.rstd[r] = rstd;
    }
  }
}

template <typename T, int V, bool RAGGED, int G, int S>
__global__ __launch_bounds__(G > 256 ? G : 256, G < 1024 ? 3 : 4) void k_norm_bwd(NormArgs a) {
  constexpr int B = G > 256 ? G : 256, RPB = B / G, P = 4 * V;
  constexpr int COLS = RPB > 1 ? 2 * P * G * S : 1;             // the workgroup's sums of dw, db over its row groups
  __shared__ float lds[G > kWave ? 4 * (B / kWave) : 1];
  __shared__ float acc_lds[2 * COLS];
  int turn = 0;
  const int own = row_of_lane<G>(), d = a.d;
  const float cols = (float)d;
  const uint32_t step = a.drop ? drop_step_of(a.dr) : 0u;
  float aw[2 * S][P] = {}, ab[2 * S][P] = {};
  // a row is kept as it was read: xh and gh = gy * w are made from 16-bit pieces twice, fp32 pieces give way to them (KEEP).
  // AHEAD: the next row is read behind this one's stores, so that all its loads leave together; at the top of the loop the compiler
  // moves some down to their use (16384 x 2048 bf16 94 against 68 us; fp32 2048 x 16384 143 against 163: no registers to spare).
  // Reading it earlier, while this row's sums go round the group, takes the registers of a third workgroup on the CU: 73 us.
  constexpr bool KEEP = sizeof(T) == 4, AHEAD = sizeof(T) == 2 && S == 1;
  struct Row {
    Raw<T, V> x[2 * S], g[2 * S], s[2 * S];
    float mean, rstd;
  };
  auto read = [&](int64_t rb, Row& row) {
    const int64_t at = rb + own, r = fresh_row<T, G>(at < a.n ? at : a.n - 1);
    const int lane = fresh_lane<G>();
    row.mean = a.mean[r];
    row.rstd = a.rstd[r];
#pragma unroll
    for (int k = 0; k < 2 * S; ++k) {
      const int c = unit_col<V>(lane + k / 2 * G) + 256 * (k & 1);
      load_raw<T, V, RAGGED>((const T*)a.x + r * a.xs, c, d, row.x[k]);
      load_raw<T, V, RAGGED>((const T*)a.gy + r * a.gys, c, d, row.g[k]);
      if (a.gs) load_raw<T, V, RAGGED>((const T*)a.gs + r * a.gss, c, d, row.s[k]);
    }
  };
  auto hats = [&](const Row& row, int k, int c, float (&xh)[P], float (&gy)[P]) {
    unpack<T, V>(row.x[k], xh);
    unpack<T, V>(row.g[k], gy);
    // columns behind the row's end have gy = 0 and must not meet an infinite xh there
#pragma unroll
    for (int i = 0; i < P; ++i) xh[i] = (RAGGED ? c + i < d : c < d) ? (xh[i] - row.mean) * row.rstd : 0.f;
  };
  const int64_t stride = (int64_t)gridDim.x * RPB;
  Row row;
  if constexpr (AHEAD) read((int64_t)blockIdx.x * RPB, row);
  for (int64_t rb = (int64_t)blockIdx.x * RPB; rb < a.n; rb += stride) {
    const bool on = rb + own < a.n;
    const int64_t r = fresh_row<T, G>(on ? rb + own : a.n - 1);
    if constexpr (!AHEAD) read(rb, row);
    float sum[2] = {0.f, 0.f};
    int lane = fresh_lane<G>();
#pragma unroll
    for (int k = 0; k < 2 * S; ++k) {
      const int c = unit_col<V>(lane + k / 2 * G) + 256 * (k & 1);
      float xh[P], gh[P], w[P];
      hats(row, k, c, xh, gh);
      load_param<T, V, RAGGED>(a.w, a.w_f32, c, d, 1.f, w);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        if (on) {
          ab[k][i] += gh[i];
          aw[k][i] += gh[i] * xh[i];
        }
        gh[i] *= w[i];
        sum[0] += gh[i];
        sum[1] += gh[i] * xh[i];
      }
      if constexpr (KEEP) {
        __builtin_memcpy(&row.x[k], xh, sizeof(xh));
        __builtin_memcpy(&row.g[k], gh, sizeof(gh));
      } else {
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    group_sum<G, 2>(sum, lds, turn);
    lane = fresh_lane<G>();
    if constexpr (!KEEP) {
#pragma unroll
      for (int k = 0; k < 2 * S; ++k) {
        keep_packed<T, V>(row.x[k]);
        keep_packed<T, V>(row.g[k]);
      }
    }
    if (on) {
      const float s1 = sum[0] / cols, s2 = sum[1] / cols;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        UnitMask m[V];
        if (a.drop) draw_unit<V>(a.dr, step, (uint32_t)r, lane + s * G, m);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = 2 * s + h, c = unit_col<V>(lane + s * G) + 256 * h;
          if (c >= d) continue;
          float xh[P], gh[P], ds[P] = {};
          if constexpr (KEEP) {
            unpack<T, V>(row.x[k], xh);
            unpack<T, V>(row.g[k], gh);
          } else {
            float w[P];
            hats(row, k, c, xh, gh);
            load_param<T, V, RAGGED>(a.w, a.w_f32, c, d, 1.f, w);
#pragma unroll
            for (int i = 0; i < P; ++i) gh[i] *= w[i];
          }
          if (a.gs) unpack<T, V>(row.s[k], ds);
#pragma unroll
          for (int i = 0; i < P; ++i) ds[i] += row.rstd * (gh[i] - s1 - xh[i] * s2);
          if (a.dres) store_piece<T, V, RAGGED>((T*)a.dres + r * a.drs, c, d, ds);
          if (a.dx) {
            if (a.drop) drop_piece<V>(ds, m, h, a.dr.thr, a.dr.scale);
            store_piece<T, V, RAGGED>((T*)a.dx + r * a.dxs, c, d, ds);
          }
          if constexpr (!KEEP) __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    if (AHEAD && rb + stride < a.n) read(rb + stride, row);
  }
  if (!a.part) return;
  const int lane = threadIdx.x % G;
  float* out = a.part + (int64_t)blockIdx.x * 2 * d;
  if constexpr (RPB > 1) {
    // lanes G apart in a wave hold the same columns: those first, then the waves (pairs of waves) one after the other
    if constexpr (G < kWave) {
#pragma unroll
      for (int k = 0; k < 2 * S; ++k)
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
          for (int o = kWave / 2; o >= G; o >>= 1) {
            aw[k][i] += __shfl_xor(aw[k][i], o, kWave);
            ab[k][i] += __shfl_xor(ab[k][i], o, kWave);
          }
    }
    constexpr int L = G < kWave ? kWave : G;                    // lanes that hold one group of sums
    for (int g = 0; g < B / L; ++g) {
      if ((int)threadIdx.x / L == g && threadIdx.x % L < G)
#pragma unroll
        for (int k = 0; k < 2 * S; ++k)
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const int at = (k * P + i) * G + lane;
            acc_lds[at] = (g ? acc_lds[at] : 0.f) + aw[k][i];
            acc_lds[COLS + at] = (g ? acc_lds[COLS + at] : 0.f) + ab[k][i];
          }
      __syncthreads();
    }
    for (int at = threadIdx.x; at < COLS; at += B) {
      const int k = at / G / P, i = at / G % P, l = at % G;
      const int c = unit_col<V>(l + k / 2 * G) + 256 * (k & 1) + i;
      if (c < d) {
        out[c] = acc_lds[at];
        out[d + c] = acc_lds[COLS + at];
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < 2 * S; ++k)
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int c = unit_col<V>(lane + k / 2 * G) + 256 * (k & 1) + i;
        if (c < d) {
          out[c] = aw[k][i];
          out[d + c] = ab[k][i];
        }
      }
  }
}

// dw, db = the workgroups' partial rows added up in a fixed order: 16 columns per block, 64 lanes of four columns over the rows
template <typename TW>
__global__ __launch_bounds__(256) void k_norm_reduce(const float* __restrict__ part, int32_t rows, int d, TW* __restrict__ dw,
                                                     TW* __restrict__ db) {
  __shared__ float s[64][17];
  TW* out = blockIdx.y ? db : dw;
  if (!out) return;
  const int c0 = blockIdx.x * 16, c = c0 + threadIdx.x % 4 * 4, l = threadIdx.x / 4;
  const float* p = part + (int64_t)blockIdx.y * d + c;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int r = l; r < rows; r += 64) {
    float v[4];
    load4_tail(p + (int64_t)r * 2 * d, d - c, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += v[i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) s[l][threadIdx.x % 4 * 4 + i] = acc[i];
  __syncthreads();
  const int col = threadIdx.x % 16, g = threadIdx.x / 16;
  float t = s[4 * g][col] + s[4 * g + 1][col] + s[4 * g + 2][col] + s[4 * g + 3][col];
  __syncthreads();
  s[g][col] = t;
  __syncthreads();
  if (g == 0 && c0 + col < d) {
    t = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += s[i][col];
    out[c0 + col] = (TW)t;
  }
}

// 16-bit rows of whole 16-byte pieces move 16 bytes a lane
inline int norm_v(int64_t d, int32_t dtype) { return dtype != PG_DTYPE_F32 && d % 8 == 0 ? 2 : 1; }

// lanes per row: some 16 elements of a row per lane (more lanes idle on narrower rows, more registers on wider ones)
inline int norm_lanes(int64_t d, int v) {
  const int u = (row_pairs(d) + v - 1) / v;
  if (u <= 64) return u <= 16 ? 16 : u <= 32 ? 32 : 64;
  const int per = v == 2 ? 1 : 2;                                // units per lane above 64 units
  const int g = (u + per - 1) / per;
  return g <= 64 ? 64 : g <= 128 ? 128 : g <= 256 ? 256 : g <= 512 ? 512 : 1024;
}

// workgroups of the backward pass: each leaves one partial row of 2 d floats, so each walks 8 rows at least, which keeps that
// traffic to a tenth of the rows' own. At most the three of 256 threads that a CU holds at once (registers): a second, partly filled round
// of them took as long as the first (1024 workgroups 117 us, 768 89 us at 16384 x 2048 bf16 with dropout and residual, before rows were
// kept as read). Of 512 and 1024 threads a CU holds one, and 768 workgroups are three rounds
inline int64_t norm_bwd_blocks(int64_t n, int64_t d, int32_t dtype) {
  const int g = norm_lanes(d, norm_v(d, dtype)), rpb = g >= 256 ? 1 : 256 / g;
  const int64_t rows = rpb > 8 ? rpb : 8, b = ceil_div<int64_t>(n, rows);
  return b < 1 ? 1 : b > 768 ? 768 : b;
}

template <typename T, int V, bool RAGGED, int G, int S>
int launch_norm(const NormArgs& a, int64_t bwd_blocks, hipStream_t st) {
  constexpr int B = G > 256 ? G : 256;
  if (bwd_blocks) {
    hipLaunchKernelGGL((k_norm_bwd<T, V, RAGGED, G, S>), dim3((unsigned)bwd_blocks), dim3(B), 0, st, a);
  } else {
    const int64_t b = ceil_div<int64_t>(a.n, B / G);
    hipLaunchKernelGGL((k_norm_fwd<T, V, RAGGED, G, S>), dim3((unsigned)(b > 8192 ? 8192 : b)), dim3(B), 0, st, a);
  }
  PG_LAUNCH_CHECK();
  return PG_OK;
}

template <typename T, int V, bool RAGGED>
int dispatch_norm_v(const NormArgs& a, int64_t bwd, hipStream_t st) {
  const int u = (row_pairs(a.d) + V - 1) / V, g = norm_lanes(a.d, V);
  constexpr int S = V == 2 ? 1 : 2;
  if (g == 16) return launch_norm<T, V, RAGGED, 16, 1>(a, bwd, st);
  if (g == 32) return launch_norm<T, V, RAGGED, 32, 1>(a, bwd, st);
  if (u <= 64) return launch_norm<T, V, RAGGED, 64, 1>(a, bwd, st);
  if (g == 64) return launch_norm<T, V, RAGGED, 64, S>(a, bwd, st);
  if (g == 128) return launch_norm<T, V, RAGGED, 128, S>(a, bwd, st);
  if (g == 256) return launch_norm<T, V, RAGGED, 256, S>(a, bwd, st);
  if (g == 512) return launch_norm<T, V, RAGGED, 512, S>(a, bwd, st);
  if (u <= 1024 * S) return launch_norm<T, V, RAGGED, 1024, S>(a, bwd, st);
  return launch_norm<T, V, RAGGED, 1024, 2 * S>(a, bwd, st);
}

template <typename T>
int dispatch_norm(const NormArgs& a, int64_t bwd, hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (a.d % 8 == 0) return dispatch_norm_v<T, 2, false>(a, bwd, st);
  } else {
    if (a.d % 4 == 0) return dispatch_norm_v<T, 1, false>(a, bwd, st);
  }
  return dispatch_norm_v<T, 1, true>(a, bwd, st);
}

template <typename T>
void launch_dropout(const void* x, int64_t xs, void* y, int64_t ys, int64_t n, int64_t d, const DropArgs& dr, uint64_t* used, hipStream_t st) {
  // one unit a thread where a row has at most 128 of them, up to two below 256 (fewer idle threads): with two everywhere, too few
  // workgroups for the card on short batches (six inputs in turn: 6000 x 602 fp32 7.8 against 7.3 us, 65536 x 17 fp16 4.7 against 4.1;
  // 16384 x 2048 bf16, which fills it either way, 25.4 against 26.6)
  const int v = sizeof(T) == 2 && d % 8 == 0 ? 2 : 1, units = (row_pairs(d) + v - 1) / v;
  const int rows = units >= 256 ? 1 : units > 128 ? 512 / units : 256 / units;
  const int64_t blocks = ceil_div<int64_t>(n, rows);
  const dim3 grid((unsigned)(blocks > 65536 ? 65536 : blocks));
  const float inv = 1.f / (float)units;
  if (v == 2)
    hipLaunchKernelGGL((k_dropout<T, 2, false>), grid, dim3(256), 0, st, (const T*)x, xs, (T*)y, ys, n, (int)d, units, rows, inv, dr, used);
  else if (d % 4 == 0)
    hipLaunchKernelGGL((k_dropout<T, 1, false>), grid, dim3(256), 0, st, (const T*)x, xs, (T*)y, ys, n, (int)d, units, rows, inv, dr, used);
  else
    hipLaunchKernelGGL((k_dropout<T, 1, true>), grid, dim3(256), 0, st, (const T*)x, xs, (T*)y, ys, n, (int)d, units, rows, inv, dr, used);
}

int norm_args(const pg_norm_desc_t* p, NormArgs* a) {
  if (!p || p->n < 0 || p->d <= 0 || p->dtype < PG_DTYPE_F32 || p->dtype > PG_DTYPE_F16) return PG_ERR_INVALID;
  if (p->d > PG_NORM_MAX_COLUMNS) return PG_ERR_UNSUPPORTED;
  if (p->param_dtype != p->dtype && p->param_dtype != PG_DTYPE_F32) return PG_ERR_INVALID;
  if (p->n > (int64_t)0xffffffffll) return PG_ERR_UNSUPPORTED;          // the mask's row counter has 32 bits
  *a = NormArgs{};
  a->n = p->n;
  a->d = (int)p->d;
  a->w = p->weight;
  a->b = p->bias;
  a->w_f32 = p->param_dtype == PG_DTYPE_F32;
  a->eps = p->eps;
  a->mean = p->mean;
  a->rstd = p->rstd;
  if (p->has_drop) a->drop = drop_args(&p->drop, &a->dr) ? 1 : 0;
  return PG_OK;
}

inline bool bad_stride(const void* p, int64_t stride, int64_t d) { return p && stride < d && stride != 0; }

}  // namespace pg

using namespace pg;

extern "C" {

int pg_dropout_apply(const void* x, int64_t x_stride, void* y, int64_t y_stride, int64_t n, int64_t d, int32_t dtype,
                     const pg_dropout_t* drop, uint64_t* step_used, pg_stream_t stream) {
  if (n < 0 || d <= 0 || dtype < PG_DTYPE_F32 || dtype > PG_DTYPE_F16 || y_stride < d || bad_stride(x, x_stride, d)) return PG_ERR_INVALID;
  if (n > (int64_t)0xffffffffll || d > (int64_t)0x7ffffc00ll) return PG_ERR_UNSUPPORTED;      // the mask's counters have 32 bits
  DropArgs dr;
  if (!drop || !drop_args(drop, &dr)) return PG_ERR_INVALID;
  if (n == 0) return PG_OK;
  if (!x || !y) return PG_ERR_INVALID;
  if (dtype == PG_DTYPE_F32) launch_dropout<float>(x, x_stride, y, y_stride, n, d, dr, step_used, as_stream(stream));
  else if (dtype == PG_DTYPE_BF16) launch_dropout<bf16_t>(x, x_stride, y, y_stride, n, d, dr, step_used, as_stream(stream));
  else launch_dropout<f16_t>(x, x_stride, y, y_stride, n, d, dr, step_used, as_stream(stream));
  PG_LAUNCH_CHECK();
  return PG_OK;
}

int pg_layer_norm_fwd(const pg_norm_desc_t* p, pg_stream_t stream) {
  NormArgs a;
  const int rc = norm_args(p, &a);
  if (rc != PG_OK) return rc;
  if ((p->residual != nullptr) != (p->sum != nullptr) || (p->mean != nullptr) != (p->rstd != nullptr)) return PG_ERR_INVALID;
  if (a.drop && !p->residual) return PG_ERR_INVALID;
  if (p->y_stride < p->d || bad_stride(p->x, p->x_stride, p->d) || bad_stride(p->residual, p->residual_stride, p->d)
      || (p->sum && p->sum_stride < p->d)) return PG_ERR_INVALID;
  if (p->n == 0) return PG_OK;
  if (!p->x || !p->y) return PG_ERR_INVALID;
  a.x = p->x; a.xs = p->x_stride;
  a.res = p->residual; a.rs = p->residual_stride;
  a.sum = p->sum; a.ss = p->sum_stride;
  a.y = p->y; a.ys = p->y_stride;
  a.step_used = p->step_used;
  if (p->dtype == PG_DTYPE_F32) return dispatch_norm<float>(a, 0, as_stream(stream));
  if (p->dtype == PG_DTYPE_BF16) return dispatch_norm<bf16_t>(a, 0, as_stream(stream));
  return dispatch_norm<f16_t>(a, 0, as_stream(stream));
}

int64_t pg_layer_norm_scratch(int64_t n, int64_t d, int32_t dtype) {
  if (n < 0 || d <= 0 || d > PG_NORM_MAX_COLUMNS) return 0;
  return norm_bwd_blocks(n, d, dtype) * 2 * d;
}

int pg_layer_norm_bwd(const pg_norm_desc_t* p, pg_stream_t stream) {
  NormArgs a;
  const int rc = norm_args(p, &a);
  if (rc != PG_OK) return rc;
  const bool params = p->dw || p->db;
  if (params && !p->partials) return PG_ERR_INVALID;
  if (bad_stride(p->sum, p->sum_stride, p->d) || bad_stride(p->gy, p->gy_stride, p->d) || bad_stride(p->gsum, p->gsum_stride, p->d)
      || (p->dx && p->dx_stride < p->d) || (p->dres && p->dres_stride < p->d)) return PG_ERR_INVALID;
  if (p->n > 0 && (!p->sum || !p->gy || !p->mean || !p->rstd)) return PG_ERR_INVALID;
  a.x = p->sum; a.xs = p->sum_stride;               // the rows that were normalised
  a.gy = p->gy; a.gys = p->gy_stride;
  a.gs = p->gsum; a.gss = p->gsum_stride;
  a.dx = p->dx; a.dxs = p->dx_stride;
  a.dres = p->dres; a.drs = p->dres_stride;
  a.part = params ? p->partials : nullptr;
  int r = PG_OK;
  const int64_t blocks = norm_bwd_blocks(p->n, p->d, p->dtype);
  if (p->n > 0) {
    if (p->dtype == PG_DTYPE_F32) r = dispatch_norm<float>(a, blocks, as_stream(stream));
    else if (p->dtype == PG_DTYPE_BF16) r = dispatch_norm<bf16_t>(a, blocks, as_stream(stream));
    else r = dispatch_norm<f16_t>(a, blocks, as_stream(stream));
  }
  if (r != PG_OK || !params) return r;
  const int32_t rows = p->n > 0 ? (int32_t)blocks : 0;     // no rows: the sums are zeros
  const dim3 grid((unsigned)ceil_div<int64_t>(p->d, 16), 2);
  if (p->param_dtype == PG_DTYPE_F32)
    hipLaunchKernelGGL(k_norm_reduce<float>, grid, dim3(256), 0, as_stream(stream), p->partials, rows, (int)p->d, (float*)p->dw, (float*)p->db);
  else if (p->param_dtype == PG_DTYPE_BF16)
    hipLaunchKernelGGL(k_norm_reduce<bf16_t>, grid, dim3(256), 0, as_stream(stream), p->partials, rows, (int)p->d, (bf16_t*)p->dw, (bf16_t*)p->db);
  else
    hipLaunchKernelGGL(k_norm_reduce<f16_t>, grid, dim3(256), 0, as_stream(stream), p->partials, rows, (int)p->d, (f16_t*)p->dw, (f16_t*)p->db);
  PG_LAUNCH_CHECK();
  return PG_OK;
}

}  // extern "C"
