// Dropout as an operator of its own, and layer norm with the residual sum and the dropout in front of it.
//
// Dropout: y = keep * x * 65536 / (65536 - threshold) with the keep mask of pg_dropout_t (include/pagraph_hip.h): the mask is a
// function of (row, column, seed, tag, step), is never stored, and is the one the fused aggregations draw for the same row — the
// backward pass draws it again. One Philox4x32-10 call makes eight 16-bit words: the columns 4p..4p+3 and 4p+256..4p+259 of one
// row, so a thread owns those eight columns ("a pair of pieces") and no word is drawn twice. Ten rounds of two 32x32 products are
// what the ALU pays; the bound is HBM (each element read once, written once).
//
// Layer norm: s = dropout(x) + residual, y = (s - mean) * rstd * w + b, biased variance. A row lives in the registers of G lanes
// (S pairs of pieces each), so mean and variance are two exact passes over registers and the row is read once. Backward:
//   gh = gy * w, xh = (s - mean) * rstd, ds = rstd * (gh - mean(gh) - xh * mean(gh * xh)) + gs
// in one pass over (gy, s, gs); dw = sum_r gy * xh and db = sum_r gy accumulate in registers over the rows a group walks, are
// added up inside the workgroup and leave as one partial row per workgroup, which a second launch sums in a fixed order
// (deterministic: no atomics). Bound: HBM.
#include "pg_elem.h"

namespace pg {

// pairs of pieces of a row of d columns (the counter's second word runs over [0, pairs))
__host__ __device__ inline int64_t row_pairs(int64_t d) {
  const int64_t rem = d % 512, last = (rem + 3) / 4;
  return d / 512 * 64 + (last > 64 ? 64 : last);
}
__device__ __forceinline__ int64_t pair_col(int64_t q) { return (q >> 6) * 512 + (q & 63) * 4; }

__device__ __forceinline__ void drop4(float (&v)[4], uint32_t w0, uint32_t w1, uint32_t thr, float scale) {
  v[0] = (w0 & 0xffffu) >= thr ? v[0] * scale : 0.f;
  v[1] = (w0 >> 16) >= thr ? v[1] * scale : 0.f;
  v[2] = (w1 & 0xffffu) >= thr ? v[2] * scale : 0.f;
  v[3] = (w1 >> 16) >= thr ? v[3] * scale : 0.f;
}

template <typename T>
__global__ __launch_bounds__(256) void k_dropout(const T* __restrict__ x, int64_t xs, T* __restrict__ y, int64_t ys, int64_t n,
                                                 int64_t d, int64_t nq, int32_t rows_per_block, float inv_nq, DropArgs dr,
                                                 uint64_t* step_used) {
  const uint32_t step = drop_step_of(dr);
  if (step_used && blockIdx.x == 0 && threadIdx.x == 0) *step_used = step;
  for (int64_t r0 = (int64_t)blockIdx.x * rows_per_block; r0 < n; r0 += (int64_t)gridDim.x * rows_per_block) {
    const int64_t rows = n - r0 < rows_per_block ? n - r0 : rows_per_block;
    const int64_t total = rows * nq;
    for (int64_t i = threadIdx.x; i < total; i += 256) {
      // (several rows per block only while rows * nq <= 2048: the quotient in floating point is then exact)
      const int64_t lr = rows_per_block > 1 ? (int64_t)(((float)(int32_t)i + 0.5f) * inv_nq) : 0;
      const int64_t q = i - lr * nq, r = r0 + lr, c0 = pair_col(q), c1 = c0 + 256;
      float a[4], b[4];
      load4_tail(x + r * xs + c0, d - c0, a);
      if (c1 < d) load4_tail(x + r * xs + c1, d - c1, b);
      uint32_t o[4];
      Philox::gen((uint32_t)r, (uint32_t)q, dr.tag, step, dr.k0, dr.k1, o);
      drop4(a, o[0], o[1], dr.thr, dr.scale);
      store4_tail(y + r * ys + c0, d - c0, a);
      if (c1 < d) {
        drop4(b, o[2], o[3], dr.thr, dr.scale);
        store4_tail(y + r * ys + c1, d - c1, b);
      }
    }
  }
}

struct NormArgs {
  const void *x, *res, *w, *b, *gy, *gs;
  void *sum, *y, *dx, *dres;
  float *mean, *rstd, *part;
  uint64_t* step_used;
  int64_t n, d, xs, rs, ss, ys, gys, gss, dxs, drs;
  float eps;
  int32_t w_f32, drop;
  DropArgs dr;
};

// sum over the G lanes of a row's group; above one wave through LDS (two slots in turn: a call may start while slow waves
// still read the previous one's)
template <int G>
__device__ __forceinline__ float group_sum(float v, float* lds, int& turn) {
#pragma unroll
  for (int o = (G < kWave ? G : kWave) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  if constexpr (G > kWave) {
    constexpr int W = G / kWave;
    float* s = lds + turn * W;
    turn ^= 1;
    if ((threadIdx.x & (kWave - 1)) == 0) s[threadIdx.x / kWave] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) v += s[i];
  }
  return v;
}

template <typename T>
__device__ __forceinline__ void load_param(const void* p, int f32, int64_t c, int64_t d, float fill, float (&v)[4]) {
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = fill;
  } else if (f32) {
    load4_tail((const float*)p + c, d - c, v);
  } else {
    load4_tail((const T*)p + c, d - c, v);
  }
}

// G lanes per row, S pairs of pieces per lane: rows of up to 8 * G * S columns (4 * G * S below 256 columns)
template <typename T, int G, int S>
__global__ __launch_bounds__(G > 256 ? G : 256) void k_norm_fwd(NormArgs a) {
  constexpr int B = G > 256 ? G : 256, RPB = B / G;
  __shared__ float lds[G > kWave ? 2 * (G / kWave) : 1];
  int turn = 0;
  const int lane = threadIdx.x % G;
  const float cols = (float)a.d;
  const uint32_t step = a.drop ? drop_step_of(a.dr) : 0u;
  if (a.drop && a.step_used && blockIdx.x == 0 && threadIdx.x == 0) *a.step_used = step;
  for (int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / G; r < a.n; r += (int64_t)gridDim.x * RPB) {
    const T* x = (const T*)a.x + r * a.xs;
    float v[2 * S][4];
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int64_t q = lane + (int64_t)s * G, c0 = pair_col(q);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t c = c0 + 256 * h;
        load4_tail(x + c, a.d - c, v[2 * s + h]);
      }
      if (a.drop && c0 < a.d) {
        uint32_t o[4];
        Philox::gen((uint32_t)r, (uint32_t)q, a.dr.tag, step, a.dr.k0, a.dr.k1, o);
        drop4(v[2 * s], o[0], o[1], a.dr.thr, a.dr.scale);
        drop4(v[2 * s + 1], o[2], o[3], a.dr.thr, a.dr.scale);
      }
      if (a.res) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int64_t c = c0 + 256 * h;
          float t[4];
          load4_tail((const T*)a.res + r * a.rs + c, a.d - c, t);
          // the sum is handed on in T: what is normalised is that rounded row, which the backward pass reads back
#pragma unroll
          for (int i = 0; i < 4; ++i) v[2 * s + h][i] = (float)(T)(v[2 * s + h][i] + t[i]);
          if (c < a.d) store4_tail((T*)a.sum + r * a.ss + c, a.d - c, v[2 * s + h]);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += v[2 * s + h][i];
    }
    const float mean = group_sum<G>(sum, lds, turn) / cols;
    float var = 0.f;
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t c = pair_col(lane + (int64_t)s * G) + 256 * h;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float t = v[2 * s + h][i] - mean;
          var += c + i < a.d ? t * t : 0.f;
        }
      }
    var = group_sum<G>(var, lds, turn) / cols;
    const float rstd = 1.f / sqrtf(var + a.eps);
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t c = pair_col(lane + (int64_t)s * G) + 256 * h;
        if (c < a.d) {
          float w[4], b[4], y[4];
          load_param<T>(a.w, a.w_f32, c, a.d, 1.f, w);
          load_param<T>(a.b, a.w_f32, c, a.d, 0.f, b);
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = (v[2 * s + h][i] - mean) * rstd * w[i] + b[i];
          store4_tail((T*)a.y + r * a.ys + c, a.d - c, y);
        }
      }
    if (a.mean && lane == 0) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
  }
}

template <typename T, int G, int S>
__global__ __launch_bounds__(G > 256 ? G : 256) void k_norm_bwd(NormArgs a) {
  constexpr int B = G > 256 ? G : 256, RPB = B / G;
  constexpr int COLS = G <= kWave ? 8 * G * S : 1;               // the workgroup's sum of dw, db (one row group per wave or less)
  __shared__ float lds[G > kWave ? 2 * (G / kWave) : 1];
  __shared__ float acc_lds[2 * COLS];
  int turn = 0;
  const int lane = threadIdx.x % G;
  const float cols = (float)a.d;
  const uint32_t step = a.drop ? drop_step_of(a.dr) : 0u;
  float aw[2 * S][4] = {}, ab[2 * S][4] = {};
  for (int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / G; r < a.n; r += (int64_t)gridDim.x * RPB) {
    const float mean = a.mean[r], rstd = a.rstd[r];
    float xh[2 * S][4], gh[2 * S][4];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = 2 * s + h;
        const int64_t c = pair_col(lane + (int64_t)s * G) + 256 * h;
        load4_tail((const T*)a.x + r * a.xs + c, a.d - c, xh[k]);
        load4_tail((const T*)a.gy + r * a.gys + c, a.d - c, gh[k]);
      }
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = 2 * s + h;
        const int64_t c = pair_col(lane + (int64_t)s * G) + 256 * h;
        float w[4];
        load_param<T>(a.w, a.w_f32, c, a.d, 1.f, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // (columns behind the row's end have gy = 0: they add nothing to any sum)
          xh[k][i] = (xh[k][i] - mean) * rstd;
          ab[k][i] += gh[k][i];
          aw[k][i] += c + i < a.d ? gh[k][i] * xh[k][i] : 0.f;
          gh[k][i] *= w[i];
          s1 += gh[k][i];
          s2 += c + i < a.d ? gh[k][i] * xh[k][i] : 0.f;
        }
      }
    s1 = group_sum<G>(s1, lds, turn) / cols;
    s2 = group_sum<G>(s2, lds, turn) / cols;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int64_t q = lane + (int64_t)s * G, c0 = pair_col(q);
      uint32_t o[4];
      if (a.drop && c0 < a.d) Philox::gen((uint32_t)r, (uint32_t)q, a.dr.tag, step, a.dr.k0, a.dr.k1, o);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = 2 * s + h;
        const int64_t c = c0 + 256 * h;
        if (c >= a.d) continue;
        float ds[4];
        if (a.gs)
          load4_tail((const T*)a.gs + r * a.gss + c, a.d - c, ds);
        else
          ds[0] = ds[1] = ds[2] = ds[3] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) ds[i] += rstd * (gh[k][i] - s1 - xh[k][i] * s2);
        if (a.dres) store4_tail((T*)a.dres + r * a.drs + c, a.d - c, ds);
        if (a.dx) {
          if (a.drop) drop4(ds, o[2 * h], o[2 * h + 1], a.dr.thr, a.dr.scale);
          store4_tail((T*)a.dx + r * a.dxs + c, a.d - c, ds);
        }
      }
    }
  }
  if (!a.part) return;
  float* out = a.part + (int64_t)blockIdx.x * 2 * a.d;
  if constexpr (G <= kWave) {
    // the wave's groups first (lanes G apart hold the same columns), then the four waves one after the other
#pragma unroll
    for (int k = 0; k < 2 * S; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int o = kWave / 2; o >= G; o >>= 1) {
          aw[k][i] += __shfl_xor(aw[k][i], o, kWave);
          ab[k][i] += __shfl_xor(ab[k][i], o, kWave);
        }
    for (int w = 0; w < B / kWave; ++w) {
      if ((int)threadIdx.x / kWave == w && (threadIdx.x & (kWave - 1)) < G)
#pragma unroll
        for (int k = 0; k < 2 * S; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at = (k * G + lane) * 4 + i;
            acc_lds[at] = (w ? acc_lds[at] : 0.f) + aw[k][i];
            acc_lds[COLS + at] = (w ? acc_lds[COLS + at] : 0.f) + ab[k][i];
          }
      __syncthreads();
    }
    for (int at = threadIdx.x; at < COLS; at += B) {
      const int k = at / (4 * G), l = at / 4 % G;
      const int64_t c = pair_col(l + (int64_t)(k / 2) * G) + 256 * (k & 1) + (at & 3);
      if (c < a.d) {
        out[c] = acc_lds[at];
        out[a.d + c] = acc_lds[COLS + at];
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < 2 * S; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t c = pair_col(lane + (int64_t)(k / 2) * G) + 256 * (k & 1) + i;
        if (c < a.d) {
          out[c] = aw[k][i];
          out[a.d + c] = ab[k][i];
        }
      }
  }
}

// dw, db = the workgroups' partial rows added up in a fixed order: 16 columns x 16 lanes over the rows per block
template <typename TW>
__global__ __launch_bounds__(256) void k_norm_reduce(const float* __restrict__ part, int32_t rows, int64_t d, TW* __restrict__ dw,
                                                     TW* __restrict__ db) {
  __shared__ float s[16][17];
  const int64_t c = (int64_t)blockIdx.x * 16 + (threadIdx.x & 15);
  const int l = threadIdx.x >> 4;
  TW* out = blockIdx.y ? db : dw;
  if (!out) return;
  const float* p = part + (int64_t)blockIdx.y * d + c;
  float acc = 0.f;
  if (c < d) {
#pragma unroll 8
    for (int r = l; r < rows; r += 16) acc += p[(int64_t)r * 2 * d];
  }
  s[l][threadIdx.x & 15] = acc;
  __syncthreads();
  if (l == 0 && c < d) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += s[i][threadIdx.x & 15];
    out[c] = (TW)t;
  }
}

// workgroups of the backward pass: enough to fill the card twice over; each leaves one partial row of 2 d floats
inline int64_t norm_bwd_blocks(int64_t n, int64_t d) {
  const int64_t nq = row_pairs(d);
  const int64_t rpb = nq <= 16 ? 16 : nq <= 32 ? 8 : nq <= 256 ? 4 : 1;
  const int64_t b = ceil_div<int64_t>(n, rpb);
  return b < 1 ? 1 : b > 512 ? 512 : b;
}

template <typename T, int G, int S>
int launch_norm(const NormArgs& a, bool bwd, hipStream_t st) {
  constexpr int B = G > 256 ? G : 256;
  if (bwd) {
    hipLaunchKernelGGL((k_norm_bwd<T, G, S>), dim3((unsigned)norm_bwd_blocks(a.n, a.d)), dim3(B), 0, st, a);
  } else {
    const int64_t b = ceil_div<int64_t>(a.n, B / G);
    hipLaunchKernelGGL((k_norm_fwd<T, G, S>), dim3((unsigned)(b > 4096 ? 4096 : b)), dim3(B), 0, st, a);
  }
  PG_LAUNCH_CHECK();
  return PG_OK;
}

// lanes per row and pairs per lane by the row's width: a row stays in registers, with as few idle lanes as a power of two allows
template <typename T>
int dispatch_norm(const NormArgs& a, bool bwd, hipStream_t st) {
  const int64_t nq = row_pairs(a.d);
  if (nq <= 16) return launch_norm<T, 16, 1>(a, bwd, st);
  if (nq <= 32) return launch_norm<T, 32, 1>(a, bwd, st);
  if (nq <= 64) return launch_norm<T, 64, 1>(a, bwd, st);
  if (nq <= 128) return launch_norm<T, 64, 2>(a, bwd, st);
  if (nq <= 256) return launch_norm<T, 64, 4>(a, bwd, st);
  if (nq <= 512) return launch_norm<T, 256, 2>(a, bwd, st);
  if (nq <= 1024) return launch_norm<T, 256, 4>(a, bwd, st);
  return launch_norm<T, 1024, 4>(a, bwd, st);
}

int norm_args(const pg_norm_desc_t* p, NormArgs* a) {
  if (!p || p->n < 0 || p->d <= 0 || p->dtype < PG_DTYPE_F32 || p->dtype > PG_DTYPE_F16) return PG_ERR_INVALID;
  if (p->d > PG_NORM_MAX_COLUMNS) return PG_ERR_UNSUPPORTED;
  if (p->param_dtype != p->dtype && p->param_dtype != PG_DTYPE_F32) return PG_ERR_INVALID;
  if (p->n > (int64_t)0xffffffffll) return PG_ERR_UNSUPPORTED;          // the mask's row counter has 32 bits
  *a = NormArgs{};
  a->n = p->n;
  a->d = p->d;
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
  if (n > (int64_t)0xffffffffll || d > (int64_t)0x7fffffffll) return PG_ERR_UNSUPPORTED;      // the mask's counters have 32 bits
  DropArgs dr;
  if (!drop || !drop_args(drop, &dr)) return PG_ERR_INVALID;
  if (n == 0) return PG_OK;
  if (!x || !y) return PG_ERR_INVALID;
  const int64_t nq = row_pairs(d);
  const int32_t rows = nq >= 1024 ? 1 : (int32_t)(1024 / nq);
  const int64_t blocks = ceil_div<int64_t>(n, rows);
  const dim3 grid((unsigned)(blocks > 16384 ? 16384 : blocks));
  const float inv = 1.f / (float)nq;
  if (dtype == PG_DTYPE_F32)
    hipLaunchKernelGGL(k_dropout<float>, grid, dim3(256), 0, as_stream(stream), (const float*)x, x_stride, (float*)y, y_stride, n, d, nq, rows, inv, dr, step_used);
  else if (dtype == PG_DTYPE_BF16)
    hipLaunchKernelGGL(k_dropout<bf16_t>, grid, dim3(256), 0, as_stream(stream), (const bf16_t*)x, x_stride, (bf16_t*)y, y_stride, n, d, nq, rows, inv, dr, step_used);
  else
    hipLaunchKernelGGL(k_dropout<f16_t>, grid, dim3(256), 0, as_stream(stream), (const f16_t*)x, x_stride, (f16_t*)y, y_stride, n, d, nq, rows, inv, dr, step_used);
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
  if (p->dtype == PG_DTYPE_F32) return dispatch_norm<float>(a, false, as_stream(stream));
  if (p->dtype == PG_DTYPE_BF16) return dispatch_norm<bf16_t>(a, false, as_stream(stream));
  return dispatch_norm<f16_t>(a, false, as_stream(stream));
}

int64_t pg_layer_norm_scratch(int64_t n, int64_t d) {
  if (n < 0 || d <= 0 || d > PG_NORM_MAX_COLUMNS) return 0;
  return norm_bwd_blocks(n, d) * 2 * d;
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
  if (p->n > 0) {
    if (p->dtype == PG_DTYPE_F32) r = dispatch_norm<float>(a, true, as_stream(stream));
    else if (p->dtype == PG_DTYPE_BF16) r = dispatch_norm<bf16_t>(a, true, as_stream(stream));
    else r = dispatch_norm<f16_t>(a, true, as_stream(stream));
  }
  if (r != PG_OK || !params) return r;
  const int32_t rows = p->n > 0 ? (int32_t)norm_bwd_blocks(p->n, p->d) : 0;     // no rows: the sums are zeros
  const dim3 grid((unsigned)ceil_div<int64_t>(p->d, 16), 2);
  if (p->param_dtype == PG_DTYPE_F32)
    hipLaunchKernelGGL(k_norm_reduce<float>, grid, dim3(256), 0, as_stream(stream), p->partials, rows, p->d, (float*)p->dw, (float*)p->db);
  else if (p->param_dtype == PG_DTYPE_BF16)
    hipLaunchKernelGGL(k_norm_reduce<bf16_t>, grid, dim3(256), 0, as_stream(stream), p->partials, rows, p->d, (bf16_t*)p->dw, (bf16_t*)p->db);
  else
    hipLaunchKernelGGL(k_norm_reduce<f16_t>, grid, dim3(256), 0, as_stream(stream), p->partials, rows, p->d, (f16_t*)p->dw, (f16_t*)p->db);
  PG_LAUNCH_CHECK();
  return PG_OK;
}

}  // extern "C"
