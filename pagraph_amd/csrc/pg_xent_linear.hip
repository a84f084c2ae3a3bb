// Softmax cross entropy of a class head z = h W^T + b of any width, without its logits:
//   m_r = max_c z_rc,  s_r = sum_c exp(z_rc - m_r),  loss_r = m_r - z_r,label + log s_r,
//   G = (exp(z - m) / s - onehot(label)) * (row factor),  dh = G W,  dW = G^T h,  db = sum_r G.
// The logits [n, C] exist only as tiles in registers. Forward: every workgroup leaves (maximum, sum of exponentials) of its tile's
// rows, a second launch joins them. Backward: the logits are computed again in pieces of the vocabulary; a piece's G leaves in
// 16-bit parts and feeds the two gradient products before the next piece overwrites it. 8 n K C operations instead of the 6 n K C
// with kept logits, against 8 bytes of fp32 logit traffic per element of [n, C].
//
// All three products run on one tile engine (pg_mm.h) with fp32 accumulation. Its operands are 16-bit parts in rows padded to
// whole tiles: 16-bit rows that are so already are used in place, others are packed first (k_lx_pack). fp32 values are split
// into three bf16 parts (x = x0 + x1 + x2 exactly, each at most 2^-8 of the one before) and six of the nine partial products are
// summed; the three left out, x1 y2 + x2 y1 + x2 y2, are below 2^-22.9 of the product. 2.5 PF / 6 where the fp32 matrix
// instructions reach 0.157 PF. An infinite element has parts that are NaN, and so are the logits it enters.
// G of 16-bit operands is held in 16 bits: |G| <= 1 and each element is off by half a step (bf16 2^-8, fp16 2^-11 relative),
// independently per element, as are the outputs, which leave in the same type. fp16 G is held times 2^14 so that a probability
// of 2^-28 is still a normal number.
// Measured at bf16 8192 x 1024 -> 65536 (2 n K C = 1.1 TFLOP a product; the library's 16384^3 product reaches 1.47 PF on the same
// card): statistics 1.09 ms, G 1.32 ms, dh 1.01 ms, dW 0.95 ms, that is 1.01, 0.83, 1.09, 1.15 PF, 4.3 ms with gradients.
#include "pg_xent_narrow.h"

namespace pg {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;
constexpr float kLowest = -3.402823466e38f;                // what a finite logit is at least, in base 2
constexpr float kTopBf16 = 3.38953139e38f;                 // bf16's largest

// how an operand type is multiplied: the parts' type and number, G's scale
template <typename T> struct Mul;
template <> struct Mul<float>  { typedef bf16_t E; static constexpr int NP = 3; static constexpr float G = 1.f; };
template <> struct Mul<bf16_t> { typedef bf16_t E; static constexpr int NP = 1; static constexpr float G = 1.f; };
template <> struct Mul<f16_t>  { typedef f16_t E;  static constexpr int NP = 1; static constexpr float G = 16384.f; };

struct LxArgs {
  const void *h, *w, *bias;                // operands in parts: h [parts][h_rows][h_ld], w [parts][w_rows][w_ld]
  int64_t h_ld, h_part, h_rows, w_ld, w_part;
  const int64_t* labels;
  int64_t n, K, Kp, C, ignore;             // Kp: K padded to whole tiles
  float2* part;                            // [n][tiles] maximum, sum of exponentials
  float *zlab, *top, *sum, *row_loss, *meta;
  int64_t tiles;
  // backward
  const float* rowf;                       // row factors: the normalised incoming gradients (NULL: 1 for rows that count)
  const float *f1, *f2;                    // the outputs' factor = *f1 * *f2 (NULL = 1)
  void* g;                                 // a piece of G: [parts][g_rows][ldg], zeros beyond n and beyond c_hi
  int64_t ldg, g_rows, c_lo, c_hi;         // the piece's classes
  float* acc;                              // fp32 partial products [split][rows][K]
  float* dbp;                              // [row tiles][C] partial sums of G
  const float *bias2, *top2, *inv2, *rowf2;        // side arrays (SideArgs)
  const int32_t* lab2;
  int32_t scaled, late;                    // G carries the row factors; dh's rows get them behind the product
  void *dh, *dw, *db;
  int64_t range;                           // reduction range of one split
  int32_t splits, first, direct;           // direct: one split and one piece, the product itself is the output
};

__device__ __forceinline__ bool label_ok(int64_t lab, const LxArgs& a) { return lab != a.ignore && lab >= 0 && lab < a.C; }
__device__ __forceinline__ float out_factor(const LxArgs& a) { return (a.f1 ? *a.f1 : 1.f) * (a.f2 ? *a.f2 : 1.f); }

// rows of T as padded rows of parts: dst [NP][rows_p][ldp]; columns beyond K, rows beyond `rows` and (labels != NULL) rows that do
// not count are zeros, whatever the source holds there
struct PackArgs {
  const void* src;
  void* dst;
  int64_t rows, rows_p, K, ld, ldp;
  const int64_t* labels;
  int64_t ignore, C;
};
// what the products' epilogues read beside the operands, padded past the last class / row (see NxArgs): base-2 biases, labels as int32,
// and for the gradients the rows' largest logits, the inverses of their sums (times G's scale) and their factors. The two stay apart:
// in one number, log2 of the sum would be lost beside a large logit (rows of nothing but masked classes: exponentials of 1 each
// instead of one C-th)
struct SideArgs {
  const void* bias;
  float *bias2, *top2, *inv2, *rowf2;      // bias2 == NULL: nothing to do; top2 == NULL: no gradients
  int32_t* lab;
  const float *top, *sum, *rowf;
  const int64_t* labels;
  int64_t n, rows_p, C, classes_p, ignore;
};
template <typename T>
__device__ __forceinline__ void lx_side(const SideArgs& a) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.classes_p || i < a.rows_p; i += (int64_t)gridDim.x * 256) {
    if (i < a.classes_p) {
      float b = i < a.C ? 0.f : -INFINITY;
      if (i < a.C && a.bias) {
        b = (float)((const T*)a.bias)[i];
        // (a finite lowest value stays finite: a row of nothing else is uniform, as in natural units)
        b = b == -INFINITY ? b : b * kLog2e < kLowest ? kLowest : b * kLog2e;
      }
      a.bias2[i] = b;
    }
    if (i < a.rows_p) {
      const int64_t lab = i < a.n ? a.labels[i] : -1;
      const bool ok = i < a.n && lab != a.ignore && lab >= 0 && lab < a.C;
      if (a.top2) {
        const float f = !ok ? 0.f : a.rowf ? a.rowf[i] : 1.f;
        a.top2[i] = f != 0.f ? a.top[i] : INFINITY;          // rows without a gradient: exponentials of 0
        a.inv2[i] = f != 0.f ? Mul<T>::G / a.sum[i] : 0.f;
        a.rowf2[i] = f;
        a.lab[i] = f != 0.f ? (int32_t)lab : -1;
      } else {
        a.lab[i] = ok ? (int32_t)lab : -1;
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void k_lx_pack(PackArgs a0, PackArgs a1, SideArgs side) {
  typedef typename Mul<T>::E E;
  if (blockIdx.y == 2) {
    if (side.bias2) lx_side<T>(side);
    return;
  }
  const PackArgs& a = blockIdx.y ? a1 : a0;
  if (!a.dst) return;
  const int64_t ch = a.ldp / 8, total = a.rows_p * ch;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
    const int64_t r = t / ch, c = (t - r * ch) * 8;
    bool ok = r < a.rows;
    if (ok && a.labels) {
      const int64_t lab = a.labels[r];
      ok = lab != a.ignore && lab >= 0 && lab < a.C;
    }
    const T* s = (const T*)a.src + r * a.ld + c;
    T v[8];
    if (ok && c + 8 <= a.K) {
      __builtin_memcpy(v, s, sizeof(v));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = ok && c + i < a.K ? s[i] : (T)0.f;
    }
    E o[8];
    E* d = (E*)a.dst + r * a.ldp + c;
    if constexpr (Mul<T>::NP == 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = (E)v[i];
      __builtin_memcpy(d, o, sizeof(o));
    } else {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = v[i];
#pragma unroll
      for (int p = 0; p < 3; ++p) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          o[i] = (E)x[i];
          // (a finite value above bf16's largest would round to infinity: its first part is the largest)
          if (p == 0 && fabsf(x[i]) < INFINITY && fabsf((float)o[i]) == INFINITY) o[i] = (E)copysignf(kTopBf16, x[i]);
          x[i] -= (float)o[i];                       // exact
        }
        __builtin_memcpy(d + p * a.rows_p * a.ldp, o, sizeof(o));
      }
    }
  }
}

// One BM-class x BN-row tile of logits; a lane holds one row's classes in registers: row = 32 j + lane % 32 of its wave's rows,
// class = 32 i + 8 (e / 4) + 4 (lane / 32) + e % 4 of its wave's classes, so a row's maximum and sum are taken in registers.
// The tile's exponentials, and G's LDS trip, follow its product: at bf16 8192 x 1024 -> 65536 the statistics take 8 % longer than a
// product of this size without them (k_lx_dh), G 31 %. The matrix units are busy in 56 and 44 % of the cycles: mm_run bounds both.
// PIECE: writes G (through LDS: whole 16-byte pieces of rows) and the column sums of the tile, else the tile's row statistics.
template <typename T, typename S, bool PIECE>
__global__ __launch_bounds__(S::THREADS, 2) void k_lx_logits(LxArgs a) {
  typedef typename S::E E;
  constexpr int BM = S::BM, BN = S::BN, WM = BM / S::WR, WN = BN / S::WC;
  // behind the tile buffers: the tile's biases (base 2, -inf beyond the last class: their exponentials are 0), the waves' statistics
  PG_MM_LDS(S, buf, 2 * BM + (PIECE ? 0 : 4 * S::WR * BN));
  float* bias = reinterpret_cast<float*>(buf + S::NB * S::TILE);
  float2(*red)[BN] = reinterpret_cast<float2(*)[BN]>(bias + BM);
  const uint32_t row_tiles = (uint32_t)ceil_div<int64_t>(a.n, BN), c_tiles = (uint32_t)ceil_div<int64_t>(a.c_hi - a.c_lo, BM);
  // an XCD's 32 CUs work on 8 row tiles x 4 class tiles at a time
  const uint32_t t = xcd_run(blockIdx.x, gridDim.x), group = t / (8 * c_tiles);
  const uint32_t in_group = row_tiles - group * 8 < 8 ? row_tiles - group * 8 : 8, u = t - group * 8 * c_tiles;
  const int ct = uniform((int)(u / in_group)), rt = uniform((int)(group * 8 + u % in_group));
  const int64_t r0 = (int64_t)rt * BN, c0 = a.c_lo + (int64_t)ct * BM;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / S::WC, wn = wave % S::WC;
  for (int c = tid; c < BM; c += S::THREADS) bias[c] = a.bias2[c0 + c];
  f32x16 acc[S::FI][S::FJ] = {};
  mm_product<S, ROWS, ROWS>(Operand{a.w, a.w_ld, a.w_part, c0, a.C, 0}, Operand{a.h, a.h_ld, a.h_part, r0, a.h_rows, 0}, 0, a.Kp, buf, acc);
  const int cw = wm * WM + 4 * (lane >> 5);                  // the lane's first class within the tile
  int at[S::FJ];                                             // the rows' labels, counted from there
  float top[S::FJ], inv[S::FJ];
#pragma unroll
  for (int j = 0; j < S::FJ; ++j) {
    const int64_t r = r0 + wn * WN + j * 32 + (lane & 31);   // (the side arrays are padded to whole tiles of rows)
    at[j] = a.lab2[r] - (int)c0 - cw;
    top[j] = PIECE ? a.top2[r] : 0.f;
    inv[j] = PIECE ? a.inv2[r] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < S::FI; ++i) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4 b = *reinterpret_cast<const float4*>(bias + cw + i * 32 + 8 * q);
#pragma unroll
      for (int j = 0; j < S::FJ; ++j) {
        acc[i][j][4 * q] = fmaf(acc[i][j][4 * q], kLog2e, b.x);
        acc[i][j][4 * q + 1] = fmaf(acc[i][j][4 * q + 1], kLog2e, b.y);
        acc[i][j][4 * q + 2] = fmaf(acc[i][j][4 * q + 2], kLog2e, b.z);
        acc[i][j][4 * q + 3] = fmaf(acc[i][j][4 * q + 3], kLog2e, b.w);
      }
    }
#pragma unroll
    for (int j = 0; j < S::FJ; ++j) {
      if constexpr (PIECE) {
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = lx_exp(acc[i][j][e] - top[j]) * inv[j];
      }
      if (__any((unsigned)(at[j] - 32 * i) < 32u)) {         // does any of the wave's rows have its label among these 32 classes?
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (at[j] == i * 32 + 8 * (e / 4) + e % 4) {
            if constexpr (PIECE)
              acc[i][j][e] -= Mul<T>::G;
            else
              a.zlab[r0 + wn * WN + j * 32 + (lane & 31)] = acc[i][j][e];
          }
      }
    }
  }
  if constexpr (!PIECE) {
#pragma unroll
    for (int j = 0; j < S::FJ; ++j) {
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < S::FI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) m = fmaxf(m, acc[i][j][e]);
      m = fmaxf(m, __shfl_xor(m, 32, kWave));
      const float base = m == -INFINITY ? 0.f : m;         // nothing but -inf so far: every exponential is 0
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < S::FI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) s += __builtin_amdgcn_exp2f(acc[i][j][e] - base);
      s += __shfl_xor(s, 32, kWave);
      if (lane < 32) red[wm][wn * WN + j * 32 + lane] = make_float2(m, s);
    }
    __syncthreads();
    for (int rl = tid; rl < BN; rl += S::THREADS)
      if (r0 + rl < a.n) {
        float m = red[0][rl].x, s = 0.f;
#pragma unroll
        for (int i = 1; i < S::WR; ++i) m = fmaxf(m, red[i][rl].x);
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int i = 0; i < S::WR; ++i) s += red[i][rl].y * __builtin_amdgcn_exp2f(red[i][rl].x - base);
        a.part[(r0 + rl) * a.tiles + ct] = make_float2(m, s);
      }
  } else {
    if (a.scaled) {                                          // rows with factors of their own
#pragma unroll
      for (int j = 0; j < S::FJ; ++j) {
        const float f = a.rowf2[r0 + wn * WN + j * 32 + (lane & 31)];
#pragma unroll
        for (int i = 0; i < S::FI; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[i][j][e] = f == 0.f ? 0.f : acc[i][j][e] * f;
      }
    }
    // [BN rows][BM classes] of one part in the tile buffers, 16-byte chunks swizzled by the row
    constexpr int CH = BM / 8, RP = S::THREADS / CH;
    static_assert(BM * BN <= S::NB * S::TILE, "a part of G fits the tile buffers");
    static_assert(RP * BM * 2 <= S::NB * S::TILE, "and so do its column sums");
    float sum[8] = {};
#pragma unroll 1
    for (int part = 0; part < S::NP; ++part) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < S::FJ; ++j) {
        const int rl = wn * WN + j * 32 + (lane & 31);
#pragma unroll
        for (int i = 0; i < S::FI; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            E o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              o[e] = (E)acc[i][j][q * 4 + e];
              acc[i][j][q * 4 + e] -= (float)o[e];
            }
            const int chunk = (wm * WM + i * 32 + 8 * q) / 8;
            __builtin_memcpy(buf + rl * BM + ((chunk ^ (rl & (CH - 1))) << 3) + 4 * (lane >> 5), o, 8);
          }
      }
      __syncthreads();
      const int ch = tid % CH;
      E* g = (E*)a.g + part * a.g_rows * a.ldg + r0 * a.ldg + (c0 - a.c_lo) + ch * 8;
      for (int rl = tid / CH; rl < BN; rl += RP) {
        E o[8];
        __builtin_memcpy(o, buf + rl * BM + ((ch ^ (rl & (CH - 1))) << 3), 16);
        __builtin_memcpy(g + rl * a.ldg, o, 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += (float)o[e];
      }
    }
    __syncthreads();
    float* cs = (float*)buf;
#pragma unroll
    for (int e = 0; e < 8; ++e) cs[(tid / CH) * BM + tid % CH * 8 + e] = sum[e];
    __syncthreads();
    for (int c = tid; c < BM; c += S::THREADS)
      if (c0 + c < a.c_hi) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < RP; ++i) s += cs[i * BM + c];
        a.dbp[rt * a.C + c0 + c] = s;
      }
  }
}

// a wave per row: joins the tiles' (narrow form: the splits') statistics, in base 2
template <typename T>
__global__ __launch_bounds__(256) void k_lx_rows(LxArgs a) {
  const int lane = threadIdx.x & 63;
  for (int64_t r = (int64_t)blockIdx.x * 4 + threadIdx.x / 64; r < a.n; r += (int64_t)gridDim.x * 4) {
    float m = -INFINITY, s = 0.f;
    for (int64_t t = lane; t < a.tiles; t += 64) {
      const float2 x = a.part[r * a.tiles + t];
      const float mm = fmaxf(m, x.x), base = mm == -INFINITY ? 0.f : mm;
      s = s * __builtin_amdgcn_exp2f(m - base) + x.y * __builtin_amdgcn_exp2f(x.x - base);
      m = mm;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const float om = __shfl_xor(m, o, kWave), os = __shfl_xor(s, o, kWave);
      const float mm = fmaxf(m, om), base = mm == -INFINITY ? 0.f : mm;
      s = s * __builtin_amdgcn_exp2f(m - base) + os * __builtin_amdgcn_exp2f(om - base);
      m = mm;
    }
    if (lane == 0) {
      const bool ok = label_ok(a.labels[r], a);
      a.top[r] = m;
      a.sum[r] = !ok ? 0.f : s > 0.f ? s : NAN;             // (a row of nothing but -inf counts, and its loss is NaN)
      float loss = 0.f;
      if (ok) {
        const float z = a.zlab[r];
        loss = ((m - z) + log2f(s)) * kLn2;
        // the label's own class is masked by a finite bias that base 2 cannot hold (lx_side), another class is not: beside such a
        // bias h W is lost, the logit is the bias
        if (z == kLowest && m > kLowest && a.bias) {
          const float b = (float)((const T*)a.bias)[a.labels[r]];
          if (b * kLog2e < kLowest) loss = (m + log2f(s)) * kLn2 - b;
        }
      }
      a.row_loss[r] = loss;
    }
  }
}
template <typename T>
int lx_rows(const LxArgs& a, hipStream_t st) {
  const int64_t blocks = ceil_div<int64_t>(a.n, 4);
  hipLaunchKernelGGL(k_lx_rows<T>, dim3((unsigned)(blocks > 65536 ? 65536 : blocks)), dim3(256), 0, st, a);
  PG_LAUNCH_CHECK();
  return PG_OK;
}

// one block, fixed order: the loss (mean or sum) and meta = 1 / counted rows
__global__ __launch_bounds__(1024) void k_lx_mean(const float* __restrict__ row_loss, const float* __restrict__ sum, int64_t n,
                                                  int mean, float* __restrict__ loss, float* __restrict__ meta) {
  __shared__ float ss[1024];
  __shared__ int sc[1024];
  float s = 0.f;
  int c = 0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) {
    s += row_loss[i];
    c += sum[i] != 0.f;
  }
  ss[threadIdx.x] = s;
  sc[threadIdx.x] = c;
  __syncthreads();
  for (int o = 512; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) {
      ss[threadIdx.x] += ss[threadIdx.x + o];
      sc[threadIdx.x] += sc[threadIdx.x + o];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    *loss = !mean ? ss[0] : sc[0] > 0 ? ss[0] / (float)sc[0] : NAN;       // as ops.cross_entropy: a mean over no rows
    *meta = sc[0] > 0 ? 1.f / (float)sc[0] : 0.f;
  }
}

// incoming gradients of single rows: row factors g / max|g| (G then uses its type's range whatever the caller's scale), the
// maximum becomes the outputs' factor. Of the finite ones: an infinite or NaN gradient stays that, in its own row
__global__ __launch_bounds__(1024) void k_lx_row_factors(const float* __restrict__ g, int64_t gs, const float* __restrict__ sum,
                                                         int64_t n, float* __restrict__ rowf, float* __restrict__ top) {
  __shared__ float ss[1024];
  float m = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += 1024)
    if (sum[i] != 0.f && fabsf(g[i * gs]) < INFINITY) m = fmaxf(m, fabsf(g[i * gs]));
  ss[threadIdx.x] = m;
  __syncthreads();
  for (int o = 512; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) ss[threadIdx.x] = fmaxf(ss[threadIdx.x], ss[threadIdx.x + o]);
    __syncthreads();
  }
  m = ss[0] > 0.f ? ss[0] : 1.f;
  for (int64_t i = threadIdx.x; i < n; i += 1024) rowf[i] = sum[i] != 0.f ? g[i * gs] / m : 0.f;
  if (threadIdx.x == 0) *top = m;
}

// f(row, column, value) for the values a lane holds that lie inside rows x cols of the tile
template <typename S, typename F>
__device__ __forceinline__ void each_output(const f32x16 (&acc)[S::FI][S::FJ], int row, int col, int rows, int cols, F f) {
#pragma unroll
  for (int j = 0; j < S::FJ; ++j)
    if (col + 32 * j < cols) {
#pragma unroll
      for (int i = 0; i < S::FI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int r = row + i * 32 + 8 * (e / 4) + e % 4;
          if (r < rows) f(r, col + 32 * j, acc[i][j][e]);
        }
    }
}

// G [rows x classes] W: G's rows are read as they stand, W through the transposing reads. Matrix units busy in 59 % of the cycles (mm_run).
// dh: acc[split][r][k] (+)= sum over the split's classes of G[r][c] W[c][k]
template <typename T, typename S>
__global__ __launch_bounds__(S::THREADS, 2) void k_lx_dh(LxArgs a) {
  constexpr int WM = S::BM / S::WR, WN = S::BN / S::WC;
  PG_MM_LDS(S, buf, 0);
  const uint32_t row_tiles = (uint32_t)ceil_div<int64_t>(a.n, S::BM), k_tiles = (uint32_t)ceil_div<int64_t>(a.K, S::BN);
  const uint32_t t = xcd_run(blockIdx.x, gridDim.x);
  const int kt = uniform((int)(t % k_tiles)), rt = uniform((int)(t / k_tiles % row_tiles)), sp = uniform((int)(t / k_tiles / row_tiles));
  const int64_t r0 = (int64_t)rt * S::BM, n0 = (int64_t)kt * S::BN, len = (a.c_hi - a.c_lo + kPad - 1) / kPad * kPad;
  const int64_t lo = sp * a.range, hi = lo + a.range < len ? lo + a.range : len;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / S::WC, wn = wave % S::WC;
  const int rl = wm * WM + 4 * (lane >> 5), kl = wn * WN + (lane & 31);       // the lane's first row, first column of the tile
  const int rows = (int)(a.n - r0 < S::BM ? a.n - r0 : S::BM), cols = (int)(a.K - n0 < S::BN ? a.K - n0 : S::BN);
  float* sum = a.acc + sp * a.n * a.K + r0 * a.K + n0;
  f32x16 acc[S::FI][S::FJ] = {};
  if (!a.first) {                              // on top of the earlier pieces' sum (before the product: all loads at once)
#pragma unroll
    for (int j = 0; j < S::FJ; ++j) {
      const int k = kl + 32 * j < cols ? kl + 32 * j : cols - 1;
#pragma unroll
      for (int i = 0; i < S::FI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int r = rl + i * 32 + 8 * (e / 4) + e % 4;
          acc[i][j][e] = sum[(r < rows ? r : rows - 1) * a.K + k];
        }
    }
  }
  mm_product<S, ROWS, COLS>(Operand{a.g, a.ldg, a.g_rows * a.ldg, r0, a.g_rows, 0},
                            Operand{(const short*)a.w + a.c_lo * a.w_ld, a.w_ld, a.w_part, n0, 0, a.Kp}, lo, hi, buf, acc);
  // (rows that do not count leave as zeros, whatever W holds; the row factors are padded to whole tiles)
  const float f = a.direct ? out_factor(a) / Mul<T>::G : 1.f;
  const bool late = a.late && a.c_hi == a.C;               // behind the last piece's share
  T* out = (T*)a.dh + r0 * a.K + n0;
#pragma unroll
  for (int i = 0; i < S::FI; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4 v4 = *reinterpret_cast<const float4*>(a.rowf2 + r0 + rl + i * 32 + 8 * q);
      const float rf[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = rl + i * 32 + 8 * q + e;
        if (r >= rows) continue;
        const float fr = late ? rf[e] * f : f;
#pragma unroll
        for (int j = 0; j < S::FJ; ++j) {
          const int k = kl + 32 * j;
          if (k >= cols) continue;
          const float v = rf[e] == 0.f ? 0.f : acc[i][j][4 * q + e] * fr;
          if (a.direct) out[r * a.K + k] = (T)v;
          else sum[r * a.K + k] = v;
        }
      }
    }
}

// partial sums added in order: out[i] = (sum over splits of acc[split][i]) * factor. Up to three such sums a launch
struct SumArgs {
  const float* acc;
  void* out;
  int64_t total, splits;
};
template <typename T>
__global__ __launch_bounds__(256) void k_lx_sums(SumArgs a0, SumArgs a1, SumArgs a2, const float* f1, const float* f2) {
  const SumArgs& a = blockIdx.y == 0 ? a0 : blockIdx.y == 1 ? a1 : a2;
  if (!a.out) return;
  const float f = (f1 ? *f1 : 1.f) * (f2 ? *f2 : 1.f) / Mul<T>::G;
  for (int64_t t = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; t < a.total; t += (int64_t)gridDim.x * 1024) {
    float s[4] = {0.f, 0.f, 0.f, 0.f}, v[4];
#pragma unroll 4
    for (int64_t i = 0; i < a.splits; ++i) {
      load4_tail(a.acc + i * a.total + t, a.total - t, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += v[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] *= f;
    store4_tail((T*)a.out + t, a.total - t, s);
  }
}
template <typename T>
int lx_sums(const SumArgs& a, const SumArgs& b, const SumArgs& c, const LxArgs& x, hipStream_t st) {
  int64_t most = a.out ? a.total : 0;
  if (b.out && b.total > most) most = b.total;
  if (c.out && c.total > most) most = c.total;
  if (most == 0) return PG_OK;
  const int64_t blocks = ceil_div<int64_t>(most, 1024);
  hipLaunchKernelGGL(k_lx_sums<T>, dim3((unsigned)(blocks > 4096 ? 4096 : blocks), c.out ? 3 : b.out ? 2 : 1), dim3(256), 0, st, a, b, c, x.f1, x.f2);
  PG_LAUNCH_CHECK();
  return PG_OK;
}

// G^T h, both through the transposing reads (neither is ever transposed in memory). Matrix units busy in 59 % of the cycles (mm_run).
// dW rows of a piece: sum over the split's rows of G[r][c] h[r][k]
template <typename T, typename S>
__global__ __launch_bounds__(S::THREADS, 2) void k_lx_dw(LxArgs a) {
  constexpr int WM = S::BM / S::WR, WN = S::BN / S::WC;
  PG_MM_LDS(S, buf, 0);
  const int64_t len = a.c_hi - a.c_lo, rows = (a.n + kPad - 1) / kPad * kPad;
  const uint32_t c_tiles = (uint32_t)ceil_div<int64_t>(len, S::BM), k_tiles = (uint32_t)ceil_div<int64_t>(a.K, S::BN), t = xcd_run(blockIdx.x, gridDim.x);
  const int kt = uniform((int)(t % k_tiles)), ct = uniform((int)(t / k_tiles % c_tiles)), sp = uniform((int)(t / k_tiles / c_tiles));
  const int64_t c0 = (int64_t)ct * S::BM, n0 = (int64_t)kt * S::BN;
  const int64_t lo = sp * a.range, hi = lo + a.range < rows ? lo + a.range : rows;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / S::WC, wn = wave % S::WC;
  f32x16 acc[S::FI][S::FJ] = {};
  mm_product<S, COLS, COLS>(Operand{a.g, a.ldg, a.g_rows * a.ldg, c0, 0, a.ldg},
                            Operand{a.h, a.h_ld, a.h_part, n0, 0, a.Kp}, lo, hi, buf, acc);
  const int cl = wm * WM + 4 * (lane >> 5), kl = wn * WN + (lane & 31);
  const int cs = (int)(len - c0 < S::BM ? len - c0 : S::BM), cols = (int)(a.K - n0 < S::BN ? a.K - n0 : S::BN);
  if (a.splits > 1) {
    float* out = a.acc + (sp * len + c0) * a.K + n0;
    each_output<S>(acc, cl, kl, cs, cols, [&](int c, int k, float v) { out[c * a.K + k] = v; });
  } else {
    const float f = out_factor(a) / Mul<T>::G;
    T* out = (T*)a.dw + (a.c_lo + c0) * a.K + n0;
    each_output<S>(acc, cl, kl, cs, cols, [&](int c, int k, float v) { out[c * a.K + k] = (T)(v * f); });
  }
}

inline int64_t up(int64_t v, int64_t m) { return ceil_div(v, m) * m; }
inline bool launchable(int64_t blocks, int64_t threads) { return blocks * threads < (int64_t(1) << 32); }

// tile shapes (BM x BN): one workgroup of 256 x 256 tiles fills a CU's LDS or registers, two of the others do
enum { BIG = 0, TALL = 1, MID = 2 };

// sizes of one call: everything follows from the shapes, types and alignments of the operands, so that the scratch the caller
// allocates (for packed operands always) fits the launches
struct LxPlan {
  int64_t Kp, h_rows, w_rows, tiles, row_tiles, piece, ldg, g_rows;
  int64_t h_bytes, w_bytes, part_bytes, g_bytes, acc_dh, acc_dw, dbp_bytes;
  int32_t dh_splits, dw_splits, pieces;
  int64_t dh_range, dw_range;
  int logits, dh, dw;                       // tile shapes
  // narrow form
  int narrow, xt_stats, xt_grad, yt;
  int32_t nx_stats, nx_dh, nx_dw;           // splits
  int64_t rs_stats, rs_dh, rs_dw;           // their ranges
  int64_t classes_p, rows_p, side_bytes;
  bool fits;                                // every launch has fewer than 2^32 threads
};

// splits of the narrow form's y for t tiles of x: every CU gets the same number of workgroups, or nearly, and at least two of them
// where there is that much work; a split adds a partial result to write and to sum
inline void narrow_split(int64_t t, int64_t y_tiles, int32_t* splits, int64_t* range, int64_t yt) {
  int64_t best = 1;
  double cost = 1e30;
  for (int64_t s = 1; s <= 512 && s * 4 <= y_tiles + 3; ++s) {
    const double c = (double)ceil_div<int64_t>(t * s, 256) / (double)s + (t * s < 512 ? 0.25 * (double)t / 256. : 0.) + 0.002 * (double)(t * s) / 256.;
    if (c < cost) { cost = c; best = s; }
  }
  const int64_t r = ceil_div<int64_t>(y_tiles, best);
  *range = r * yt;
  *splits = (int32_t)ceil_div<int64_t>(y_tiles, r);
}

inline LxPlan lx_plan(int64_t n, int64_t K, int64_t C, int32_t dtype, bool backward) {
  LxPlan p{};
  const int64_t np = dtype == PG_DTYPE_F32 ? 3 : 1;
  p.Kp = up(K, kPad);
  p.h_rows = up(n, 256);
  p.h_bytes = up(np * p.h_rows * p.Kp * 2, 256);
  p.w_rows = up(C, kPad);
  p.w_bytes = up(np * p.w_rows * p.Kp * 2, 256);
  p.classes_p = up(C, 256) + 64;
  p.rows_p = p.h_rows + 64;
  p.side_bytes = up(p.classes_p * 4, 256) + 4 * up(p.rows_p * 4, 256);
  // (us, narrow against wide. fp32 6000 -> 50000: 64 columns forward 223, 343, with gradients 998, 2645; 128: 424, 501 and 1970,
  // 3464. bf16 8192 -> 65536: 128 columns 188, 264 and 763, 1408; 192: 239, 325 and 1025, 1712; 256: forward 269, 390, but the
  // gradients alone 1652, 1478, since 256 columns of operands and sums do not fit the registers of a wave)
  p.narrow = p.Kp <= (np == 3 ? 128 : backward ? 192 : 256);
  if (p.narrow) {
    p.xt_stats = 128 * narrow_xb((int)np, (int)p.Kp, NX_STATS);
    p.xt_grad = 128 * narrow_xb((int)np, (int)p.Kp, NX_DH);
    p.yt = np * p.Kp <= 256 ? 64 : 32;
    const int64_t classes = ceil_div<int64_t>(C, p.yt);
    narrow_split(ceil_div<int64_t>(n, p.xt_stats), classes, &p.nx_stats, &p.rs_stats, p.yt);
    narrow_split(ceil_div<int64_t>(n, p.xt_grad), classes, &p.nx_dh, &p.rs_dh, p.yt);
    narrow_split(ceil_div<int64_t>(C, p.xt_grad), ceil_div<int64_t>(n, p.yt), &p.nx_dw, &p.rs_dw, p.yt);
    p.part_bytes = up(n * p.nx_stats * 8, 256);
    p.acc_dh = p.nx_dh > 1 ? up((int64_t)p.nx_dh * n * K * 4, 256) : 0;
    p.acc_dw = p.nx_dw > 1 ? up((int64_t)p.nx_dw * C * (K + 1) * 4, 256) : 0;
    p.fits = backward ? launchable(ceil_div<int64_t>(n, p.xt_grad) * p.nx_dh, 256) && launchable(ceil_div<int64_t>(C, p.xt_grad) * p.nx_dw, 256)
                      : launchable(ceil_div<int64_t>(n, p.xt_stats) * p.nx_stats, 256);
    return p;
  }
  // 256 x 256 tiles need a quarter less LDS traffic and two thirds of the loads of 128 x 128 ones, and fill the card from 256 tiles
  // on: at half of that 128 x 128 ones, two to a CU, are ahead (fp16 777 x 602 -> 1153, 20 against 70 tiles: logits 22 -> 12.5 us).
  // 256 x 128 tiles, two to a CU, hide one tile's exponentials behind the other's products, which pays while the exponentials are
  // a good part of a tile (us with gradients, 256 x 256 against 256 x 128: bf16 8192 x 320 -> 65536 2125, 2050; 8192 x 512 -> 32768
  // 1259, 1188; 8192 x 768 -> 32768 1971, 1936; 8192 x 1024 -> 65536 4204, 4288; fp32, six products a tile: 4096 x 1024 -> 16384
  // 2849, 3059)
  const bool big = ceil_div<int64_t>(n, 256) * ceil_div<int64_t>(C, 256) >= 192;
  p.logits = !big ? MID : np == 1 && p.Kp <= 768 ? TALL : BIG;
  p.tiles = ceil_div<int64_t>(C, big ? 256 : 128);
  p.row_tiles = ceil_div<int64_t>(n, p.logits == BIG ? 256 : 128);
  p.part_bytes = up(n * p.tiles * 8, 256);
  // a piece of G: half a GB (128 MB, 256 MB, half a GB: 4690, 4363, 4280 us at bf16 8192 x 1024 -> 65536, 3005, 2847, 2680 at fp16
  // 16384 x 512 -> 32768: fewer launches with a ragged end each, and fewer passes over dh's running sum)
  p.g_rows = up(n, 256);
  int64_t cols = (int64_t(512) << 20) / (np * 2 * p.g_rows) / 256 * 256;
  if (cols < 256) cols = 256;
  if (cols > (1 << 18)) cols = 1 << 18;
  p.pieces = (int32_t)ceil_div<int64_t>(C, cols);
  p.piece = up(ceil_div<int64_t>(C, p.pieces), 256);
  p.pieces = (int32_t)ceil_div<int64_t>(C, p.piece);
  p.ldg = p.piece + 64;        // (rows a power of two apart would share their memory channels: dh 296 -> 279 us at 8192 x 1024 -> 65536)
  p.g_bytes = up(np * p.g_rows * p.ldg * 2, 256);
  // A gradient's tiles and the splits of its reduction: the cheapest by a count of rounds of workgroups over the card, in units of a
  // round of 256 x 256 tiles. For the same product 256 x 128 tiles take 1.13 times as long as those and 128 x 128 ones 1.31 times
  // (bf16 8192 x 1024 -> 65536 gradients 2069, 2342, 2714 us; fp32 4096 x 1024 -> 16384 1474, 1662, 1943), but they leave less of
  // the card idle: bf16 3000 x 300 -> 40000 with gradients 538 us with 256 x 256 alone, 494 so; fp16 777 x 602 -> 1153 165, 143
  p.fits = launchable((backward ? ceil_div<int64_t>(p.piece, big ? 256 : 128) : p.tiles) * p.row_tiles, p.logits == BIG ? 512 : 256);
  auto split = [&](int64_t rows, int64_t len, int* shape, int32_t* s, int64_t* range) {
    const struct { int64_t bm, bn, slots; double unit; } shapes[] = {{256, 256, 256, 1.}, {256, 128, 512, 1.13}, {128, 128, 512, 0.65}};
    // a split's partial result, written and read at 5 TB/s, in units of a round
    const double extra = (double)rows * (double)K / (double)len * 6.7e-5 / (np == 3 ? 6. : 1.);
    double best = 1e30;
    for (int i = BIG; i <= MID; ++i) {
      const int64_t tiles = ceil_div<int64_t>(rows, shapes[i].bm) * ceil_div<int64_t>(K, shapes[i].bn);
      for (int64_t k = 1; k <= 64 && (k == 1 || k * 4 * kPad <= len); ++k) {
        const double cost = shapes[i].unit * (double)ceil_div<int64_t>(tiles * k, shapes[i].slots) / (double)k + (k > 1 ? extra * (double)k : 0.);
        if (cost < best * 0.999) { best = cost; *shape = i; *s = (int32_t)k; }
      }
    }
    *range = up(ceil_div<int64_t>(len, *s), kPad);
    *s = (int32_t)ceil_div<int64_t>(len, *range);
    if (backward)
      p.fits = p.fits && launchable(ceil_div<int64_t>(rows, shapes[*shape].bm) * ceil_div<int64_t>(K, shapes[*shape].bn) * *s, *shape == BIG ? 512 : 256);
  };
  split(n, p.piece, &p.dh, &p.dh_splits, &p.dh_range);
  split(p.piece, up(n, kPad), &p.dw, &p.dw_splits, &p.dw_range);
  p.acc_dh = p.dh_splits > 1 || p.pieces > 1 ? up((int64_t)p.dh_splits * n * K * 4, 256) : 0;
  p.acc_dw = p.dw_splits > 1 ? up((int64_t)p.dw_splits * p.piece * K * 4, 256) : 0;
  p.dbp_bytes = up(p.row_tiles * C * 4, 256);
  return p;
}

template <typename T> using BigTile = Shape<typename Mul<T>::E, Mul<T>::NP, 256, 256, 2, 4, 4>;
template <typename T> using TallTile = Shape<typename Mul<T>::E, Mul<T>::NP, 256, 128, 2, 2, 3>;
template <typename T> using MidTile = Shape<typename Mul<T>::E, Mul<T>::NP, 128, 128, 2, 2, 4>;

// operands in parts: in place where they are padded 16-bit rows already, else packed into h_dst / w_dst by one launch
template <typename T>
int lx_operands(LxArgs& a, const pg_linear_xent_desc_t* d, const LxPlan& p, char* h_dst, char* w_dst, bool mask, const SideArgs& side, hipStream_t st) {
  constexpr int NP = Mul<T>::NP;
  auto fits = [&](const void* q, int64_t ld) { return NP == 1 && d->K == p.Kp && ld % 8 == 0 && ld < (1 << 21) && (uintptr_t)q % 16 == 0; };
  PackArgs h{}, w{};
  if (!mask && fits(d->h, d->h_stride)) {
    a.h = d->h; a.h_ld = d->h_stride; a.h_rows = d->n;
  } else {
    h = PackArgs{d->h, h_dst, d->n, p.h_rows, d->K, d->h_stride, p.Kp, d->labels, d->ignore_index, d->C};
    a.h = h_dst; a.h_ld = p.Kp; a.h_rows = p.h_rows; a.h_part = p.h_rows * p.Kp;
  }
  // (dh's product reads whole tiles of classes: in the wide form's backward pass only a table of such is used in place)
  if (fits(d->W, d->w_stride) && (p.narrow || !mask || d->C % kPad == 0)) {
    a.w = d->W; a.w_ld = d->w_stride;
  } else {
    w = PackArgs{d->W, w_dst, d->C, p.w_rows, d->K, d->w_stride, p.Kp, nullptr, 0, 0};
    a.w = w_dst; a.w_ld = p.Kp; a.w_part = p.w_rows * p.Kp;
  }
  if (!h.dst && !w.dst && !side.bias2) return PG_OK;
  const int64_t most = (w.dst && (!h.dst || p.w_rows > p.h_rows) ? p.w_rows : h.dst ? p.h_rows : 32) * (p.Kp / 8);
  const int64_t sides = p.classes_p > p.rows_p ? p.classes_p : p.rows_p, blocks = ceil_div<int64_t>(most > sides ? most : sides, 256);
  if (!h.dst) { h = w; w = PackArgs{}; }
  hipLaunchKernelGGL(k_lx_pack<T>, dim3((unsigned)(blocks > 4096 ? 4096 : blocks), side.bias2 ? 3 : w.dst ? 2 : 1), dim3(256), 0, st, h, w, side);
  PG_LAUNCH_CHECK();
  return PG_OK;
}

template <typename T, int KP, int MODE>
int launch_narrow_kp(const NxArgs& n, hipStream_t st) {
  constexpr int XB = narrow_xb(Mul<T>::NP, KP, MODE);
  hipLaunchKernelGGL((k_lx_narrow<T, KP, XB, MODE>), dim3((unsigned)(ceil_div<int64_t>(n.nx, 128 * XB) * n.splits)), dim3(256), 0, st, n);
  PG_LAUNCH_CHECK();
  return PG_OK;
}
template <typename T, int MODE>
int launch_narrow(const NxArgs& n, const LxPlan& p, hipStream_t st) {
  if (p.Kp == 64) return launch_narrow_kp<T, 64, MODE>(n, st);
  if constexpr (Mul<T>::NP == 1) {
    if (p.Kp == 192) return launch_narrow_kp<T, 192, MODE>(n, st);
    if constexpr (MODE == NX_STATS)
      if (p.Kp == 256) return launch_narrow_kp<T, 256, MODE>(n, st);
  }
  return launch_narrow_kp<T, 128, MODE>(n, st);
}

// the side arrays at s, in the order bias2 | labels | largest logits | inverse sums | row factors
inline SideArgs lx_side_arrays(const LxArgs& a, const LxPlan& p, char* s, bool grads) {
  SideArgs side{};
  const int64_t rows = up(p.rows_p * 4, 256);
  side.bias = a.bias; side.labels = a.labels; side.ignore = a.ignore;
  side.n = a.n; side.rows_p = p.rows_p; side.C = a.C; side.classes_p = p.classes_p;
  side.bias2 = (float*)s;
  side.lab = (int32_t*)(s + up(p.classes_p * 4, 256));
  if (grads) {
    side.top2 = (float*)((char*)side.lab + rows);
    side.inv2 = (float*)((char*)side.lab + 2 * rows);
    side.rowf2 = (float*)((char*)side.lab + 3 * rows);
    side.top = a.top; side.sum = a.sum; side.rowf = a.rowf;
  }
  return side;
}

inline NxArgs narrow_args(const LxArgs& a, bool classes_are_x) {
  NxArgs n{};
  if (classes_are_x) {
    n.x = a.w; n.x_ld = a.w_ld; n.x_part = a.w_part; n.x_rows = a.C; n.nx = a.C;
    n.y = a.h; n.y_ld = a.h_ld; n.y_part = a.h_part; n.y_rows = a.h_rows; n.ny = a.n;
  } else {
    n.x = a.h; n.x_ld = a.h_ld; n.x_part = a.h_part; n.x_rows = a.h_rows; n.nx = a.n;
    n.y = a.w; n.y_ld = a.w_ld; n.y_part = a.w_part; n.y_rows = a.C; n.ny = a.C;
  }
  n.K = a.K; n.f1 = a.f1; n.f2 = a.f2;
  return n;
}

template <typename T>
int narrow_forward(LxArgs& a, const pg_linear_xent_desc_t* d, const LxPlan& p, char* s, hipStream_t st) {
  a.part = (float2*)s;
  a.zlab = (float*)(s + p.part_bytes);
  char* h = s + p.part_bytes + up(4 * a.n, 256);
  const SideArgs side = lx_side_arrays(a, p, h + p.h_bytes + p.w_bytes, false);
  int rc = lx_operands<T>(a, d, p, h, h + p.h_bytes, false, side, st);
  if (rc != PG_OK) return rc;
  NxArgs n = narrow_args(a, false);
  n.side0 = side.bias2; n.xlab = side.lab; n.part = a.part; n.zlab = a.zlab;
  n.splits = p.nx_stats; n.range = p.rs_stats;
  rc = launch_narrow<T, NX_STATS>(n, p, st);
  if (rc != PG_OK) return rc;
  a.tiles = p.nx_stats;
  return lx_rows<T>(a, st);
}

template <typename T>
int narrow_backward(LxArgs& a, const pg_linear_xent_desc_t* d, const LxPlan& p, char* s, hipStream_t st) {
  float* acc_dh = (float*)s;
  s += p.acc_dh;
  float* acc_dw = (float*)s;
  s += p.acc_dw;
  const SideArgs side = lx_side_arrays(a, p, s + p.h_bytes + p.w_bytes, true);
  int rc = lx_operands<T>(a, d, p, s, s + p.h_bytes, true, side, st);
  if (rc != PG_OK) return rc;
  SumArgs dh{}, dw{}, db{};
  if (a.dh) {
    NxArgs n = narrow_args(a, false);
    n.side0 = side.bias2; n.xa = side.top2; n.xi = side.inv2; n.xb = side.rowf2; n.xlab = side.lab;
    n.splits = p.nx_dh; n.range = p.rs_dh; n.acc = acc_dh; n.out = a.dh;
    rc = launch_narrow<T, NX_DH>(n, p, st);
    if (rc != PG_OK) return rc;
    if (n.splits > 1) dh = SumArgs{acc_dh, a.dh, a.n * a.K, n.splits};
  }
  if (a.dw || a.db) {
    NxArgs n = narrow_args(a, true);
    n.side0 = side.top2; n.side1 = (const float*)side.lab; n.side2 = side.rowf2; n.side3 = side.inv2; n.xa = side.bias2;
    n.scaled = a.rowf != nullptr;
    n.splits = p.nx_dw; n.range = p.rs_dw; n.acc = acc_dw; n.accb = acc_dw + (int64_t)p.nx_dw * a.C * a.K; n.out = a.dw; n.outb = a.db;
    rc = launch_narrow<T, NX_DW>(n, p, st);
    if (rc != PG_OK) return rc;
    if (n.splits > 1) {
      if (a.dw) dw = SumArgs{acc_dw, a.dw, a.C * a.K, n.splits};
      if (a.db) db = SumArgs{n.accb, a.db, a.C, n.splits};
    }
  }
  return lx_sums<T>(dh, dw, db, a, st);
}

template <typename T, bool PIECE>
void lx_launch_logits(const LxArgs& a, const LxPlan& p, dim3 grid, hipStream_t st) {
  if (p.logits == BIG) {
    hipLaunchKernelGGL((k_lx_logits<T, BigTile<T>, PIECE>), grid, dim3(BigTile<T>::THREADS), 0, st, a);
    return;
  }
  if constexpr (Mul<T>::NP == 1)
    if (p.logits == TALL) {
      hipLaunchKernelGGL((k_lx_logits<T, TallTile<T>, PIECE>), grid, dim3(TallTile<T>::THREADS), 0, st, a);
      return;
    }
  hipLaunchKernelGGL((k_lx_logits<T, MidTile<T>, PIECE>), grid, dim3(MidTile<T>::THREADS), 0, st, a);
}

template <typename T>
int lx_forward(LxArgs& a, const pg_linear_xent_desc_t* d, const LxPlan& p, char* s, hipStream_t st) {
  if (p.narrow) return narrow_forward<T>(a, d, p, s, st);
  a.part = (float2*)s;
  a.zlab = (float*)(s + p.part_bytes);
  char* h = s + p.part_bytes + up(4 * a.n, 256);
  const SideArgs side = lx_side_arrays(a, p, h + p.h_bytes + p.w_bytes, false);
  const int rc = lx_operands<T>(a, d, p, h, h + p.h_bytes, false, side, st);
  if (rc != PG_OK) return rc;
  a.bias2 = side.bias2; a.lab2 = side.lab;
  a.tiles = p.tiles;
  a.c_lo = 0;
  a.c_hi = a.C;
  const dim3 grid((unsigned)(p.tiles * p.row_tiles));
  lx_launch_logits<T, false>(a, p, grid, st);
  PG_LAUNCH_CHECK();
  return lx_rows<T>(a, st);
}

template <typename T, typename S>
int lx_launch_dh(const LxArgs& a, hipStream_t st) {
  const int64_t tiles = ceil_div<int64_t>(a.n, S::BM) * ceil_div<int64_t>(a.K, S::BN) * a.splits;
  hipLaunchKernelGGL((k_lx_dh<T, S>), dim3((unsigned)tiles), dim3(S::THREADS), 0, st, a);
  PG_LAUNCH_CHECK();
  return PG_OK;
}
template <typename T, typename S>
int lx_launch_dw(const LxArgs& a, hipStream_t st) {
  const int64_t tiles = ceil_div<int64_t>(a.c_hi - a.c_lo, S::BM) * ceil_div<int64_t>(a.K, S::BN) * a.splits;
  hipLaunchKernelGGL((k_lx_dw<T, S>), dim3((unsigned)tiles), dim3(S::THREADS), 0, st, a);
  PG_LAUNCH_CHECK();
  return PG_OK;
}

// one piece's G, and its share of the gradients
template <typename T>
int lx_piece(const LxArgs& a, const LxPlan& p, hipStream_t st) {
  const dim3 grid((unsigned)(ceil_div<int64_t>(a.c_hi - a.c_lo, p.logits == MID ? 128 : 256) * p.row_tiles));
  lx_launch_logits<T, true>(a, p, grid, st);
  PG_LAUNCH_CHECK();
  return PG_OK;
}
template <typename T>
int lx_piece_dh(LxArgs& a, const LxPlan& p, float* acc, hipStream_t st) {
  a.acc = acc;
  a.splits = p.dh_splits;
  a.range = p.dh_range;
  a.first = a.c_lo == 0;
  a.direct = p.dh_splits == 1 && p.pieces == 1;
  return p.dh == BIG ? lx_launch_dh<T, BigTile<T>>(a, st) : p.dh == TALL ? lx_launch_dh<T, TallTile<T>>(a, st) : lx_launch_dh<T, MidTile<T>>(a, st);
}
template <typename T>
int lx_piece_dw(LxArgs& a, const LxPlan& p, float* acc, hipStream_t st) {
  a.acc = acc;
  a.splits = p.dw_splits;
  a.range = p.dw_range;
  const int rc = p.dw == BIG ? lx_launch_dw<T, BigTile<T>>(a, st) : p.dw == TALL ? lx_launch_dw<T, TallTile<T>>(a, st) : lx_launch_dw<T, MidTile<T>>(a, st);
  if (rc != PG_OK || a.splits == 1 || p.pieces == 1) return rc;
  return lx_sums<T>(SumArgs{acc, (T*)a.dw + a.c_lo * a.K, (a.c_hi - a.c_lo) * a.K, a.splits}, SumArgs{}, SumArgs{}, a, st);
}

template <typename T>
int lx_backward(LxArgs& a, const pg_linear_xent_desc_t* d, const LxPlan& p, char* s, hipStream_t st) {
  if (p.narrow) return narrow_backward<T>(a, d, p, s, st);
  a.g = s;
  s += p.g_bytes;
  float* acc_dh = (float*)s;
  s += p.acc_dh;
  float* acc_dw = (float*)s;
  s += p.acc_dw;
  a.dbp = (float*)s;
  s += p.dbp_bytes;
  const SideArgs side = lx_side_arrays(a, p, s + p.h_bytes + p.w_bytes, true);
  int rc = lx_operands<T>(a, d, p, s, s + p.h_bytes, true, side, st);
  if (rc != PG_OK) return rc;
  a.bias2 = side.bias2; a.lab2 = side.lab; a.top2 = side.top2; a.inv2 = side.inv2; a.rowf2 = side.rowf2;
  a.ldg = p.ldg;
  a.g_rows = p.g_rows;
  // Rows with factors of their own in fp16: below 2^-14 of the largest one, G times its factor begins to leave the type's range, and
  // dh, which has the row to itself, would lose those bits. Its G carries no factors, its rows get them behind the product. dW and
  // db sum over the rows, largest ones beside them: their G carries the factors, and is made a second time where both are wanted
  const bool scaled = a.rowf != nullptr, head = a.dw || a.db;
  a.late = scaled && Mul<T>::G != 1.f;
  for (a.c_lo = 0; a.c_lo < a.C; a.c_lo = a.c_hi) {
    a.c_hi = a.c_lo + p.piece < a.C ? a.c_lo + p.piece : a.C;
    if (a.dh) {
      a.scaled = scaled && !a.late;
      rc = lx_piece<T>(a, p, st);
      if (rc == PG_OK) rc = lx_piece_dh<T>(a, p, acc_dh, st);
      if (rc != PG_OK) return rc;
    }
    if (head && (!a.dh || a.late)) {
      a.scaled = scaled;
      rc = lx_piece<T>(a, p, st);
      if (rc != PG_OK) return rc;
    }
    if (a.dw) {
      rc = lx_piece_dw<T>(a, p, acc_dw, st);
      if (rc != PG_OK) return rc;
    }
  }
  const bool direct = p.dh_splits == 1 && p.pieces == 1;
  return lx_sums<T>(SumArgs{acc_dh, direct ? nullptr : a.dh, a.n * a.K, p.dh_splits}, SumArgs{a.dbp, a.db, a.C, p.row_tiles},
                    SumArgs{acc_dw, p.dw_splits > 1 && p.pieces == 1 ? a.dw : nullptr, a.C * a.K, p.dw_splits}, a, st);
}

// a tile's offsets have 32 bits (that the launches fit their grids: LxPlan::fits)
inline int lx_check(int64_t n, int64_t K, int64_t C, int32_t dtype) {
  if (n < 0 || K <= 0 || C <= 0 || dtype < PG_DTYPE_F32 || dtype > PG_DTYPE_F16) return PG_ERR_INVALID;
  if (n > (int64_t(1) << 31) || K > (int64_t(1) << 20) || C > (int64_t(1) << 31)) return PG_ERR_UNSUPPORTED;
  if (ceil_div<int64_t>(n, 128) * ceil_div<int64_t>(C, 128) > 0x7fffffffll / 2) return PG_ERR_UNSUPPORTED;
  return PG_OK;
}

int lx_args(const pg_linear_xent_desc_t* d, LxArgs* a) {
  if (!d) return PG_ERR_INVALID;
  const int rc = lx_check(d->n, d->K, d->C, d->dtype);
  if (rc != PG_OK) return rc;
  if ((d->h_stride < d->K && d->h_stride != 0) || d->w_stride < d->K) return PG_ERR_INVALID;
  if (!d->W || !d->meta || (d->n > 0 && (!d->h || !d->labels || !d->top || !d->sum || !d->scratch))) return PG_ERR_INVALID;
  if ((uintptr_t)d->scratch % 16) return PG_ERR_INVALID;            // packed rows and G move 16 bytes a lane
  *a = LxArgs{};
  a->bias = d->bias; a->labels = d->labels;
  a->n = d->n; a->K = d->K; a->Kp = up(d->K, kPad); a->C = d->C; a->ignore = d->ignore_index;
  a->top = d->top; a->sum = d->sum; a->meta = d->meta;
  return PG_OK;
}

}  // namespace pg

using namespace pg;

extern "C" {

int64_t pg_linear_xent_scratch(int64_t n, int64_t K, int64_t C, int32_t dtype, int32_t backward) {
  if (lx_check(n, K, C, dtype) != PG_OK) return -1;
  if (n == 0) return 0;
  const LxPlan p = lx_plan(n, K, C, dtype, backward != 0);
  if (!p.fits) return -1;
  const int64_t ops = p.h_bytes + p.w_bytes + p.side_bytes;
  return backward ? p.g_bytes + p.acc_dh + p.acc_dw + p.dbp_bytes + ops + up(4 * n, 256) + 256 : p.part_bytes + 2 * up(4 * n, 256) + ops;
}

int pg_linear_xent_fwd(const pg_linear_xent_desc_t* d, pg_stream_t stream) {
  LxArgs a;
  int rc = lx_args(d, &a);
  if (rc != PG_OK) return rc;
  hipStream_t st = as_stream(stream);
  if (d->reduction < PG_XENT_MEAN || d->reduction > PG_XENT_NONE) return PG_ERR_INVALID;
  const bool rows = d->reduction == PG_XENT_NONE;
  if (rows ? a.n > 0 && !d->row_loss : !d->loss) return PG_ERR_INVALID;
  if (a.n > 0) {
    const LxPlan p = lx_plan(a.n, a.K, a.C, d->dtype, false);
    if (!p.fits) return PG_ERR_UNSUPPORTED;
    char* s = (char*)d->scratch;
    a.row_loss = rows ? d->row_loss : (float*)s;
    s += up(4 * a.n, 256);
    rc = d->dtype == PG_DTYPE_F32 ? lx_forward<float>(a, d, p, s, st) : d->dtype == PG_DTYPE_BF16 ? lx_forward<bf16_t>(a, d, p, s, st)
                                                                                                  : lx_forward<f16_t>(a, d, p, s, st);
    if (rc != PG_OK) return rc;
  }
  if (!rows) {
    hipLaunchKernelGGL(k_lx_mean, dim3(1), dim3(1024), 0, st, a.row_loss, a.sum, a.n, d->reduction == PG_XENT_MEAN ? 1 : 0, d->loss, a.meta);
    PG_LAUNCH_CHECK();
  }
  return PG_OK;
}

int pg_linear_xent_bwd(const pg_linear_xent_desc_t* d, pg_stream_t stream) {
  LxArgs a;
  const int rc = lx_args(d, &a);
  if (rc != PG_OK) return rc;
  if (!d->grad || d->reduction < PG_XENT_MEAN || d->reduction > PG_XENT_NONE) return PG_ERR_INVALID;
  if (a.n == 0) return PG_ERR_INVALID;            // no row, no gradient to compute: the caller's zeros
  hipStream_t st = as_stream(stream);
  const LxPlan p = lx_plan(a.n, a.K, a.C, d->dtype, true);
  if (!p.fits) return PG_ERR_UNSUPPORTED;
  char* s = (char*)d->scratch;
  a.dh = d->dh; a.dw = d->dW; a.db = d->db;
  if (d->reduction == PG_XENT_NONE) {
    float* rowf = (float*)s;
    float* top = (float*)(s + up(4 * a.n, 256));
    hipLaunchKernelGGL(k_lx_row_factors, dim3(1), dim3(1024), 0, st, d->grad, d->grad_stride, a.sum, a.n, rowf, top);
    PG_LAUNCH_CHECK();
    a.rowf = rowf;
    a.f1 = top;
  } else {
    a.f1 = d->grad;
    a.f2 = d->reduction == PG_XENT_MEAN ? a.meta : nullptr;
  }
  s += up(4 * a.n, 256) + 256;
  return d->dtype == PG_DTYPE_F32 ? lx_backward<float>(a, d, p, s, st) : d->dtype == PG_DTYPE_BF16 ? lx_backward<bf16_t>(a, d, p, s, st)
                                                                                                   : lx_backward<f16_t>(a, d, p, s, st);
}

}  // extern "C"
