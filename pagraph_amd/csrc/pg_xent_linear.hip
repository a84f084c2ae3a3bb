// Softmax cross entropy of a class head z = h W^T + b of any width, without its logits:
//   lse_r = log sum_c exp z_rc,  loss_r = lse_r - z_r,label,
//   G = (exp(z - lse) - onehot(label)) * (row factor),  dh = G W,  dW = G^T h,  db = sum_r G.
// The logits [n, C] exist only as tiles in registers. Forward: every workgroup leaves (maximum, sum of exponentials) of its tile's
// rows, a second launch joins them. Backward: the logits are computed again in pieces of the vocabulary; a piece's G leaves in
// the operands' 16 bits (fp32 for fp32 operands) and feeds the two gradient products before the next piece overwrites it.
// 8 n K C operations instead of the 6 n K C with kept logits, against 8 bytes of fp32 logit traffic per element of [n, C].
//
// Products run on the matrix cores with fp32 accumulation. fp32 operands: each value is split into three bf16 parts
// (x = x0 + x1 + x2 to 24 bits) and six of the nine partial products are summed, what is left out is below 2^-24 of the product —
// 2.5 PF / 6 where the fp32 matrix instructions reach 0.157 PF.
// G in 16 bits: |G| <= 1 and each element is off by half a step (bf16 2^-9, fp16 2^-12 relative), independently per element, as
// are the outputs, which leave in the same type. fp16 G is held times 2^14 so that a probability of 2^-28 is still a normal number.
#include "pg_elem.h"

namespace pg {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.44269504088896340736f;

// how an operand type is multiplied: parts per value, the parts' type, depth of a tile
template <typename T> struct Mul;
template <> struct Mul<float>  { typedef bf16_t E; typedef bf16x8 V; static constexpr int NP = 3, BK = 32, MB = 2; };
template <> struct Mul<bf16_t> { typedef bf16_t E; typedef bf16x8 V; static constexpr int NP = 1, BK = 64, MB = 4; };
template <> struct Mul<f16_t>  { typedef f16_t E;  typedef f16x8 V;  static constexpr int NP = 1, BK = 64, MB = 4; };

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// LDS tile [rows][BK] of one part: 16-byte chunks, chunk index XORed with bits of the row so that the 8 lanes of a read phase
// (consecutive rows) and of a transposing write (rows 4 resp. 2 apart) meet different banks
template <int BK>
__device__ __forceinline__ int lds_at(int row, int chunk) {
  return BK == 64 ? row * 64 + ((chunk ^ ((row ^ (row >> 2)) & 7)) << 3) : row * 32 + ((chunk ^ ((row >> 1) & 3)) << 3);
}

template <typename T>
__device__ __forceinline__ void split_write(typename Mul<T>::E* tile, int part_stride, int at, const T (&v)[8]) {
  typename Mul<T>::V o;
  if constexpr (Mul<T>::NP == 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = v[i];
    *reinterpret_cast<typename Mul<T>::V*>(tile + at) = o;
  } else {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = v[i];
#pragma unroll
    for (int p = 0; p < 3; ++p) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        o[i] = (bf16_t)x[i];
        x[i] -= (float)o[i];                       // exact
      }
      *reinterpret_cast<bf16x8*>(tile + p * part_stride + at) = o;
    }
  }
}

// Operand whose reduction index is contiguous: p[row * ld + k]. Rows >= nrows and k >= K read as 0.
template <typename T, int ROWS>
struct LoadK {
  static constexpr int BK = Mul<T>::BK, CH = BK / 8, U = ROWS * CH / 256;
  const T* p;
  int64_t ld, row0, nrows, K;
  T v[U][8];
  __device__ __forceinline__ void load(int64_t k0, int tid) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int id = tid + u * 256, row = id / CH, ch = id % CH;
      const int64_t k = k0 + ch * 8, r = row0 + row;
      const T* s = p + r * ld + k;
      if (r < nrows && k + 8 <= K) {
        __builtin_memcpy(v[u], s, sizeof(v[u]));
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] = r < nrows && k + i < K ? s[i] : (T)0.f;
      }
    }
  }
  __device__ __forceinline__ void store(typename Mul<T>::E* tile, int tid) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int id = tid + u * 256;
      split_write<T>(tile, ROWS * BK, lds_at<BK>(id / CH, id % CH), v[u]);
    }
  }
};

// Operand whose row index is contiguous: p[k * ld + row], transposed on its way into LDS: a thread holds MB rows x 8 k.
// flag (may be NULL): k with flag[k] == 0 read as 0 without being read (ignored rows may hold anything)
template <typename T, int ROWS>
struct LoadM {
  static constexpr int BK = Mul<T>::BK, MB = Mul<T>::MB, UR = ROWS / MB, UNITS = UR * (BK / 8);
  const T* p;
  int64_t ld, row0, nrows, K;
  const float* flag;
  T v[8][MB];
  __device__ __forceinline__ void load(int64_t k0, int tid) {
    if (UNITS < 256 && tid >= UNITS) return;
    const int64_t r = row0 + (tid % UR) * MB;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t k = k0 + (tid / UR) * 8 + j;
      const bool ok = k < K && (!flag || flag[k] != 0.f);
      const T* s = p + k * ld + r;
      if (ok && r + MB <= nrows) {
        __builtin_memcpy(v[j], s, sizeof(v[j]));
      } else {
#pragma unroll
        for (int i = 0; i < MB; ++i) v[j][i] = ok && r + i < nrows ? s[i] : (T)0.f;
      }
    }
  }
  __device__ __forceinline__ void store(typename Mul<T>::E* tile, int tid) {
    if (UNITS < 256 && tid >= UNITS) return;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
      T c[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = v[j][i];
      split_write<T>(tile, ROWS * BK, lds_at<BK>((tid % UR) * MB + i, tid / UR), c);
    }
  }
};

struct NoSide { __device__ __forceinline__ void operator()() const {} };

// acc[i][j] += A(64-row slab wm of BM) x B(slab wn of BN): 4 waves, 2 x 2; reduction over [k_lo, k_hi). One register-staged tile
// ahead, two LDS buffers, one barrier per step. side() runs once per loaded A tile (its values are in la.v).
template <typename T, int BM, int BN, typename LA, typename LB, typename Side>
__device__ __forceinline__ void product(LA& la, LB& lb, int64_t k_lo, int64_t k_hi, typename Mul<T>::E* lds,
                                        f32x16 (&acc)[BM / 64][BN / 64], Side side) {
  typedef typename Mul<T>::E E;
  typedef typename Mul<T>::V V;
  constexpr int BK = Mul<T>::BK, NP = Mul<T>::NP, STAGE = NP * (BM + BN) * BK;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
  int buf = 0;
  la.load(k_lo, tid);
  lb.load(k_lo, tid);
  for (int64_t k0 = k_lo; k0 < k_hi; k0 += BK) {
    E* ta = lds + buf * STAGE;
    E* tb = ta + NP * BM * BK;
    side();
    la.store(ta, tid);
    lb.store(tb, tid);
    if (k0 + BK < k_hi) {
      la.load(k0 + BK, tid);
      lb.load(k0 + BK, tid);
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < BK / 16; ++kk) {
      const int chunk = kk * 2 + (lane >> 5);
      V a[NP][BM / 64], b[NP][BN / 64];
#pragma unroll
      for (int p = 0; p < NP; ++p) {
#pragma unroll
        for (int i = 0; i < BM / 64; ++i)
          a[p][i] = *reinterpret_cast<const V*>(ta + p * BM * BK + lds_at<BK>(wm * (BM / 2) + i * 32 + (lane & 31), chunk));
#pragma unroll
        for (int j = 0; j < BN / 64; ++j)
          b[p][j] = *reinterpret_cast<const V*>(tb + p * BN * BK + lds_at<BK>(wn * (BN / 2) + j * 32 + (lane & 31), chunk));
      }
#pragma unroll
      for (int i = 0; i < BM / 64; ++i)
#pragma unroll
        for (int j = 0; j < BN / 64; ++j) {
          if constexpr (NP == 3) {                 // smallest first
            acc[i][j] = mma(a[2][i], b[0][j], acc[i][j]);
            acc[i][j] = mma(a[1][i], b[1][j], acc[i][j]);
            acc[i][j] = mma(a[0][i], b[2][j], acc[i][j]);
            acc[i][j] = mma(a[1][i], b[0][j], acc[i][j]);
            acc[i][j] = mma(a[0][i], b[1][j], acc[i][j]);
          }
          acc[i][j] = mma(a[0][i], b[0][j], acc[i][j]);
        }
    }
    buf ^= 1;                                      // the other buffer's readers have passed the barrier above
  }
}

struct LxArgs {
  const void *h, *w, *bias;
  const int64_t* labels;
  int64_t n, K, C, hs, ws, ignore;
  float2* part;            // [n][tiles] maximum, sum of exponentials
  float *zlab, *lse, *row_loss, *flag, *meta;
  int64_t tiles;
  // backward
  const float *rowf;       // row factors: flag, or the normalised incoming gradients
  const float *f1, *f2;    // the outputs' factor = *f1 * *f2 (NULL = 1)
  void* g;                 // a piece of G: [n][ldg]
  int64_t ldg, c_lo, c_hi; // the piece's classes
  float* acc;              // fp32 partial products [split][rows][K]
  float* accb;
  void *dh, *dw, *db;
  int64_t k_split;         // reduction range of one split
  int32_t splits, first;
};

template <typename T> struct GScale { static constexpr float v = 1.f; };
template <> struct GScale<f16_t> { static constexpr float v = 16384.f; };

__device__ __forceinline__ bool label_ok(int64_t lab, const LxArgs& a) { return lab != a.ignore && lab >= 0 && lab < a.C; }
__device__ __forceinline__ float out_factor(const LxArgs& a) { return (a.f1 ? *a.f1 : 1.f) * (a.f2 ? *a.f2 : 1.f); }

// Workgroups go round the 8 XCDs in turn: give each XCD a contiguous run of tiles, so that its own L2 sees a tile's neighbours
__device__ __forceinline__ int64_t xcd_run(int64_t b, int64_t total) {
  const int64_t per = total / 8, rest = total % 8, x = b % 8, i = b / 8;
  return x * per + (x < rest ? x : rest) + i;
}

// One 128-class x BN-row tile of logits; a lane holds one row's classes in registers: row = wn * BN/2 + 32 j + lane % 32,
// class = wm * 64 + 32 i + 8 (e / 4) + 4 (lane / 32) + e % 4. PIECE: writes G, else the tile's row statistics.
template <typename T, int BN, bool PIECE>
__global__ __launch_bounds__(256) void k_lx_logits(LxArgs a) {
  typedef typename Mul<T>::E E;
  constexpr int BM = 128, BK = Mul<T>::BK, NP = Mul<T>::NP;
  __shared__ __align__(16) E lds[2 * NP * (BM + BN) * BK];
  __shared__ float2 red[2][BN];
  const int64_t row_tiles = ceil_div<int64_t>(a.n, BN), c_tiles = ceil_div<int64_t>(a.c_hi - a.c_lo, BM);
  const int64_t t = xcd_run(blockIdx.x, row_tiles * c_tiles);
  const int64_t ct = t / row_tiles, r0 = t % row_tiles * BN, c0 = a.c_lo + ct * BM;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
  f32x16 acc[2][BN / 64] = {};
  LoadK<T, BM> la{(const T*)a.w, a.ws, c0, a.c_hi, a.K};
  LoadK<T, BN> lb{(const T*)a.h, a.hs, r0, a.n, a.K};
  product<T, BM, BN>(la, lb, 0, a.K, lds, acc, NoSide{});
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int64_t c = c0 + wm * 64 + i * 32 + 8 * (e / 4) + 4 * (lane >> 5) + e % 4;
      float b = c < a.c_hi ? 0.f : -INFINITY;
      if (a.bias && c < a.c_hi) b = (float)((const T*)a.bias)[c];
#pragma unroll
      for (int j = 0; j < BN / 64; ++j) acc[i][j][e] += b;
    }
#pragma unroll
  for (int j = 0; j < BN / 64; ++j) {
    const int rl = wn * (BN / 2) + j * 32 + (lane & 31);
    const int64_t r = r0 + rl;
    const int64_t lab = r < a.n ? a.labels[r] : -1;
    if constexpr (!PIECE) {
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          m = fmaxf(m, acc[i][j][e]);
          const int64_t c = c0 + wm * 64 + i * 32 + 8 * (e / 4) + 4 * (lane >> 5) + e % 4;
          if (c == lab && r < a.n) a.zlab[r] = acc[i][j][e];
        }
      m = fmaxf(m, __shfl_xor(m, 32, kWave));
      const float base = m == -INFINITY ? 0.f : m;         // nothing but -inf so far: every exponential is 0
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) s += __builtin_amdgcn_exp2f((acc[i][j][e] - base) * kLog2e);
      s += __shfl_xor(s, 32, kWave);
      if (lane < 32) red[wm][rl] = make_float2(m, s);
    } else if (r < a.n) {
      const float lse = a.lse[r], f = a.rowf[r] * GScale<T>::v;
      T* g = (T*)a.g + r * a.ldg + (c0 - a.c_lo) + wm * 64 + 4 * (lane >> 5);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int64_t c = c0 + wm * 64 + i * 32 + 8 * q + 4 * (lane >> 5) + e;
            const float pr = __builtin_amdgcn_exp2f((acc[i][j][q * 4 + e] - lse) * kLog2e) - (c == lab ? 1.f : 0.f);
            o[e] = f == 0.f || c >= a.c_hi ? 0.f : pr * f;
          }
          store4(g + i * 32 + 8 * q, o);
        }
    }
  }
  if constexpr (!PIECE) {
    __syncthreads();
    for (int rl = tid; rl < BN; rl += 256)
      if (r0 + rl < a.n) {
        const float2 x = red[0][rl], y = red[1][rl];
        const float m = fmaxf(x.x, y.x), base = m == -INFINITY ? 0.f : m;
        a.part[(r0 + rl) * a.tiles + ct] =
            make_float2(m, x.y * __builtin_amdgcn_exp2f((x.x - base) * kLog2e) + y.y * __builtin_amdgcn_exp2f((y.x - base) * kLog2e));
      }
  }
}

// a wave per row: joins the tiles' statistics
__global__ __launch_bounds__(256) void k_lx_rows(LxArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
  if (r >= a.n) return;
  float m = -INFINITY, s = 0.f;
  for (int64_t t = lane; t < a.tiles; t += 64) {
    const float2 x = a.part[r * a.tiles + t];
    const float mm = fmaxf(m, x.x), base = mm == -INFINITY ? 0.f : mm;
    s = s * __builtin_amdgcn_exp2f((m - base) * kLog2e) + x.y * __builtin_amdgcn_exp2f((x.x - base) * kLog2e);
    m = mm;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float om = __shfl_xor(m, o, kWave), os = __shfl_xor(s, o, kWave);
    const float mm = fmaxf(m, om), base = mm == -INFINITY ? 0.f : mm;
    s = s * __builtin_amdgcn_exp2f((m - base) * kLog2e) + os * __builtin_amdgcn_exp2f((om - base) * kLog2e);
    m = mm;
  }
  if (lane == 0) {
    const float lse = m + logf(s);
    const bool ok = label_ok(a.labels[r], a);
    a.lse[r] = lse;
    a.flag[r] = ok ? 1.f : 0.f;
    a.row_loss[r] = ok ? lse - a.zlab[r] : 0.f;
  }
}

// one block, fixed order: meta = {mean, 1 / counted rows, sum}
__global__ __launch_bounds__(1024) void k_lx_mean(const float* __restrict__ row_loss, const float* __restrict__ flag, int64_t n,
                                                  float* __restrict__ meta) {
  __shared__ float ss[1024];
  __shared__ int sc[1024];
  float s = 0.f;
  int c = 0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) {
    s += row_loss[i];
    c += flag[i] != 0.f;
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
    meta[0] = sc[0] > 0 ? ss[0] / (float)sc[0] : NAN;       // as ops.cross_entropy: a mean over no rows
    meta[1] = sc[0] > 0 ? 1.f / (float)sc[0] : 0.f;
    meta[2] = ss[0];
  }
}

// incoming gradients of single rows: row factors g / max|g| (G then uses its type's range whatever the caller's scale), the
// maximum becomes the outputs' factor
__global__ __launch_bounds__(1024) void k_lx_row_factors(const float* __restrict__ g, int64_t gs, const float* __restrict__ flag,
                                                         int64_t n, float* __restrict__ rowf, float* __restrict__ top) {
  __shared__ float ss[1024];
  float m = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += 1024)
    if (flag[i] != 0.f) m = fmaxf(m, fabsf(g[i * gs]));
  ss[threadIdx.x] = m;
  __syncthreads();
  for (int o = 512; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) ss[threadIdx.x] = fmaxf(ss[threadIdx.x], ss[threadIdx.x + o]);
    __syncthreads();
  }
  m = ss[0];
  for (int64_t i = threadIdx.x; i < n; i += 1024) rowf[i] = flag[i] != 0.f && m > 0.f ? g[i * gs] / m : 0.f;
  if (threadIdx.x == 0) *top = m;
}

// dh partials: acc[split][r][k] (+)= sum over the split's classes of G[r][c] W[c][k]
template <typename T, int BN>
__global__ __launch_bounds__(256) void k_lx_dh(LxArgs a) {
  typedef typename Mul<T>::E E;
  constexpr int BM = 128, BK = Mul<T>::BK, NP = Mul<T>::NP;
  __shared__ __align__(16) E lds[2 * NP * (BM + BN) * BK];
  const int64_t row_tiles = ceil_div<int64_t>(a.n, BM), k_tiles = ceil_div<int64_t>(a.K, BN);
  const int64_t t = xcd_run(blockIdx.x, row_tiles * k_tiles * a.splits);
  const int64_t kt = t % k_tiles, rt = t / k_tiles % row_tiles, sp = t / k_tiles / row_tiles;
  const int64_t r0 = rt * BM, n0 = kt * BN, len = a.c_hi - a.c_lo;
  const int64_t lo = sp * a.k_split, hi = lo + a.k_split < len ? lo + a.k_split : len;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
  f32x16 acc[2][BN / 64] = {};
  if (lo < hi) {
    LoadK<T, BM> la{(const T*)a.g, a.ldg, r0, a.n, hi};
    LoadM<T, BN> lb{(const T*)a.w + a.c_lo * a.ws, a.ws, n0, a.K, hi, nullptr};
    product<T, BM, BN>(la, lb, lo, hi, lds, acc, NoSide{});
  }
  float* out = a.acc + sp * a.n * a.K;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < BN / 64; ++j) {
      const int64_t k = n0 + wn * (BN / 2) + j * 32 + (lane & 31);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int64_t r = r0 + wm * 64 + i * 32 + 8 * (e / 4) + 4 * (lane >> 5) + e % 4;
        if (r < a.n && k < a.K) {
          float* p = out + r * a.K + k;
          *p = (a.first ? 0.f : *p) + acc[i][j][e];
        }
      }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void k_lx_dh_out(LxArgs a) {
  const float f = out_factor(a) / GScale<T>::v;
  const int64_t total = a.n * a.K;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
    float s = 0.f;
    for (int i = 0; i < a.splits; ++i) s += a.acc[i * total + t];
    ((T*)a.dh)[t] = a.rowf[t / a.K] == 0.f ? (T)0.f : (T)(s * f);
  }
}

// dW rows of a piece: sum over the split's rows of G[r][c] h[r][k]; db rides along in the workgroups of the first column tile
template <typename T, int BN>
__global__ __launch_bounds__(256) void k_lx_dw(LxArgs a) {
  typedef typename Mul<T>::E E;
  constexpr int BM = 128, BK = Mul<T>::BK, NP = Mul<T>::NP, MB = Mul<T>::MB;
  __shared__ __align__(16) E lds[2 * NP * (BM + BN) * BK];
  __shared__ float sdb[BK / 8][BM];
  const int64_t len = a.c_hi - a.c_lo, c_tiles = ceil_div<int64_t>(len, BM), k_tiles = ceil_div<int64_t>(a.K, BN);
  const int64_t t = xcd_run(blockIdx.x, c_tiles * k_tiles * a.splits);
  const int64_t kt = t % k_tiles, ct = t / k_tiles % c_tiles, sp = t / k_tiles / c_tiles;
  const int64_t c0 = ct * BM, n0 = kt * BN;
  const int64_t lo = sp * a.k_split, hi = lo + a.k_split < a.n ? lo + a.k_split : a.n;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
  f32x16 acc[2][BN / 64] = {};
  float bsum[MB] = {};
  LoadM<T, BM> la{(const T*)a.g, a.ldg, c0, a.ldg, hi, nullptr};
  LoadM<T, BN> lb{(const T*)a.h, a.hs, n0, a.K, hi, a.rowf};
  if (lo < hi)
    product<T, BM, BN>(la, lb, lo, hi, lds, acc, [&] {
      if (kt == 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int i = 0; i < MB; ++i) bsum[i] += (float)la.v[j][i];
      }
    });
  const float f = out_factor(a) / GScale<T>::v;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < BN / 64; ++j) {
      const int64_t k = n0 + wn * (BN / 2) + j * 32 + (lane & 31);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int64_t c = c0 + wm * 64 + i * 32 + 8 * (e / 4) + 4 * (lane >> 5) + e % 4;
        if (c < len && k < a.K) {
          if (a.splits > 1)
            a.acc[(sp * len + c) * a.K + k] = acc[i][j][e];
          else if (a.dw)
            ((T*)a.dw)[(a.c_lo + c) * a.K + k] = (T)(acc[i][j][e] * f);
        }
      }
    }
  if (kt == 0 && (a.db || a.accb)) {
    constexpr int UR = BM / MB;
#pragma unroll
    for (int i = 0; i < MB; ++i) sdb[tid / UR][tid % UR * MB + i] = bsum[i];
    __syncthreads();
    if (tid < BM && c0 + tid < len) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < BK / 8; ++i) s += sdb[i][tid];
      if (a.splits == 1)
        ((T*)a.db)[a.c_lo + c0 + tid] = (T)(s * f);
      else
        a.accb[sp * len + c0 + tid] = s;
    }
  }
}

// the splits of one piece's dW (rows x K) and db added in order
template <typename T>
__global__ __launch_bounds__(256) void k_lx_dw_out(LxArgs a) {
  const float f = out_factor(a) / GScale<T>::v;
  const int64_t len = a.c_hi - a.c_lo, total = len * a.K;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total + len; t += (int64_t)gridDim.x * 256) {
    float s = 0.f;
    if (t < total) {
      if (!a.dw) continue;
      for (int i = 0; i < a.splits; ++i) s += a.acc[i * total + t];
      ((T*)a.dw)[a.c_lo * a.K + t] = (T)(s * f);
    } else if (a.db) {
      for (int i = 0; i < a.splits; ++i) s += a.accb[i * len + t - total];
      ((T*)a.db)[a.c_lo + t - total] = (T)(s * f);
    }
  }
}

inline int64_t up(int64_t v, int64_t m) { return ceil_div(v, m) * m; }

// sizes of one call: everything follows from (n, K, C, type) alone, so that the scratch the caller allocates fits the launches
struct LxPlan {
  int64_t tiles, piece, ldg, part_bytes, g_bytes, acc_bytes;
  int32_t dh_splits, dw_splits;
  int64_t dh_range, dw_range;
  int bn_rows, bn_cols;
};

inline LxPlan lx_plan(int64_t n, int64_t K, int64_t C, int32_t dtype) {
  LxPlan p{};
  const int64_t e = dtype == PG_DTYPE_F32 ? 4 : 2, bk = dtype == PG_DTYPE_F32 ? 32 : 64;
  p.tiles = ceil_div<int64_t>(C, 128);
  p.bn_rows = n <= 64 ? 64 : 128;
  p.bn_cols = K <= 64 ? 64 : 128;
  p.part_bytes = n * p.tiles * 8;
  // a piece of G within 128 MB: the 256 MB memory-side cache then holds it between the three products
  int64_t cols = (int64_t(128) << 20) / (e * (n > 0 ? n : 1)) / 128 * 128;
  if (cols < 128) cols = 128;
  const int64_t pieces = ceil_div<int64_t>(C, cols);
  p.piece = up(ceil_div<int64_t>(C, pieces), 128);
  p.ldg = p.piece;
  p.g_bytes = n * p.ldg * e;
  // splits of the reductions: at least two workgroups per CU, ranges of at least eight tile depths
  auto split = [&](int64_t tiles, int64_t len, int32_t* s, int64_t* range) {
    int64_t want = ceil_div<int64_t>(512, tiles), most = len / (8 * bk);
    if (want > most) want = most;
    if (want < 1) want = 1;
    *range = up(ceil_div<int64_t>(len, want), bk);
    *s = (int32_t)ceil_div<int64_t>(len, *range);
  };
  split(ceil_div<int64_t>(n, 128) * ceil_div<int64_t>(K, p.bn_cols), p.piece, &p.dh_splits, &p.dh_range);
  split(p.piece / 128 * ceil_div<int64_t>(K, p.bn_cols), n > 0 ? n : 1, &p.dw_splits, &p.dw_range);
  const int64_t a = (int64_t)p.dh_splits * n * K * 4, b = p.dw_splits > 1 ? (int64_t)p.dw_splits * p.piece * (K + 1) * 4 : 0;
  p.acc_bytes = up(a, 256) + up(b, 256);
  return p;
}

template <typename T>
int lx_forward(LxArgs& a, const LxPlan& p, hipStream_t st) {
  a.c_lo = 0;
  a.c_hi = a.C;
  const dim3 grid((unsigned)(p.tiles * ceil_div<int64_t>(a.n, p.bn_rows)));
  if (p.bn_rows == 64)
    hipLaunchKernelGGL((k_lx_logits<T, 64, false>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((k_lx_logits<T, 128, false>), grid, dim3(256), 0, st, a);
  PG_LAUNCH_CHECK();
  hipLaunchKernelGGL(k_lx_rows, dim3((unsigned)ceil_div<int64_t>(a.n, 4)), dim3(256), 0, st, a);
  PG_LAUNCH_CHECK();
  return PG_OK;
}

template <typename T>
int lx_backward(LxArgs& a, const LxPlan& p, char* scratch, hipStream_t st) {
  a.g = scratch;
  float* acc_dh = (float*)(scratch + up(p.g_bytes, 256));
  float* acc_dw = (float*)((char*)acc_dh + up((int64_t)p.dh_splits * a.n * a.K * 4, 256));
  a.ldg = p.ldg;
  const int64_t row_tiles = ceil_div<int64_t>(a.n, 128), k_tiles = ceil_div<int64_t>(a.K, p.bn_cols);
  for (a.c_lo = 0; a.c_lo < a.C; a.c_lo = a.c_hi) {
    a.c_hi = a.c_lo + p.piece < a.C ? a.c_lo + p.piece : a.C;
    const int64_t len = a.c_hi - a.c_lo, c_tiles = ceil_div<int64_t>(len, 128);
    const dim3 g1((unsigned)(c_tiles * ceil_div<int64_t>(a.n, p.bn_rows)));
    if (p.bn_rows == 64)
      hipLaunchKernelGGL((k_lx_logits<T, 64, true>), g1, dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((k_lx_logits<T, 128, true>), g1, dim3(256), 0, st, a);
    PG_LAUNCH_CHECK();
    if (a.dh) {
      a.acc = acc_dh;
      a.splits = p.dh_splits;
      a.k_split = p.dh_range;
      a.first = a.c_lo == 0;
      const dim3 g2((unsigned)(row_tiles * k_tiles * a.splits));
      if (p.bn_cols == 64)
        hipLaunchKernelGGL((k_lx_dh<T, 64>), g2, dim3(256), 0, st, a);
      else
        hipLaunchKernelGGL((k_lx_dh<T, 128>), g2, dim3(256), 0, st, a);
      PG_LAUNCH_CHECK();
    }
    if (a.dw || a.db) {
      a.acc = acc_dw;
      a.accb = p.dw_splits > 1 ? acc_dw + (int64_t)p.dw_splits * len * a.K : nullptr;
      a.splits = p.dw_splits;
      a.k_split = p.dw_range;
      const dim3 g3((unsigned)(c_tiles * k_tiles * a.splits));
      if (p.bn_cols == 64)
        hipLaunchKernelGGL((k_lx_dw<T, 64>), g3, dim3(256), 0, st, a);
      else
        hipLaunchKernelGGL((k_lx_dw<T, 128>), g3, dim3(256), 0, st, a);
      PG_LAUNCH_CHECK();
      if (a.splits > 1) {
        const int64_t b = ceil_div<int64_t>(len * (a.K + 1), 256);
        hipLaunchKernelGGL(k_lx_dw_out<T>, dim3((unsigned)(b > 4096 ? 4096 : b)), dim3(256), 0, st, a);
        PG_LAUNCH_CHECK();
      }
    }
  }
  if (a.dh) {
    a.acc = acc_dh;
    a.splits = p.dh_splits;
    const int64_t b = ceil_div<int64_t>(a.n * a.K, 256);
    hipLaunchKernelGGL(k_lx_dh_out<T>, dim3((unsigned)(b > 4096 ? 4096 : b)), dim3(256), 0, st, a);
    PG_LAUNCH_CHECK();
  }
  return PG_OK;
}

// the grids are one-dimensional: every product's tile count has to fit
inline int lx_check(int64_t n, int64_t K, int64_t C, int32_t dtype) {
  if (n < 0 || K <= 0 || C <= 0 || dtype < PG_DTYPE_F32 || dtype > PG_DTYPE_F16) return PG_ERR_INVALID;
  if (n > (int64_t(1) << 31) || K > (int64_t(1) << 24) || C > (int64_t(1) << 31)) return PG_ERR_UNSUPPORTED;
  if (ceil_div<int64_t>(n, 64) * ceil_div<int64_t>(C, 128) > 0x7fffffffll / 2) return PG_ERR_UNSUPPORTED;
  return PG_OK;
}

int lx_args(const pg_linear_xent_desc_t* d, LxArgs* a) {
  if (!d) return PG_ERR_INVALID;
  const int rc = lx_check(d->n, d->K, d->C, d->dtype);
  if (rc != PG_OK) return rc;
  if (d->h_stride < d->K || d->w_stride < d->K) return PG_ERR_INVALID;
  if (!d->W || !d->meta || (d->n > 0 && (!d->h || !d->labels || !d->lse || !d->flag))) return PG_ERR_INVALID;
  *a = LxArgs{};
  a->h = d->h; a->w = d->W; a->bias = d->bias; a->labels = d->labels;
  a->n = d->n; a->K = d->K; a->C = d->C; a->hs = d->h_stride; a->ws = d->w_stride; a->ignore = d->ignore_index;
  a->lse = d->lse; a->flag = d->flag; a->row_loss = d->row_loss; a->meta = d->meta;
  return PG_OK;
}

}  // namespace pg

using namespace pg;

extern "C" {

int64_t pg_linear_xent_scratch(int64_t n, int64_t K, int64_t C, int32_t dtype, int32_t backward) {
  if (lx_check(n, K, C, dtype) != PG_OK) return -1;
  if (n == 0) return 0;
  const LxPlan p = lx_plan(n, K, C, dtype);
  return backward ? up(p.g_bytes, 256) + p.acc_bytes + up(4 * n, 256) + 256 : up(p.part_bytes, 256) + up(4 * n, 256);
}

int pg_linear_xent_fwd(const pg_linear_xent_desc_t* d, pg_stream_t stream) {
  LxArgs a;
  int rc = lx_args(d, &a);
  if (rc != PG_OK) return rc;
  hipStream_t st = as_stream(stream);
  if (a.n > 0) {
    if (!d->row_loss || !d->scratch) return PG_ERR_INVALID;
    const LxPlan p = lx_plan(a.n, a.K, a.C, d->dtype);
    a.part = (float2*)d->scratch;
    a.zlab = (float*)((char*)d->scratch + up(p.part_bytes, 256));
    a.tiles = p.tiles;
    rc = d->dtype == PG_DTYPE_F32 ? lx_forward<float>(a, p, st) : d->dtype == PG_DTYPE_BF16 ? lx_forward<bf16_t>(a, p, st) : lx_forward<f16_t>(a, p, st);
    if (rc != PG_OK) return rc;
  }
  hipLaunchKernelGGL(k_lx_mean, dim3(1), dim3(1024), 0, st, a.row_loss, a.flag, a.n, a.meta);
  PG_LAUNCH_CHECK();
  return PG_OK;
}

int pg_linear_xent_bwd(const pg_linear_xent_desc_t* d, pg_stream_t stream) {
  LxArgs a;
  int rc = lx_args(d, &a);
  if (rc != PG_OK) return rc;
  if (!d->grad || d->reduction < PG_XENT_MEAN || d->reduction > PG_XENT_NONE) return PG_ERR_INVALID;
  if (a.n == 0) return PG_ERR_INVALID;            // no row, no gradient to compute: the caller's zeros
  if (!d->scratch) return PG_ERR_INVALID;
  hipStream_t st = as_stream(stream);
  const LxPlan p = lx_plan(a.n, a.K, a.C, d->dtype);
  char* s = (char*)d->scratch;
  a.dh = d->dh; a.dw = d->dW; a.db = d->db;
  if (d->reduction == PG_XENT_NONE) {
    float* rowf = (float*)(s + up(p.g_bytes, 256) + p.acc_bytes);
    float* top = (float*)((char*)rowf + up(4 * a.n, 256));
    hipLaunchKernelGGL(k_lx_row_factors, dim3(1), dim3(1024), 0, st, d->grad, d->grad_stride, a.flag, a.n, rowf, top);
    PG_LAUNCH_CHECK();
    a.rowf = rowf;
    a.f1 = top;
  } else {
    a.rowf = a.flag;
    a.f1 = d->grad;
    a.f2 = d->reduction == PG_XENT_MEAN ? a.meta + 1 : nullptr;
  }
  return d->dtype == PG_DTYPE_F32 ? lx_backward<float>(a, p, s, st) : d->dtype == PG_DTYPE_BF16 ? lx_backward<bf16_t>(a, p, s, st) : lx_backward<f16_t>(a, p, s, st);
}

}  // extern "C"
