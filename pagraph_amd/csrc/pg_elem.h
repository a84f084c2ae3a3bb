// Element types of the operators that take fp32, bf16 and fp16 rows (pg_norm.hip, pg_xent_linear.hip). Arithmetic is always
// fp32; a row leaves with one round-to-nearest-even conversion per element.
#pragma once
#include "pg_common.h"

namespace pg {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// four consecutive elements as floats. The memcpy has the element's own alignment: gfx950's global loads and stores take any
// alignment, so a row of 602 floats (2408 bytes: not a multiple of 16) still moves 16 bytes per lane.
template <typename T>
__device__ __forceinline__ void load4(const T* __restrict__ p, float (&v)[4]) {
  T t[4];
  __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (float)t[i];
}
template <typename T>
__device__ __forceinline__ void store4(T* __restrict__ p, const float (&v)[4]) {
  T t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = (T)v[i];
  __builtin_memcpy(p, t, sizeof(t));
}
// ... of a row that ends inside them (left = columns from p to the row's end): what lies behind it reads as 0, is not written
template <typename T>
__device__ __forceinline__ void load4_tail(const T* __restrict__ p, int64_t left, float (&v)[4]) {
  if (left >= 4) {
    load4(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? (float)p[i] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store4_tail(T* __restrict__ p, int64_t left, const float (&v)[4]) {
  if (left >= 4) {
    store4(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i] = (T)v[i];
  }
}

}  // namespace pg
