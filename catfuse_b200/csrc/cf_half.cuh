// cf_half.cuh — fp16 / bf16 element access shared by the attention kernels.
#pragma once

#include "cf_common.cuh"

#include <cuda_bf16.h>

namespace cf {

__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// Whether the rows of an output (d elements; n of them st apart, of each h heads sh
// apart) share no element: where they do, the value left would be either writer's.
inline bool rows_apart(int64_t n, int64_t st, int64_t h, int64_t sh, int64_t d) {
  st = st < 0 ? -st : st;
  sh = sh < 0 ? -sh : sh;
  if (n <= 1) return n == 0 || h <= 1 || sh >= d;
  if (h <= 1) return st >= d;
  return st < sh ? st >= d && (n - 1) <= (sh - d) / st : sh >= d && (h - 1) <= (st - d) / sh;
}

// A head's decay l = exp(log_decay) as hi + lo, so that l s is
// fma(hi, s, lo s): with l rounded to fp32 alone, a state that forgets slowly
// would drift by 2^-25 of itself at every token.
__device__ __forceinline__ float2 decay_hi_lo(float log_decay) {
  const double l = exp((double)log_decay);
  const float hi = (float)l;
  return make_float2(hi, isfinite(hi) ? (float)(l - (double)hi) : 0.f);
}

// Whether a head's state outlives a token.  What enters one that keeps nothing
// (log_decay = -inf) is not looked at: it may be anything, and 0 * inf is no zero.
__device__ __forceinline__ bool keeps_state(float log_decay) { return log_decay != -INFINITY; }

}  // namespace cf
