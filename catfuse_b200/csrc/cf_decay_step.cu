// cf_decay_step.cu — decayed linear attention for one token per sequence:
//
//   S = l S + k^T v,   o = scale q S,   l = exp(log_decay[h])
//
// per head that owns a state S [Dk][Dv] (fp32); its Hq / Hk query heads all read
// that state.  The state crosses HBM once each way (8 Dk Dv bytes per head),
// which is what bounds the operator: q, k, v and o are a hundredth of it.
//
// A CTA takes 32 columns of one state: eight lanes cover a row's 128 bytes, so
// every request is whole sectors, and columns are independent, so no sums cross
// CTAs and the result does not depend on the grid.
//
// Measured: 128 sequences of 32 states of 128 x 128, 85 us = 6.4 TB/s, 0.97 of the
// measured copy bandwidth (256 threads with half the rows each: 90 us, 64 with twice
// as many: 89 us); 512 sequences of 64 x 64, 98 us of a floor of 83 (130 with 256).
#include "cf_half.cuh"

namespace cf {
namespace {

constexpr int kStepThreads = 128;
constexpr int kStepCols = 32;   // state columns of a CTA
constexpr int kStepMaxDim = 128;
static_assert(kStepThreads >= kStepMaxDim, "a thread loads one entry of q and k");
constexpr int kStepRowGroups = kStepThreads / (kStepCols / 4);
constexpr int kStepRows = kStepMaxDim / kStepRowGroups;  // state rows of a thread

struct StepArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  const float* log_decay;
  const float* s_in;
  float* s_out;
  const int32_t* slots;
  int64_t n_slots, q_st, q_sh, k_st, k_sh, v_st, v_sh, o_st, o_sh;
  int Hq, Hk, Dk, Dv, n_slices;
  float scale;
};

template <typename T>
__global__ void __launch_bounds__(kStepThreads) decay_step_kernel(const __grid_constant__ StepArgs a) {
  __shared__ float s_k[kStepMaxDim];
  __shared__ float s_q[kStepMaxDim];
  __shared__ float2 s_decay;
  __shared__ __align__(16) float s_o[kStepThreads / 32][kStepCols];
  const int slice = blockIdx.x % a.n_slices;
  const int64_t bh = blockIdx.x / a.n_slices;
  const int h = (int)(bh % a.Hk);
  const int64_t b = bh / a.Hk;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = a.Hq / a.Hk;
  const int64_t slot = a.slots ? a.slots[b] : b;
  const int c0 = slice * kStepCols;
  T* out = static_cast<T*>(a.out) + b * a.o_st;
  if (slot < 0 || slot >= a.n_slots) {  // padding: no state behind this row
    for (int i = tid; i < G * kStepCols; i += kStepThreads) {
      const int c = c0 + i % kStepCols;
      if (c < a.Dv) out[(int64_t)(h * G + i / kStepCols) * a.o_sh + c] = from_f<T>(0.f);
    }
    return;
  }
  const int c = c0 + (tid & 7) * 4;
  const int rg = tid >> 3;
  const bool on = c < a.Dv;
  const int64_t base = (slot * a.Hk + h) * a.Dk * a.Dv + c;
  float4 s[kStepRows];
#pragma unroll
  for (int i = 0; i < kStepRows; ++i) {
    const int r = i * kStepRowGroups + rg;
    s[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (on && r < a.Dk) s[i] = __ldcs(reinterpret_cast<const float4*>(a.s_in + base + (int64_t)r * a.Dv));
  }
  if (tid < a.Dk) s_k[tid] = to_f(static_cast<const T*>(a.k)[b * a.k_st + h * a.k_sh + tid]);
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (on) {
    const T* pv = static_cast<const T*>(a.v) + b * a.v_st + h * a.v_sh + c;
    v = make_float4(to_f(pv[0]), to_f(pv[1]), to_f(pv[2]), to_f(pv[3]));
  }
  if (tid == 0) {
    const float ld = a.log_decay[h];
    s_decay = keeps_state(ld) ? decay_hi_lo(ld) : make_float2(-1.f, 0.f);
  }
  __syncthreads();
  const float2 decay = s_decay;
  // -1: nothing is kept, and what was loaded may be anything; masked to zeros
  const uint32_t kept = decay.x == -1.f ? 0u : ~0u;
  auto held = [&](float x) { return __uint_as_float(__float_as_uint(x) & kept); };
#pragma unroll
  for (int i = 0; i < kStepRows; ++i) {
    const int r = i * kStepRowGroups + rg;
    if (on && r < a.Dk) {
      const float k = s_k[r];
      const float4 e = make_float4(held(s[i].x), held(s[i].y), held(s[i].z), held(s[i].w));
      s[i].x = fmaf(decay.x, e.x, fmaf(decay.y, e.x, k * v.x));
      s[i].y = fmaf(decay.x, e.y, fmaf(decay.y, e.y, k * v.y));
      s[i].z = fmaf(decay.x, e.z, fmaf(decay.y, e.z, k * v.z));
      s[i].w = fmaf(decay.x, e.w, fmaf(decay.y, e.w, k * v.w));
      __stcs(reinterpret_cast<float4*>(a.s_out + base + (int64_t)r * a.Dv), s[i]);
    }
  }
  for (int g = 0; g < G; ++g) {
    const int64_t hq = (int64_t)h * G + g;
    if (tid < a.Dk) s_q[tid] = to_f(static_cast<const T*>(a.q)[b * a.q_st + hq * a.q_sh + tid]);
    __syncthreads();
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kStepRows; ++i) {
      const int r = i * kStepRowGroups + rg;
      if (r < a.Dk) {
        const float q = s_q[r];
        o.x += q * s[i].x; o.y += q * s[i].y; o.z += q * s[i].z; o.w += q * s[i].w;
      }
    }
#pragma unroll
    for (int m = 8; m <= 16; m <<= 1) {
      o.x += __shfl_xor_sync(0xffffffffu, o.x, m);
      o.y += __shfl_xor_sync(0xffffffffu, o.y, m);
      o.z += __shfl_xor_sync(0xffffffffu, o.z, m);
      o.w += __shfl_xor_sync(0xffffffffu, o.w, m);
    }
    if (lane < 8) *reinterpret_cast<float4*>(&s_o[warp][lane * 4]) = o;
    __syncthreads();
    if (tid < kStepCols && c0 + tid < a.Dv) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kStepThreads / 32; ++w) sum += s_o[w][tid];
      out[hq * a.o_sh + c0 + tid] = from_f<T>(sum * a.scale);
    }
    __syncthreads();
  }
}

}  // namespace
}  // namespace cf

using namespace cf;

extern "C" int cf_decay_attention_step(const void* q, const void* k, const void* v, void* out,
                                       int fmt, const float* log_decay, const float* s_in,
                                       float* s_out, const int32_t* slots, int64_t n_slots,
                                       int64_t B, int64_t Hq, int64_t Hk, int64_t Dk, int64_t Dv,
                                       int64_t q_st, int64_t q_sh, int64_t k_st, int64_t k_sh,
                                       int64_t v_st, int64_t v_sh, int64_t o_st, int64_t o_sh,
                                       float scale, void* stream) {
  if (B < 0 || Hq <= 0 || Hk <= 0 || Hq % Hk || Dk <= 0 || Dv <= 0 || n_slots < 0)
    return fail(CF_ERR_INVALID_ARG, "bad attention shape (Hq must be a multiple of Hk)");
  if (fmt != CF_FMT_F16 && fmt != CF_FMT_BF16)
    return fail(CF_ERR_INVALID_ARG, "q, k and v must be fp16 or bf16");
  if (Dk % 8 || Dv % 8 || Dk > kStepMaxDim || Dv > kStepMaxDim)
    return fail(CF_ERR_UNSUPPORTED, "head dimensions must be multiples of 8 and at most %d", kStepMaxDim);
  if (B == 0) return CF_OK;
  if (!q || !k || !v || !out || !log_decay || !s_in || !s_out)
    return fail(CF_ERR_INVALID_ARG, "q, k, v, out, log_decay and the states must not be NULL");
  if (!slots && n_slots < B) return fail(CF_ERR_INVALID_ARG, "fewer states than sequences");
  if ((reinterpret_cast<uintptr_t>(s_in) | reinterpret_cast<uintptr_t>(s_out)) & 15)
    return fail(CF_ERR_UNSUPPORTED, "states must be 16-byte aligned");
  const int64_t slices = (Dv + kStepCols - 1) / kStepCols;
  if (Hq > 65536 || B > 0x7FFFFFFF / (Hk * slices))
    return fail(CF_ERR_UNSUPPORTED, "too many sequences or heads");
  if (slices > 1 && (out == q || out == k))  // other CTAs of a head read them while one writes
    return fail(CF_ERR_INVALID_ARG, "out must not be q or k");
  if (!rows_apart(B, o_st, Hq, o_sh, Dv))
    return fail(CF_ERR_INVALID_ARG, "rows of out overlap");
  if (int rc = require_sm100()) return rc;
  StepArgs a{q, k, v, out, log_decay, s_in, s_out, slots, n_slots, q_st, q_sh, k_st, k_sh,
             v_st, v_sh, o_st, o_sh, (int)Hq, (int)Hk, (int)Dk, (int)Dv, (int)slices, scale};
  const unsigned grid = (unsigned)(B * Hk * slices);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (fmt == CF_FMT_F16) decay_step_kernel<__half><<<grid, kStepThreads, 0, st>>>(a);
  else decay_step_kernel<__nv_bfloat16><<<grid, kStepThreads, 0, st>>>(a);
  return check_launch("decay_attention_step launch");
}
