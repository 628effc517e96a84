// cf_decay.cu — decayed linear attention over whole prompts:
//
//   S_t = l S_{t-1} + k_t^T v_t,   o_t = scale q_t S_t,   l = exp(log_decay[h])
//
// The plain recurrence: a CTA takes 32 columns of the state of one (sequence,
// head) and walks its tokens, 16 at a time through shared memory.  A lane owns a
// column, a warp an eighth of its rows, in registers.
#include "cf_half.cuh"

namespace cf {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kCols = 32;
constexpr int kTok = 16;
constexpr int kMaxDim = 128;
constexpr int kRows = kMaxDim / kWarps;

struct DecayArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  const float* log_decay;
  const float* s_in;
  float* s_out;
  const int32_t* slots;
  const int32_t* cu;
  int64_t n_slots, L, N, q_st, q_sh, k_st, k_sh, v_st, v_sh, o_st, o_sh;
  int Hq, Hk, Dk, Dv, n_slices;
  float scale;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) decay_recurrent_kernel(const __grid_constant__ DecayArgs a) {
  __shared__ float s_k[kTok][kMaxDim], s_q[kTok][kMaxDim], s_v[kTok][kCols];
  __shared__ float s_o[kWarps][kTok][kCols];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int slice = blockIdx.x % a.n_slices;
  const int64_t sh = blockIdx.x / a.n_slices;
  const int h = (int)(sh % a.Hk);
  const int64_t seq = sh / a.Hk;
  const int G = a.Hq / a.Hk;
  int64_t t0 = seq * a.L, t1 = t0 + a.L;
  if (a.cu) {
    t0 = min(max((int64_t)a.cu[seq], (int64_t)0), a.N);
    t1 = min(max((int64_t)a.cu[seq + 1], t0), a.N);
  }
  const int64_t slot = a.slots ? a.slots[seq] : seq;
  const bool has_slot = slot >= 0 && slot < a.n_slots;
  const int c = slice * kCols + lane;
  const bool on = c < a.Dv;
  const float2 decay = decay_hi_lo(a.log_decay[h]);
  const int64_t base = (slot * a.Hk + h) * a.Dk * a.Dv + c;
  float s[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = i * kWarps + warp;
    s[i] = (on && r < a.Dk && a.s_in && has_slot) ? a.s_in[base + (int64_t)r * a.Dv] : 0.f;
  }
  for (int64_t t = t0; t < t1; t += kTok) {
    const int n = t1 - t < kTok ? (int)(t1 - t) : kTok;
    __syncthreads();
    for (int i = threadIdx.x; i < n * a.Dk; i += kThreads)
      s_k[i / a.Dk][i % a.Dk] = to_f(static_cast<const T*>(a.k)[(t + i / a.Dk) * a.k_st + h * a.k_sh + i % a.Dk]);
    for (int i = threadIdx.x; i < n * kCols; i += kThreads) {
      const int cc = slice * kCols + i % kCols;
      s_v[i / kCols][i % kCols] = cc < a.Dv ? to_f(static_cast<const T*>(a.v)[(t + i / kCols) * a.v_st + h * a.v_sh + cc]) : 0.f;
    }
    float s0[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) s0[i] = s[i];
    for (int g = 0; g < G; ++g) {
      const int64_t hq = (int64_t)h * G + g;
      for (int i = threadIdx.x; i < n * a.Dk; i += kThreads)
        s_q[i / a.Dk][i % a.Dk] = to_f(static_cast<const T*>(a.q)[(t + i / a.Dk) * a.q_st + hq * a.q_sh + i % a.Dk]);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kRows; ++i) s[i] = s0[i];
      for (int j = 0; j < n; ++j) {
        const float v = s_v[j][lane];
        float o = 0.f;
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const int r = i * kWarps + warp;
          if (r < a.Dk) {
            s[i] = fmaf(decay.x, s[i], fmaf(decay.y, s[i], s_k[j][r] * v));
            o += s_q[j][r] * s[i];
          }
        }
        s_o[warp][j][lane] = o;
      }
      __syncthreads();
      for (int i = threadIdx.x; i < n * kCols; i += kThreads) {
        const int j = i / kCols, cc = slice * kCols + i % kCols;
        float sum = 0.f;
        for (int w = 0; w < kWarps; ++w) sum += s_o[w][j][i % kCols];
        if (cc < a.Dv)
          static_cast<T*>(a.out)[(t + j) * a.o_st + hq * a.o_sh + cc] = from_f<T>(sum * a.scale);
      }
      __syncthreads();
    }
  }
  if (a.s_out && has_slot && on) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int r = i * kWarps + warp;
      if (r < a.Dk) a.s_out[base + (int64_t)r * a.Dv] = s[i];
    }
  }
}

}  // namespace
}  // namespace cf

using namespace cf;

extern "C" int64_t cf_decay_attention_workspace(int64_t S, int64_t N, int64_t Hk, int64_t Dk, int64_t Dv) {
  if (S < 0 || N < 0 || Hk <= 0 || Dk <= 0 || Dv <= 0)
    return fail(CF_ERR_INVALID_ARG, "bad attention shape");
  return 0;
}

extern "C" int cf_decay_attention(const void* q, const void* k, const void* v, void* out, int fmt,
                                  const float* log_decay, const float* s_in, float* s_out,
                                  const int32_t* slots, int64_t n_slots, const int32_t* cu_seqlens,
                                  int64_t S, int64_t L, int64_t N, int64_t Hq, int64_t Hk, int64_t Dk,
                                  int64_t Dv, int64_t q_st, int64_t q_sh, int64_t k_st, int64_t k_sh,
                                  int64_t v_st, int64_t v_sh, int64_t o_st, int64_t o_sh, float scale,
                                  void* workspace, int64_t workspace_bytes, void* stream) {
  if (S < 0 || N < 0 || Hq <= 0 || Hk <= 0 || Hq % Hk || Dk <= 0 || Dv <= 0 || n_slots < 0)
    return fail(CF_ERR_INVALID_ARG, "bad attention shape (Hq must be a multiple of Hk)");
  if (!cu_seqlens && (L < 0 || (L ? N / L != S || N % L : N != 0)))
    return fail(CF_ERR_INVALID_ARG, "N must be S * L without cu_seqlens");
  if (fmt != CF_FMT_F16 && fmt != CF_FMT_BF16)
    return fail(CF_ERR_INVALID_ARG, "q, k and v must be fp16 or bf16");
  if (Dk % 8 || Dv % 8 || Dk > kMaxDim || Dv > kMaxDim)
    return fail(CF_ERR_UNSUPPORTED, "head dimensions must be multiples of 8 and at most %d", kMaxDim);
  if (S == 0) return CF_OK;
  if (!log_decay || (N && (!q || !k || !v || !out)))
    return fail(CF_ERR_INVALID_ARG, "q, k, v, out and log_decay must not be NULL");
  if (!slots && (s_in || s_out) && n_slots < S)
    return fail(CF_ERR_INVALID_ARG, "fewer states than sequences");
  const int64_t slices = (Dv + kCols - 1) / kCols;
  if (Hq > 65536 || S > 0x7FFFFFFF / (Hk * slices))
    return fail(CF_ERR_UNSUPPORTED, "too many sequences or heads");
  if (int rc = require_sm100()) return rc;
  DecayArgs a{q, k, v, out, log_decay, s_in, s_out, slots, cu_seqlens, n_slots, L, N, q_st, q_sh,
              k_st, k_sh, v_st, v_sh, o_st, o_sh, (int)Hq, (int)Hk, (int)Dk, (int)Dv, (int)slices, scale};
  const unsigned grid = (unsigned)(S * Hk * slices);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (fmt == CF_FMT_F16) decay_recurrent_kernel<__half><<<grid, kThreads, 0, st>>>(a);
  else decay_recurrent_kernel<__nv_bfloat16><<<grid, kThreads, 0, st>>>(a);
  return check_launch("decay_attention launch");
}
