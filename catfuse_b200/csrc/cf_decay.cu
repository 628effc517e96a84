// cf_decay.cu — decayed linear attention over whole prompts (host side and the
// small kernels; the tensor-core kernel is in cf_decay_kernels.cuh).
//
//   S_t = l S_{t-1} + k_t^T v_t,   o_t = scale q_t S_t,   l = exp(log_decay[h])
//
// A prompt is walked chunk by chunk by one CTA per (sequence, head).  Where that
// leaves the GPU idle, sequences are cut into segments: one launch sums each
// segment's own state from its k and v, a small one turns them into the states
// that enter the segments, and the walk then runs per segment.
//
// Measured (launches one by one): 4095 tokens of 32 heads of 128 x 128, states summed
// in 22 us, entered in 4 us, walked in 45 us (floor 21 us without the second reading
// of k and v); 65536 tokens of 16 heads of 64 x 64, 64 + 7 + 159 us (floor 82 us).
#include "cf_decay_kernels.cuh"

#include <cmath>
#include <mutex>

namespace cf {
namespace decayk {
// cf_decay_tc_{f16,bf16}.cu
template <typename T>
int launch_chunks(bool out, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                  const DecayArgs& a, int sms, cudaStream_t s);
extern template int launch_chunks<__half>(bool, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&,
                                          const DecayArgs&, int, cudaStream_t);
extern template int launch_chunks<__nv_bfloat16>(bool, const CUtensorMap&, const CUtensorMap&,
                                                 const CUtensorMap&, const DecayArgs&, int, cudaStream_t);
}  // namespace decayk

namespace {
using namespace decayk;

constexpr int kMaxDim = 128;

// --------------------------------------------------------------------------
// Rows that a TMA load cannot start on (not 16-byte aligned): the recurrence
// itself.  A CTA takes 32 columns of the state of one (sequence, head) and walks
// its tokens, 16 at a time through shared memory.  A lane owns a column, a warp
// an eighth of its rows, in registers.  Bound by the walk itself, 0.8 us a token
// and CTA: 4095 tokens of 32 heads of 128 x 128 took 3.2 ms.
// --------------------------------------------------------------------------
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kCols = 32;
constexpr int kTok = 16;
constexpr int kRows = kMaxDim / kWarps;

template <typename T>
__global__ void __launch_bounds__(kThreads) decay_recurrent_kernel(const __grid_constant__ DecayArgs a,
                                                               int n_slices) {
  __shared__ float s_k[kTok][kMaxDim], s_q[kTok][kMaxDim], s_v[kTok][kCols];
  __shared__ float s_o[kWarps][kTok][kCols];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int slice = blockIdx.x % n_slices;
  const int64_t sh = blockIdx.x / n_slices;
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
  const bool carried = a.s_in && has_slot && (t0 == t1 || keeps_state(a.log_decay[h]));
  const int64_t base = (slot * a.Hk + h) * a.Dk * a.Dv + c;
  float s[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = i * kWarps + warp;
    s[i] = (on && r < a.Dk && carried) ? a.s_in[base + (int64_t)r * a.Dv] : 0.f;
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

// --------------------------------------------------------------------------
// segments
// --------------------------------------------------------------------------

template <typename I>
__device__ __forceinline__ I warp_scan(I x) {  // over the lanes up to this one
  for (int m = 1; m < 32; m <<= 1) {
    const I y = __shfl_up_sync(0xffffffffu, x, m);
    if ((threadIdx.x & 31) >= m) x += y;
  }
  return x;
}

// The segments of packed sequences, in order: every sequence has one at least, and
// those with more have a row of seg_states for each (first: the first of them).
// Entries that are left over have seq = -1.  Sums over more than a warp's sequences (2^23
// segments each at most) are 64 bits wide: overlapping boundaries can ask for far more
// segments and rows than there are, and get no more.
__global__ void __launch_bounds__(1024) decay_segments_kernel(const int32_t* cu, int S, int64_t N, int64_t seg_len,
                                                              Seg* segs, int32_t* first, int64_t n_segs,
                                                              int64_t n_rows) {
  __shared__ int32_t s_n[32], s_rows[32];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t base = 0, row_base = 0;
  for (int s0 = 0; s0 < S; s0 += 1024) {
    const int s = s0 + threadIdx.x;
    int64_t t0 = 0, t1 = 0;
    int32_t n = 0;
    if (s < S) {
      t0 = min(max((int64_t)cu[s], (int64_t)0), N);
      t1 = min(max((int64_t)cu[s + 1], t0), N);
      n = t1 > t0 ? (int32_t)((t1 - t0 + seg_len - 1) / seg_len) : 1;
    }
    const int32_t own_rows = n > 1 ? n : 0;
    const int32_t n_to = warp_scan(n), rows_to = warp_scan(own_rows);
    if (lane == 31) {
      s_n[warp] = n_to;
      s_rows[warp] = rows_to;
    }
    __syncthreads();
    const int64_t n_all = warp_scan((int64_t)s_n[lane]), rows_all = warp_scan((int64_t)s_rows[lane]);
    int64_t at = base + n_to - n, row = row_base + rows_to - own_rows;
    const int64_t n_before = __shfl_sync(0xffffffffu, n_all, (warp + 31) & 31);
    const int64_t rows_before = __shfl_sync(0xffffffffu, rows_all, (warp + 31) & 31);
    if (warp > 0) {
      at += n_before;
      row += rows_before;
    }
    if (s < S) {
      first[s] = (int32_t)min(row, n_rows);
      for (int i = 0; i < n && at < n_segs; ++i, ++at, ++row) {
        const int64_t b = t0 + i * seg_len;
        const bool in = n == 1 || row < n_rows;
        segs[at] = Seg{(int32_t)b, (int32_t)min(b + seg_len, t1), in ? s : -1,
                       (n == 1 ? 0 : (int32_t)min(row, n_rows) * 2) + (i == n - 1)};
      }
    }
    base += __shfl_sync(0xffffffffu, n_all, 31);
    row_base += __shfl_sync(0xffffffffu, rows_all, 31);
    __syncthreads();
  }
  for (int64_t i = base + threadIdx.x; i < n_segs; i += 1024) segs[i] = Seg{0, 0, -1, 0};
  if (threadIdx.x == 0) first[S] = (int32_t)min(row_base, n_rows);
}

// A segment's own state L_r becomes the state that enters it:
// E_0 = s_in, E_{r+1} = l^{seg_len} E_r + L_r.  One thread per four entries of a
// (sequence, head).  The chain runs in fp64: with the power rounded to fp32 a state that
// decays slowly drifted by 2.6 x 2^-18 of itself over 256 segments.
__global__ void __launch_bounds__(256) decay_enter_kernel(const __grid_constant__ DecayArgs a,
                                                          const int32_t* first) {
  griddep_wait();
  griddep_launch_dependents();
  const int dd = a.Dk * a.Dv, parts = (dd + 1023) / 1024;
  const int e = (int)(blockIdx.x % parts * 256 + threadIdx.x) * 4;
  const int h = (int)(blockIdx.x / parts % a.Hk);
  const int64_t seq = blockIdx.x / parts / a.Hk;
  if (e >= dd) return;
  const int64_t r0 = a.segs ? first[seq] : seq * a.n_seg;
  const int n = a.segs ? first[seq + 1] - first[seq] : a.n_seg;
  if (n < 2) return;
  const int64_t slot = a.slots ? a.slots[seq] : seq;
  const bool carried = a.s_in && slot >= 0 && slot < a.n_slots;
  const int64_t step = (int64_t)a.Hk * dd;
  float* p = a.seg_states + (r0 * a.Hk + h) * dd + e;
  double run[4] = {0.0, 0.0, 0.0, 0.0};
  if (carried && keeps_state(a.log_decay[h])) {
    const float4 x = *reinterpret_cast<const float4*>(a.s_in + (slot * a.Hk + h) * dd + e);
    run[0] = x.x, run[1] = x.y, run[2] = x.z, run[3] = x.w;
  }
  const double l = exp((double)a.log_decay[h] * (double)a.seg_len);
  auto put = [&](float* to) {
    *reinterpret_cast<float4*>(to) = make_float4((float)run[0], (float)run[1], (float)run[2], (float)run[3]);
  };
  constexpr int kAhead = 4;  // own states in flight
  for (int r = 0; r + 1 < n; r += kAhead) {
    float4 own[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (r + i + 1 < n) own[i] = *reinterpret_cast<const float4*>(p + i * step);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (r + i + 1 < n) {
        if (r + i > 0 || carried) put(p + i * step);
        run[0] = fma(l, run[0], (double)own[i].x);
        run[1] = fma(l, run[1], (double)own[i].y);
        run[2] = fma(l, run[2], (double)own[i].z);
        run[3] = fma(l, run[3], (double)own[i].w);
      }
    }
    p += kAhead * step;
  }
  put(a.seg_states + ((r0 + n - 1) * a.Hk + h) * dd + e);
}

// --------------------------------------------------------------------------
// host side
// --------------------------------------------------------------------------
int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    return 148;
  }
  return n;
}

struct Plan {
  int64_t seg_len, n_segs, n_rows, state_bytes, bytes;  // n_rows: states of cut sequences' segments
  int n_seg;  // segments of each sequence (dense)
  bool split;
};

// How long the segments are.  Times in units of one chunk of a single query
// head: the walk takes 1 for a chunk and its first query head and about 0.7 for
// every further one, the pass that sums states 0.6; a segment costs 5 on top (its
// state comes and goes, its pipeline fills), a cut call's two more launches 8.
Plan make_plan(int64_t S, int64_t N, int64_t Hq, int64_t Hk, int64_t Dk, int64_t Dv, bool packed, int sms) {
  Plan p{};
  const double t_walk = 1.0 + 0.7 * ((double)Hq / Hk - 1.0), t_sum = 0.6, t_cut = 8.0, t_unit = 5.0;
  const int64_t units = S * Hk, ctas = (Dk <= 64 && Dv <= 64) ? 2 * sms : sms;
  p.n_segs = S;
  p.n_seg = 1;
  p.seg_len = N > kC ? (N + kC - 1) / kC * kC : kC;
  if (S > 0 && N > 0) {
    if (!packed) {
      const int64_t ch = (N / S + kC - 1) / kC;
      double best = 0;
      for (int64_t n = 1; n <= ch && n <= 256; ++n) {
        const int64_t len = (ch + n - 1) / n;
        if ((ch + len - 1) / len != n) continue;
        const double waves = (double)((units * n + ctas - 1) / ctas);
        const double waves_s = (double)((units * (n - 1) + ctas - 1) / ctas);
        const double t = waves * (len * t_walk + t_unit) + (n > 1 ? waves_s * (len * t_sum + t_unit) + t_cut : 0.0);
        if (n == 1 || t < best) {
          best = t;
          p.n_seg = (int)n;
          p.seg_len = len * kC;
        }
      }
      p.n_segs = p.n_rows = S * p.n_seg;
      p.split = p.n_seg > 1;
    } else {
      // Lengths are on the device.  The shorter the segments, the more evenly
      // they spread (half a segment is lost at the end), and the more of them
      // there are to set up: of c chunks for each CTA, c / len segments.
      const double c = (double)(N / kC + S) * Hk / ctas;
      int64_t len = (int64_t)sqrt(2.0 * c * t_unit / t_walk) + 1;
      if (len < 4) len = 4;
      if (N > len * kC) {
        p.seg_len = len * kC;
        p.n_segs = S + N / p.seg_len;
        // a cut sequence has more than seg_len tokens, and one segment that is not full
        p.n_rows = N / p.seg_len + (S < N / p.seg_len ? S : N / p.seg_len);
        p.split = true;
      }
    }
  }
  if (p.split) {
    p.state_bytes = p.n_rows * Hk * Dk * Dv * 4;
    p.bytes = p.state_bytes + (packed ? p.n_segs * (int64_t)sizeof(Seg) + (S + 1) * 4 : 0);
    p.bytes = (p.bytes + 15) / 16 * 16;
  }
  return p;
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// x[N][H][D] by strides, in boxes of 64 tokens x 64 channels of one head.  Heads
// of a multiple of 64 channels bring their panels in one load.
int make_map(CUtensorMap* m, int fmt, const void* x, int64_t N, int64_t H, int64_t D, int64_t st,
             int64_t sh, int* panels) {
  const bool whole = D % 64 == 0;
  *panels = whole ? (int)(D / 64) : 1;
  if (N == 1) st = 8;  // an axis of one entry: its stride is never taken
  if (H == 1) sh = D;
  cuuint64_t dims[4] = {(cuuint64_t)(whole ? 64 : D), (cuuint64_t)N, (cuuint64_t)*panels, (cuuint64_t)H};
  cuuint64_t strides[3] = {(cuuint64_t)st * 2, 128, (cuuint64_t)sh * 2};
  cuuint32_t box[4] = {64, (cuuint32_t)kC, (cuuint32_t)*panels, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  auto encode = encode_fn();
  if (!encode) return fail(CF_ERR_CUDA, "cuTensorMapEncodeTiled entry point unavailable");
  const CUresult r = encode(m, fmt == CF_FMT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                            4, const_cast<void*>(x), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(CF_ERR_CUDA, "tensor map (attention) failed: %d", (int)r);
  return CF_OK;
}

// Whether TMA can read rows: 16-byte address and strides, strides within the
// tensor map's range.
bool tma_rows(const void* p, int64_t N, int64_t H, int64_t st, int64_t sh) {
  const int64_t lim = (int64_t)1 << 38;
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (N == 1 || (st % 8 == 0 && st > 0 && st < lim)) &&
         (H == 1 || (sh % 8 == 0 && sh > 0 && sh < lim));
}

template <typename Kern, typename... Args>
int launch_after(Kern kernel, dim3 grid, int threads, cudaStream_t s, const char* what, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, args...), what);
}

}  // namespace
}  // namespace cf

using namespace cf;

extern "C" int64_t cf_decay_attention_workspace(int64_t S, int64_t N, int64_t Hq, int64_t Hk, int64_t Dk,
                                                int64_t Dv, int packed) {
  if (S < 0 || N < 0 || Hk <= 0 || Hq <= 0 || Hq % Hk || Dk <= 0 || Dv <= 0 || Dk > kMaxDim || Dv > kMaxDim)
    return fail(CF_ERR_INVALID_ARG, "bad attention shape");
  return make_plan(S, N, Hq, Hk, Dk, Dv, packed != 0, sm_count()).bytes;
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
  if (Hq > 65535 || N > 0x7FFFFFC0 || S > 0x7FFFFFFF / (Hk * 16))
    return fail(CF_ERR_UNSUPPORTED, "too many tokens, sequences or heads");
  for (const void* p : {(const void*)s_in, (const void*)s_out, (const void*)workspace})
    if (reinterpret_cast<uintptr_t>(p) & 15)
      return fail(CF_ERR_UNSUPPORTED, "states and workspace must be 16-byte aligned");
  if (!rows_apart(N, o_st, Hq, o_sh, Dv))
    return fail(CF_ERR_INVALID_ARG, "rows of out overlap");
  const bool recurrence = N == 0 || !tma_rows(q, N, Hq, q_st, q_sh) || !tma_rows(k, N, Hk, k_st, k_sh) ||
                          !tma_rows(v, N, Hk, v_st, v_sh);
  if (N && recurrence && Dv > kCols && (out == q || out == k))  // other CTAs of a head read them while one writes
    return fail(CF_ERR_INVALID_ARG, "out must not be q or k where rows are off 16 bytes");
  if (int rc = require_sm100()) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  DecayArgs a{};
  a.q = q; a.k = k; a.v = v; a.out = out; a.log_decay = log_decay; a.s_in = s_in; a.s_out = s_out;
  a.slots = slots; a.cu = cu_seqlens; a.n_slots = n_slots; a.L = L; a.N = N;
  a.q_st = q_st; a.q_sh = q_sh; a.k_st = k_st; a.k_sh = k_sh; a.v_st = v_st; a.v_sh = v_sh;
  a.o_st = o_st; a.o_sh = o_sh; a.Hq = (int)Hq; a.Hk = (int)Hk; a.Dk = (int)Dk; a.Dv = (int)Dv;
  a.S = (int)S; a.scale = scale; a.n_seg = 1;

  if (recurrence) {
    const int slices = (int)((Dv + kCols - 1) / kCols);
    const unsigned grid = (unsigned)(S * Hk * slices);
    if (fmt == CF_FMT_F16) decay_recurrent_kernel<__half><<<grid, kThreads, 0, st>>>(a, slices);
    else decay_recurrent_kernel<__nv_bfloat16><<<grid, kThreads, 0, st>>>(a, slices);
    return check_launch("decay_attention launch");
  }

  const int sms = sm_count();
  const Plan p = make_plan(S, N, Hq, Hk, Dk, Dv, cu_seqlens != nullptr, sms);
  if (p.n_segs > 0x7FFFFFFF / Hk) return fail(CF_ERR_UNSUPPORTED, "too many tokens, sequences or heads");
  if (p.split && (!workspace || workspace_bytes < p.bytes))
    return fail(CF_ERR_INVALID_ARG, "the workspace must have %lld bytes", (long long)p.bytes);
  a.max_polls = wait_limit();
  a.err = device_error_word();
  if (!a.err) return fail(CF_ERR_CUDA, "device error word is not addressable");
  a.drop_load = take_stalled_load();
  a.n_seg = p.n_seg;
  a.seg_len = p.seg_len;
  a.seg_states = static_cast<float*>(workspace);
  a.o_vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && o_st % 8 == 0 && o_sh % 8 == 0;
  CUtensorMap mq, mk, mv;
  if (int rc = make_map(&mq, fmt, q, N, Hq, Dk, q_st, q_sh, &a.qp)) return rc;
  if (int rc = make_map(&mk, fmt, k, N, Hk, Dk, k_st, k_sh, &a.kp)) return rc;
  if (int rc = make_map(&mv, fmt, v, N, Hk, Dv, v_st, v_sh, &a.vp)) return rc;
  auto chunks = [&](bool with_out) {
    return fmt == CF_FMT_F16 ? launch_chunks<__half>(with_out, mq, mk, mv, a, sms, st)
                             : launch_chunks<__nv_bfloat16>(with_out, mq, mk, mv, a, sms, st);
  };
  if (p.split) {
    int32_t* first = nullptr;
    if (cu_seqlens) {
      Seg* segs = reinterpret_cast<Seg*>(static_cast<char*>(workspace) + p.state_bytes);
      first = reinterpret_cast<int32_t*>(segs + p.n_segs);
      a.segs = segs;
      if (int rc = launch_after(decay_segments_kernel, dim3(1), 1024, st, "decay segments launch", cu_seqlens,
                                (int)S, N, p.seg_len, segs, first, p.n_segs, p.n_rows))
        return rc;
    }
    a.n_units = (uint32_t)((cu_seqlens ? p.n_segs : S * (p.n_seg - 1)) * Hk);
    if (int rc = chunks(false)) return rc;
    const dim3 grid((unsigned)((Dk * Dv + 1023) / 1024 * S * Hk));
    if (int rc = launch_after(decay_enter_kernel, grid, 256, st, "decay states launch", a, (const int32_t*)first))
      return rc;
  }
  a.n_units = (uint32_t)(p.n_segs * Hk);
  return chunks(true);
}
