// cf_rope.cu — per-head RMS norm of queries and keys with the position
// rotation in the same pass, so that each element crosses HBM once each way.
//
//   y = x / sqrt(mean(x^2) + eps) * w          (norm; optional)
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = pos[axis(p)] * inv_freq[p]
//
// for the pairs p of the first `rot` channels of a head; channels from `rot` on
// pass through.  A pair is (p, p + rot/2) or (2p, 2p + 1).  Each pair belongs to
// one of up to four position axes (text: one; images: height and width; video:
// time, height and width).
//
// The angle is reduced in fp64 (turns = pos * inv_freq / 2 pi, minus the nearest
// whole number): in fp32 the product alone is 2e-3 radians off at position
// 32768, more than bf16 rounds away.  One sine and cosine per (token, pair) is
// put into shared memory and serves all heads of the token.
#include "cf_half.cuh"

namespace cf {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxDim = 256;
constexpr int kRopeMaxAxes = 4;
constexpr int kRopeMaxTokens = 16;      // tokens of one CTA
constexpr int kRopeTableBytes = 16 << 10;  // cosines and sines of one CTA

struct RopeArgs {
  const void* q;
  const void* k;
  void* q_out;
  void* k_out;
  int64_t q_st, q_sh, k_st, k_sh, qo_st, qo_sh, ko_st, ko_sh;  // token and head strides
  const void* pos;
  int64_t pos_stride;  // elements between two position axes
  int pos64;
  const float* inv_freq;
  const float* q_weight;
  const float* k_weight;
  int64_t N;
  int Hq, Hk, D, rot, half_pairs, norm, tok;  // half_pairs: pairs are (p, p + rot/2)
  float eps;
  uint8_t axis[kRopeMaxDim / 2];
};

template <typename T, int V>
struct RopeVec;
template <typename T>
struct RopeVec<T, 8> { using type = uint4; };
template <typename T>
struct RopeVec<T, 4> { using type = uint2; };
template <typename T>
struct RopeVec<T, 2> { using type = uint32_t; };
template <typename T>
struct RopeVec<T, 1> { using type = uint16_t; };

template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&f)[V]) {
  typename RopeVec<T, V>::type raw = *reinterpret_cast<const typename RopeVec<T, V>::type*>(p);
  const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = to_f(e[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[V]) {
  typename RopeVec<T, V>::type raw;
  T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
  for (int i = 0; i < V; ++i) e[i] = from_f<T>(f[i]);
  *reinterpret_cast<typename RopeVec<T, V>::type*>(p) = raw;
}

__device__ __forceinline__ void turn(float& a, float& b, float2 cs) {
  const float u = a, v = b;
  a = u * cs.x - v * cs.y;
  b = v * cs.x + u * cs.y;
}

// A lane owns U units of a row, a unit being two vectors of V channels that
// hold V whole pairs (or 2V channels that pass through); lpr <= 32 lanes own a row.
template <typename T, int V, int U>
__global__ void __launch_bounds__(kRopeThreads) qk_norm_rope_kernel(const __grid_constant__ RopeArgs a,
                                                                   int lpr) {
  extern __shared__ float2 s_cs[];  // [tokens of this CTA][rot / 2]
  const int P = a.rot / 2;
  const int64_t t0 = (int64_t)blockIdx.x * a.tok;
  const int nt = a.N - t0 < a.tok ? (int)(a.N - t0) : a.tok;
  for (int i = threadIdx.x; i < nt * P; i += kRopeThreads) {
    const int t = i / P, p = i - t * P;
    const int64_t at = a.axis[p] * a.pos_stride + t0 + t;
    const double pos = a.pos64 ? (double)static_cast<const int64_t*>(a.pos)[at]
                               : (double)static_cast<const int32_t*>(a.pos)[at];
    const double turns = pos * (double)a.inv_freq[p] * 0.15915494309189533577;
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    s_cs[i] = make_float2(c, s);
  }
  __syncthreads();

  const int H = a.Hq + a.Hk;
  const int lane = threadIdx.x & (lpr - 1);
  const int rows_at_once = kRopeThreads / lpr;
  const int RU = a.rot / (2 * V), NU = a.D / (2 * V);
  // every lane of a warp takes part in the row sums, also beyond the last row
  const int n_rows = nt * H;
  for (int r0 = 0; r0 < n_rows; r0 += rows_at_once) {
    const int r = r0 + threadIdx.x / lpr;
    const bool on = r < n_rows;
    const int t = on ? r / H : 0;
    const int h = on ? r - t * H : 0;
    const bool is_q = h < a.Hq;
    const int hh = is_q ? h : h - a.Hq;
    const T* src = is_q ? static_cast<const T*>(a.q) + (t0 + t) * a.q_st + hh * a.q_sh
                        : static_cast<const T*>(a.k) + (t0 + t) * a.k_st + hh * a.k_sh;
    T* dst = is_q ? static_cast<T*>(a.q_out) + (t0 + t) * a.qo_st + hh * a.qo_sh
                  : static_cast<T*>(a.k_out) + (t0 + t) * a.ko_st + hh * a.ko_sh;
    float x[U][V], y[U][V];
    int ca[U], cb[U];  // first channels of the two vectors
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int unit = lane + j * 32;
      const bool split = a.half_pairs && unit < RU;
      ca[j] = split ? unit * V : 2 * unit * V;
      cb[j] = split ? ca[j] + P : ca[j] + V;
#pragma unroll
      for (int i = 0; i < V; ++i) x[j][i] = y[j][i] = 0.f;
      if (on && unit < NU) {
        load_vec<T, V>(src + ca[j], x[j]);
        load_vec<T, V>(src + cb[j], y[j]);
      }
    }
    if (a.norm) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < U; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) ss += x[j][i] * x[j][i] + y[j][i] * y[j][i];
      for (int m = lpr >> 1; m; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
      const float inv = 1.f / sqrtf(ss / (float)a.D + a.eps);
      const float* w = is_q ? a.q_weight : a.k_weight;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        if (lane + j * 32 >= NU) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          x[j][i] *= w ? inv * __ldg(w + ca[j] + i) : inv;
          y[j][i] *= w ? inv * __ldg(w + cb[j] + i) : inv;
        }
      }
    }
    if (!on) continue;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int unit = lane + j * 32;
      if (unit >= NU) continue;
      if (unit < RU) {
        const float2* cs = s_cs + t * P + unit * V;
        if (a.half_pairs || V == 1) {
#pragma unroll
          for (int i = 0; i < V; ++i) turn(x[j][i], y[j][i], cs[i]);
        } else {
#pragma unroll
          for (int i = 0; i + 1 < V; i += 2) {
            turn(x[j][i], x[j][i + 1], cs[i / 2]);
            turn(y[j][i], y[j][i + 1], cs[V / 2 + i / 2]);
          }
        }
      }
      store_vec<T, V>(dst + ca[j], x[j]);
      store_vec<T, V>(dst + cb[j], y[j]);
    }
  }
}

template <typename T, int V>
int launch_rope(const RopeArgs& a, cudaStream_t s) {
  constexpr int U = kRopeMaxDim / (2 * V) > 32 ? kRopeMaxDim / (2 * V) / 32 : 1;
  int lpr = 1;
  while (lpr < 32 && lpr < a.D / (2 * V)) lpr <<= 1;
  const int64_t grid = (a.N + a.tok - 1) / a.tok;
  qk_norm_rope_kernel<T, V, U>
      <<<(unsigned)grid, kRopeThreads, (size_t)a.tok * (a.rot / 2) * 8, s>>>(a, lpr);
  return check_launch("qk_norm_rope launch");
}

template <typename T>
int launch_rope_v(const RopeArgs& a, int V, cudaStream_t s) {
  switch (V) {
    case 8: return launch_rope<T, 8>(a, s);
    case 4: return launch_rope<T, 4>(a, s);
    case 2: return launch_rope<T, 2>(a, s);
    default: return launch_rope<T, 1>(a, s);
  }
}

}  // namespace
}  // namespace cf

using namespace cf;

extern "C" int cf_qk_norm_rope(const void* q, const void* k, void* q_out, void* k_out, int fmt,
                               int64_t N, int64_t Hq, int64_t Hk, int64_t D, int64_t q_st,
                               int64_t q_sh, int64_t k_st, int64_t k_sh, int64_t qo_st,
                               int64_t qo_sh, int64_t ko_st, int64_t ko_sh, const void* positions,
                               int pos_bits, int64_t pos_stride, const float* inv_freq,
                               int64_t rot, const int32_t* sections, int axes, int axis_order,
                               int pairing, const float* q_weight, const float* k_weight, int norm,
                               float eps, void* stream) {
  if (N < 0 || Hq <= 0 || Hk <= 0 || D <= 0 || rot < 0 || axes < 1)
    return fail(CF_ERR_INVALID_ARG, "bad rotation shape");
  if (fmt != CF_FMT_F16 && fmt != CF_FMT_BF16)
    return fail(CF_ERR_INVALID_ARG, "q and k must be fp16 or bf16");
  if (D > kRopeMaxDim || (D & 1))
    return fail(CF_ERR_UNSUPPORTED, "head_dim must be even and at most %d", kRopeMaxDim);
  if (rot > D || (rot & 1))
    return fail(CF_ERR_INVALID_ARG, "the rotated channels must be even and at most head_dim");
  if (axes > kRopeMaxAxes)
    return fail(CF_ERR_UNSUPPORTED, "at most %d position axes", kRopeMaxAxes);
  if (!sections) return fail(CF_ERR_INVALID_ARG, "sections must not be NULL");
  if (pos_bits != 32 && pos_bits != 64)
    return fail(CF_ERR_INVALID_ARG, "positions must have 32 or 64 bits");
  if ((axis_order != CF_AXES_BLOCKS && axis_order != CF_AXES_CYCLIC) ||
      (pairing != CF_PAIR_HALF && pairing != CF_PAIR_ADJACENT))
    return fail(CF_ERR_INVALID_ARG, "unknown axis order or pairing");
  if (Hq + Hk > 65536) return fail(CF_ERR_UNSUPPORTED, "too many heads");
  RopeArgs a{};
  int left[kRopeMaxAxes];
  int64_t sum = 0;
  for (int i = 0; i < axes; ++i) {
    if (sections[i] < 0 || sections[i] > rot / 2)
      return fail(CF_ERR_INVALID_ARG, "sections must be between 0 and rot / 2");
    left[i] = sections[i];
    sum += sections[i];
  }
  if (sum != rot / 2) return fail(CF_ERR_INVALID_ARG, "sections must add up to rot / 2");
  for (int p = 0, ax = 0; p < rot / 2;) {
    if (left[ax]) {
      --left[ax];
      a.axis[p++] = (uint8_t)ax;
      if (axis_order == CF_AXES_BLOCKS) continue;
    }
    ax = ax + 1 == axes ? 0 : ax + 1;
  }
  if (N == 0) return CF_OK;
  if (!q || !k || !q_out || !k_out || (rot && (!positions || !inv_freq)))
    return fail(CF_ERR_INVALID_ARG, "q, k, their outputs, positions and inv_freq must not be NULL");

  // the widest vector that divides the pairs, what passes through, and every
  // row's address
  int V = 8;
  const int64_t st[] = {q_st, q_sh, k_st, k_sh, qo_st, qo_sh, ko_st, ko_sh};
  const void* ptrs[] = {q, k, q_out, k_out};
  for (; V > 1; V >>= 1) {
    const int per_side = pairing == CF_PAIR_HALF ? V : 2 * V;  // channels of a vector or a unit
    bool ok = (pairing == CF_PAIR_HALF ? rot / 2 : rot) % per_side == 0 && (D - rot) % (2 * V) == 0;
    for (int64_t x : st) ok = ok && x % V == 0;
    for (const void* p : ptrs) ok = ok && reinterpret_cast<uintptr_t>(p) % (2 * V) == 0;
    if (ok) break;
  }
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) & 1)
      return fail(CF_ERR_UNSUPPORTED, "q, k and their outputs must be aligned to their type");
  if (int rc = require_sm100()) return rc;

  a.q = q; a.k = k; a.q_out = q_out; a.k_out = k_out;
  a.q_st = q_st; a.q_sh = q_sh; a.k_st = k_st; a.k_sh = k_sh;
  a.qo_st = qo_st; a.qo_sh = qo_sh; a.ko_st = ko_st; a.ko_sh = ko_sh;
  a.pos = positions; a.pos_stride = pos_stride; a.pos64 = pos_bits == 64;
  a.inv_freq = inv_freq; a.q_weight = q_weight; a.k_weight = k_weight;
  a.N = N; a.Hq = (int)Hq; a.Hk = (int)Hk; a.D = (int)D; a.rot = (int)rot;
  a.half_pairs = pairing == CF_PAIR_HALF; a.norm = norm; a.eps = eps;
  a.tok = 4;
  if (a.tok * (rot / 2) * 8 > kRopeTableBytes) a.tok = 1;
  if ((N + a.tok - 1) / a.tok > 0x7FFFFFFF) return fail(CF_ERR_UNSUPPORTED, "too many tokens");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return fmt == CF_FMT_F16 ? launch_rope_v<__half>(a, V, s) : launch_rope_v<__nv_bfloat16>(a, V, s);
}
