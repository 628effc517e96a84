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
// 32768, more than bf16 rounds away.
//
// A warp owns a token (or a share of its heads where tokens are few): each lane
// takes the sine and cosine of a few pairs and the warp exchanges them once.  Every
// lane then keeps, for its own channels, sines and cosines times the norm's weights
// in registers for all heads of the token:
//
//   a' = inv (a (wa cos) - b (wb sin)),   b' = inv (b (wb cos) + a (wa sin))
//
// so a head costs one load, one sum over the row's lanes, two products of two values
// at a time per pair, and one store, with the next two rows' loads in flight.
// (With weights and rotation applied one after the other and a rounded square root
// and division, four rows of 128 channels took 390 instructions and the case below 64 us.)
//
// Measured: 8192 tokens of 32 + 8 heads of 128 in bf16, 46 us = 3.6 TB/s; 12544 tokens of
// 16 + 16 heads of 80 in fp16 on three axes (4-byte vectors, since half of 60 rotated
// channels is no multiple of 8 bytes), 54 us = 2.4 TB/s.  Bound by its instructions: 21 and 35
// an element where converting, summing, turning and storing need about 4; a scheduler issues in
// 0.57 and 0.62 of its cycles with 14 warps an SM (123 registers; capped at 80 it
// spilled and lost more than the occupancy gained).
#include "cf_half.cuh"

namespace cf {
namespace {

constexpr int kRopeThreads = 128;
constexpr int kRopeMaxDim = 256;
constexpr int kRopeMaxAxes = 4;

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
  int Hq, Hk, D, rot, half_pairs, norm;  // half_pairs: pairs are (p, p + rot/2)
  int partial;      // some channels pass through
  int lpr, splits;  // lanes of a row, warps of a token
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
__device__ __forceinline__ void to_floats(const typename RopeVec<T, V>::type& raw, float* f) {
  const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = to_f(e[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float* f) {
  typename RopeVec<T, V>::type raw;
  T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
  for (int i = 0; i < V; ++i) e[i] = from_f<T>(f[i]);
  *reinterpret_cast<typename RopeVec<T, V>::type*>(p) = raw;
}

// Two fp32 values at a time, in a register pair.
typedef unsigned long long F2;
__device__ __forceinline__ F2 pack2(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpack2(F2 a, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a));
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// A lane owns U units of a row, a unit being two vectors of V channels that
// hold V whole pairs (or 2V channels that pass through); lpr lanes own a row.
template <typename T, int V, int U>
__global__ void __launch_bounds__(kRopeThreads) qk_norm_rope_kernel(const __grid_constant__ RopeArgs a) {
  __shared__ float2 s_cs[kRopeThreads / 32][kRopeMaxDim / 2];
  __shared__ __align__(16) float s_w[2][kRopeMaxDim];
  using Vec = typename RopeVec<T, V>::type;
  const int lane = threadIdx.x & 31;
  const int64_t id = (int64_t)blockIdx.x * (kRopeThreads / 32) + (threadIdx.x >> 5);
  const int64_t t = min(id / a.splits, a.N - 1);
  const int split = (int)(id - id / a.splits * a.splits);
  const int P = a.rot / 2, RU = a.rot / (2 * V), NU = a.D / (2 * V);
  const int lpr = a.lpr, sub = lane & (lpr - 1), rows = 32 / lpr;
  const int itq = (a.Hq + rows - 1) / rows, its = itq + (a.Hk + rows - 1) / rows;
  const int first = its * split / a.splits, end = id / a.splits < a.N ? its * (split + 1) / a.splits : 0;
  int ca[U], cb[U];  // first channels of the two vectors
#pragma unroll
  for (int j = 0; j < U; ++j) {
    const int unit = sub + j * lpr;
    const bool apart = a.half_pairs && unit < RU;
    ca[j] = apart ? unit * V : 2 * unit * V;
    cb[j] = apart ? ca[j] + P : ca[j] + V;
  }
  const T* const q = static_cast<const T*>(a.q) + t * a.q_st;
  const T* const k = static_cast<const T*>(a.k) + t * a.k_st;
  T* const qo = static_cast<T*>(a.q_out) + t * a.qo_st;
  T* const ko = static_cast<T*>(a.k_out) + t * a.ko_st;
  // rows it * rows .. of the queries, then of the keys
  auto head = [&](int it) { return (it < itq ? it : it - itq) * rows + lane / lpr; };
  auto on = [&](int it) { return it < end && head(it) < (it < itq ? a.Hq : a.Hk); };
  auto load = [&](int it, Vec (&x)[U], Vec (&y)[U]) {
    const T* src = it < itq ? q + head(it) * a.q_sh : k + head(it) * a.k_sh;
    const bool in = on(it);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      x[j] = y[j] = Vec{};
      if (in && sub + j * lpr < NU) {
        x[j] = *reinterpret_cast<const Vec*>(src + ca[j]);
        y[j] = *reinterpret_cast<const Vec*>(src + cb[j]);
      }
    }
  };
  constexpr int B = 2;  // rows of a batch; the next batch is loaded while one is worked on
  Vec nx[B][U], ny[B][U];
#pragma unroll
  for (int b = 0; b < B; ++b) load(first + b, nx[b], ny[b]);

  for (int i = threadIdx.x; i < 2 * a.D; i += kRopeThreads) {
    const float* w = a.norm ? (i < a.D ? a.q_weight : a.k_weight) : nullptr;
    const int c = i < a.D ? i : i - a.D;
    s_w[i >= a.D][c] = w ? w[c] : 1.f;
  }
  float2* cs = s_cs[threadIdx.x >> 5];
  for (int p = lane; p < P; p += 32) {
    const int64_t at = a.axis[p] * a.pos_stride + t;
    const double pos = a.pos64 ? (double)static_cast<const int64_t*>(a.pos)[at]
                               : (double)static_cast<const int32_t*>(a.pos)[at];
    const double turns = pos * (double)a.inv_freq[p] * 0.15915494309189533577;
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    cs[p] = make_float2(c, s);
  }
  __syncthreads();

  // Coefficients of x and y, the lane's two vectors, two values at a time:
  // pairs across the vectors: x' = x c0 + y c1, y' = y c2 + x c3;
  // pairs within a vector:    x' = x c0 + swap(x) c1, y' = y c2 + swap(y) c3.
  // One value in place of two where V = 1 (the second is unused).
  constexpr int H = V > 1 ? V / 2 : 1;
  F2 c0[U][H], c1[U][H], c2[U][H], c3[U][H];
  auto coefficients = [&](const float* wt) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int unit = sub + j * lpr;
      const bool in = unit < NU, turned = unit < RU;
      float wa[2 * H], wb[2 * H], c[2 * H], s[2 * H];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        wa[i] = in ? wt[ca[j] + i] : 0.f;
        wb[i] = in ? wt[cb[j] + i] : 0.f;
        const float2 z = turned ? cs[unit * V + i] : make_float2(1.f, 0.f);
        c[i] = z.x;
        s[i] = z.y;
      }
      if (V == 1) wa[1] = wb[1] = c[1] = s[1] = 0.f;
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const int e = 2 * i, f = 2 * i + 1;
        if (a.half_pairs || V == 1) {
          c0[j][i] = pack2(wa[e] * c[e], wa[f] * c[f]);
          c1[j][i] = pack2(-wb[e] * s[e], -wb[f] * s[f]);
          c2[j][i] = pack2(wb[e] * c[e], wb[f] * c[f]);
          c3[j][i] = pack2(wa[e] * s[e], wa[f] * s[f]);
        } else {  // vector x holds pairs 0 .. V/2 - 1, y the others
          const float cx = c[i], sx = s[i], cy = c[V / 2 + i], sy = s[V / 2 + i];
          c0[j][i] = pack2(wa[e] * cx, wa[f] * cx);
          c1[j][i] = pack2(-wa[f] * sx, wa[e] * sx);
          c2[j][i] = pack2(wb[e] * cy, wb[f] * cy);
          c3[j][i] = pack2(-wb[f] * sy, wb[e] * sy);
        }
      }
    }
  };
  const float inv_d = 1.f / (float)a.D;
  bool keys = first >= itq;
  coefficients(s_w[keys]);
  for (int it = first; it < end; it += B) {
    Vec rx[B][U], ry[B][U];
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int j = 0; j < U; ++j) {
        rx[b][j] = nx[b][j];
        ry[b][j] = ny[b][j];
      }
#pragma unroll
    for (int b = 0; b < B; ++b) load(it + B + b, nx[b], ny[b]);
#pragma unroll
    for (int b = 0; b < B; ++b) {
      if (it + b >= end) break;
      if (!keys && it + b >= itq) {
        keys = true;
        coefficients(s_w[1]);
      }
      F2 x[U][H], y[U][H];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        float e[2 * H], f[2 * H];
        e[2 * H - 1] = f[2 * H - 1] = 0.f;
        to_floats<T, V>(rx[b][j], e);
        to_floats<T, V>(ry[b][j], f);
#pragma unroll
        for (int i = 0; i < H; ++i) {
          x[j][i] = pack2(e[2 * i], e[2 * i + 1]);
          y[j][i] = pack2(f[2 * i], f[2 * i + 1]);
        }
      }
      float inv = 1.f;
      if (a.norm) {
        F2 sum = 0;
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
          for (int i = 0; i < H; ++i) sum = fma2(x[j][i], x[j][i], fma2(y[j][i], y[j][i], sum));
        float ss, s1;
        unpack2(sum, ss, s1);
        ss += s1;
        for (int m = lpr >> 1; m; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
        inv = rsqrtf(fmaf(ss, inv_d, a.eps));
      }
      const F2 inv2 = pack2(inv, inv);
      const bool put = on(it + b);
      T* dst = it + b < itq ? qo + head(it + b) * a.qo_sh : ko + head(it + b) * a.ko_sh;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        float e[2 * H], f[2 * H];
#pragma unroll
        for (int i = 0; i < H; ++i) {
          F2 p = x[j][i], r = y[j][i];  // what meets c1 and c3
          if (a.half_pairs || V == 1) {
            p = y[j][i];
            r = x[j][i];
          } else {
            float u, v;
            unpack2(p, u, v);
            p = pack2(v, u);
            unpack2(r, u, v);
            r = pack2(v, u);
          }
          F2 u = mul2(x[j][i], c0[j][i]), v = mul2(y[j][i], c2[j][i]);
          if (!a.partial || sub + j * lpr < RU) {  // else no partner: 0 * inf must not appear
            u = fma2(p, c1[j][i], u);
            v = fma2(r, c3[j][i], v);
          }
          unpack2(mul2(u, inv2), e[2 * i], e[2 * i + 1]);
          unpack2(mul2(v, inv2), f[2 * i], f[2 * i + 1]);
        }
        if (put && sub + j * lpr < NU) {
          store_vec<T, V>(dst + ca[j], e);
          store_vec<T, V>(dst + cb[j], f);
        }
      }
    }
  }
}

template <typename T, int V, int U>
int launch_rope(const RopeArgs& a, cudaStream_t s) {
  constexpr int kWarps = kRopeThreads / 32;
  const int64_t grid = (a.N * a.splits + kWarps - 1) / kWarps;
  qk_norm_rope_kernel<T, V, U><<<(unsigned)grid, kRopeThreads, 0, s>>>(a);
  return check_launch("qk_norm_rope launch");
}

// As few lanes a row as keep U V <= 8: more rows a warp, and more loads in
// flight a lane (80 channels in 4-byte vectors: 8 lanes x 3 units instead of 32 x 1).
template <typename T>
int launch_rope_v(RopeArgs a, int V, cudaStream_t s) {
  const int units = a.D / (2 * V);
  a.lpr = 1;
  while (a.lpr < 32 && a.lpr * (8 / V) < units) a.lpr <<= 1;
  const int U = (units + a.lpr - 1) / a.lpr, rows = 32 / a.lpr;
  // Tokens that do not fill the GPU share their heads out over more warps.
  const int its = (a.Hq + rows - 1) / rows + (a.Hk + rows - 1) / rows;
  const int64_t want = (148 * 16 + a.N - 1) / a.N;
  a.splits = (int)(want < its ? want : its);
  if (V == 8) return launch_rope<T, 8, 1>(a, s);
  if (V == 4) return U == 1 ? launch_rope<T, 4, 1>(a, s) : launch_rope<T, 4, 2>(a, s);
  if (V == 2)
    return U == 1 ? launch_rope<T, 2, 1>(a, s) : U == 2 ? launch_rope<T, 2, 2>(a, s)
         : U == 3 ? launch_rope<T, 2, 3>(a, s) : launch_rope<T, 2, 4>(a, s);
  return launch_rope<T, 1, 8>(a, s);
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
  if (!rows_apart(N, qo_st, Hq, qo_sh, D) || !rows_apart(N, ko_st, Hk, ko_sh, D))
    return fail(CF_ERR_INVALID_ARG, "rows of an output overlap");
  if (int rc = require_sm100()) return rc;

  a.q = q; a.k = k; a.q_out = q_out; a.k_out = k_out;
  a.q_st = q_st; a.q_sh = q_sh; a.k_st = k_st; a.k_sh = k_sh;
  a.qo_st = qo_st; a.qo_sh = qo_sh; a.ko_st = ko_st; a.ko_sh = ko_sh;
  a.pos = positions; a.pos_stride = pos_stride; a.pos64 = pos_bits == 64;
  a.inv_freq = inv_freq; a.q_weight = q_weight; a.k_weight = k_weight;
  a.N = N; a.Hq = (int)Hq; a.Hk = (int)Hk; a.D = (int)D; a.rot = (int)rot;
  a.half_pairs = pairing == CF_PAIR_HALF; a.partial = rot < D; a.norm = norm; a.eps = eps;
  if (N > 0x7FFFFFFF) return fail(CF_ERR_UNSUPPORTED, "too many tokens");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return fmt == CF_FMT_F16 ? launch_rope_v<__half>(a, V, s) : launch_rope_v<__nv_bfloat16>(a, V, s);
}
