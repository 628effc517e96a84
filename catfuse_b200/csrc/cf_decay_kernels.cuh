// cf_decay_kernels.cuh — decayed linear attention over whole prompts on the
// 5th-generation tensor cores (tcgen05, sm_100a).
//
//   S_t = l S_{t-1} + k_t^T v_t,   o_t = scale q_t S_t,   l = exp(log_decay[h])
//
// Chunks of C = 64 tokens turn the recurrence into matrix products.  With S
// entering a chunk (tokens i, j counted from 0, n of them):
//
//   o_i = scale ( l^{i+1} q_i S + sum_{j <= i} l^{i-j} (q_i . k_j) v_j )
//   S'  = l^n S + sum_j l^{n-1-j} k_j^T v_j
//
// One CTA walks the chunks of one (segment, head); the Hq / Hk query heads of a
// head follow each other inside a chunk, so k, v and the state are read once for
// all of them.  S stays in registers in fp32 for the whole walk.
//
// Products per chunk (D = accumulator in TMEM, fp32):
//   QK  [64 i][64 j]    A = Q (K-major),        B = K (K-major)
//   KV  [dv][dk]        A = V' (MN-major),      B = K (MN-major)   V'_j = l^{n-1-j} v_j
//   QS  [dv][64 i]      A = S^T (K-major),      B = Q (K-major)
//   PV  [dv][64 i]      A = V (MN-major),       B = P (K-major)    P_ij = l^{i-j} QK_ij, j <= i
// The outputs are built transposed (channels in lanes): with 64 tokens as M the
// same products run at half rate.
//
// What is rounded to 16 bits on its way through a product, and how: V' carries
// the state's precision, so it goes as three bf16 parts (24 bits) or two fp16
// parts (22 bits); S and P only reach the 16-bit outputs and go as two parts, which
// leaves the outputs' own rounding as their only error of that size (one part each
// made it 1.4 times as large).  fp16 parts are scaled by powers of two (V' per chunk,
// S per channel, P per row), so that neither a full state nor a small one leaves
// fp16's range; bf16 has fp32's range.
//
// Warp roles: P warps (QK -> P), O warps (outputs), state warps (V', S), one TMA
// warp, one MMA warp.
#pragma once

#include "cf_half.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

namespace cf {
namespace decayk {

constexpr int kC = 64;            // tokens of a chunk
constexpr int kTileBytes = kC * 128;  // 64 tokens x 64 channels of 16 bits, 128-byte swizzle
constexpr int kSmallBytes = 3072;  // barriers and tables

enum : int32_t {
  ERR_SITE_DECAY_LOAD = 16,
  ERR_SITE_DECAY_MMA = 17,
  ERR_SITE_DECAY_P = 18,
  ERR_SITE_DECAY_O = 19,
  ERR_SITE_DECAY_STATE = 20,
  ERR_SITE_DECAY_ALIGN = 21,
};

struct Seg {  // one segment of one packed sequence
  int32_t t0, t1, seq, last;
};

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
  const Seg* segs;    // packed sequences in segments, else NULL
  float* seg_states;  // [segment][Hk][Dk][Dv]: a segment's own state, then the one that enters it
  int64_t n_slots, L, N, seg_len;  // seg_len: tokens of a segment, a multiple of 64 (or >= every length)
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, o_st, o_sh;
  int64_t n_units;    // segments x heads
  int n_seg;          // segments of each sequence (dense)
  int Hq, Hk, Dk, Dv, S;
  int kp, vp, qp;     // panels of 64 channels that one load brings
  float scale;
  uint32_t max_polls;
  int32_t* err;
  int drop_load;      // test hook: CTA 0 skips its first load
};

struct Wait {
  uint32_t max_polls;
  int32_t* err;
  volatile int* abort;
};

// One lane waits.
__device__ __forceinline__ bool lane_wait(uint64_t* bar, uint32_t parity, int32_t site, const Wait& w) {
  for (uint32_t i = 0; i < w.max_polls; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 255u && *w.abort) return false;
  }
  atomicCAS(w.err, 0, site);
  *w.abort = 1;
  return false;
}
// A whole warp waits (uniform result).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int32_t site, const Wait& w) {
  for (uint32_t i = 0; i < w.max_polls; ++i) {
    if (__any_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if ((i & 255u) == 255u && __any_sync(0xffffffffu, *w.abort != 0)) return false;
  }
  if ((threadIdx.x & 31) == 0) {
    atomicCAS(w.err, 0, site);
    *w.abort = 1;
  }
  __syncwarp();
  return false;
}
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}
__device__ __forceinline__ void fence_async_shared() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void tma_load_4d(void* dst, const void* tmap, uint64_t* bar, int c0, int c1,
                                            int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
      "l"(tmap), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}

// 16 columns of an accumulator.  M = 128: lane = row of the warp's quarter.
// M = 64: the quarter's 16 rows sit in lanes 0-15; the upper half-warp takes
// the columns 32 further on.
template <int M>
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&r)[16]) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  if constexpr (M == 128) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]),
          "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]),
          "=r"(u[14]), "=r"(u[15])
        : "r"(taddr)
        : "memory");
  } else {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x32bx2.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16], 32;\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]),
          "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]),
          "=r"(u[14]), "=r"(u[15])
        : "r"(taddr)
        : "memory");
  }
}

// Descriptor of an operand whose contiguous axis is M or N: panels of 64
// elements (128 bytes, swizzled) `panel` bytes apart, tokens as rows.
__device__ __forceinline__ uint64_t make_smem_desc_mn(uint32_t saddr, uint32_t panel) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFFu) >> 4);
  d |= (uint64_t)((panel >> 4) & 0x3FFFu) << 16;  // between panels
  d |= (uint64_t)(1024 >> 4) << 32;               // between groups of 8 tokens
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

template <typename T>
__host__ __device__ constexpr uint32_t idesc(int M, int N, int a_mn, int b_mn) {
  return (1u << 4) | ((std::is_same<T, __half>::value ? 0u : 1u) << 7) |
         ((std::is_same<T, __half>::value ? 0u : 1u) << 10) | ((uint32_t)a_mn << 15) |
         ((uint32_t)b_mn << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

template <typename T>
struct Half2;
template <>
struct Half2<__half> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
  // nonzero if one of the two is an infinity or NaN
  static __device__ __forceinline__ uint32_t non_finite(uint32_t u) {
    return ((u & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
  }
};
template <>
struct Half2<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
  }
  static __device__ __forceinline__ uint32_t non_finite(uint32_t u) {
    return ((u & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
  }
};

// x (two values) as `parts` 16-bit parts, largest first.
template <typename T, int PARTS>
__device__ __forceinline__ void split2(float a, float b, uint32_t (&out)[PARTS]) {
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    out[p] = Half2<T>::pack(a, b);
    if (p + 1 < PARTS) {
      const float2 h = Half2<T>::unpack(out[p]);
      a -= h.x;
      b -= h.y;
    }
  }
}

// Exponent e for which 2^e brings a positive finite m into [2^14, 2^15).
__device__ __forceinline__ int fp16_shift(float m) {
  if (!(m > 0.f) || !isfinite(m)) return 0;
  const int e = 14 - ilogbf(m);
  return e > 120 ? 120 : (e < -120 ? -120 : e);
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((127 + e) << 23); }

// l^n for n >= 0; 0^0 = 1 (log2 decays below -1e4 are one that keeps nothing).
__device__ __forceinline__ float log2_decay(float log_decay) {
  const float l2 = log_decay * 1.4426950408889634f;
  return l2 < -1e4f ? -1e4f : l2;
}
// l^n as hi + lo, for the factor that a state meets chunk after chunk.
__device__ __forceinline__ float2 pow_hi_lo(float log_decay, int64_t n) {
  if (n == 0) return make_float2(1.f, 0.f);
  const double p = exp((double)log_decay * (double)n);
  const float hi = (float)p;
  return make_float2(hi, isfinite(hi) ? (float)(p - (double)hi) : 0.f);
}

template <typename T, int DK, int DV, bool OUT>
struct Cfg {
  static constexpr bool kFp16 = std::is_same<T, __half>::value;
  static constexpr int kVParts = kFp16 ? 2 : 3;
  static constexpr int kCg = DK / 64;          // state warps per lane quarter
  static constexpr int kStateWarps = 4 * kCg;
  static constexpr int kOutWarps = OUT ? 8 : 0;  // P warps, then O warps
  static constexpr int kWarps = kOutWarps + kStateWarps + 2;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kKBytes = DK / 64 * kTileBytes;
  static constexpr int kVBytes = DV / 64 * kTileBytes;
  static constexpr int kSPart = DV * DK * 2;
  static constexpr int kKvStages = OUT ? 2 : 3;
  static constexpr int kQStages = OUT ? 2 : 0;
  static constexpr int kVp = OUT ? 1 : 2;       // V' buffers
  static constexpr int kScaleBytes = (OUT && kFp16) ? 4096 : 0;
  static constexpr int kSmem = kKvStages * (kKBytes + kVBytes) + kQStages * kKBytes +
                               kVp * kVParts * kVBytes + kScaleBytes +
                               (OUT ? 2 * kSPart + 2 * kTileBytes : 0) + kSmallBytes;
  static constexpr int kCtas = (OUT && DK == 64 && DV == 64) ? 2 : 1;
  // TMEM columns: QK 64 | O from S 64 | O from P 64 | KV buffers
  static constexpr int kColOs = 64, kColOp = 128, kColKv = OUT ? 192 : 0;
  static constexpr int kColsUsed = kColKv + kVp * DK;
  static constexpr int kCols = kColsUsed <= 64 ? 64 : kColsUsed <= 128 ? 128 : kColsUsed <= 256 ? 256 : 512;
};

struct Unit {
  int64_t t0;
  int len, h, seq;
  const float* start;  // state that enters, NULL = zeros
  float* end;          // where the last state goes, or NULL
};

// Unit u of the grid (heads fastest).  Returns false if there is nothing in it.
template <bool OUT>
__device__ __forceinline__ bool get_unit(const DecayArgs& a, int64_t u, Unit& x) {
  const int64_t sg = u / a.Hk;
  x.h = (int)(u - sg * a.Hk);
  bool first, last;
  int64_t seg = sg;  // row of seg_states
  if (a.segs) {
    const Seg s = a.segs[sg];
    if (s.seq < 0) return false;
    x.seq = s.seq;
    x.t0 = s.t0;
    x.len = s.t1 - s.t0;
    last = s.last != 0;
    first = sg == 0 || a.segs[sg - 1].seq != s.seq;
  } else if (a.cu) {
    x.seq = (int)sg;
    x.t0 = min(max((int64_t)a.cu[sg], (int64_t)0), a.N);
    x.len = (int)(min(max((int64_t)a.cu[sg + 1], x.t0), a.N) - x.t0);
    first = last = true;
  } else {
    const int per = OUT ? a.n_seg : a.n_seg - 1;
    x.seq = (int)(sg / per);
    const int i = (int)(sg - (int64_t)x.seq * per);
    seg = (int64_t)x.seq * a.n_seg + i;
    const int64_t off = (int64_t)i * a.seg_len;
    x.t0 = x.seq * a.L + off;
    x.len = (int)min(a.seg_len, a.L - off);
    first = i == 0;
    last = i == a.n_seg - 1;
  }
  const int64_t dd = (int64_t)a.Dk * a.Dv;
  float* mine = a.seg_states + (seg * a.Hk + x.h) * dd;
  if (!OUT) {
    x.start = nullptr;
    x.end = mine;
    return !last;
  }
  const int64_t slot = a.slots ? a.slots[x.seq] : x.seq;
  const bool has_slot = slot >= 0 && slot < a.n_slots;
  const int64_t row = (slot * a.Hk + x.h) * dd;
  x.start = !first ? mine : (a.s_in && has_slot) ? a.s_in + row : nullptr;
  x.end = (last && a.s_out && has_slot) ? a.s_out + row : nullptr;
  return true;
}

template <typename T, int DK, int DV, bool OUT>
__global__ void __launch_bounds__(Cfg<T, DK, DV, OUT>::kThreads, Cfg<T, DK, DV, OUT>::kCtas)
    decay_chunk_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const __grid_constant__ DecayArgs a) {
  using K = Cfg<T, DK, DV, OUT>;
  constexpr bool FP16 = K::kFp16;
  constexpr int VP = K::kVp;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sK = smem;
  uint8_t* sV = sK + K::kKvStages * K::kKBytes;
  uint8_t* sQ = sV + K::kKvStages * K::kVBytes;
  uint8_t* sVp = sQ + K::kQStages * K::kKBytes;
  float* s_sscale = reinterpret_cast<float*>(sVp + VP * K::kVParts * K::kVBytes);  // fp16 only:
  float* s_pscale = s_sscale + 256;  // [2][128] S's scales by chunk parity, [2][64] P's by item parity,
  float* s_smax = s_pscale + 128;    // [2][2][128] maxima of half a channel of S
  uint8_t* sS = sVp + VP * K::kVParts * K::kVBytes + K::kScaleBytes;
  uint8_t* sP = sS + (OUT ? 2 * K::kSPart : 0);
  uint8_t* small = sP + (OUT ? 2 * kTileBytes : 0);
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(small);
  uint64_t* kv_empty = kv_full + 4;
  uint64_t* q_full = kv_empty + 4;
  uint64_t* q_empty = q_full + 4;
  uint64_t* vp_full = q_empty + 4;
  uint64_t* ds_full = vp_full + 2;
  uint64_t* qk_full = ds_full + 2;
  uint64_t* p_full = qk_full + 1;
  uint64_t* o_full = p_full + 1;
  uint64_t* o_empty = o_full + 1;
  uint64_t* s_full = o_empty + 1;
  uint64_t* s_empty = s_full + 1;
  uint64_t* p_sync = s_empty + 1;
  uint64_t* st_sync = p_sync + 1;
  uint64_t* done_bar = st_sync + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile uint32_t* s_badany = reinterpret_cast<volatile uint32_t*>(tmem_slot + 2);  // [3]
  float* s_vmax = reinterpret_cast<float*>(tmem_slot + 6);                    // [2][8] state warps
  float* s_pow = reinterpret_cast<float*>(small + 512);                       // [2][128]: l^{n - 63}
  // [3][DV]: chunk + 1 and, as 63 - j, the first token whose v is not finite in a
  // channel.  Three, since v of chunk c + 2 may be looked at while chunk c is put out.
  uint32_t* s_bad = reinterpret_cast<uint32_t*>(small + 1536);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Wait w{a.max_polls, a.err, abort_flag};
  const int G = a.Hq / a.Hk;
  (void)s_sscale, (void)s_pscale, (void)s_smax;

  if (smem_u32(smem) & 1023u) {  // the swizzle is by address: without this alignment nothing may run
    if (threadIdx.x == 0) atomicCAS(a.err, 0, ERR_SITE_DECAY_ALIGN);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&vp_full[i], K::kStateWarps);
      mbar_init(&ds_full[i], 1);
    }
    for (int i = 0; i < 3; ++i) s_badany[i] = 0;
    mbar_init(qk_full, 1);
    mbar_init(p_full, 4);
    mbar_init(o_full, 1);
    mbar_init(o_empty, 4);
    mbar_init(s_full, K::kStateWarps);
    mbar_init(s_empty, 1);
    mbar_init(p_sync, 4);
    mbar_init(st_sync, K::kStateWarps);
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  for (int i = threadIdx.x; i < 3 * DV; i += K::kThreads) s_bad[i] = 0;
  constexpr int kTmaWarp = K::kWarps - 2, kMmaWarp = K::kWarps - 1;
  if (warp == kTmaWarp && lane == 0) {
    if (OUT) prefetch_tmap(&tmQ);
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, K::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_wait();
  griddep_launch_dependents();
  const uint32_t tmem = *tmem_slot;

  if (warp == kTmaWarp) {
    // ------------------------------------------------------------ loads
    uint32_t cc = 0, it = 0;
    uint32_t kv_used = 0, q_used = 0;  // parity of each stage's last load, + 2 once there was one
    auto mark = [](uint32_t& used, int s, uint32_t parity) {
      used = (used & ~(3u << (2 * s))) | ((2u | parity) << (2 * s));
    };
    bool ok = true, drop = a.drop_load && blockIdx.x == 0;
    for (int64_t u = blockIdx.x; u < a.n_units && ok; u += gridDim.x) {
      Unit x;
      if (!get_unit<OUT>(a, u, x)) continue;
      for (int c = 0; c < x.len && ok; c += kC, ++cc) {
        const int st = cc % K::kKvStages;
        if (!(ok = warp_wait(&kv_empty[st], ((cc / K::kKvStages) & 1) ^ 1, ERR_SITE_DECAY_LOAD, w))) break;
        const int t = (int)(x.t0 + c);
        if (lane == 0 && !drop) {
          mbar_arrive_expect_tx(&kv_full[st], K::kKBytes + K::kVBytes);
          for (int p = 0; p < DK / 64; p += a.kp)
            tma_load_4d(sK + st * K::kKBytes + p * kTileBytes, &tmK, &kv_full[st], a.kp == 1 ? 64 * p : 0, t, 0, x.h);
          for (int p = 0; p < DV / 64; p += a.vp)
            tma_load_4d(sV + st * K::kVBytes + p * kTileBytes, &tmV, &kv_full[st], a.vp == 1 ? 64 * p : 0, t, 0, x.h);
        }
        if (!drop) mark(kv_used, st, (cc / K::kKvStages) & 1);
        drop = false;
        __syncwarp();
        if constexpr (OUT) {
          for (int g = 0; g < G; ++g, ++it) {
            const int qs = it % K::kQStages;
            if (!(ok = warp_wait(&q_empty[qs], ((it / K::kQStages) & 1) ^ 1, ERR_SITE_DECAY_LOAD, w))) break;
            if (lane == 0) {
              mbar_arrive_expect_tx(&q_full[qs], K::kKBytes);
              for (int p = 0; p < DK / 64; p += a.qp)
                tma_load_4d(sQ + qs * K::kKBytes + p * kTileBytes, &tmQ, &q_full[qs], a.qp == 1 ? 64 * p : 0, t, 0,
                            x.h * G + g);
            }
            mark(q_used, qs, (it / K::kQStages) & 1);
            __syncwarp();
          }
        }
      }
    }
    if (!ok) {
      // the loads in flight land before the CTA ends
      for (int s = 0; s < 4; ++s) {
        for (uint32_t i = 0; (kv_used >> (2 * s) & 2u) && i < (1u << 16); ++i)
          if (mbar_try_wait(&kv_full[s], kv_used >> (2 * s) & 1u)) break;
        for (uint32_t i = 0; (q_used >> (2 * s) & 2u) && i < (1u << 16); ++i)
          if (mbar_try_wait(&q_full[s], q_used >> (2 * s) & 1u)) break;
      }
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t kIdQk = idesc<T>(64, 64, 0, 0);
      constexpr uint32_t kIdKv = idesc<T>(DV, DK, 1, 1);
      constexpr uint32_t kIdQs = idesc<T>(DV, 64, 0, 0);
      constexpr uint32_t kIdPv = idesc<T>(DV, 64, 1, 0);
      const uint64_t dQ = make_smem_desc(smem_u32(sQ), 128);
      const uint64_t dKk = make_smem_desc(smem_u32(sK), 128);
      const uint64_t dKm = make_smem_desc_mn(smem_u32(sK), kTileBytes);
      const uint64_t dVm = make_smem_desc_mn(smem_u32(sV), kTileBytes);
      const uint64_t dVpm = make_smem_desc_mn(smem_u32(sVp), kTileBytes);
      const uint64_t dS = make_smem_desc(smem_u32(sS), 128);
      const uint64_t dP = make_smem_desc(smem_u32(sP), 128);
      const uint32_t dQk = tmem, dOs = tmem + K::kColOs, dOp = tmem + K::kColOp, dKv = tmem + K::kColKv;
      uint32_t cc = 0, it = 0, ns = 0;
      bool ok = true, qk_early = false;
      auto issue_qk = [&](uint32_t qs, uint32_t st) {
        uint64_t ad = dQ + (uint64_t)(qs * (K::kKBytes >> 4)), bd = dKk + (uint64_t)(st * (K::kKBytes >> 4));
#pragma unroll
        for (int p = 0; p < DK / 64; ++p)
#pragma unroll
          for (int s = 0; s < 4; ++s)
            umma_f16(dQk, ad + p * (kTileBytes >> 4) + s * 2, bd + p * (kTileBytes >> 4) + s * 2, kIdQk, p + s > 0);
        umma_commit(qk_full);
      };
      for (int64_t u = blockIdx.x; u < a.n_units && ok; u += gridDim.x) {
        Unit x;
        if (!get_unit<OUT>(a, u, x)) continue;
        for (int c = 0; c < x.len && ok; c += kC, ++cc) {
          const uint32_t st = cc % K::kKvStages;
          const uint32_t vb = cc % VP;
          if (!(ok = lane_wait(&kv_full[st], (cc / K::kKvStages) & 1, ERR_SITE_DECAY_MMA, w))) break;
          auto issue_kv = [&]() {
            const uint64_t ad = dVpm + (uint64_t)(vb * K::kVParts * (K::kVBytes >> 4));
            const uint64_t bd = dKm + (uint64_t)(st * (K::kKBytes >> 4));
#pragma unroll
            for (int p = K::kVParts - 1; p >= 0; --p)  // the small parts first
#pragma unroll
              for (int s = 0; s < 4; ++s)
                umma_f16(dKv + vb * DK, ad + p * (K::kVBytes >> 4) + s * 128, bd + s * 128, kIdKv,
                         p < K::kVParts - 1 || s > 0);
            umma_commit(&ds_full[vb]);
          };
          if constexpr (!OUT) {
            if (!(ok = lane_wait(&vp_full[vb], (cc / VP) & 1, ERR_SITE_DECAY_MMA, w))) break;
            tc_fence_after();
            issue_kv();
            umma_commit(&kv_empty[st]);
          } else {
            const bool has_s = c > 0 || x.start != nullptr;
            for (int g = 0; g < G; ++g, ++it) {
              const uint32_t qs = it % K::kQStages;
              if (!qk_early) {
                if (!(ok = lane_wait(&q_full[qs], (it / K::kQStages) & 1, ERR_SITE_DECAY_MMA, w))) break;
                tc_fence_after();
                issue_qk(qs, st);
              }
              qk_early = false;
              if (g == 0) {
                if (!(ok = lane_wait(&vp_full[vb], (cc / VP) & 1, ERR_SITE_DECAY_MMA, w))) break;
                tc_fence_after();
                issue_kv();
              }
              if (!(ok = lane_wait(o_empty, (it & 1) ^ 1, ERR_SITE_DECAY_MMA, w))) break;
              if (has_s) {
                if (g == 0 && !(ok = lane_wait(s_full, ns & 1, ERR_SITE_DECAY_MMA, w))) break;
                tc_fence_after();
                const uint64_t bd = dQ + (uint64_t)(qs * (K::kKBytes >> 4));
#pragma unroll
                for (int part = 1; part >= 0; --part)
#pragma unroll
                  for (int p = 0; p < DK / 64; ++p)
#pragma unroll
                    for (int s = 0; s < 4; ++s)
                      umma_f16(dOs, dS + part * (K::kSPart >> 4) + p * (DV * 128 >> 4) + s * 2,
                               bd + p * (kTileBytes >> 4) + s * 2, kIdQs, part < 1 || p + s > 0);
                if (g == G - 1) {
                  umma_commit(s_empty);
                  ++ns;
                }
              }
              if (!(ok = lane_wait(p_full, it & 1, ERR_SITE_DECAY_MMA, w))) break;
              tc_fence_after();
              // the next product with the queries, if its operands are there: it
              // runs while the P warps of this one are done and PV is under way
              {
                const uint32_t nq = (it + 1) % K::kQStages;
                const bool same = g + 1 < G;
                const uint32_t nst = same ? st : (cc + 1) % K::kKvStages;
                if ((same || c + kC < x.len) &&
                    mbar_test_wait(&q_full[nq], ((it + 1) / K::kQStages) & 1) &&
                    (same || mbar_test_wait(&kv_full[nst], ((cc + 1) / K::kKvStages) & 1))) {
                  issue_qk(nq, nst);
                  qk_early = true;
                }
              }
              const uint64_t ad = dVm + (uint64_t)(st * (K::kVBytes >> 4));
#pragma unroll
              for (int part = 1; part >= 0; --part)
#pragma unroll
                for (int s = 0; s < 4; ++s)
                  umma_f16(dOp, ad + s * 128, dP + part * (kTileBytes >> 4) + s * 2, kIdPv, part < 1 || s > 0);
              umma_commit(o_full);
              umma_commit(&q_empty[qs]);
              if (g == G - 1) umma_commit(&kv_empty[st]);
            }
          }
        }
      }
      umma_commit(done_bar);
      for (uint32_t p = 0; p < kMaxPolls; ++p)
        if (mbar_try_wait(done_bar, 0)) break;
    }
  } else if (OUT && warp < 4) {
    // ------------------------------------------------------------ QK -> P
    // Lane: row i = 16 warp + lane % 16, columns 32 (lane / 16) + 0..31.
    if constexpr (OUT) {
      uint32_t it = 0, nu = 0;
      bool ok = true;
      const int i = warp * 16 + (lane & 15), j0 = (lane >> 4) * 32;
      for (int64_t u = blockIdx.x; u < a.n_units && ok; u += gridDim.x) {
        Unit x;
        if (!get_unit<OUT>(a, u, x) || x.len == 0) continue;
        float* pw = s_pow + (nu & 1) * 128;
        for (int c = 0; c < x.len && ok; c += kC) {
          for (int g = 0; g < G; ++g, ++it) {
            if (!(ok = warp_wait(qk_full, it & 1, ERR_SITE_DECAY_P, w))) break;
            tc_fence_after();
            float r[32];
            {
              float(&lo)[16] = *reinterpret_cast<float(*)[16]>(&r[0]);
              float(&hi)[16] = *reinterpret_cast<float(*)[16]>(&r[16]);
              tmem_ld16<64>(tmem + ((uint32_t)(warp * 32) << 16), lo);
              tmem_ld16<64>(tmem + ((uint32_t)(warp * 32) << 16) + 16, hi);
            }
            tc_fence_before();
            // PV of the item before has read P, and the O warps the table two units back
            if (it > 0 && !(ok = warp_wait(o_full, (it - 1) & 1, ERR_SITE_DECAY_P, w))) break;
            if (c == 0 && g == 0) {
              const float l2 = log2_decay(a.log_decay[x.h]);
              const int n = threadIdx.x - 63;
              pw[threadIdx.x] = n < 0 ? 0.f : exp2f(l2 * (float)n);
              warp_arrive(p_sync);
              if (!(ok = warp_wait(p_sync, nu & 1, ERR_SITE_DECAY_P, w))) break;
            }
            const float* f = pw + 63 + i - j0;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float y = f[-j];
              r[j] = y != 0.f ? r[j] * y : 0.f;  // never 0 * inf: what is masked is not looked at
            }
            if constexpr (FP16) {
              float m = 0.f;
#pragma unroll
              for (int j = 0; j < 32; ++j) m = fmaxf(m, fabsf(r[j]));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
              const int e = fp16_shift(m);
              const float up = pow2i(e);
#pragma unroll
              for (int j = 0; j < 32; ++j) r[j] *= up;
              if (lane < 16) s_pscale[(it & 1) * 64 + i] = pow2i(-e);
            }
#pragma unroll
            for (int ch = 0; ch < 4; ++ch) {
              uint32_t p[4][2];
#pragma unroll
              for (int z = 0; z < 4; ++z) split2<T, 2>(r[ch * 8 + 2 * z], r[ch * 8 + 2 * z + 1], p[z]);
              const int off = i * 128 + (((j0 >> 3) + ch) ^ (i & 7)) * 16;
              *reinterpret_cast<uint4*>(sP + off) = make_uint4(p[0][0], p[1][0], p[2][0], p[3][0]);
              *reinterpret_cast<uint4*>(sP + kTileBytes + off) = make_uint4(p[0][1], p[1][1], p[2][1], p[3][1]);
            }
            fence_async_shared();
            warp_arrive(p_full);
          }
        }
        ++nu;
      }
    }
  } else if (OUT && warp < 8) {
    // ------------------------------------------------------------ outputs
    // DV = 128: lane = channel, all 64 tokens.  DV = 64: lane % 16 = channel,
    // tokens 32 (lane / 16) + 0..31.
    if constexpr (OUT) {
      uint32_t it = 0, cc = 0, nu = 0;
      bool ok = true;
      const int qd = warp & 3;
      const int dv = DV == 128 ? qd * 32 + lane : qd * 16 + (lane & 15);
      const int i0 = DV == 128 ? 0 : (lane >> 4) * 32;
      const uint32_t ta = tmem + ((uint32_t)(qd * 32) << 16);
      T* const out = static_cast<T*>(a.out);
      for (int64_t u = blockIdx.x; u < a.n_units && ok; u += gridDim.x) {
        Unit x;
        if (!get_unit<OUT>(a, u, x) || x.len == 0) continue;
        const float* pw = s_pow + (nu & 1) * 128 + 64;  // l^{i+1}
        for (int c = 0; c < x.len && ok; c += kC, ++cc) {
          const bool has_s = c > 0 || x.start != nullptr;
          const int n = min(kC, x.len - c);
          for (int g = 0; g < G; ++g, ++it) {
            if (!(ok = warp_wait(o_full, it & 1, ERR_SITE_DECAY_O, w))) break;
            tc_fence_after();
            T* const row = out + (x.t0 + c) * a.o_st + (int64_t)(x.h * G + g) * a.o_sh + dv;
            float ss = a.scale;
            if constexpr (FP16) ss *= s_sscale[(cc & 1) * 128 + dv];
            int bad = kC;  // first token of the chunk whose v is not finite in this channel
            if (s_badany[cc % 3] == cc + 1) {
              const uint32_t b = s_bad[(cc % 3) * DV + dv];
              if ((b >> 6) == cc + 1) bad = 63 - (int)(b & 63);
            }
            constexpr int NB = DV == 128 ? 4 : 2;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              float r[16], s[16];
              tmem_ld16<DV>(ta + K::kColOp + b * 16, r);
              if (has_s) tmem_ld16<DV>(ta + K::kColOs + b * 16, s);
              const int t = i0 + b * 16;
              float o[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                float pr = a.scale;
                if constexpr (FP16) pr *= s_pscale[(it & 1) * 64 + t + j];
                o[j] = pr * r[j];
                if (has_s) o[j] = fmaf(ss * pw[t + j], s[j], o[j]);
              }
              if (b == NB - 1) {
                tc_fence_before();
                warp_arrive(o_empty);
              }
              if (bad < kC) {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  if (t + j >= bad) o[j] = __int_as_float(0x7FFFFFFF);
              }
              if (dv < a.Dv) {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  if (t + j < n) row[(int64_t)(t + j) * a.o_st] = from_f<T>(o[j]);
              }
            }
          }
        }
        ++nu;
      }
    }
  } else {
    // ------------------------------------------------------------ state
    // Lane: channel dv as in the outputs, NC of the 64 dk columns of its group.
    constexpr int NC = DV == 128 ? 64 : 32;
    constexpr int NT = K::kStateWarps * 32;
    const int sw = warp - K::kOutWarps, stid = threadIdx.x - K::kOutWarps * 32;
    const int qd = sw & 3, cg = sw >> 2;
    // the warp's TMEM lanes are those of its number modulo 4
    const int dv = DV == 128 ? qd * 32 + lane : qd * 16 + (lane & 15);
    const int c0 = cg * 64 + (DV == 128 ? 0 : (lane >> 4) * 32);
    uint32_t cc = 0, ns = 0, nsync = 0;
    bool ok = true;
    const uint32_t ta = tmem + ((uint32_t)(qd * 32) << 16) + K::kColKv + cg * 64;
    float S[NC];

    // all state warps meet (bounded, as every wait)
    auto meet = [&]() -> bool {
      warp_arrive(st_sync);
      return warp_wait(st_sync, nsync++ & 1, ERR_SITE_DECAY_STATE, w);
    };
    // S^T as two 16-bit parts in shared memory, for the product with the queries
    auto put_s = [&](uint32_t chunk) -> bool {
      if constexpr (OUT) {
        float up = 1.f, undo = 1.f;
        if constexpr (FP16) {
          // the channel's largest entry sits in up to two warps and two half-warps
          float m = 0.f;
#pragma unroll
          for (int j = 0; j < NC; ++j) m = fmaxf(m, fabsf(S[j]));
          if (DV == 64) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
          float* mx = s_smax + (chunk & 1) * 256;
          if (K::kCg > 1) {
            mx[cg * 128 + dv] = m;
            if (!meet()) return false;
            m = fmaxf(mx[dv], mx[128 + dv]);
          }
          const int e = fp16_shift(m);
          up = pow2i(e);
          undo = pow2i(-e);
        }
        // the product with the S before it is done, so chunk - 2 has been put out
        if (!warp_wait(s_empty, (ns & 1) ^ 1, ERR_SITE_DECAY_STATE, w)) return false;
        if (FP16 && cg == 0) s_sscale[(chunk & 1) * 128 + dv] = undo;
        uint8_t* base = sS + (c0 >> 6) * (DV * 128) + dv * 128;
#pragma unroll
        for (int ch = 0; ch < NC / 8; ++ch) {
          uint32_t p[4][2];
#pragma unroll
          for (int z = 0; z < 4; ++z) split2<T, 2>(S[ch * 8 + 2 * z] * up, S[ch * 8 + 2 * z + 1] * up, p[z]);
          const int off = ((((c0 & 63) >> 3) + ch) ^ (dv & 7)) * 16;
          *reinterpret_cast<uint4*>(base + off) = make_uint4(p[0][0], p[1][0], p[2][0], p[3][0]);
          *reinterpret_cast<uint4*>(base + K::kSPart + off) = make_uint4(p[0][1], p[1][1], p[2][1], p[3][1]);
        }
        fence_async_shared();
        warp_arrive(s_full);
        ++ns;
      }
      return true;
    };
    // V' of chunk `chunk` (n tokens) into its buffer; returns fp16's power of two
    auto put_v = [&](uint32_t chunk, int n, float l2, float& down) -> bool {
      const uint32_t st = chunk % K::kKvStages;
      if (!warp_wait(&kv_full[st], (chunk / K::kKvStages) & 1, ERR_SITE_DECAY_STATE, w)) return false;
      uint8_t* v = sV + st * K::kVBytes;
      uint8_t* dst = sVp + (chunk % VP) * K::kVParts * K::kVBytes;
      constexpr int NV = K::kVBytes / 16 / NT;
      if (n < kC) {
        // tokens beyond the segment's end belong to others: zeros in their place
        uint8_t* k = sK + st * K::kKBytes;
        for (int e = stid; e < K::kKBytes / 16; e += NT)
          if (((e >> 3) & 63) >= n) *reinterpret_cast<uint4*>(k + e * 16) = make_uint4(0, 0, 0, 0);
      }
      uint4 raw[NV];
      uint32_t odd = 0, top = 0;
#pragma unroll
      for (int z = 0; z < NV; ++z) {
        const int e = stid + z * NT, j = (e >> 3) & 63;
        uint4 r = *reinterpret_cast<const uint4*>(v + e * 16);
        if (j >= n) {
          r = make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(v + e * 16) = r;
        }
        raw[z] = r;
        odd |= Half2<T>::non_finite(r.x) | Half2<T>::non_finite(r.y) | Half2<T>::non_finite(r.z) |
               Half2<T>::non_finite(r.w);
        if constexpr (FP16) {
          top = __vmaxu2(top, __vmaxu2(__vmaxu2(r.x & 0x7FFF7FFFu, r.y & 0x7FFF7FFFu),
                                       __vmaxu2(r.z & 0x7FFF7FFFu, r.w & 0x7FFF7FFFu)));
        }
      }
      if (odd) {
        // An infinity or NaN in v: zero in its place for PV, where earlier tokens
        // would meet it as 0 * inf; the O warps write NaN from its token on.
#pragma unroll
        for (int z = 0; z < NV; ++z) {
          const int e = stid + z * NT, j = (e >> 3) & 63;
          const int d0 = (e >> 9) * 64 + ((e & 7) ^ (j & 7)) * 8;
          uint32_t q[4] = {raw[z].x, raw[z].y, raw[z].z, raw[z].w};
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            const uint32_t half = (q[y >> 1] >> (16 * (y & 1))) & 0xFFFFu;
            if (Half2<T>::non_finite(half)) {
              q[y >> 1] &= (y & 1) ? 0x0000FFFFu : 0xFFFF0000u;
              atomicMax(&s_bad[(chunk % 3) * DV + d0 + y], ((chunk + 1) << 6) + (63 - j));
              s_badany[chunk % 3] = chunk + 1;
            }
          }
          *reinterpret_cast<uint4*>(v + e * 16) = make_uint4(q[0], q[1], q[2], q[3]);
        }
      }
      float up = 1.f;
      down = 1.f;
      if constexpr (FP16) {
        uint32_t m = max(top & 0xFFFFu, top >> 16);
        m = __reduce_max_sync(0xffffffffu, m);
        float* vm = s_vmax + (chunk & 1) * 8;
        if (lane == 0) vm[sw] = __half2float(__ushort_as_half((unsigned short)min(m, 0x7BFFu)));
        if (!meet()) return false;
        float f = 0.f;
#pragma unroll
        for (int z = 0; z < K::kStateWarps; ++z) f = fmaxf(f, vm[z]);
        const int e = fp16_shift(f);
        up = pow2i(e);
        down = pow2i(-e);
      }
#pragma unroll
      for (int z = 0; z < NV; ++z) {
        const int e = stid + z * NT, j = (e >> 3) & 63;
        const float f = j < n ? exp2f(l2 * (float)(n - 1 - j)) * up : 0.f;
        const uint32_t q[4] = {raw[z].x, raw[z].y, raw[z].z, raw[z].w};
        uint32_t p[4][K::kVParts];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float2 g = Half2<T>::unpack(q[y]);
          split2<T, K::kVParts>(g.x * f, g.y * f, p[y]);
        }
#pragma unroll
        for (int y = 0; y < K::kVParts; ++y)
          *reinterpret_cast<uint4*>(dst + y * K::kVBytes + e * 16) = make_uint4(p[0][y], p[1][y], p[2][y], p[3][y]);
      }
      fence_async_shared();
      warp_arrive(&vp_full[chunk % VP]);
      return true;
    };

    for (int64_t u = blockIdx.x; u < a.n_units && ok; u += gridDim.x) {
      Unit x;
      if (!get_unit<OUT>(a, u, x)) continue;
      const float ld = a.log_decay[x.h];
      const float l2 = log2_decay(ld);
      const int64_t at = (int64_t)c0 * a.Dv + dv;
#pragma unroll
      for (int j = 0; j < NC; ++j)
        S[j] = (x.start && dv < a.Dv && c0 + j < a.Dk) ? x.start[at + (int64_t)j * a.Dv] : 0.f;
      if (x.len > 0) {
        if (x.start && !(ok = put_s(cc))) break;
        float2 dec = pow_hi_lo(ld, min(kC, x.len));
        float down = 1.f, next = 1.f;  // fp16's power of two of this chunk's V' and the next's
        if (VP == 2 && !(ok = put_v(cc, min(kC, x.len), l2, next))) break;
        for (int c = 0; c < x.len; c += kC, ++cc) {
          const int n = min(kC, x.len - c);
          if (n < kC && c > 0) dec = pow_hi_lo(ld, n);
          if (VP == 1) {
            if (!(ok = put_v(cc, n, l2, down))) break;
          } else {
            down = next;
            if (c + kC < x.len && !(ok = put_v(cc + 1, min(kC, x.len - c - kC), l2, next))) break;
          }
          if (!(ok = warp_wait(&ds_full[cc % VP], (cc / VP) & 1, ERR_SITE_DECAY_STATE, w))) break;
          tc_fence_after();
#pragma unroll
          for (int b = 0; b < NC / 16; ++b) {
            float r[16];
            tmem_ld16<DV>(ta + (cc % VP) * DK + b * 16, r);
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              float& s = S[b * 16 + j];
              const float add = FP16 ? r[j] * down : r[j];
              s = fmaf(dec.x, s, fmaf(dec.y, s, add));
            }
          }
          tc_fence_before();
          if (OUT && c + kC < x.len && !(ok = put_s(cc + 1))) break;
        }
        if (!ok) break;
      }
      if (x.end && dv < a.Dv) {
#pragma unroll
        for (int j = 0; j < NC; ++j)
          if (c0 + j < a.Dk) x.end[at + (int64_t)j * a.Dv] = S[j];
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, K::kCols);
  }
}

}  // namespace decayk
}  // namespace cf
