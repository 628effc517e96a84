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
//   QS  [dv][64 i]      A = S^T,                B = Q (K-major)
//   PV  [dv][64 i]      A = V (MN-major),       B = P (K-major)    P_ij = l^{i-j} QK_ij, j <= i
// The outputs are built transposed (channels in lanes): with 64 tokens as M the
// same products run at half rate.  Channels are padded to 64 or 128 with the
// zeros that TMA fills in.  With 128 of them V' and S^T go to the products from
// TMEM: from shared memory, a chunk's 460 KB of tile writes and operand reads alone
// took 3600 cycles at its 128 bytes a cycle, against the 2850 in which HBM brings the
// chunk; from TMEM they are 220 KB.  With 64 channels an M = 64 product takes them
// from shared memory and two CTAs share the SM.
//
// What is rounded to 16 bits on its way through a product, and how: V' carries
// the state's precision, so it goes as three bf16 parts (24 bits) or two fp16
// parts (22 bits).  S and P reach only the 16-bit outputs and are rounded once,
// which makes the outputs' error 1.42 times that of their own rounding alone.
// In fp16 every row of V', S and P is scaled by a power of two of its own, so that
// neither a full state nor a small one leaves the type's range; bf16 has fp32's.  What lies
// far below its row's largest is held to 2^-39 of that: terms of V' below 2^-17, of S and P below
// 2^-28 of it.
//
// Warpgroups: P (QK -> P), O (outputs), S (state), V (V'; in the walk with 64 channels
// the S warps do it), and one with the TMA and the MMA warp.
//
// Measured on one B200 (2048 tokens of 148 sequences x heads, one of each a CTA, as graphs back
// to back; HBM floor at 6547 GB/s in brackets): bf16 128 x 128 channels 77 us (50), with four
// query heads a state 165 us (122), fp16 105 us (50); 296 of 64 x 64 channels, bf16 90 us,
// fp16 97 us (49).  A chunk takes 3000 cycles of the 2850 that HBM needs with
// 128 channels in bf16; the rest of the 77 us is the ends: launch, 64 KB of state in
// and out, the first chunk through a cold pipeline.  In fp16 the row scales lengthen
// the S and V roles by a third; with 64 channels the S warps' chain V' -> KV -> S
// takes 2700 a chunk and SM, where HBM would need 1430.  The roles wait for
// instructions and for each other more than for any pipe (tensor pipe 29 %, shared
// memory 14 %, a scheduler issues in 0.34 of its cycles).
#pragma once

#include "cf_half.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

namespace cf {
namespace decayk {

constexpr int kC = 64;            // tokens of a chunk
constexpr int kTileBytes = kC * 128;  // 64 tokens x 64 channels of 16 bits, 128-byte swizzle
constexpr int kSmallBytes = 4096;  // barriers and tables

enum : int32_t {
  ERR_SITE_DECAY_LOAD = 16,
  ERR_SITE_DECAY_MMA = 17,
  ERR_SITE_DECAY_P = 18,
  ERR_SITE_DECAY_O = 19,
  ERR_SITE_DECAY_STATE = 20,
  ERR_SITE_DECAY_V = 21,
  ERR_SITE_DECAY_ALIGN = 22,
};

struct Seg {  // one segment of one packed sequence
  int32_t t0, t1, seq, row_last;  // its row of seg_states (if the sequence is cut) * 2 + whether it is the last
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
  float* seg_states;  // [row][Hk][Dk][Dv]: a segment's own state, then the one that enters it
  int64_t n_slots, L, N, seg_len;  // seg_len: tokens of a segment, a multiple of 64 (or >= every length)
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, o_st, o_sh;
  uint32_t n_units;   // segments x heads, below 2^31
  int n_seg;          // segments of each sequence (dense)
  int Hq, Hk, Dk, Dv, S;
  int kp, vp, qp;     // panels of 64 channels that one load brings
  int o_vec;          // rows of out start on 16 bytes
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

// A whole warp waits (uniform result).  False: the limit ran out, or another role
// gave up; the role then leaves its loop and reports its site (give_up).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const Wait& w) {
  uint32_t i = w.max_polls;
#pragma unroll 1
  do {
    if (__any_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  } while (--i && !__any_sync(0xffffffffu, *w.abort != 0));
  return false;
}
__device__ __forceinline__ void give_up(int32_t site, const Wait& w) {
  if ((threadIdx.x & 31) == 0 && !*w.abort) {
    atomicCAS(w.err, 0, site);
    *w.abort = 1;
  }
}
__device__ __forceinline__ bool warp_test(uint64_t* bar, uint32_t parity) {
  return __any_sync(0xffffffffu, mbar_test_wait(bar, parity));
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

// Accumulator fragments.  One 16x256b load brings 16 lanes (rows) x 8 columns:
// thread t of the warp holds row t / 4, columns 2 (t % 4) and + 1, then row
// t / 4 + 8, the same columns; xN repeats that for the next columns.
__device__ __forceinline__ void tmem_ld_frag8(uint32_t taddr, float (&r)[32]) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]),
        "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]),
        "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]),
        "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]),
        "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(taddr)
      : "memory");
}
// 32 columns, without waiting; tmem_wait16 hands the registers over.
__device__ __forceinline__ void tmem_ld_frag4(uint32_t taddr, float (&r)[16]) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]),
        "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]),
        "=r"(u[14]), "=r"(u[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait16(float (&r)[16]) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(u[0]), "+r"(u[1]), "+r"(u[2]), "+r"(u[3]), "+r"(u[4]), "+r"(u[5]), "+r"(u[6]),
                 "+r"(u[7]), "+r"(u[8]), "+r"(u[9]), "+r"(u[10]), "+r"(u[11]), "+r"(u[12]), "+r"(u[13]),
                 "+r"(u[14]), "+r"(u[15])::"memory");
}
// 8 N columns of two accumulators (of the first alone if !both), one wait.
template <int N>
__device__ __forceinline__ void tmem_ld_pair(uint32_t ta, uint32_t tb, bool both, float (&x)[4 * N], float (&y)[4 * N]) {
  uint32_t* u = reinterpret_cast<uint32_t*>(x);
  uint32_t* v = reinterpret_cast<uint32_t*>(y);
  if constexpr (N == 4) {
    tmem_ld_frag4(ta, x);
    if (both) tmem_ld_frag4(tb, y);
    tmem_wait16(x);
    tmem_wait16(y);
  } else {
#define CF_LD8(R, A)                                                                                              \
  asm volatile(                                                                                                   \
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "                                                                   \
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"                                                   \
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"                                  \
      : "=r"(R[0]), "=r"(R[1]), "=r"(R[2]), "=r"(R[3]), "=r"(R[4]), "=r"(R[5]), "=r"(R[6]), "=r"(R[7]),           \
        "=r"(R[8]), "=r"(R[9]), "=r"(R[10]), "=r"(R[11]), "=r"(R[12]), "=r"(R[13]), "=r"(R[14]), "=r"(R[15]),     \
        "=r"(R[16]), "=r"(R[17]), "=r"(R[18]), "=r"(R[19]), "=r"(R[20]), "=r"(R[21]), "=r"(R[22]), "=r"(R[23]),   \
        "=r"(R[24]), "=r"(R[25]), "=r"(R[26]), "=r"(R[27]), "=r"(R[28]), "=r"(R[29]), "=r"(R[30]), "=r"(R[31])    \
      : "r"(A)                                                                                                    \
      : "memory")
#define CF_WAIT16(R, O, S)                                                                                        \
  asm volatile(S : "+r"(R[O]), "+r"(R[O + 1]), "+r"(R[O + 2]), "+r"(R[O + 3]), "+r"(R[O + 4]), "+r"(R[O + 5]),    \
                   "+r"(R[O + 6]), "+r"(R[O + 7]), "+r"(R[O + 8]), "+r"(R[O + 9]), "+r"(R[O + 10]),               \
                   "+r"(R[O + 11]), "+r"(R[O + 12]), "+r"(R[O + 13]), "+r"(R[O + 14]), "+r"(R[O + 15])::"memory")
    CF_LD8(u, ta);
    if (both) CF_LD8(v, tb);
    CF_WAIT16(u, 0, "tcgen05.wait::ld.sync.aligned;");
    CF_WAIT16(u, 16, "");
    CF_WAIT16(v, 0, "");
    CF_WAIT16(v, 16, "");
#undef CF_LD8
#undef CF_WAIT16
  }
}
// 16 rows x 32 words of a packed 16-bit operand: thread t holds row t / 4, word
// t % 4 of every four, then row t / 4 + 8 (the fragment above, packed in pairs).
__device__ __forceinline__ void tmem_st_frag8(uint32_t taddr, const uint32_t (&u)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%16], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(u[0]),
      "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]),
      "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Four 8x8 blocks of 16-bit values; lane 8 m + r gives the address of row r of
// block m.  A thread's registers are the fragment above; `_t`: transposed.
__device__ __forceinline__ void stm4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b),
               "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ void stm4_t(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a),
               "r"(b), "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ void ldm4_t(uint32_t addr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(a), "=r"(b), "=r"(c), "=r"(d)
               : "r"(addr)
               : "memory");
}

// The MMA warp runs its loop with all lanes and one of them issues (`one`): in a
// single lane's branch the compiler cannot keep descriptors in uniform registers,
// and moving them there took 100 cycles a product.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t e;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(e));
  return e;
}
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }
// D[tmem] (+)= A[smem] * B[smem]^T.
__device__ __forceinline__ void mma_ss(uint32_t one, uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(one)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]^T.
__device__ __forceinline__ void mma_ts(uint32_t one, uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(one)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t one, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "setp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(one)
      : "memory");
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
__device__ __forceinline__ F2 sub2(F2 a, F2 b) { return fma2(b, pack2(-1.f, -1.f), a); }

// Registers move between warpgroups: the sum stays within the launch's share.
template <int N>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
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
  static __device__ __forceinline__ uint32_t pack(F2 v) {
    float a, b;
    unpack2(v, a, b);
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ F2 unpack(uint32_t u) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
    return pack2(f.x, f.y);
  }
  static constexpr uint32_t kInf = 0x7C00;
};
template <>
struct Half2<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(F2 v) {
    float a, b;
    unpack2(v, a, b);
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ F2 unpack(uint32_t u) {
    return pack2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
  }
  static constexpr uint32_t kInf = 0x7F80;
};

// Two values as PARTS 16-bit parts each, largest first.
template <typename T, int PARTS>
__device__ __forceinline__ void split2(F2 a, uint32_t (&out)[PARTS]) {
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    out[p] = Half2<T>::pack(a);
    if (p + 1 < PARTS) a = sub2(a, Half2<T>::unpack(out[p]));
  }
}

// Exponent e for which 2^e brings a positive finite m into [2^14, 2^15).
__device__ __forceinline__ int fp16_shift(float m) {
  if (!(m > 0.f) || !isfinite(m)) return 0;
  const int e = 14 - ilogbf(m);
  return e > 120 ? 120 : (e < -120 ? -120 : e);
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((127 + e) << 23); }

__device__ __forceinline__ float exp2_fast(float x) {  // within 2^-22, and 1 at 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// l^n for n >= 0; 0^0 = 1 (log2 decays below -1e4 are one that keeps nothing).
__device__ __forceinline__ float log2_decay(float log_decay) {
  const float l2 = log_decay * 1.4426950408889634f;
  return l2 < -1e4f ? -1e4f : l2;
}
// The factors of V' reach the state: l^d for 0 <= d < 64 within 2^-21.  log2(l) stands as
// hi + lo, since one rounding of an exponent near 100 alone is 2^-18 of the power.
__device__ __forceinline__ float2 log2_decay_hi_lo(float log_decay) {
  const float hi = log_decay * 1.4426950408889634f;
  if (!(hi >= -1e4f)) return make_float2(hi < -1e4f ? -1e4f : hi, 0.f);
  return make_float2(hi, fmaf(log_decay, 1.925963e-8f, fmaf(log_decay, 1.4426950408889634f, -hi)));
}
__device__ __forceinline__ float decay_power(float2 l2, float d) {
  const float x = l2.x * d, rest = fmaf(l2.y, d, fmaf(l2.x, d, -x));
  const float p = exp2_fast(x);
  return fmaf(p, rest * 0.69314718f, p);
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
  static constexpr bool kTm = DV == 128;       // V' and S^T in TMEM, V' by warps of its own
  static constexpr int kHalves = DV / 64;      // 16-row halves of a warp's lanes
  static constexpr int kCg = DK / 64;          // groups of 64 state columns
  // warpgroups
  static constexpr int kP = 0, kO = OUT ? 1 : -1, kS = OUT ? 2 : 0, kV = (kTm || !OUT) ? kS + 1 : kS;
  static constexpr int kCtl = kV + 1;
  static constexpr int kThreads = 128 * (kCtl + 1);
  static constexpr int kCtas = DV == 64 && DK == 64 ? 2 : 1;
  static constexpr int kKBytes = DK / 64 * kTileBytes;
  static constexpr int kVBytes = DV / 64 * kTileBytes;
  static constexpr int kSPart = DV * DK * 2;
  static constexpr int kVp = OUT ? 1 : 2;  // V' and KV buffers
  // Chunks whose V' scales (fp16) are held.  V writes those of chunk c before it waits for a
  // buffer of V': KV of chunk c - kVp - 1 is done by then, so S has let go of the accumulator
  // of c - 2 kVp - 1, but may still read its last scales.  That takes 2 kVp + 2 slots.
  static constexpr int kVScales = OUT ? 4 : 8;
  static_assert(kVScales >= 2 * kVp + 2, "slots of V' scales");
  static constexpr int kKvStages = kCtas == 1 ? 4 : OUT ? 2 : 3;
  static constexpr int kQStages = OUT ? (kCtas > 1 ? 2 : 4) : 0;
  static constexpr int kScaleBytes = kFp16 ? 4096 : 0;
  static constexpr int kVpBytes = kTm ? 0 : kVp * kVParts * kVBytes;
  static constexpr int kSBytes = (OUT && !kTm) ? kSPart : 0;
  static constexpr int kStage = OUT ? kC * DV * 2 : 0;  // outputs on their way out
  static constexpr int kSmem = kKvStages * (kKBytes + kVBytes) + kQStages * kKBytes + kVpBytes + kSBytes +
                               (OUT ? kTileBytes : 0) + kStage + kScaleBytes + kSmallBytes;
  // TMEM columns: QK 64 | O from S 64 | O from P 64 | KV | S | V'
  static constexpr int kColOs = 64, kColOp = 128, kColKv = OUT ? 192 : 0;
  static constexpr int kColS = kColKv + kVp * DK;
  static constexpr int kColV = kColS + ((OUT && kTm) ? DK / 2 : 0);
  static constexpr int kColsUsed = kColV + (kTm ? kVp * kVParts * 32 : 0);
  static constexpr int kCols = kColsUsed <= 64 ? 64 : kColsUsed <= 128 ? 128 : kColsUsed <= 256 ? 256 : 512;
  // Registers of each warpgroup where the launch's even share does not do
  // (threads x registers at launch, over 128: 5 x 96 and 4 x 64).
  static constexpr bool kMove = OUT && (kTm || kCtas == 2);
  static constexpr int kRegP = kTm ? 96 : 80, kRegO = kTm ? (kFp16 ? 112 : 96) : 64, kRegS = kTm ? 168 : 88,
                       kRegV = kFp16 ? 80 : 96, kRegCtl = 24;
  static_assert(!kMove || kRegP + kRegO + kRegS + kRegCtl + (kTm ? kRegV : 0) <= (kTm ? 5 * 96 : 4 * 64), "registers");
};

struct Unit {
  int64_t t0;
  int len, h, seq;
  const float* start;  // state that enters, NULL = zeros
  float* end;          // where the last state goes, or NULL
};

// Unit u of the grid (heads fastest).  Returns false if there is nothing in it.
template <bool OUT>
__device__ __forceinline__ bool get_unit(const DecayArgs& a, uint32_t u, Unit& x) {
  const uint32_t sg = u / (uint32_t)a.Hk;
  x.h = (int)(u - sg * (uint32_t)a.Hk);
  bool first, last;
  int64_t seg = sg;  // row of seg_states
  if (a.segs) {
    const Seg s = a.segs[sg];
    if (s.seq < 0) return false;
    x.seq = s.seq;
    x.t0 = s.t0;
    x.len = s.t1 - s.t0;
    seg = s.row_last >> 1;
    last = s.row_last & 1;
    first = sg == 0 || a.segs[sg - 1].seq != s.seq;
  } else if (a.cu) {
    x.seq = (int)sg;
    x.t0 = min(max((int64_t)a.cu[sg], (int64_t)0), a.N);
    x.len = (int)(min(max((int64_t)a.cu[sg + 1], x.t0), a.N) - x.t0);
    first = last = true;
  } else {
    const uint32_t per = OUT ? a.n_seg : a.n_seg - 1;
    x.seq = (int)(sg / per);
    const int i = (int)(sg - x.seq * per);
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
  // Where s_out is s_in, a sequence's last segment may be done before its first
  // begins: several segments all start from their own copies.
  const bool carried = a.s_in && has_slot;
  x.start = !first || (carried && !last) ? mine : carried ? a.s_in + row : nullptr;
  x.end = (last && a.s_out && has_slot) ? a.s_out + row : nullptr;
  return true;
}

// The infinities and NaN among n channels of a tile of v: zeros in their place,
// where PV would meet them as 0 * inf for earlier tokens; the O warps write NaN
// from their token on.
template <typename T>
__device__ __forceinline__ void mark_non_finite(uint8_t* v, int d0, int n, uint32_t chunk, uint32_t* bad,
                                                volatile uint32_t* any) {
#pragma unroll 1
  for (int e = threadIdx.x & 31; e < kC * n; e += 32) {
    const int j = e / n, d = d0 + e % n;
    uint16_t* at = reinterpret_cast<uint16_t*>(v + (d >> 6) * kTileBytes + j * 128 +
                                               ((((d & 63) >> 3) ^ (j & 7)) << 4) + (d & 7) * 2);
    if ((*at & 0x7FFFu) >= Half2<T>::kInf) {
      *at = 0;
      atomicMax(&bad[d], ((chunk + 1) << 6) + (63 - j));
      *any = chunk + 1;
    }
  }
  fence_async_shared();
}

// A warp's part of a chunk's outputs on its way out: kRow bytes of each token,
// 16-byte vectors spread over all banks.
template <int kRow>
__device__ __forceinline__ int out_at(int row, int v) {
  return row * kRow + ((v ^ ((row / (128 / kRow)) & (kRow / 16 - 1))) << 4);
}
template <int kRow>
__device__ __forceinline__ void spoil_outputs(uint8_t* stage, const uint32_t* bad, uint32_t chunk) {
  __syncwarp();
#pragma unroll 1
  for (int e = threadIdx.x & 31; e < kC * kRow / 2; e += 32) {
    const int row = e / (kRow / 2), d = e % (kRow / 2);
    const uint32_t b = bad[d];
    if ((b >> 6) == chunk + 1 && row >= 63 - (int)(b & 63))
      *reinterpret_cast<uint16_t*>(stage + out_at<kRow>(row, d >> 3) + (d & 7) * 2) = 0x7FFF;
  }
}
template <typename T, int kRow>
__device__ __forceinline__ void store_unaligned(const uint8_t* stage, T* to, int64_t st, int rows, int channels) {
#pragma unroll 1
  for (int e = threadIdx.x & 31; e < rows * (kRow / 2); e += 32) {
    const int row = e / (kRow / 2), d = e % (kRow / 2);
    if (d < channels)
      to[(int64_t)row * st + d] = *reinterpret_cast<const T*>(stage + out_at<kRow>(row, d >> 3) + (d & 7) * 2);
  }
}

template <typename T, int DK, int DV, bool OUT>
__global__ void __launch_bounds__(Cfg<T, DK, DV, OUT>::kThreads, Cfg<T, DK, DV, OUT>::kCtas)
    decay_chunk_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const __grid_constant__ DecayArgs a) {
  using K = Cfg<T, DK, DV, OUT>;
  constexpr bool FP16 = K::kFp16, TM = K::kTm;
  constexpr int VP = K::kVp, NH = K::kHalves;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sK = smem;
  uint8_t* sV = sK + K::kKvStages * K::kKBytes;
  uint8_t* sQ = sV + K::kKvStages * K::kVBytes;
  uint8_t* sVp = sQ + K::kQStages * K::kKBytes;
  uint8_t* sS = sVp + K::kVpBytes;
  uint8_t* sP = sS + K::kSBytes;
  uint8_t* sOut = sP + (OUT ? kTileBytes : 0);
  float* s_sscale = reinterpret_cast<float*>(sOut + K::kStage);  // fp16 only: [2][128] S's scales by put,
  float* s_pscale = s_sscale + (OUT ? 256 : 0);                  // [2][64] P's by item (both in the walk),
  float* s_vscale = s_pscale + (OUT ? 128 : 0);                  // [kVScales][128] V's by chunk
  static_assert(!FP16 || ((OUT ? 384 : 0) + K::kVScales * 128) * 4 <= K::kScaleBytes, "scales");
  constexpr uint32_t kVMask = K::kVScales - 1;
  uint8_t* small = sOut + K::kStage + K::kScaleBytes;
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(small);
  uint64_t* kv_empty = kv_full + 4;
  uint64_t* q_full = kv_empty + 4;
  uint64_t* q_empty = q_full + 4;
  uint64_t* vp_full = q_empty + 4;
  uint64_t* ds_full = vp_full + 2;
  uint64_t* ds_empty = ds_full + 2;
  uint64_t* qk_full = ds_empty + 2;
  uint64_t* p_full = qk_full + 1;
  uint64_t* p_empty = p_full + 1;
  uint64_t* o_full = p_empty + 1;
  uint64_t* o_empty = o_full + 1;
  uint64_t* s_full = o_empty + 1;
  uint64_t* s_empty = s_full + 1;
  uint64_t* done_bar = s_empty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile uint32_t* s_badany = reinterpret_cast<volatile uint32_t*>(tmem_slot + 2);  // [4]
  // [4][DV]: chunk + 1 and, as 63 - j, the first token whose v is not finite in a
  // channel.  More than one, since v is looked at ahead of the outputs.
  uint32_t* s_bad = reinterpret_cast<uint32_t*>(small + 512);

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int wg = warp >> 2, wq = warp & 3;  // warpgroup; the warp's TMEM lanes are 32 wq ..
  const Wait w{a.max_polls, a.err, abort_flag};
  const int G = a.Hq / a.Hk;
  (void)s_sscale, (void)s_pscale, (void)s_vscale;

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
      s_badany[i] = 0;
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&vp_full[i], 4);
      mbar_init(&ds_full[i], 1);
      mbar_init(&ds_empty[i], 4);
    }
    mbar_init(qk_full, 1);
    mbar_init(p_full, 4);
    mbar_init(p_empty, 1);
    mbar_init(o_full, 1);
    mbar_init(o_empty, 4);
    mbar_init(s_full, 4);
    mbar_init(s_empty, 1);
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  for (int i = threadIdx.x; i < 4 * DV; i += K::kThreads) s_bad[i] = 0;
  constexpr int kTmaWarp = K::kCtl * 4, kMmaWarp = kTmaWarp + 1;
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
  const uint32_t tlane = tmem + ((uint32_t)(wq * 32) << 16);
  const int fr = lane >> 2, fc = (lane & 3) * 2;  // a fragment's row and first column

  if (wg == K::kCtl) {
    if constexpr (K::kMove) regs_down<K::kRegCtl>();
    if (warp == kTmaWarp) {
      // ---------------------------------------------------------- loads
      uint32_t cc = 0, it = 0;
      uint32_t kv_used = 0, q_used = 0;  // parity of each stage's last load, + 2 once there was one
      auto mark = [](uint32_t& used, int s, uint32_t parity) {
        used = (used & ~(3u << (2 * s))) | ((2u | parity) << (2 * s));
      };
      bool ok = true, drop = a.drop_load && blockIdx.x == 0;
      for (uint32_t u = blockIdx.x; u < a.n_units && ok; u += gridDim.x) {
        Unit x;
        if (!get_unit<OUT>(a, u, x)) continue;
        for (int c = 0; c < x.len && ok; c += kC, ++cc) {
          const int st = cc % K::kKvStages;
          if (!(ok = warp_wait(&kv_empty[st], ((cc / K::kKvStages) & 1) ^ 1, w))) break;
          const int t = (int)(x.t0 + c);
          if (lane == 0 && !drop) {
            mbar_arrive_expect_tx(&kv_full[st], K::kKBytes + K::kVBytes);
            for (int p = 0; p < DK / 64; p += a.kp)
              tma_load_4d(sK + st * K::kKBytes + p * kTileBytes, &tmK, &kv_full[st], a.kp == 1 ? 64 * p : 0, t, 0,
                          x.h);
            for (int p = 0; p < DV / 64; p += a.vp)
              tma_load_4d(sV + st * K::kVBytes + p * kTileBytes, &tmV, &kv_full[st], a.vp == 1 ? 64 * p : 0, t, 0,
                          x.h);
          }
          if (!drop) mark(kv_used, st, (cc / K::kKvStages) & 1);
          drop = false;
          __syncwarp();
          if constexpr (OUT) {
            for (int g = 0; g < G; ++g, ++it) {
              const int qs = it % K::kQStages;
              if (!(ok = warp_wait(&q_empty[qs], ((it / K::kQStages) & 1) ^ 1, w))) break;
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
        give_up(ERR_SITE_DECAY_LOAD, w);
        // the loads in flight land before the CTA ends
        for (int s = 0; s < 4; ++s) {
          for (uint32_t i = 0; (kv_used >> (2 * s) & 2u) && i < (1u << 16); ++i)
            if (mbar_try_wait(&kv_full[s], kv_used >> (2 * s) & 1u)) break;
          for (uint32_t i = 0; (q_used >> (2 * s) & 2u) && i < (1u << 16); ++i)
            if (mbar_try_wait(&q_full[s], q_used >> (2 * s) & 1u)) break;
        }
      }
    } else if (warp == kMmaWarp) {
      // ---------------------------------------------------------- MMA issuer
      // Per chunk: KV, then for each query head PV, the next head's QK as soon
      // as its operands are there, and QS.  P and V' of a chunk are ready early
      // (QK of it ran in the chunk before), S last.
      constexpr uint32_t kIdQk = idesc<T>(64, 64, 0, 0);
      constexpr uint32_t kIdKv = idesc<T>(DV, DK, TM ? 0 : 1, 1);
      constexpr uint32_t kIdQs = idesc<T>(DV, 64, 0, 0);
      constexpr uint32_t kIdPv = idesc<T>(DV, 64, 1, 0);
      const uint64_t dQ = make_smem_desc(smem_u32(sQ), 128);
      const uint64_t dKk = make_smem_desc(smem_u32(sK), 128);
      const uint64_t dKm = make_smem_desc_mn(smem_u32(sK), kTileBytes);
      const uint64_t dVm = make_smem_desc_mn(smem_u32(sV), kTileBytes);
      const uint64_t dVpm = make_smem_desc_mn(smem_u32(sVp), kTileBytes);
      const uint64_t dS = make_smem_desc(smem_u32(sS), 128);
      const uint64_t dP = make_smem_desc(smem_u32(sP), 128);
      const uint32_t one = elect_one();
      const uint32_t tm = uniform(tmem);
      uint32_t cc = 0, it = 0, ns = 0;
      bool ok = true, qk_early = false;
      auto issue_qk = [&](uint32_t qs, uint32_t st) {
        const uint64_t ad = dQ + (uint64_t)(qs * (K::kKBytes >> 4)), bd = dKk + (uint64_t)(st * (K::kKBytes >> 4));
#pragma unroll 1
        for (int p = 0; p < DK / 64; ++p)
#pragma unroll
          for (int s = 0; s < 4; ++s)
            mma_ss(one, tm, ad + p * (kTileBytes >> 4) + s * 2, bd + p * (kTileBytes >> 4) + s * 2, kIdQk, p + s > 0);
        mma_commit(one, qk_full);
      };
      for (uint32_t u = blockIdx.x; u < a.n_units && ok; u += gridDim.x) {
        Unit x;
        if (!get_unit<OUT>(a, u, x)) continue;
        const int len = uniform(x.len), started = uniform(x.start != nullptr);
        for (int c = 0; c < len && ok; c += kC, ++cc) {
          const uint32_t st = cc % K::kKvStages;
          const uint32_t vb = cc % VP;
          if (!(ok = warp_wait(&kv_full[st], (cc / K::kKvStages) & 1, w))) break;
          if constexpr (OUT) {
            if (!qk_early) {
              const uint32_t qs = it % K::kQStages;
              if (!(ok = warp_wait(&q_full[qs], (it / K::kQStages) & 1, w))) break;
              tc_fence_after();
              issue_qk(qs, st);
            }
            qk_early = false;
          }
          if (!(ok = warp_wait(&vp_full[vb], (cc / VP) & 1, w))) break;
          if (!(ok = warp_wait(&ds_empty[vb], ((cc / VP) & 1) ^ 1, w))) break;
          tc_fence_after();
          {
            const uint64_t ad = dVpm + (uint64_t)(vb * K::kVParts * (K::kVBytes >> 4));
            const uint32_t at = tm + K::kColV + vb * K::kVParts * 32;
            const uint64_t bd = dKm + (uint64_t)(st * (K::kKBytes >> 4));
            const uint32_t d = tm + K::kColKv + vb * DK;
#pragma unroll 1
            for (int p = K::kVParts - 1; p >= 0; --p)  // the small parts first
#pragma unroll
              for (int s = 0; s < 4; ++s) {
                const uint32_t acc = p < K::kVParts - 1 || s > 0;
                if constexpr (TM) mma_ts(one, d, at + p * 32 + s * 8, bd + s * 128, kIdKv, acc);
                else mma_ss(one, d, ad + p * (K::kVBytes >> 4) + s * 128, bd + s * 128, kIdKv, acc);
              }
            mma_commit(one, &ds_full[vb]);
          }
          if constexpr (!OUT) {
            mma_commit(one, &kv_empty[st]);
          } else {
            const bool has_s = c > 0 || started;
            for (int g = 0; g < G; ++g, ++it) {
              const uint32_t qs = it % K::kQStages;
              if (!(ok = warp_wait(p_full, it & 1, w))) break;
              if (!(ok = warp_wait(o_empty, (it & 1) ^ 1, w))) break;
              tc_fence_after();
              {
                const uint64_t ad = dVm + (uint64_t)(st * (K::kVBytes >> 4));
#pragma unroll
                for (int s = 0; s < 4; ++s)
                  mma_ss(one, tm + K::kColOp, ad + s * 128, dP + s * 2, kIdPv, s > 0);
                mma_commit(one, p_empty);
              }
              // QK's accumulator is free: P of this head is written
              const bool same = g + 1 < G;
              const uint32_t nq = (it + 1) % K::kQStages;
              const uint32_t nst = same ? st : (cc + 1) % K::kKvStages;
              if (same && !(ok = warp_wait(&q_full[nq], ((it + 1) / K::kQStages) & 1, w))) break;
              if (same || (c + kC < len && warp_test(&q_full[nq], ((it + 1) / K::kQStages) & 1) &&
                           warp_test(&kv_full[nst], ((cc + 1) / K::kKvStages) & 1))) {
                issue_qk(nq, nst);
                qk_early = !same;
              }
              if (!same) mma_commit(one, &kv_empty[st]);
              if (has_s) {
                if (g == 0 && !(ok = warp_wait(s_full, ns & 1, w))) break;
                tc_fence_after();
                const uint64_t bd = dQ + (uint64_t)(qs * (K::kKBytes >> 4));
#pragma unroll 1
                for (int p = 0; p < DK / 64; ++p)
#pragma unroll
                  for (int s = 0; s < 4; ++s) {
                    const uint64_t b = bd + p * (kTileBytes >> 4) + s * 2;
                    if constexpr (TM) mma_ts(one, tm + K::kColOs, tm + K::kColS + p * 32 + s * 8, b, kIdQs, p + s > 0);
                    else mma_ss(one, tm + K::kColOs, dS + p * (DV * 128 >> 4) + s * 2, b, kIdQs, p + s > 0);
                  }
                if (!same) {
                  mma_commit(one, s_empty);
                  ++ns;
                }
              }
              mma_commit(one, o_full);
              mma_commit(one, &q_empty[qs]);
            }
          }
        }
      }
      if (!ok) give_up(ERR_SITE_DECAY_MMA, w);
      mma_commit(one, done_bar);
      for (uint32_t p = 0; p < kMaxPolls; ++p)
        if (mbar_try_wait(done_bar, 0)) break;
    }
  } else if (OUT && wg == K::kP) {
    // ------------------------------------------------------------ QK -> P
    // Rows i = 16 wq + fr and + 8, columns j = 8 n + fc and + 1.
    if constexpr (K::kMove) {
      if constexpr (K::kRegP > (TM ? 96 : 64)) regs_up<K::kRegP>();
    }
    if constexpr (OUT) {
      uint32_t it = 0;
      bool ok = true;
      const int i = wq * 16 + fr;
      // where the lane's row of an 8x8 block goes: block m = lane / 8 holds rows
      // 8 (m % 2).., columns 8 (m / 2)..
      const int si = wq * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
      const uint32_t prow = smem_u32(sP) + si * 128;
      for (uint32_t u = blockIdx.x; u < a.n_units && ok; u += gridDim.x) {
        Unit x;
        if (!get_unit<OUT>(a, u, x) || x.len == 0) continue;
        const float l2 = log2_decay(a.log_decay[x.h]);
        F2 f[8][2];  // scale l^{i-j}, 0 above the diagonal
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int d = i + 8 * r - 8 * n - fc;
            f[n][r] = pack2(d < 0 ? 0.f : a.scale * exp2_fast(l2 * (float)d),
                            d < 1 ? 0.f : a.scale * exp2_fast(l2 * (float)(d - 1)));
          }
        const int items = (x.len + kC - 1) / kC * G;
        for (int k = 0; k < items; ++k, ++it) {
          if (!(ok = warp_wait(qk_full, it & 1, w))) break;
          tc_fence_after();
          float q[32];
          tmem_ld_frag8(tlane, q);
          tc_fence_before();
#pragma unroll
          for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const F2 y = mul2(pack2(q[4 * n + 2 * r], q[4 * n + 2 * r + 1]), f[n][r]);
              unpack2(y, q[4 * n + 2 * r], q[4 * n + 2 * r + 1]);
              // above the diagonal 0 * inf must not appear
              if (i - fc < 8 * n - 8 * r) q[4 * n + 2 * r] = 0.f;
              if (i - fc < 8 * n - 8 * r + 1) q[4 * n + 2 * r + 1] = 0.f;
            }
          float undo[2] = {1.f, 1.f};
          if constexpr (FP16) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              float m = 0.f;
#pragma unroll
              for (int n = 0; n < 8; ++n) m = fmaxf(m, fmaxf(fabsf(q[4 * n + 2 * r]), fabsf(q[4 * n + 2 * r + 1])));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
              const int e = fp16_shift(m);
              const float up = pow2i(e);
              undo[r] = pow2i(-e);
#pragma unroll
              for (int n = 0; n < 8; ++n) {
                q[4 * n + 2 * r] *= up;
                q[4 * n + 2 * r + 1] *= up;
              }
            }
          }
          // PV of the item before has read P
          if (!(ok = warp_wait(p_empty, (it & 1) ^ 1, w))) break;
          if (FP16 && (lane & 3) == 0) {
            s_pscale[(it & 1) * 64 + i] = undo[0];
            s_pscale[(it & 1) * 64 + i + 8] = undo[1];
          }
#pragma unroll
          for (int n = 0; n < 8; n += 2) {
            uint32_t p[4];
#pragma unroll
            for (int z = 0; z < 4; ++z) p[z] = Half2<T>::pack(pack2(q[4 * n + 2 * z], q[4 * n + 2 * z + 1]));
            stm4(prow + (((n + (lane >> 4)) ^ (si & 7)) << 4), p[0], p[1], p[2], p[3]);
          }
          fence_async_shared();
          warp_arrive(p_full);
        }
      }
      if (!ok) give_up(ERR_SITE_DECAY_P, w);
    }
  } else if (OUT && wg == K::kO) {
    if constexpr (K::kMove && K::kRegO > 96) regs_up<K::kRegO>();
    // ------------------------------------------------------------ outputs
    // Channels dv = (DV / 4) wq + 16 hh + fr and + 8, tokens 8 n + fc and + 1; put
    // out through shared memory as rows of a token.
    if constexpr (OUT) {
      uint32_t it = 0, cc = 0, ns = 0;
      bool ok = true;
      constexpr int kRow = DV / 4 * 2;       // bytes of a token's row of this warp: 64 or 32
      constexpr int kVec = kRow / 16;        // 16-byte vectors of it
      uint8_t* stage = sOut + wq * kC * kRow;
      const uint32_t stage_u = smem_u32(stage);
      T* const out = static_cast<T*>(a.out);
      for (uint32_t u = blockIdx.x; u < a.n_units && ok; u += gridDim.x) {
        Unit x;
        if (!get_unit<OUT>(a, u, x) || x.len == 0) continue;
        const float l2 = log2_decay(a.log_decay[x.h]);
        F2 grow[8];  // scale l^{i+1}
#pragma unroll
        for (int n = 0; n < 8; ++n)
          grow[n] = pack2(a.scale * exp2_fast(l2 * (float)(8 * n + fc + 1)),
                          a.scale * exp2_fast(l2 * (float)(8 * n + fc + 2)));
        for (int c = 0; c < x.len && ok; c += kC, ++cc) {
          const bool has_s = c > 0 || x.start != nullptr;
          const int n_tok = min(kC, x.len - c);
          for (int g = 0; g < G; ++g, ++it) {
            if (!(ok = warp_wait(o_full, it & 1, w))) break;
            tc_fence_after();
            // 16 channels x 64 tokens at a time; 32 tokens where registers are few
            constexpr int NO = K::kCtas == 2 ? 4 : 8;
            auto put = [&](int hh, auto half) {
              constexpr int n0 = decltype(half)::value * NO;
              float p[4 * NO], z[4 * NO];
              const uint32_t ta = tlane + ((uint32_t)(hh * 16) << 16) + n0 * 8;
              tmem_ld_pair<NO>(ta + K::kColOp, ta + K::kColOs, has_s, p, z);
              const bool last = hh == NH - 1 && n0 + NO == 8;
              if (!FP16 && last) {
                tc_fence_before();
                warp_arrive(o_empty);
              }
              [[maybe_unused]] F2 ss[2];
              if constexpr (FP16) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                  const float e = s_sscale[(ns & 1) * 128 + wq * (DV / 4) + hh * 16 + fr + 8 * r];
                  ss[r] = pack2(e, e);
                }
              }
              uint32_t o[NO][2];
#pragma unroll
              for (int n = 0; n < NO; ++n) {
                [[maybe_unused]] F2 pf = 0;
                if constexpr (FP16) pf = *reinterpret_cast<const F2*>(&s_pscale[(it & 1) * 64 + 8 * (n0 + n) + fc]);
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                  F2 y = pack2(p[4 * n + 2 * r], p[4 * n + 2 * r + 1]);
                  if constexpr (FP16) y = mul2(y, pf);
                  if (has_s) {
                    F2 x2 = pack2(z[4 * n + 2 * r], z[4 * n + 2 * r + 1]);
                    if constexpr (FP16) x2 = mul2(x2, ss[r]);
                    y = fma2(grow[n0 + n], x2, y);
                  }
                  o[n][r] = Half2<T>::pack(y);
                }
              }
              if (FP16 && last) {  // accumulators and scales are read
                tc_fence_before();
                warp_arrive(o_empty);
              }
              // block m = lane / 8: tokens 8 (n + m / 2).., channels 8 (m % 2)..
#pragma unroll
              for (int n = 0; n < NO; n += 2)
                stm4_t(stage_u + out_at<kRow>(8 * (n0 + n + (lane >> 4)) + (lane & 7), hh * 2 + ((lane >> 3) & 1)),
                       o[n][0], o[n][1], o[n + 1][0], o[n + 1][1]);
            };
#pragma unroll 1
            for (int hh = 0; hh < NH; ++hh) {
              put(hh, std::integral_constant<int, 0>{});
              if constexpr (NO == 4) put(hh, std::integral_constant<int, 1>{});
            }
            if (s_badany[cc & 3] == cc + 1)
              spoil_outputs<kRow>(stage, s_bad + (cc & 3) * DV + wq * (DV / 4), cc);
            __syncwarp();
            constexpr int kRows = 32 / kVec;  // rows of a warp's store
            const int v = lane % kVec, row0 = lane / kVec, dv = wq * (DV / 4) + v * 8;
            T* dst = out + (x.t0 + c) * a.o_st + (int64_t)(x.h * G + g) * a.o_sh + wq * (DV / 4);
            if (a.o_vec) {
              dst += (int64_t)row0 * a.o_st + v * 8;
              const int64_t step = (int64_t)kRows * a.o_st;
              const int left = dv < a.Dv ? n_tok - row0 : 0;
              uint4 val[kC / kRows];
#pragma unroll
              for (int z = 0; z < kC / kRows; ++z)
                val[z] = *reinterpret_cast<const uint4*>(stage + out_at<kRow>(z * kRows + row0, v));
#pragma unroll
              for (int z = 0; z < kC / kRows; ++z, dst += step)
                if (z * kRows < left) *reinterpret_cast<uint4*>(dst) = val[z];
            } else {
              store_unaligned<T, kRow>(stage, dst, a.o_st, n_tok, a.Dv - wq * (DV / 4));
            }
            __syncwarp();
          }
          ns += has_s;
        }
      }
      if (!ok) give_up(ERR_SITE_DECAY_O, w);
    }
  } else {
    // ------------------------------------------------------------ state and V'
    // S: rows dv as in the outputs, columns dk = 64 cg + 8 n + fc and + 1.
    bool ok = true;
    const int dv0 = wq * (DV / 4) + fr;

    // V' of chunk `chunk` (n tokens): v comes transposed from its tile (rows dv,
    // tokens 8 m + fc and + 1), meets f (l^{n-1-j}), and goes out in parts.
    auto factors = [&](float2 l2, int n, F2 (&f)[8]) {
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        const int d = n - 1 - 8 * m - fc;
        f[m] = pack2(d < 0 ? 0.f : decay_power(l2, (float)d), d < 1 ? 0.f : decay_power(l2, (float)(d - 1)));
      }
    };
    auto put_v = [&](uint32_t chunk, int n, const F2 (&f)[8]) -> bool {
      const uint32_t st = chunk % K::kKvStages;
      if (!warp_wait(&kv_full[st], (chunk / K::kKvStages) & 1, w)) return false;
      uint8_t* v = sV + st * K::kVBytes;
      const uint32_t vu = smem_u32(v);
      if (n < kC) {
        // Tokens beyond the segment's end belong to others: zeros in their place,
        // in k for KV and in v for V' and PV (each warp in its own channels of v).
        uint8_t* k = sK + st * K::kKBytes;
#pragma unroll 1
        for (int e = wq * 32 + lane; e < K::kKBytes / 16; e += 128)
          if (((e >> 3) & 63) >= n) *reinterpret_cast<uint4*>(k + e * 16) = make_uint4(0, 0, 0, 0);
        constexpr int kV8 = DV / 32;  // vectors of a token in the warp's channels
#pragma unroll 1
        for (int e = n * kV8 + lane; e < kC * kV8; e += 32) {
          const int j = e / kV8, d8 = wq * kV8 + e % kV8;
          *reinterpret_cast<uint4*>(v + (d8 >> 3) * kTileBytes + j * 128 + (((d8 & 7) ^ (j & 7)) << 4)) =
              make_uint4(0, 0, 0, 0);
        }
        fence_async_shared();
        __syncwarp();
      }
      bool odd = false;
#pragma unroll 1
      for (int hh = 0; hh < NH; ++hh) {
        const int d0 = wq * (DV / 4) + hh * 16;  // 16 channels
        // block m = lane / 8 of a load: tokens 8 (2 z + m / 2).., channels d0 + 8 (m % 2)..
        const int ch = ((d0 & 63) >> 3) + ((lane >> 3) & 1), tr = (lane & 7) + (lane >> 4) * 8;
        const uint32_t at = vu + (d0 >> 6) * kTileBytes + tr * 128 + ((ch ^ (lane & 7)) << 4);
        uint32_t raw[16];  // [token octet][row half]
        uint32_t top = 0;  // largest magnitudes, as bits
#pragma unroll
        for (int z = 0; z < 4; ++z) ldm4_t(at + z * 2048, raw[4 * z], raw[4 * z + 1], raw[4 * z + 2], raw[4 * z + 3]);
#pragma unroll
        for (int y = 0; y < 16; y += 2)
          top = __vimax3_u16x2(top, raw[y] & 0x7FFF7FFFu, raw[y + 1] & 0x7FFF7FFFu);
        odd = odd || max(top & 0xFFFFu, top >> 16) >= Half2<T>::kInf;
        float up[2] = {1.f, 1.f};
        if constexpr (FP16) {
          // Row scales come from the largest |V'|, not |v|: under a steep decay the largest v
          // may be all but gone.  Where the S warps do this (64 channels: the longest
          // chain), products in fp16 do for most rows: they are off by 2^-9 at most
          // (factors and results below 2^-14), a quarter of 2^-7; only rows below that take
          // fp32.  (65536 tokens of 16 heads of 64: 240 us; 269 with fp32 everywhere, 256 with
          // fp16 first everywhere, which took 128 channels from 104 to 117.)
          float m[2];
          bool small = true;
          if constexpr (K::kV == K::kS) {
            uint32_t live[2] = {0, 0};
            __half2 p[2] = {__half2(), __half2()};
#pragma unroll
            for (int y = 0; y < 8; ++y) {
              const uint32_t fu = Half2<__half>::pack(f[y]);
              const __half2 fh = *reinterpret_cast<const __half2*>(&fu);
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                live[r] |= raw[2 * y + r];
                p[r] = __hmax2(p[r], __habs2(__hmul2(*reinterpret_cast<const __half2*>(&raw[2 * y + r]), fh)));
              }
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              p[r] = __hmax2(p[r], __shfl_xor_sync(0xffffffffu, p[r], 1));
              p[r] = __hmax2(p[r], __shfl_xor_sync(0xffffffffu, p[r], 2));
              m[r] = fmaxf(__low2float(p[r]), __high2float(p[r]));
            }
            small = __any_sync(0xffffffffu, (m[0] < 0x1p-7f && (live[0] & 0x7FFF7FFFu)) ||
                                                (m[1] < 0x1p-7f && (live[1] & 0x7FFF7FFFu)));
          }
          if (small) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              m[r] = 0.f;
#pragma unroll
              for (int y = 0; y < 8; ++y) {
                float a0, a1;
                unpack2(mul2(Half2<T>::unpack(raw[2 * y + r]), f[y]), a0, a1);
                m[r] = fmaxf(m[r], fmaxf(fabsf(a0), fabsf(a1)));
              }
              m[r] = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], 1));
              m[r] = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], 2));
            }
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int e = fp16_shift(m[r]);
            up[r] = pow2i(e);
            if ((lane & 3) == 0) s_vscale[(chunk & kVMask) * 128 + d0 + fr + 8 * r] = pow2i(-e);
          }
        }
        auto split8 = [&](int h, uint32_t (*part)[16], int o) {
          F2 g[8];
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            g[y] = mul2(Half2<T>::unpack(raw[h + y]), f[(h + y) >> 1]);
            if constexpr (FP16) g[y] = mul2(g[y], pack2(up[y & 1], up[y & 1]));
          }
#pragma unroll
          for (int p = 0; p < K::kVParts; ++p)
#pragma unroll
            for (int y = 0; y < 8; ++y) {
              part[p][o + y] = Half2<T>::pack(g[y]);
              if (p + 1 < K::kVParts) g[y] = sub2(g[y], Half2<T>::unpack(part[p][o + y]));
            }
        };
        uint32_t part[K::kVParts][16];
        if constexpr (TM) {
          split8(0, part, 0);
          split8(8, part, 8);
        }
        // KV of the chunk before in this buffer has read its V'
        if (hh == 0) {
          if (!warp_wait(&ds_full[chunk % VP], ((chunk / VP) & 1) ^ 1, w)) return false;
          tc_fence_after();
        }
        if constexpr (TM) {
#pragma unroll
          for (int q = 0; q < K::kVParts; ++q)
            tmem_st_frag8(tlane + ((uint32_t)(hh * 16) << 16) + K::kColV + ((chunk % VP) * K::kVParts + q) * 32, part[q]);
        } else {
#pragma unroll
          for (int h = 0; h < 16; h += 8) {
            split8(h, part, 0);
#pragma unroll
            for (int q = 0; q < K::kVParts; ++q) {
              const uint32_t to = smem_u32(sVp) + ((chunk % VP) * K::kVParts + q) * K::kVBytes + (at - vu) + h * 512;
              stm4_t(to, part[q][0], part[q][1], part[q][2], part[q][3]);
              stm4_t(to + 2048, part[q][4], part[q][5], part[q][6], part[q][7]);
            }
          }
        }
      }
      if (__any_sync(0xffffffffu, odd))
        mark_non_finite<T>(v, wq * (DV / 4), DV / 4, chunk, s_bad + (chunk & 3) * DV, &s_badany[chunk & 3]);
      if constexpr (TM) {
        tmem_st_wait();
        tc_fence_before();
      } else {
        fence_async_shared();
      }
      warp_arrive(&vp_full[chunk % VP]);
      return true;
    };

    if (K::kV != K::kS && wg == K::kV) {
      if constexpr (K::kMove && K::kRegV < 96) regs_down<K::kRegV>();
      uint32_t cc = 0;
      for (uint32_t u = blockIdx.x; u < a.n_units && ok; u += gridDim.x) {
        Unit x;
        if (!get_unit<OUT>(a, u, x)) continue;
        const float2 l2 = log2_decay_hi_lo(a.log_decay[x.h]);
        F2 f[8];
        for (int c = 0; c < x.len && ok; c += kC, ++cc) {
          const int n = min(kC, x.len - c);
          if (c == 0 || n < kC) factors(l2, n, f);
          ok = put_v(cc, n, f);
        }
      }
    } else {
      if constexpr (K::kMove) regs_up<K::kRegS>();
      uint32_t cc = 0, ns = 0;
      F2 S[NH][K::kCg][16];  // pair y of 64 columns: octet y / 2, row half y % 2
      for (uint32_t u = blockIdx.x; u < a.n_units && ok; u += gridDim.x) {
        Unit x;
        if (!get_unit<OUT>(a, u, x)) continue;
        const float ld = a.log_decay[x.h];
        const float2 l2 = log2_decay_hi_lo(ld);
        const float2 whole = pow_hi_lo(ld, kC), tail = pow_hi_lo(ld, x.len & (kC - 1));
        const int64_t at = (int64_t)fc * a.Dv + dv0;
        if (x.start && a.Dk == DK && a.Dv == DV) {  // all loads in flight at once
          const float* src = x.start + fc * DV + dv0;
          float e[NH][K::kCg][32];
#pragma unroll
          for (int hh = 0; hh < NH; ++hh)
#pragma unroll
            for (int cg = 0; cg < K::kCg; ++cg)
#pragma unroll
              for (int y = 0; y < 32; ++y)
                e[hh][cg][y] = src[(cg * 64 + (y >> 2) * 8 + (y & 1)) * DV + hh * 16 + (y >> 1 & 1) * 8];
#pragma unroll
          for (int hh = 0; hh < NH; ++hh)
#pragma unroll
            for (int cg = 0; cg < K::kCg; ++cg)
#pragma unroll
              for (int y = 0; y < 16; ++y) S[hh][cg][y] = pack2(e[hh][cg][2 * y], e[hh][cg][2 * y + 1]);
        } else {
#pragma unroll
          for (int hh = 0; hh < NH; ++hh)
#pragma unroll
            for (int cg = 0; cg < K::kCg; ++cg)
#pragma unroll
              for (int y = 0; y < 16; ++y) S[hh][cg][y] = 0;
          if (x.start) {
#pragma unroll
            for (int hh = 0; hh < NH; ++hh)
#pragma unroll
              for (int cg = 0; cg < K::kCg; ++cg)
#pragma unroll
                for (int y = 0; y < 16; ++y) {
                  const int dk = cg * 64 + (y >> 1) * 8, dv = hh * 16 + (y & 1) * 8;
                  if (dk < a.Dk && dv0 + dv < a.Dv) {
                    const float* src = x.start + at + dk * a.Dv + dv;
                    S[hh][cg][y] = pack2(src[0], src[a.Dv]);
                  }
                }
          }
        }
        if (x.len > 0 && !keeps_state(ld)) {
#pragma unroll
          for (int hh = 0; hh < NH; ++hh)
#pragma unroll
            for (int cg = 0; cg < K::kCg; ++cg)
#pragma unroll
              for (int y = 0; y < 16; ++y) S[hh][cg][y] = 0;
        }
        F2 f[8];
        for (int c = 0; c < x.len; c += kC, ++cc) {
          const int n = min(kC, x.len - c);
          if constexpr (K::kV == K::kS) {  // before S, so that KV runs while S is put
            if (c == 0 || n < kC) factors(l2, n, f);
            if (!(ok = put_v(cc, n, f))) break;
          }
          if (OUT && (c > 0 || x.start)) {
            // S^T in 16 bits, for the product with the queries; the one before it
            // is done when s_empty comes round.  The scales' slots go by puts: the product
            // with put ns - 1 was issued after the O warps were done with put ns - 2, whose
            // slot this is.  By chunks nothing would order the two, since a chunk that
            // starts from zeros puts no S.
            if (!(ok = warp_wait(s_empty, (ns & 1) ^ 1, w))) break;
            tc_fence_after();
#pragma unroll
            for (int hh = 0; hh < NH; ++hh) {
              float up[2] = {1.f, 1.f};
              if constexpr (FP16) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                  float m = 0.f;
#pragma unroll
                  for (int cg = 0; cg < K::kCg; ++cg)
#pragma unroll
                    for (int y = 0; y < 8; ++y) {
                      float e, g;
                      unpack2(S[hh][cg][2 * y + r], e, g);
                      m = fmaxf(m, fmaxf(fabsf(e), fabsf(g)));
                    }
                  m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                  m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                  const int e = fp16_shift(m);
                  up[r] = pow2i(e);
                  if ((lane & 3) == 0) s_sscale[(ns & 1) * 128 + dv0 + hh * 16 + 8 * r] = pow2i(-e);
                }
              }
#pragma unroll
              for (int cg = 0; cg < K::kCg; ++cg) {
                uint32_t p[16];
#pragma unroll
                for (int y = 0; y < 16; ++y) {
                  F2 z = S[hh][cg][y];
                  if constexpr (FP16) z = mul2(z, pack2(up[y & 1], up[y & 1]));
                  p[y] = Half2<T>::pack(z);
                }
                if constexpr (TM) {
                  tmem_st_frag8(tlane + ((uint32_t)(hh * 16) << 16) + K::kColS + cg * 32, p);
                } else {
                  // block m = lane / 8: rows dv + 8 (m % 2).., columns 8 (m / 2)..
                  const int row = wq * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
                  const uint32_t to = smem_u32(sS) + cg * (DV * 128) + row * 128;
#pragma unroll
                  for (int z = 0; z < 4; ++z)
                    stm4(to + (((2 * z + (lane >> 4)) ^ (row & 7)) << 4), p[4 * z], p[4 * z + 1], p[4 * z + 2],
                         p[4 * z + 3]);
                }
              }
            }
            if constexpr (TM) {
              tmem_st_wait();
              tc_fence_before();
            } else {
              fence_async_shared();
            }
            warp_arrive(s_full);
            ++ns;
          }
          if (!(ok = warp_wait(&ds_full[cc % VP], (cc / VP) & 1, w))) break;
          tc_fence_after();
          const float2 dec = n == kC ? whole : tail;
          const F2 hi = pack2(dec.x, dec.x), lo = pack2(dec.y, dec.y);
          constexpr int NQ = NH * 2 * K::kCg;  // groups of 16 rows x 32 columns, one load ahead
          const uint32_t ta = tlane + K::kColKv + (cc % VP) * DK;
          auto group = [&](int q) { return ta + ((uint32_t)(q / (2 * K::kCg) * 16) << 16) + q % (2 * K::kCg) * 32; };
          float r[2][16];
          tmem_ld_frag4(group(0), r[0]);
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            tmem_wait16(r[q & 1]);
            if (q + 1 < NQ) {
              tmem_ld_frag4(group(q + 1), r[(q + 1) & 1]);
            } else {
              tc_fence_before();
              warp_arrive(&ds_empty[cc % VP]);
            }
            const int hh = q / (2 * K::kCg);
            float dn[2] = {1.f, 1.f};
            if constexpr (FP16) {
              dn[0] = s_vscale[(cc & kVMask) * 128 + dv0 + hh * 16];
              dn[1] = s_vscale[(cc & kVMask) * 128 + dv0 + hh * 16 + 8];
            }
#pragma unroll
            for (int y = 0; y < 8; ++y) {
              F2 add = pack2(r[q & 1][2 * y], r[q & 1][2 * y + 1]);
              if constexpr (FP16) add = mul2(add, pack2(dn[y & 1], dn[y & 1]));
              F2& e = S[hh][q / 2 % K::kCg][(q & 1) * 8 + y];
              e = fma2(hi, e, fma2(lo, e, add));
            }
          }
        }
        if (!ok) break;
        if (x.end) {
#pragma unroll
          for (int hh = 0; hh < NH; ++hh)
#pragma unroll
            for (int cg = 0; cg < K::kCg; ++cg)
#pragma unroll
              for (int m = 0; m < 8; ++m) {
                if (cg * 64 + m * 8 >= a.Dk) continue;
                float* dst = x.end + at + (cg * 64 + m * 8) * a.Dv;
#pragma unroll
                for (int r = 0; r < 2; ++r)
                  if (dv0 + hh * 16 + r * 8 < a.Dv) {
                    float e, g;
                    unpack2(S[hh][cg][2 * m + r], e, g);
                    dst[hh * 16 + r * 8] = e;
                    dst[a.Dv + hh * 16 + r * 8] = g;
                  }
              }
        }
      }
    }

    if (!ok) give_up(K::kV != K::kS && wg == K::kV ? ERR_SITE_DECAY_V : ERR_SITE_DECAY_STATE, w);
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
