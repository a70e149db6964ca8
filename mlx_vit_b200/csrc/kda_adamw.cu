// AdamW over many tensors in one launch, with float32 or 8-bit states, global-norm gradient
// clipping and an exponential moving average of the parameters in the same pass:
//
//   g <- coef g,  coef = min(1, max_norm / (||g|| + 1e-6))              (clipping only)
//   m <- b1 m + (1 - b1) g;   v <- b2 v + (1 - b2) g^2
//   p <- p (1 - lr wd) - c1 m / (sqrt(v) c2 + eps),  c1 = lr / (1 - b1^t), c2 = 1 / sqrt(1 - b2^t)
//   ema <- d ema + (1 - d) p
//
// (the reference trainers' optimizer, clip and shadow average: train_mlx_k400.py:176-222,
// :379-408).  Every element is independent, so the step is bound by its bytes: float32 with
// float32 states moves 28 bytes an element (p, m, v read and written, g read), bf16 with 8-bit
// states 10.  One launch covers up to kCap tensors: their table travels in the kernel's own
// parameters, so no copy to the device precedes the launch and a captured graph holds it.  A
// CTA takes chunks of kChunk elements, chunk index -> tensor by binary search in that table.
//
// Measured on 40M elements: float32 187 us (5.99 TB/s, 91 % of a copy's rate), with the shadow average
// 239 us, bf16 with 32-bit states 145 us (6.05 TB/s); bf16 with 8-bit states 123 us, bound by its instructions
// (issue slots 73 % busy; a generic path without packing and with one pass's loads took 179 us).
//
// This file is compiled without --use_fast_math: m and v are exactly the separately rounded
// float32 products and sums written above (no contraction, subnormals kept), so that an 8-bit
// code is a function of its inputs alone and a restatement of it gives the same codes.
#include <math.h>

#include <atomic>

#include "kda_common.cuh"

namespace kda {
namespace adamw {

constexpr int kThreads = 256, kPer = 8, kBlock = 32 * kPer;
constexpr int kPass = kThreads * kPer, kChunk = 2 * kPass;  // elements a CTA takes at once; two passes a chunk
constexpr int kCap = 448, kCapSmall = 64;  // tensors a launch holds (72 bytes each; parameters end at 32764 bytes)

constexpr int kCtasPerSm = 4;       // resident CTAs the update's grid is sized for (64 registers a thread)
constexpr int kCtasPerSmRead = 8;   // and the reading kernels'

struct Entry {
  void *p;
  const void *g;
  void *m, *v;
  uint8_t *me, *ve;
  float *ema;
  int64_t n;
  uint32_t first;      // first chunk of this tensor
  uint16_t dtype, vec; // vec: every pointer allows whole-vector accesses
};
template <int CAP>
struct Table {
  uint32_t count, chunks, index0;
  uint16_t skip[2];
  Entry e[CAP];
};
// what a step multiplies by; `coef`, `c1`, `c2`, `decay` and `key` are replaced by the device's
// own (Dyn) where they are known there only
struct Hyper {
  float b1, b1c, b2, b2c, eps, ema_d, ema_c;
  float coef, c1, c2, decay;
  uint32_t key;
};
struct Dyn {
  float coef, c1, c2, decay;
  uint32_t key, pad[3];
};

// the finaliser of MurmurHash3 (32 bits, published by its author in the public domain)
__host__ __device__ __forceinline__ uint32_t mix(uint32_t h) {
  h = (h ^ (h >> 16)) * 0x85EBCA6Bu;
  h = (h ^ (h >> 13)) * 0xC2B2AE35u;
  return h ^ (h >> 16);
}

// ---- the 8-bit formats ----
// kBlock consecutive elements share an exponent byte e: 0 for a block of zeros, 255 for one that
// holds a value that is not finite (or above 2^127), else float32's exponent field of the
// block's largest magnitude plus one, so that every magnitude is below 2^(e - 127).  A code's
// magnitude is c = 8 k + f: c = 0 is zero, else (1 + f / 8) 2^(k - L + e - 127); m has a sign in
// bit 7 and L = 15, v (never negative) L = 31, which halves to m's range under the square root.
// Rounding to three bits of mantissa is stochastic: the bits cut off, read as a fraction, are the
// probability of rounding up.  Rounding to nearest would lose every change below half a
// step (3-6 %), and v changes by 0.1 % a step at b2 = 0.999: it could grow but never decay.
constexpr int kLowM = 15, kLowV = 31;
constexpr uint32_t kTiny = 1u << 23;  // smallest normal float32: magnitudes below count as zero

__device__ __forceinline__ uint32_t block_exp(uint32_t top) { return top >= kTiny ? (top >> 23) + 1 : 0; }

// One code: `a` the value's magnitude bits, `base` = (e - L) 2^23, r20 20 random bits (an odd
// multiple of 8, so that exact values stay).  (a + r20) >> 20 is exponent and three bits of
// mantissa with the carry; a value below the least code becomes that code or zero for m, unbiased,
// and the least code for v, where a zero would be divided by in a later step.
template <bool SIGNED>
__device__ __forceinline__ uint32_t encode(uint32_t a, int base, uint32_t r20) {
  uint32_t c = (a + r20 - (uint32_t)base) >> 20;
  const int least = max(base + (1 << 20), (int)kTiny);
  if ((int)a < least)
    c = a >= kTiny && (!SIGNED || __fmul_rn(__uint2float_rn(r20) * 0x1p-20f, __int_as_float(least)) < __uint_as_float(a));
  return c;
}
// Two codes, in the low bytes of w's 16-bit halves, to two values as bf16 halves (three bits of
// mantissa and float32's exponent: exact): 16 code + (e - L) 2^7 where the code is not zero.
// shift2 = |e - L| 2^7 in both halves, dir its sign; no half carries into the other.
template <bool SIGNED>
__device__ __forceinline__ uint32_t decode2(uint32_t w, uint32_t shift2, uint32_t dir) {
  const uint32_t mag = SIGNED ? w & 0x007F007Fu : w;
  const uint32_t live = __vminu2(mag, 0x00010001u) * 0xFFFFu;
  const uint32_t x = (shift2 & live) * dir + mag * 16u;
  return SIGNED ? x | ((w << 8) & 0x80008000u) : x;
}
// the eight values of u's codes in a block with exponent byte e, as bf16 pairs (e = 255: anything)
template <bool SIGNED>
__device__ __forceinline__ void decode8(uint2 u, int e, uint32_t (&x)[4]) {
  const int up = e - (SIGNED ? kLowM : kLowV);
  const uint32_t shift2 = (uint32_t)abs(up) * 0x00800080u, dir = up < 0 ? 0xFFFFFFFFu : 1u;
  if (e == 0) u = make_uint2(0, 0);
  x[0] = decode2<SIGNED>(__byte_perm(u.x, 0, 0x4140), shift2, dir);
  x[1] = decode2<SIGNED>(__byte_perm(u.x, 0, 0x4342), shift2, dir);
  x[2] = decode2<SIGNED>(__byte_perm(u.y, 0, 0x4140), shift2, dir);
  x[3] = decode2<SIGNED>(__byte_perm(u.y, 0, 0x4342), shift2, dir);
}
__device__ __forceinline__ float bf16_of(const uint32_t (&x)[4], int j) {
  return __uint_as_float(j & 1 ? x[j >> 1] & 0xFFFF0000u : x[j >> 1] << 16);
}
// byte `sel` of four words, in order
__device__ __forceinline__ uint32_t gather(uint32_t a, uint32_t b, uint32_t c, uint32_t d, bool top) {
  const uint32_t ab = __byte_perm(a, b, top ? 0x0073 : 0x0040), cd = __byte_perm(c, d, top ? 0x0073 : 0x0040);
  return __byte_perm(ab, cd, 0x5410);
}

// ---- vectors of kPer elements; float32's as one 32-byte access (two of 16 bytes take a tenth longer
// over the whole step) ----
template <typename T>
__device__ __forceinline__ void load_vec(const T *p, float (&x)[kPer]) {
  if constexpr (sizeof(T) == 4) {
    asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]) : "l"(p));
  } else {
    union { uint4 u; T t[8]; } q;
    q.u = *reinterpret_cast<const uint4 *>(p);
#pragma unroll
    for (int j = 0; j < kPer; ++j) x[j] = to_f<T>(q.t[j]);
  }
}
template <typename T>
__device__ __forceinline__ void store_vec(T *p, const float (&x)[kPer]) {
  if constexpr (sizeof(T) == 4) {
    asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 :: "l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]) : "memory");
  } else {
    union { uint4 u; T t[8]; } q;
#pragma unroll
    for (int j = 0; j < kPer; ++j) q.t[j] = from_f<T>(x[j]);
    *reinterpret_cast<uint4 *>(p) = q.u;
  }
}
// k of the kPer elements exist
template <typename T>
__device__ __forceinline__ void load_n(const T *p, float (&x)[kPer], int k, bool vec) {
  if (vec) return load_vec<T>(p, x);
#pragma unroll
  for (int j = 0; j < kPer; ++j) x[j] = j < k ? to_f<T>(p[j]) : 0.f;
}
template <typename T>
__device__ __forceinline__ void store_n(T *p, const float (&x)[kPer], int k, bool vec) {
  if (vec) return store_vec<T>(p, x);
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    if (j < k) p[j] = from_f<T>(x[j]);
}
__device__ __forceinline__ uint2 load_codes(const uint8_t *p, int k, bool vec) {
  if (vec) return *reinterpret_cast<const uint2 *>(p);
  uint32_t u[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    if (j < k) u[j >> 2] |= (uint32_t)p[j] << (8 * (j & 3));
  return make_uint2(u[0], u[1]);
}
__device__ __forceinline__ void store_codes(uint8_t *p, uint2 u, int k, bool vec) {
  if (vec) {
    *reinterpret_cast<uint2 *>(p) = u;
    return;
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    if (j < k) p[j] = (uint8_t)((j < 4 ? u.x : u.y) >> (8 * (j & 3)));
}

// sqrt(v) and the quotient by the fast units (1 and 2 units in the last place): the update is
// added to p in float32 and lies some binades below it; m and v are not touched by them.  With
// 8-bit states subnormals count as zero (and eps is not): the forms that flush them.
template <bool FLUSH>
__device__ __forceinline__ float sqrt_fast(float x) {
  float y;
  if (FLUSH) asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  else asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool FLUSH>
__device__ __forceinline__ float div_fast(float x, float d) {
  float y;
  if (FLUSH) asm("div.approx.ftz.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(d));
  else asm("div.approx.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(d));
  return y;
}

template <bool FLUSH>
__device__ __forceinline__ void moments(float &p, float g, float &m, float &v, float b1, float b2, const Hyper &h) {
  g = __fmul_rn(g, h.coef);
  m = __fadd_rn(__fmul_rn(m, b1), __fmul_rn(g, h.b1c));
  v = __fadd_rn(__fmul_rn(v, b2), __fmul_rn(__fmul_rn(g, g), h.b2c));
  p = fmaf(p, h.decay, -div_fast<FLUSH>(h.c1 * m, fmaf(sqrt_fast<FLUSH>(v), h.c2, h.eps)));
}

// one warp's block of kBlock elements; k of this lane's kPer exist
template <typename T, bool EIGHT, bool EMA>
__device__ __forceinline__ void update(const Entry &e, int64_t i, uint32_t tensor, const Hyper &h) {
  const int64_t left = e.n - i;
  const int k = left >= kPer ? kPer : left > 0 ? (int)left : 0;
  const bool vec = k == kPer && e.vec;
  float p[kPer], g[kPer], s[kPer];
  load_n(static_cast<const T *>(e.g) + i, g, k, vec);
  load_n(static_cast<const T *>(e.p) + i, p, k, vec);
  if constexpr (EMA && !EIGHT) load_n(e.ema + i, s, k, vec);
  if constexpr (EIGHT) {
    const uint2 mc = load_codes(static_cast<const uint8_t *>(e.m) + i, k, vec);
    const uint2 vc = load_codes(static_cast<const uint8_t *>(e.v) + i, k, vec);
    uint8_t *me = e.me + i / kBlock, *ve = e.ve + i / kBlock;
    const int me0 = *me, ve0 = *ve;
    uint32_t mx[4], vx[4], ma[kPer], va[kPer], mtop = 0, vtop = 0;
    decode8<true>(mc, me0, mx);
    decode8<false>(vc, ve0, vx);
    const float nan = __uint_as_float(0x7FC00000u);  // what a block that is not finite decodes to
    const float b1 = me0 == 255 ? nan : h.b1, b2 = ve0 == 255 ? nan : h.b2;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      float m = bf16_of(mx, j), v = bf16_of(vx, j);
      moments<true>(p[j], g[j], m, v, b1, b2, h);
      ma[j] = __float_as_uint(m);
      va[j] = __float_as_uint(v) & 0x7FFFFFFFu;
      if (j < k) {
        mtop = max(mtop, ma[j] & 0x7FFFFFFFu);
        vtop = max(vtop, va[j]);
      }
    }
    store_n(static_cast<T *>(e.p) + i, p, k, vec);
    // a NaN's exponent field plus one is 256
    const int me1 = min((int)block_exp(__reduce_max_sync(0xFFFFFFFFu, mtop)), 255);
    const int ve1 = min((int)block_exp(__reduce_max_sync(0xFFFFFFFFu, vtop)), 255);
    const int mbase = (me1 - kLowM) * (1 << 23), vbase = (ve1 - kLowV) * (1 << 23);
    const uint32_t key = mix(h.key ^ tensor);
    uint32_t cm[kPer], cv[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const uint32_t r = mix(((uint32_t)i + j) ^ key);
      cm[j] = encode<true>(ma[j] & 0x7FFFFFFFu, mbase, ((r & 0xFFFFu) << 4) | 8u);
      cv[j] = encode<false>(va[j], vbase, ((r >> 12) & 0xFFFF0u) | 8u);
      if (cm[j] == 0) ma[j] = 0;  // zero has no sign
    }
    const uint2 mn = make_uint2(gather(cm[0], cm[1], cm[2], cm[3], false) |
                                    (gather(ma[0], ma[1], ma[2], ma[3], true) & 0x80808080u),
                                gather(cm[4], cm[5], cm[6], cm[7], false) |
                                    (gather(ma[4], ma[5], ma[6], ma[7], true) & 0x80808080u));
    const uint2 vn = make_uint2(gather(cv[0], cv[1], cv[2], cv[3], false), gather(cv[4], cv[5], cv[6], cv[7], false));
    store_codes(static_cast<uint8_t *>(e.m) + i, mn, k, vec);
    store_codes(static_cast<uint8_t *>(e.v) + i, vn, k, vec);
    if (k > 0 && i % kBlock == 0) {
      *me = (uint8_t)me1;
      *ve = (uint8_t)ve1;
    }
  } else {
    float m[kPer], v[kPer];
    load_n(static_cast<const float *>(e.m) + i, m, k, vec);
    load_n(static_cast<const float *>(e.v) + i, v, k, vec);
#pragma unroll
    for (int j = 0; j < kPer; ++j) moments<false>(p[j], g[j], m[j], v[j], h.b1, h.b2, h);
    store_n(static_cast<T *>(e.p) + i, p, k, vec);
    store_n(static_cast<float *>(e.m) + i, m, k, vec);
    store_n(static_cast<float *>(e.v) + i, v, k, vec);
  }
  if constexpr (EMA) {
    if constexpr (EIGHT) load_n(e.ema + i, s, k, vec);  // late: registers
#pragma unroll
    for (int j = 0; j < kPer; ++j) {  // of the parameter as it is stored
      const float held = to_f<T>(from_f<T>(p[j]));
      s[j] = __fadd_rn(__fmul_rn(s[j], h.ema_d), __fmul_rn(held, h.ema_c));
    }
    store_n(e.ema + i, s, k, vec);
  }
}

// ---- a lane whose eight elements all exist and are aligned: the same with 8-bit states in fewer
// instructions.  The step is bound by them, not by its 10 bytes an element, so p's products and sums go
// two to an instruction, zero codes and values below the least code take branches of their own (rare
// but in tensors without gradients), and codes are picked from bits 20-27 by bytes. ----
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mul.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
      " fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// decode8 where no code is zero
template <bool SIGNED>
__device__ __forceinline__ void decode8_live(uint2 u, int e, uint32_t (&x)[4]) {
  const uint32_t shift = (uint32_t)(e - (SIGNED ? kLowM : kLowV)) * 0x00800080u;  // a negative one borrows nothing
  const uint32_t w[4] = {__byte_perm(u.x, 0, 0x4140), __byte_perm(u.x, 0, 0x4342), __byte_perm(u.y, 0, 0x4140),
                         __byte_perm(u.y, 0, 0x4342)};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[j] = (SIGNED ? w[j] & 0x007F007Fu : w[j]) * 16u + shift;
    if (SIGNED) x[j] |= (w[j] << 8) & 0x80008000u;
  }
}
__device__ __forceinline__ bool all_live(uint2 m, uint2 v) {  // no zero byte in m (without signs) and v
  const uint32_t a = ((m.x & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) & ((m.y & 0x7F7F7F7Fu) + 0x7F7F7F7Fu);
  const uint32_t zx = (v.x - 0x01010101u) & ~v.x, zy = (v.y - 0x01010101u) & ~v.y;
  return ((~a | zx | zy) & 0x80808080u) == 0;
}
// bits 20-27 of four words as four bytes
__device__ __forceinline__ uint32_t pick(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x7632) >> 4, __byte_perm(c, d, 0x7632) >> 4, 0x6420);
}

// what a lane reads of its eight elements, as it lies in memory: held for both passes of a chunk, so that
// the second's loads pass while the first is worked on
template <typename T>
struct Raw {
  uint4 g[sizeof(T) / 2], p[sizeof(T) / 2];
  uint2 m, v;
  int me, ve;
  __device__ __forceinline__ void load(const Entry &e, int64_t i) {
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; ++j) {
      g[j] = reinterpret_cast<const uint4 *>(static_cast<const T *>(e.g) + i)[j];
      p[j] = reinterpret_cast<const uint4 *>(static_cast<const T *>(e.p) + i)[j];
    }
    m = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(e.m) + i);
    v = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(e.v) + i);
    me = e.me[i / kBlock];
    ve = e.ve[i / kBlock];
  }
  static __device__ __forceinline__ void values(const uint4 (&u)[sizeof(T) / 2], float (&x)[kPer]) {
    const T *t = reinterpret_cast<const T *>(u);
#pragma unroll
    for (int j = 0; j < kPer; ++j) x[j] = to_f<T>(t[j]);
  }
};

template <typename T, bool EMA>
__device__ __forceinline__ void update8(const Raw<T> &in, const Entry &e, int64_t i, uint32_t tensor, const Hyper &h) {
  uint8_t *mp = static_cast<uint8_t *>(e.m) + i, *vp = static_cast<uint8_t *>(e.v) + i;
  uint8_t *me = e.me + i / kBlock, *ve = e.ve + i / kBlock;
  float p[kPer], g[kPer];
  Raw<T>::values(in.g, g);
  Raw<T>::values(in.p, p);
  const uint2 mc = in.m, vc = in.v;
  const int me0 = in.me, ve0 = in.ve;
  uint32_t mx[4], vx[4];
  if (all_live(mc, vc)) {
    decode8_live<true>(mc, me0, mx);
    decode8_live<false>(vc, ve0, vx);
  } else {
    decode8<true>(mc, me0, mx);
    decode8<false>(vc, ve0, vx);
  }
  const float nan = __uint_as_float(0x7FC00000u);  // what a block that is not finite decodes to
  const float b1 = me0 == 255 ? nan : h.b1, b2 = ve0 == 255 ? nan : h.b2;
  float m[kPer], v[kPer];
  uint32_t mtop = 0, vtop = 0;
#pragma unroll
  for (int j = 0; j < kPer; j += 2) {
    float mv[2][2];
#pragma unroll
    for (int l = 0; l < 2; ++l) {  // m and v one by one: ptxas joins a packed product and sum into one rounding
      const float gl = __fmul_rn(g[j + l], h.coef);
      mv[0][l] = __fadd_rn(__fmul_rn(bf16_of(mx, j + l), b1), __fmul_rn(gl, h.b1c));
      mv[1][l] = __fadd_rn(__fmul_rn(bf16_of(vx, j + l), b2), __fmul_rn(__fmul_rn(gl, gl), h.b2c));
    }
    const float2 mj = make_float2(mv[0][0], mv[0][1]), vj = make_float2(mv[1][0], mv[1][1]);
    const float2 d = fma2(make_float2(sqrt_fast<true>(vj.x), sqrt_fast<true>(vj.y)), both(h.c2), both(h.eps));
    const float2 s = mul2(mj, both(-h.c1));
    const float2 pj = fma2(make_float2(p[j], p[j + 1]), both(h.decay),
                           make_float2(div_fast<true>(s.x, d.x), div_fast<true>(s.y, d.y)));
    p[j] = pj.x; p[j + 1] = pj.y;
    m[j] = mj.x; m[j + 1] = mj.y;
    v[j] = vj.x; v[j + 1] = vj.y;
    mtop = max(mtop, max(__float_as_uint(mj.x) & 0x7FFFFFFFu, __float_as_uint(mj.y) & 0x7FFFFFFFu));
    vtop = max(vtop, max(__float_as_uint(vj.x), __float_as_uint(vj.y)));  // v has no sign, but for a NaN's
  }
  store_vec(static_cast<T *>(e.p) + i, p);
  const int me1 = min((int)block_exp(__reduce_max_sync(0xFFFFFFFFu, mtop)), 255);
  const int ve1 = min((int)block_exp(__reduce_max_sync(0xFFFFFFFFu, vtop)), 255);
  const int mbase = (me1 - kLowM) * (1 << 23), vbase = (ve1 - kLowV) * (1 << 23);
  const int mleast = max(mbase + (1 << 20), (int)kTiny), vleast = max(vbase + (1 << 20), (int)kTiny);
  const uint32_t at = (uint32_t)i ^ mix(h.key ^ tensor);  // i is a multiple of kPer: (i + j) ^ key = at ^ j
  uint32_t tm[kPer], tv[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const uint32_t r = mix(at ^ (uint32_t)j);
    const uint32_t rm = ((r << 4) & 0xFFFF0u) | 8u, rv = ((r >> 12) & 0xFFFF0u) | 8u;
    const uint32_t a = __float_as_uint(m[j]) & 0x7FFFFFFFu, b = __float_as_uint(v[j]);
    tm[j] = a + rm - (uint32_t)mbase;
    tv[j] = b + rv - (uint32_t)vbase;
    if ((int)a < mleast) {
      tm[j] = encode<true>(a, mbase, rm) << 20;
      if (tm[j] == 0) m[j] = 0.f;  // zero has no sign
    }
    if ((int)b < vleast) tv[j] = encode<false>(b & 0x7FFFFFFFu, vbase, rv) << 20;
  }
  uint2 mn = make_uint2(pick(tm[0], tm[1], tm[2], tm[3]), pick(tm[4], tm[5], tm[6], tm[7]));
  mn.x |= gather(__float_as_uint(m[0]), __float_as_uint(m[1]), __float_as_uint(m[2]), __float_as_uint(m[3]), true) & 0x80808080u;
  mn.y |= gather(__float_as_uint(m[4]), __float_as_uint(m[5]), __float_as_uint(m[6]), __float_as_uint(m[7]), true) & 0x80808080u;
  *reinterpret_cast<uint2 *>(mp) = mn;
  *reinterpret_cast<uint2 *>(vp) = make_uint2(pick(tv[0], tv[1], tv[2], tv[3]), pick(tv[4], tv[5], tv[6], tv[7]));
  if (i % kBlock == 0) {
    *me = (uint8_t)me1;
    *ve = (uint8_t)ve1;
  }
  if constexpr (EMA) {
    float s[kPer];
    load_vec(e.ema + i, s);
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      s[j] = __fadd_rn(__fmul_rn(s[j], h.ema_d), __fmul_rn(to_f<T>(from_f<T>(p[j])), h.ema_c));
    store_vec(e.ema + i, s);
  }
}

template <int CAP>
__device__ __forceinline__ uint32_t find_tensor(const Table<CAP> &t, uint32_t lo, uint32_t chunk) {
  uint32_t hi = t.count - 1;
  while (lo < hi) {
    const uint32_t mid = (lo + hi + 1) >> 1;
    if (t.e[mid].first <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// a thread's two passes of a chunk, from element i on
template <typename T, bool EIGHT, bool EMA>
__device__ __forceinline__ void chunk(const Entry &e, int64_t i, uint32_t tensor, const Hyper &h) {
  const int64_t warp_at = i - (threadIdx.x & 31) * kPer;
  if (EIGHT && e.vec && warp_at + kPass + kBlock <= e.n) {  // the warp's elements all exist, aligned
    Raw<T> a, b;
    a.load(e, i);
    b.load(e, i + kPass);
    update8<T, EMA>(a, e, i, tensor, h);
    update8<T, EMA>(b, e, i + kPass, tensor, h);
    return;
  }
#pragma unroll 1
  for (int pass = 0; pass < 2 && warp_at + pass * kPass < e.n; ++pass)
    update<T, EIGHT, EMA>(e, i + pass * kPass, tensor, h);
}

template <bool EIGHT, bool EMA, int CAP>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) adamw_kernel(const __grid_constant__ Table<CAP> t, Hyper h, const Dyn *dyn) {
  if (dyn) {
    h.coef = dyn->coef;
    h.c1 = dyn->c1;
    h.c2 = dyn->c2;
    h.decay = dyn->decay;
    h.key = dyn->key;
  }
  uint32_t ti = 0;
  for (uint32_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    ti = find_tensor(t, ti, c);
    const Entry &e = t.e[ti];
    const int64_t i = (int64_t)(c - e.first) * kChunk + threadIdx.x * kPer;
    const uint32_t tensor = t.index0 + ti;
    if (e.dtype == KDA_F32) chunk<float, EIGHT, EMA>(e, i, tensor, h);
    else if (e.dtype == KDA_BF16) chunk<__nv_bfloat16, EIGHT, EMA>(e, i, tensor, h);
    else chunk<__half, EIGHT, EMA>(e, i, tensor, h);
  }
}

// ---- the gradients' global norm: sums of squares in 64 bits, one partial a CTA, added in a fixed order
// (72.7M float32 gradients: 61 us, 4.8 TB/s, and 4 us to add) ----
template <typename T>
__device__ __forceinline__ double squares(const Entry &e, int64_t i) {
  const int64_t left = e.n - i;
  const int k = left >= kPer ? kPer : left > 0 ? (int)left : 0;
  float g[kPer];
  load_n(static_cast<const T *>(e.g) + i, g, k, k == kPer && e.vec);
  double s = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) s += (double)g[j] * (double)g[j];
  return s;
}
__device__ __forceinline__ double block_sum(double s) {  // the result is thread 0's
  __shared__ double red[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_down_sync(0xFFFFFFFFu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0;
  for (int w = 0; w < kThreads / 32; ++w) s += red[w];
  return s;
}
template <int CAP>
__global__ void __launch_bounds__(kThreads) squares_kernel(const __grid_constant__ Table<CAP> t, double *partial) {
  double s = 0;
  uint32_t ti = 0;
  for (uint32_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    ti = find_tensor(t, ti, c);
    const Entry &e = t.e[ti];
    const int64_t i = (int64_t)(c - e.first) * kChunk + threadIdx.x * kPer;
    if (e.dtype == KDA_F32) s += squares<float>(e, i) + squares<float>(e, i + kPass);
    else if (e.dtype == KDA_BF16) s += squares<__nv_bfloat16>(e, i) + squares<__nv_bfloat16>(e, i + kPass);
    else s += squares<__half>(e, i) + squares<__half>(e, i + kPass);
  }
  s = block_sum(s);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// what the update multiplies by, where the device alone knows it: the clip's coefficient, and
// with a device step counter (which it advances) the step's own constants
struct Prep {
  double b1, b2, lr, wd, max_norm;
  int64_t *step;
  const float *lr_dev;
  int64_t host_step;
  uint32_t seed;
  int bias, parts, norm_given;
};
__global__ void __launch_bounds__(kThreads) prep_kernel(Prep a, const double *partial, float *norm, Dyn *dyn) {
  double s = 0;
  for (int i = threadIdx.x; i < a.parts; i += kThreads) s += partial[i];
  s = block_sum(s);
  if (threadIdx.x) return;
  const double n = a.norm_given ? (double)*norm : sqrt(s);
  if (norm && !a.norm_given) *norm = (float)n;
  int64_t step = a.host_step;
  if (a.step) *a.step = step = *a.step + 1;
  if (!dyn) return;
  double coef = 1;
  if (a.max_norm > 0) {
    coef = a.max_norm / (n + 1e-6);
    if (coef > 1) coef = 1;  // a NaN stays one
  }
  const double lr = a.lr_dev ? (double)*a.lr_dev : a.lr;
  dyn->coef = (float)coef;
  dyn->c1 = (float)(a.bias ? lr / (1 - pow(a.b1, (double)step)) : lr);
  dyn->c2 = (float)(a.bias ? 1 / sqrt(1 - pow(a.b2, (double)step)) : 1);
  dyn->decay = (float)(1 - lr * a.wd);
  dyn->key = mix(a.seed + (uint32_t)step * 0x9E3779B9u);
}

// 8-bit states back to values: three bits of mantissa, so that bf16 holds them exactly (155M codes: 82 us,
// 5.7 TB/s of 3 bytes each)
template <bool SIGNED>
__global__ void __launch_bounds__(kThreads) decode_kernel(int64_t n, const uint8_t *code, const uint8_t *exp,
                                                          __nv_bfloat16 *out, bool vec_ok) {
  for (int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * kPer; i < n;
       i += (int64_t)gridDim.x * kPass) {
    const int k = n - i >= kPer ? kPer : (int)(n - i);
    const bool vec = vec_ok && k == kPer;
    const int e = exp[i / kBlock];
    uint32_t x[4];
    decode8<SIGNED>(load_codes(code + i, k, vec), e, x);
    if (e == 255) x[0] = x[1] = x[2] = x[3] = 0x7FC07FC0u;
    if (vec) {
      *reinterpret_cast<uint4 *>(out + i) = make_uint4(x[0], x[1], x[2], x[3]);
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (j < k) out[i + j] = __ushort_as_bfloat16((unsigned short)(x[j >> 1] >> (16 * (j & 1))));
    }
  }
}

// ---- host side ----
static int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < 64) {
    const int n = known[dev].load(std::memory_order_relaxed);
    if (n) return n;
  }
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}
static bool multiple(const void *p, uintptr_t a) { return ((uintptr_t)p % a) == 0; }
static int launched() {
  if (cudaGetLastError() != cudaSuccess) return KDA_ERR_CUDA;
  count_launch();
  return KDA_OK;
}

constexpr size_t kDynBytes = 256;

template <int CAP, typename F>
static int for_tables(const KdaAdamWTensor *x, int64_t count, uint32_t first, bool grads_only, bool eight, F launch) {
  static thread_local Table<CAP> t;
  int64_t at = 0;
  while (at < count) {
    t.count = 0;
    t.chunks = 0;
    t.index0 = first + (uint32_t)at;
    uint64_t chunks = 0;
    for (; at < count && t.count < CAP; ++at) {
      const KdaAdamWTensor &a = x[at];
      Entry &e = t.e[t.count];
      const uint64_t more = (uint64_t)((a.numel + kChunk - 1) / kChunk);
      if (chunks + more >= (1ull << 31)) break;  // the chunk index is 32 bits wide
      e.p = a.p; e.g = a.g; e.m = a.m; e.v = a.v; e.me = a.m_exp; e.ve = a.v_exp; e.ema = a.ema;
      e.n = a.numel;
      e.first = (uint32_t)chunks;
      e.dtype = (uint16_t)a.dtype;
      const uintptr_t own = a.dtype == KDA_F32 ? 32 : 16, state = eight ? 8 : 32;
      bool vec = multiple(a.g, own);
      if (!grads_only)
        vec = vec && multiple(a.p, own) && multiple(a.m, state) && multiple(a.v, state) && multiple(a.ema, 32);
      e.vec = vec;
      chunks += more;
      ++t.count;
    }
    t.chunks = (uint32_t)chunks;
    if (!t.count) return KDA_ERR_UNSUPPORTED;  // one tensor alone is past the chunk index
    if (chunks) {
      const int s = launch(t);
      if (s) return s;
    }
  }
  return KDA_OK;
}

static int grid_for(uint32_t chunks, int sms, int per_sm) {
  const uint32_t most = (uint32_t)(sms * per_sm);
  return (int)(chunks < most ? chunks : most);
}

template <int CAP>
static int launch_squares(const KdaAdamWTensor *x, int64_t count, double *partial, int most, int &parts, int sms,
                          cudaStream_t st) {
  return for_tables<CAP>(x, count, 0, true, false, [&](const Table<CAP> &t) {
    const int grid = grid_for(t.chunks, sms, kCtasPerSmRead);
    if (parts + grid > most) return (int)KDA_ERR_WORKSPACE;
    squares_kernel<CAP><<<grid, kThreads, 0, st>>>(t, partial + parts);
    parts += grid;
    return launched();
  });
}
template <bool EIGHT, bool EMA, int CAP>
static int launch_update(const KdaAdamWTensor *x, int64_t count, uint32_t first, const Hyper &h, const Dyn *dyn, int sms,
                         cudaStream_t st) {
  return for_tables<CAP>(x, count, first, false, EIGHT, [&](const Table<CAP> &t) {
    adamw_kernel<EIGHT, EMA, CAP><<<grid_for(t.chunks, sms, kCtasPerSm), kThreads, 0, st>>>(t, h, dyn);
    return launched();
  });
}
template <int CAP>
static int launch_update(const KdaAdamWTensor *x, int64_t count, uint32_t first, const Hyper &h, const Dyn *dyn, bool eight,
                         bool ema, int sms, cudaStream_t st) {
  if (eight)
    return ema ? launch_update<true, true, CAP>(x, count, first, h, dyn, sms, st)
               : launch_update<true, false, CAP>(x, count, first, h, dyn, sms, st);
  return ema ? launch_update<false, true, CAP>(x, count, first, h, dyn, sms, st)
             : launch_update<false, false, CAP>(x, count, first, h, dyn, sms, st);
}

static int64_t max_parts(int64_t count, int sms) {
  // launches: one per kCap tensors, and one more for every 2^31 chunks (far past any memory)
  return ((count + kCapSmall - 1) / kCapSmall + 1) * sms * kCtasPerSmRead;
}

static int check_tensors(const KdaAdamWTensor *x, int64_t count) {
  if (count < 0 || count > (1ll << 24) || (count && !x)) return KDA_ERR_INVALID_ARG;
  for (int64_t i = 0; i < count; ++i) {
    if (x[i].numel < 0 || (x[i].numel && !x[i].g)) return KDA_ERR_INVALID_ARG;
    if (x[i].dtype != KDA_F32 && x[i].dtype != KDA_BF16 && x[i].dtype != KDA_F16) return KDA_ERR_DTYPE;
    if (!multiple(x[i].g, x[i].dtype == KDA_F32 ? 4 : 2)) return KDA_ERR_MISALIGNED;
  }
  return KDA_OK;
}

}  // namespace adamw
}  // namespace kda

using namespace kda::adamw;

extern "C" {

size_t kda_adamw_workspace_bytes(int64_t count) {
  if (count <= 0 || count > (1ll << 24)) return 0;
  // the partial sums of a device of up to 256 SMs
  return kDynBytes + (size_t)max_parts(count, 256) * sizeof(double);
}

int kda_adamw_step(const KdaAdamW *a, const KdaAdamWTensor *x, int64_t count, int64_t *step_dev, const float *lr_dev,
                   float *grad_norm, void *ws, size_t ws_bytes, void *stream) {
  if (!a) return KDA_ERR_INVALID_ARG;
  const bool eight = a->state_bits == 8;
  if (!eight && a->state_bits != 32) return KDA_ERR_UNSUPPORTED;
  if (!(a->beta1 >= 0 && a->beta1 < 1) || !(a->beta2 >= 0 && a->beta2 < 1) || !(a->eps >= 0) ||
      !(a->max_grad_norm >= 0) || !(a->ema_decay >= 0 && a->ema_decay <= 1) || (!step_dev && a->step < 1) ||
      !isfinite(a->lr) || !isfinite(a->weight_decay) || (eight && a->eps < 1e-30))
    return KDA_ERR_INVALID_ARG;
  if (!multiple(step_dev, 8) || !multiple(lr_dev, 4) || !multiple(grad_norm, 4)) return KDA_ERR_MISALIGNED;
  int s = check_tensors(x, count);
  if (s) return s;
  for (int64_t i = 0; i < count; ++i) {
    const KdaAdamWTensor &t = x[i];
    if (!t.numel) continue;
    if (!t.p || !t.m || !t.v || (eight && (!t.m_exp || !t.v_exp)) || (a->use_ema && !t.ema)) return KDA_ERR_INVALID_ARG;
    if (!multiple(t.p, t.dtype == KDA_F32 ? 4 : 2) || (!eight && (!multiple(t.m, 4) || !multiple(t.v, 4))) ||
        (a->use_ema && !multiple(t.ema, 4)))
      return KDA_ERR_MISALIGNED;
  }
  const bool clip = a->max_grad_norm > 0, dynamic = clip || step_dev || lr_dev;
  const bool given = clip && a->norm_given;
  if (given && !grad_norm) return KDA_ERR_INVALID_ARG;
  if (!count && !step_dev && !grad_norm) return KDA_OK;
  const int sms = sm_count();
  if (!sms) return KDA_ERR_CUDA;
  cudaStream_t st = (cudaStream_t)stream;
  Dyn *dyn = nullptr;
  double *partial = nullptr;
  int parts = 0;
  if (dynamic || grad_norm) {
    const bool sum = (clip || grad_norm) && !given && count;
    const int64_t most = sum ? max_parts(count, sms) : 0;
    // without tensors the step's number and the norm alone are written, and no workspace is used
    if (count && (!ws || !multiple(ws, 16) || ws_bytes < kDynBytes + (size_t)most * sizeof(double))) return KDA_ERR_WORKSPACE;
    dyn = dynamic && count ? static_cast<Dyn *>(ws) : nullptr;
    partial = count ? reinterpret_cast<double *>(static_cast<char *>(ws) + kDynBytes) : nullptr;
    if (sum) {
      s = count <= kCapSmall ? launch_squares<kCapSmall>(x, count, partial, (int)most, parts, sms, st)
                             : launch_squares<kCap>(x, count, partial, (int)most, parts, sms, st);
      if (s) return s;
    }
    const Prep pr = {a->beta1, a->beta2, a->lr, a->weight_decay, a->max_grad_norm, step_dev, lr_dev,
                     a->step,  a->seed,  a->bias_correction ? 1 : 0, parts, given ? 1 : 0};
    prep_kernel<<<1, kThreads, 0, st>>>(pr, partial, grad_norm, dyn);
    if ((s = launched())) return s;
  }
  Hyper h = {};
  h.b1 = (float)a->beta1; h.b1c = (float)(1 - a->beta1);
  h.b2 = (float)a->beta2; h.b2c = (float)(1 - a->beta2);
  h.eps = (float)a->eps;
  h.ema_d = (float)a->ema_decay; h.ema_c = (float)(1 - a->ema_decay);
  h.coef = 1;
  if (!dynamic) {
    h.c1 = (float)(a->bias_correction ? a->lr / (1 - pow(a->beta1, (double)a->step)) : a->lr);
    h.c2 = (float)(a->bias_correction ? 1 / sqrt(1 - pow(a->beta2, (double)a->step)) : 1);
    h.decay = (float)(1 - a->lr * a->weight_decay);
    h.key = mix(a->seed + (uint32_t)a->step * 0x9E3779B9u);
  }
  return count <= kCapSmall ? launch_update<kCapSmall>(x, count, a->first_tensor, h, dyn, eight, a->use_ema != 0, sms, st)
                            : launch_update<kCap>(x, count, a->first_tensor, h, dyn, eight, a->use_ema != 0, sms, st);
}

int kda_grad_norm(const KdaAdamWTensor *x, int64_t count, float *norm, void *ws, size_t ws_bytes, void *stream) {
  int s = check_tensors(x, count);
  if (s) return s;
  if (!norm || !multiple(norm, 4)) return KDA_ERR_INVALID_ARG;
  const int sms = sm_count();
  if (!sms) return KDA_ERR_CUDA;
  const int64_t most = max_parts(count, sms);
  if (count && (!ws || !multiple(ws, 16) || ws_bytes < kDynBytes + (size_t)most * sizeof(double))) return KDA_ERR_WORKSPACE;
  double *partial = count ? reinterpret_cast<double *>(static_cast<char *>(ws) + kDynBytes) : nullptr;
  cudaStream_t st = (cudaStream_t)stream;
  int parts = 0;
  s = count <= kCapSmall ? launch_squares<kCapSmall>(x, count, partial, (int)most, parts, sms, st)
                         : launch_squares<kCap>(x, count, partial, (int)most, parts, sms, st);
  if (s) return s;
  Prep pr = {};
  pr.parts = parts;
  prep_kernel<<<1, kThreads, 0, st>>>(pr, partial, norm, nullptr);
  return launched();
}

int kda_decode_state8(int64_t n, int is_signed, const uint8_t *code, const uint8_t *exp, void *out, void *stream) {
  if (n < 0 || (n && (!code || !exp || !out))) return KDA_ERR_INVALID_ARG;
  if (!n) return KDA_OK;
  if (!multiple(out, 2)) return KDA_ERR_MISALIGNED;
  const int sms = sm_count();
  if (!sms) return KDA_ERR_CUDA;
  const int64_t need = (n + kPass - 1) / kPass, most = (int64_t)sms * kCtasPerSmRead;
  const int grid = (int)(need < most ? need : most);
  const bool vec = multiple(code, 8) && multiple(out, 16);
  cudaStream_t st = (cudaStream_t)stream;
  if (is_signed) decode_kernel<true><<<grid, kThreads, 0, st>>>(n, code, exp, static_cast<__nv_bfloat16 *>(out), vec);
  else decode_kernel<false><<<grid, kThreads, 0, st>>>(n, code, exp, static_cast<__nv_bfloat16 *>(out), vec);
  return launched();
}

}  // extern "C"
