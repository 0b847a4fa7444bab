// The softmax of the tensor-core attention kernels (sm_100a): a thread owns a query
// row, its scores in registers, against a lazy running maximum in base 2.
#pragma once
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include "sd_common.cuh"
#include "sd_tcgen05.cuh"

namespace sd {

constexpr float PX_HEADROOM = 8.f;           // lazy-rescale headroom of the running max (base 2)
// Largest maximum (base 2) whose scores go through fma(s, sl2, -m).  m is the float
// next to s sl2 of the largest score: from 2^31 on it may be more than 128 away
// from it, and 2^(s sl2 - m) leaves the float range; up to 2^20, 1/32.
constexpr float PX_TAME = 1048576.f;

__device__ __forceinline__ void px_max3(float& m, uint32_t a, uint32_t b) {
  asm("max.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)));
}

// (2^a, 2^b) on the FMA pipe: with a = i + f, i the nearest integer, 2^f by a
// polynomial of degree 4 on [-1/2, 1/2] (least relative error, 2.7e-6) times
// 2^i, whose bits the rounding constant leaves in place.  Held at i = -127, whose
// bits are those of 0: a masked score (-inf) weighs nothing.  A NaN stays one.
__device__ __forceinline__ unsigned long long px_exp2(float a, float b) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(-127.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(-127.f));
  const float magic = 12582912.f + 127.f;            // 1.5 * 2^23: the sum's low byte is i + 127
  const unsigned long long x2 = pair2(a, b), r2 = add2(x2, pair2(magic, magic));
  const unsigned long long i2 = add2(r2, pair2(-magic, -magic));
  const unsigned long long f2 = fma2(i2, pair2(-1.f, -1.f), x2);
  unsigned long long p2 = pair2(0.009570100344717503f, 0.009570100344717503f);
  p2 = fma2(p2, f2, pair2(0.05591785907745361f, 0.05591785907745361f));
  p2 = fma2(p2, f2, pair2(0.240247443318367f, 0.240247443318367f));
  p2 = fma2(p2, f2, pair2(0.6931217908859253f, 0.6931217908859253f));
  p2 = fma2(p2, f2, pair2(0.9999992847442627f, 0.9999992847442627f));
  float ra, rb;
  unpair(r2, ra, rb);
  return mul2(p2, pair2(__uint_as_float(__float_as_uint(ra) << 23),
                        __uint_as_float(__float_as_uint(rb) << 23)));
}

// The weights p = 2^(s sl2 - m) of 32 scores as bf16 pairs, and their sums.  A
// quarter by the FMA pipe: the exponentials of a page take 2048 cycles of the
// special-function units otherwise (shared ranges: a call of 101.3 us took 102.5
// without, 103 with half of them there).
__device__ __forceinline__ void px_weights(const uint32_t (&s)[32], uint32_t* p,
                                           unsigned long long (&sum)[2], unsigned long long sl22,
                                           unsigned long long nm2) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    float a, b;
    const unsigned long long s2 = pair2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1]));
    unpair(fma2(s2, sl22, nm2), a, b);
    const unsigned long long p2 = e % 4 == 1 ? px_exp2(a, b) : pair2(ex2f(a), ex2f(b));
    sum[e & 1] = add2(sum[e & 1], p2);
    unpair(p2, a, b);
    p[e] = pack_bf16(a, b);
  }
}

// Beyond PX_TAME the scores are scaled first, with a rounding of their own: the
// largest one's exponent is 0 again.  (Rare; px_weights then gets a factor of 1.)
__device__ __forceinline__ bool px_wild(float m) {
  return __any_sync(0xffffffffu, fabsf(m) > PX_TAME && m != -CUDART_INF_F);
}
__device__ __forceinline__ void px_scale(uint32_t (&s)[32], float sl2) {
#pragma unroll
  for (int e = 0; e < 32; ++e) s[e] = __float_as_uint(__fmul_rn(__uint_as_float(s[e]), sl2));
}

}  // namespace sd
