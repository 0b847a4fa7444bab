// Tensor-core plumbing of the attention kernels (sm_100a): shared-memory and
// instruction descriptors, tcgen05.mma / ld / st / commit, mbarriers with
// bounded waits, TMA tile loads.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace sd {

constexpr long long TC_WAIT = 1LL << 31; // cycles (~1 s) before a wait gives up

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint64_t tc_desc(uint32_t addr, uint32_t lbo, uint32_t sbo,
                                            uint32_t layout) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)((lbo >> 4) & 0x3FFF) << 16) |
         ((uint64_t)((sbo >> 4) & 0x3FFF) << 32) | ((uint64_t)1 << 46) |
         ((uint64_t)(layout & 7) << 61);
}
// kind::f16 instruction descriptor: bf16 A and B, f32 D, M x N, majors
__host__ __device__ constexpr uint32_t tc_idesc(int M, int N, int a_mn, int b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t id, int acc) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
               :: "r"(d), "l"(a), "l"(b), "r"(id), "r"(acc) : "memory");
}
__device__ __forceinline__ void tc_commit(unsigned long long* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
               :: "r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void tc_bar_init(unsigned long long* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(smem_addr(bar)), "r"(count)
               : "memory");
}
__device__ __forceinline__ void tc_arrive(unsigned long long* bar) {
  asm volatile("{\n .reg .b64 st;\n mbarrier.arrive.shared::cta.b64 st, [%0];\n}"
               :: "r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void tc_expect_tx(unsigned long long* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;"
               :: "r"(smem_addr(bar)), "r"(bytes) : "memory");
}
// Has the phase of parity `par` completed?  (non-blocking)
__device__ __forceinline__ bool tc_test(unsigned long long* bar, uint32_t par) {
  uint32_t done;
  asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
               " selp.u32 %0, 1, 0, p;\n}" : "=r"(done) : "r"(smem_addr(bar)), "r"(par)
               : "memory");
  return done != 0;
}
// Bounded wait for the phase of parity `par`; false (and the CTA's abort
// flag set) on expiry or when another thread already gave up.
__device__ __forceinline__ bool tc_wait(unsigned long long* bar, uint32_t par, int* abort_) {
  long long t0 = 0;
  while (true) {
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
                 " selp.u32 %0, 1, 0, p;\n}" : "=r"(done) : "r"(smem_addr(bar)), "r"(par)
                 : "memory");
    if (done) return true;
    if (t0 == 0) t0 = clock64();                       // (a phase already there costs no clock read)
    if (*reinterpret_cast<volatile int*>(abort_) || clock64() - t0 > TC_WAIT) {
      *reinterpret_cast<volatile int*>(abort_) = 1;
      return false;
    }
  }
}
// Warp-wide issue: every lane calls, one elected lane issues, and control flow
// stays uniform.  (Under `if (lane == 0)` the operands' way to the uniform
// registers is set up again after every wait: some 200 cycles each, while the
// tensor queue runs dry.)
__device__ __forceinline__ void tc_mma_warp(uint32_t d, uint64_t a, uint64_t b, uint32_t id,
                                            int acc) {
  asm volatile("{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
               " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
               :: "r"(d), "l"(a), "l"(b), "r"(id), "r"(acc) : "memory");
}
// A in tensor memory
__device__ __forceinline__ void tc_mma_ts_warp(uint32_t d, uint32_t a, uint64_t b, uint32_t id,
                                               int acc) {
  asm volatile("{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
               " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
               :: "r"(d), "r"(a), "l"(b), "r"(id), "r"(acc) : "memory");
}
// D[lanes that `off` leaves on] (+)= A[shared] B[shared]: a set bit of off keeps
// its accumulator lane (quarter i: bits of off[i]) as it is
__device__ __forceinline__ void tc_mma_lanes_warp(uint32_t d, uint64_t a, uint64_t b, uint32_t id,
                                                  const uint32_t (&off)[4], int acc) {
  asm volatile("{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
               " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n}"
               :: "r"(d), "l"(a), "l"(b), "r"(id), "r"(acc), "r"(off[0]), "r"(off[1]), "r"(off[2]),
                  "r"(off[3]) : "memory");
}
// The same with A in tensor memory
__device__ __forceinline__ void tc_mma_ts_lanes_warp(uint32_t d, uint32_t a, uint64_t b, uint32_t id,
                                                     const uint32_t (&off)[4], int acc) {
  asm volatile("{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
               " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n}"
               :: "r"(d), "r"(a), "l"(b), "r"(id), "r"(acc), "r"(off[0]), "r"(off[1]), "r"(off[2]),
                  "r"(off[3]) : "memory");
}
__device__ __forceinline__ void tc_commit_warp(unsigned long long* bar) {
  asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n"
               " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}"
               :: "r"(smem_addr(bar)) : "memory");
}
// tc_wait on two phases at once, by a whole warp.
__device__ __forceinline__ bool tc_wait2_warp(unsigned long long* b0, uint32_t p0,
                                              unsigned long long* b1, uint32_t p1, int* abort_) {
  long long t0 = 0;
  while (true) {
    uint32_t done;
    asm volatile("{\n .reg .pred p, q;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
                 " mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n"
                 " and.pred p, p, q;\n selp.u32 %0, 1, 0, p;\n}"
                 : "=r"(done) : "r"(smem_addr(b0)), "r"(p0), "r"(smem_addr(b1)), "r"(p1)
                 : "memory");
    if (__all_sync(0xffffffffu, done != 0u)) return true;
    if (t0 == 0) t0 = clock64();
    const bool stop = *reinterpret_cast<volatile int*>(abort_) || clock64() - t0 > TC_WAIT;
    if (__any_sync(0xffffffffu, stop)) {
      *reinterpret_cast<volatile int*>(abort_) = 1;
      return false;
    }
  }
}
__device__ __forceinline__ void tc_tma_2d(void* dst, const void* tmap, int x, int y,
                                          unsigned long long* bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
               " [%0], [%1, {%2, %3}], [%4];"
               :: "r"(smem_addr(dst)), "l"(tmap), "r"(x), "r"(y), "r"(smem_addr(bar))
               : "memory");
}
// A cache policy for data that is read once, and a load under a policy
__device__ __forceinline__ uint64_t tc_evict_first() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void tc_tma_2d(void* dst, const void* tmap, int x, int y,
                                          unsigned long long* bar, uint64_t policy) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
               ".L2::cache_hint [%0], [%1, {%2, %3}], [%4], %5;"
               :: "r"(smem_addr(dst)), "l"(tmap), "r"(x), "r"(y), "r"(smem_addr(bar)), "l"(policy)
               : "memory");
}
#define TC_LD32(r, addr)                                                                        \
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,"    \
               "%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"  \
               "%30,%31}, [%32];"                                                               \
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),        \
                 "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),     \
                 "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), \
                 "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), \
                 "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), \
                 "=r"(r[30]), "=r"(r[31])                                                      \
               : "r"(addr) : "memory")
#define TC_ST32(addr, r)                                                                        \
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,"  \
               "%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"  \
               "%30,%31,%32};"                                                                  \
               :: "r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), \
                 "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),\
                 "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),       \
                 "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),       \
                 "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),       \
                 "r"(r[31]) : "memory")
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

}  // namespace sd
