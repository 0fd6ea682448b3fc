// Pieces the tcgen05 attention kernels share: bounded waits that keep no
// registers, the exponential on both pipes, named barriers.
#pragma once

#include "common.cuh"

namespace qv {

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Bounded mbarrier wait.  Its failure bookkeeping (abort flag, status word
// pointer, timeout) is read from shared memory at `misc` only once the first
// try_wait fails, so a thread keeps no registers for it across its loop (held
// in registers, it pushed parts of a softmax thread's 128-score row to local
// memory).
__device__ __forceinline__ bool wait_slow(uint32_t bar, uint32_t parity, uint32_t misc, uint32_t code) {
  int ab;
  uint64_t status, timeout;
  asm volatile("ld.shared.u64 %0, [%1 + 8];" : "=l"(status) : "r"(misc));
  asm volatile("ld.shared.u64 %0, [%1 + 16];" : "=l"(timeout) : "r"(misc));
  const uint64_t t0 = globaltimer_ns();
#pragma unroll 1
  while (true) {
    asm volatile("ld.volatile.shared.s32 %0, [%1 + 4];" : "=r"(ab) : "r"(misc) : "memory");
    if (ab) return false;
#pragma unroll 1
    for (int k = 0; k < 16; ++k)
      if (mbar_try_wait(bar, parity)) return true;
    if (globaltimer_ns() - t0 > timeout) {
      asm volatile("st.volatile.shared.s32 [%0 + 4], 1;" ::"r"(misc) : "memory");
      if (status) atomicCAS(reinterpret_cast<uint32_t*>(status), 0u, code);
      return false;
    }
  }
}

__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, uint32_t misc, uint32_t code) {
  return mbar_try_wait(bar, parity) || wait_slow(bar, parity, misc, code);
}
__device__ __forceinline__ bool wait(const uint64_t* bar, uint32_t parity, uint32_t misc, uint32_t code) {
  return wait(smem_u32(bar), parity, misc, code);
}

// The softmax warps' wait (barrier given by its shared-memory address): all
// lanes wait; the warp proceeds only if all saw the phase complete.
__device__ __forceinline__ bool softmax_wait(uint32_t bar, uint32_t parity, uint32_t misc) {
  return __all_sync(0xffffffffu, wait(bar, parity, misc, ST_TIMEOUT_SOFTMAX));
}

__device__ __forceinline__ void fence_acq_rel_gpu() { asm volatile("fence.acq_rel.gpu;" ::: "memory"); }

// Named barrier `id` over `count` threads (whole warps).
__device__ __forceinline__ void named_bar_sync(uint32_t id, uint32_t count) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(count) : "memory");
}

__device__ __forceinline__ uint32_t atom_add_acq_rel_gpu(uint32_t* p, uint32_t v) {
  uint32_t old;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
  return old;
}

__device__ __forceinline__ void arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// tcgen05.ld writes its destination registers asynchronously: they are valid
// only after tcgen05.wait::ld.  This empty asm takes s[A..B) as in-out
// operands after the wait, so the compiler cannot move reads of them above it.
template <int A, int B, int N>
__device__ __forceinline__ void reg_fence(uint32_t (&s)[N]) {
#pragma unroll
  for (int k = A; k < B; ++k) asm volatile("" : "+r"(s[k]));
}

// 2^x for a pair of arguments on the FMA pipe (Cody-Waite range reduction:
// x = n + f, n = round(x), f in [-1/2, 1/2]; 2^f by a degree-3 polynomial
// fitted to minimise the relative error on [-1/2, 1/2] (max 7.5e-5, well under
// the fp16 rounding P gets afterwards); 2^n added into the exponent field).
// Arguments are clamped at -125 so 2^n stays a normal float; those values
// round to 0 in fp16 anyway.
__device__ __forceinline__ void exp2_poly_pair(uint64_t x2, float& p0, float& p1) {
  const uint64_t MAGIC = f2_pack(12582912.0f, 12582912.0f);        // 1.5 * 2^23: rounds to an integer
  const uint64_t NEG_MAGIC = f2_pack(-12582912.0f, -12582912.0f);
  const uint64_t NEG_ONE = f2_pack(-1.0f, -1.0f);
  const uint64_t C0 = f2_pack(0.99992806f, 0.99992806f), C1 = f2_pack(0.69326097f, 0.69326097f);
  const uint64_t C2 = f2_pack(0.24261114f, 0.24261114f), C3 = f2_pack(0.05517166f, 0.05517166f);
  float x0, x1;
  f2_unpack(x2, x0, x1);
  const uint64_t xc = f2_pack(fmaxf(x0, -125.f), fmaxf(x1, -125.f));
  const uint64_t t = f2_add(xc, MAGIC);          // low mantissa bits hold n
  const uint64_t nf = f2_add(t, NEG_MAGIC);      // n as a float
  const uint64_t f = f2_fma(nf, NEG_ONE, xc);    // x - n
  uint64_t p = f2_fma(C3, f, C2);
  p = f2_fma(p, f, C1);
  p = f2_fma(p, f, C0);
  float q0, q1, t0, t1;
  f2_unpack(p, q0, q1);
  f2_unpack(t, t0, t1);
  p0 = __int_as_float(__float_as_int(q0) + (__float_as_int(t0) << 23));
  p1 = __int_as_float(__float_as_int(q1) + (__float_as_int(t1) << 23));
}

}  // namespace qv
