// Shared pieces of the 8-bit K/V cache kernels.
#pragma once

#include <algorithm>

#include "../../include/qvggt_b200.h"
#include "common.cuh"

namespace qv {

// Smallest scale of a (block, head): keeps 1 / s and log2 s ordinary floats
// (attention adds log2 of the V scale to its scores), far under what fp16 or
// any useful bf16 value needs (codes of a block below 127 * 2^-60 lose digits).
constexpr float KV_SCALE_MIN = 8.673617379884035e-19f;   // 2^-60

// A block id outside the cache was met (the keys or rows of it are skipped).
enum : uint32_t { ST_BAD_BLOCK = 0x201, ST_BAD_LENGTH = 0x202 };

__device__ __forceinline__ void report_status(const Ctl& ctl, uint32_t code) {
  if (ctl.status) atomicCAS(ctl.status, 0u, code);
}
__device__ __forceinline__ void report_bad_block(const Ctl& ctl) { report_status(ctl, ST_BAD_BLOCK); }

template <bool BF16>
__device__ __forceinline__ float half_bits_to_f32(uint16_t u) {
  if (BF16) return __uint_as_float((uint32_t)u << 16);
  return __half2float(__ushort_as_half(u));
}

// Code of x / s, given x * (1 / s): nearest, ties to even, within +-127; NaN gives 0.
__device__ __forceinline__ int8_t kv_code(float x) {
  return f32_to_s8_rni_sat(fminf(fmaxf(x != x ? 0.f : x, -127.f), 127.f));
}

// Checks of the cache's tensors that every entry point makes; sets the error.
int check_cache(const char* name, const qvggt_kv_cache& c);

}  // namespace qv
