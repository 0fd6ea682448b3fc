// Attention over a paged K/V cache in 8 bits: what the kernels share.
//
// With code c of a key's element and the scales ks_B, vs_B of its (block,
// head), the row's result is
//   out = sum_j w_j vs_B(j) c_v[j] / sum_j w_j,   w_j = exp(scale ks_B(j) q.c_k[j]).
// Neither scale is multiplied into the rows.  With
//   x_j = (scale log2e ks_B) (q.c_k[j]) + log2 vs_B,   P_j = 2^(x_j - m),
// the products q.c_k and P.c_v have the codes themselves as operands (exact in
// fp16 and bf16), m = max x_j keeps every P_j (which now holds the V scale) in
// fp16's range, and the denominator is sum_B (1 / vs_B) sum_{j in B} P_j.
#pragma once

#include "kv_cache.cuh"

namespace qv {

struct CacheAttnArgs {
  const uint16_t* q;
  uint16_t* out;
  float* lse;                            // [heads][Tq] or null
  const int8_t *kc, *vc;
  const float *ks, *vs;
  const int32_t *table, *cu_q, *kv_lens;
  float *part_o, *part_lse;              // parts of rows, and their log2-sum-exp
  long long q_tok, q_head, o_tok, o_head, block_stride, Tq;
  int B, hq, hk, group, wide, num_blocks, bs_log2, chunk, max_q, splits;
  int row_blocks;                        // Q blocks (16-row tiles) of the longest request
  int can_split;                         // tile kernel: items may be cut, a join follows
  float scale_log2;
  uint32_t wait_tries;                   // tile kernel: bound of every wait
  Ctl ctl;
};

// Keys that query i (of ql) of a request with n keys sees.
__device__ __forceinline__ int key_limit(int i, int ql, int n, int chunk) {
  if (!chunk) return n;
  const int pos = n - ql + i;
  if (pos < 0) return 0;
  const long long lim = ((long long)(pos / chunk) + 1) * chunk;
  return lim < n ? (int)lim : n;
}

// Two codes (bytes 0 and 1, or 2 and 3 with HI, of w) as a pair of fp16 / bf16.
// fp16: the byte with its sign bit flipped (c + 128) placed under the exponent
// of 1024 reads 1024 + c + 128; subtracting 1152 is exact.
template <bool HI>
__device__ __forceinline__ uint32_t codes_f16(uint32_t flipped) {
  const uint32_t u = __byte_perm(flipped, 0x64646464u, HI ? 0x4342 : 0x4140);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&u), __float2half2_rn(1152.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// bf16 holds 7 fraction bits, one short of that: 128 + (c & 127) minus 128, or
// minus 256 where c is negative; both have the form 0x4300 | bits of c.
template <bool HI>
__device__ __forceinline__ uint32_t codes_bf16(uint32_t w) {
  const uint32_t u = __byte_perm(w, 0u, HI ? 0x4342 : 0x4140);
  const uint32_t x = (u & 0x007f007fu) | 0x43004300u, y = (u & 0x00800080u) | 0x43004300u;
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x),
                                   *reinterpret_cast<const __nv_bfloat162*>(&y));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <bool BF16, bool HI>
__device__ __forceinline__ uint32_t codes2(uint32_t w) {
  return BF16 ? codes_bf16<HI>(w) : codes_f16<HI>(w ^ 0x80808080u);
}

// attn_cache_sm100.cu (many rows): whether its TMA map can read these queries;
// the scratch for `items` (request, Q block, kv head) triples; the launches.
bool tiles_can_read(const CacheAttnArgs& a);
int64_t tiles_scratch(long long items, long long max_kv, int D);
int launch_tiles(CacheAttnArgs& a, int D, bool bf16, long long max_kv, void* scratch, cudaStream_t stream);

}  // namespace qv
