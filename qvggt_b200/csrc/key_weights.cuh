// What cached keys have gathered: what the kernels share.
#pragma once

#include "kv_cache.cuh"

namespace qv {

struct KeyWeightArgs {
  const int8_t* kc;
  const float* ks;
  const uint16_t* q;
  const float* lse;                      // [heads][Tq]
  const int32_t *table, *cu_q, *kv_lens, *fresh;   // fresh: null where all keys add to what they have
  const float* w;
  float* out;
  long long q_tok, q_head, block_stride, Tq;
  int B, hq, hk, group, wide, num_blocks, bs_log2, chunk, max_q;
  float scale_log2, decay;
  uint32_t wait_tries;                   // bound of every wait
  Ctl ctl;
};

constexpr float LOG2E = 1.4426950408889634f;

}  // namespace qv
