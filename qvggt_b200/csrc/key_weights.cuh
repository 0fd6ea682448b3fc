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
  uint32_t chunk_mul, chunk_shift;       // division by chunk
  int row_blocks;                        // 1: a request is one entry of scan_blocks
  float scale_log2, decay;
  uint32_t wait_tries;                   // bound of every wait
  Ctl ctl;
};

constexpr float LOG2E = 1.4426950408889634f;

// key_weights_sm100.cu (many rows): whether its TMA map can read these queries; the launch.
bool key_weight_tiles_can_read(const KeyWeightArgs& a);
int launch_key_weight_tiles(KeyWeightArgs& a, int D, bool bf16, cudaStream_t stream);

}  // namespace qv
