// What cached keys have gathered: for key j of a request
//   out_j = decay w_j + sum_{rows i that see j} 2^(scale log2e ks_B (q_i . c_j) - lse_i log2e),
// a row being a (token, query head of the group) pair.  The product's operands
// are the queries and the codes themselves (exact in fp16 and bf16); the scale
// of the key's (block, head) is one factor of the exponent.
#include "key_weights.cuh"
#include "attn_cache.cuh"
#include "attn_common.cuh"
#include "host.hpp"

namespace qv {
namespace {

constexpr int UNIT = 32;                 // keys a warp takes at a time: never across two blocks
constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int ROWS_MAX = 32;             // more rows of a key head go to key_weights_sm100.cu

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The codes are the M operand of mma.m16n8k16 and the rows its N: a lane reads
// 16 codes of one key at once, straight from memory into the fragments (any
// order of the dims will do, as the queries' fragments use the same), and the
// sum over rows is over a lane's registers and four lanes.  Nothing is shared
// between warps.  More than 8 NT rows are taken 8 NT at a time.
template <bool BF16, int D, int NT>
__global__ void __launch_bounds__(THREADS) key_weights_rows_kernel(KeyWeightArgs a, int ctas) {
  constexpr int KC = D / 64;             // 64-dim chunks
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int pair = blockIdx.x / ctas, kvh = pair % a.hk, b = pair / a.hk;
  const int q0 = a.cu_q[b], ql = a.cu_q[b + 1] - q0, n = a.kv_lens[b];
  if (q0 < 0 || ql < 0 || ql > a.max_q || (long long)q0 + ql > a.Tq || n < 0 || n > (a.wide << a.bs_log2)) {
    if (threadIdx.x == 0) report_status(a.ctl, ST_BAD_LENGTH);
    return;
  }
  const int fresh = a.fresh ? a.fresh[b] : n;
  const int bs = 1 << a.bs_log2, rows = ql * a.group;
  const int32_t* table = a.table + (long long)b * a.wide;
  const int units = (int)(((long long)n + UNIT - 1) / UNIT), stride = ctas * WARPS;

  uint2 qb[NT][KC][4];
  float nl[NT][2];                       // -lse log2e of rows 2t, 2t + 1 of each tile
  int lim[NT][2];                        // keys they see
  auto load_rows = [&](int row0) {
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const int row = min(row0 + 8 * x + g, rows - 1);
      const uint16_t* qp = a.q + (long long)(q0 + row / a.group) * a.q_tok + (long long)(kvh * a.group + row % a.group) * a.q_head;
#pragma unroll
      for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int s = 0; s < 4; ++s) qb[x][c][s] = *reinterpret_cast<const uint2*>(qp + 64 * c + 16 * t + 4 * s);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = row0 + 8 * x + 2 * t + e;
        const float l = r < rows ? a.lse[(long long)(kvh * a.group + r % a.group) * a.Tq + q0 + r / a.group] : INFINITY;
        nl[x][e] = -l * LOG2E;
        lim[x][e] = isfinite(l) ? key_limit(r / a.group, ql, n, a.chunk) : 0;
      }
    }
  };
  const bool once = rows <= 8 * NT;
  if (once && rows > 0) load_rows(0);

  for (int u0 = (blockIdx.x % ctas) * WARPS + warp; u0 < units; u0 += 32 * stride) {
    // lane i holds the block of unit u0 + i stride, and its scale
    const int mine = u0 + lane * stride;
    int id = -1;
    float ks = 0.f;
    if (mine < units) {
      id = table[(mine * UNIT) >> a.bs_log2];
      if (id < 0 || id >= a.num_blocks) {
        report_bad_block(a.ctl);
        id = -1;
      } else {
        ks = a.ks[(long long)id * a.hk + kvh];
      }
    }
    // the next unit's codes and old weight are on their way while one is used
    uint4 w[2][2][KC], wn[2][2][KC];     // keys 16 mt + 8 half + g
    float old = 0.f, old_n = 0.f;
    auto fetch = [&](int i) {
      const int blk = __shfl_sync(~0u, id, i);
      if (i < 32 && blk >= 0) {
        const int key0 = (u0 + i * stride) * UNIT;
        const int8_t* kp = a.kc + blk * a.block_stride + ((long long)kvh * bs + (key0 & (bs - 1))) * D;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int c = 0; c < KC; ++c)
              wn[mt][half][c] = __ldg(reinterpret_cast<const uint4*>(kp + (16 * mt + 8 * half + g) * D + 64 * c + 16 * t));
        const int key = key0 + 16 * (t / 2) + 8 * (t % 2) + g;
        old_n = key < n && key < fresh ? a.w[(((long long)blk * a.hk + kvh) << a.bs_log2) + (key & (bs - 1))] : 0.f;
      }
    };
    fetch(0);
    for (int i = 0; i < 32 && u0 + i * stride < units; ++i) {
      const int blk = __shfl_sync(~0u, id, i);
      const float ck = __shfl_sync(~0u, ks, i) * a.scale_log2;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int c = 0; c < KC; ++c) w[mt][half][c] = wn[mt][half][c];
      old = old_n * a.decay;
      fetch(i + 1);                      // (of unit 32 nothing: its lane is outside the batch)
      if (blk < 0) continue;
      const int key0 = (u0 + i * stride) * UNIT;
      // the place this lane writes: key 16 (t / 2) + 8 (t % 2) + g
      const int key = key0 + 16 * (t / 2) + 8 * (t % 2) + g;
      const long long place = (((long long)blk * a.hk + kvh) << a.bs_log2) + (key & (bs - 1));
      float sum[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
      for (int row0 = 0; row0 < rows; row0 += 8 * NT) {
        if (!once) load_rows(row0);
        float s[NT][2][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
          for (int x = 0; x < NT; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[x][mt][e] = 0.f;
#pragma unroll
          for (int c = 0; c < KC; ++c) {
            const uint32_t x0[4] = {w[mt][0][c].x, w[mt][0][c].y, w[mt][0][c].z, w[mt][0][c].w};
            const uint32_t x1[4] = {w[mt][1][c].x, w[mt][1][c].y, w[mt][1][c].z, w[mt][1][c].w};
#pragma unroll
            for (int sp = 0; sp < 4; ++sp) {
              const uint32_t ka[4] = {codes2<BF16, false>(x0[sp]), codes2<BF16, false>(x1[sp]),
                                      codes2<BF16, true>(x0[sp]), codes2<BF16, true>(x1[sp])};
#pragma unroll
              for (int x = 0; x < NT; ++x) mma16816<BF16>(s[x][mt], ka, qb[x][c][sp].x, qb[x][c][sp].y);
            }
          }
        }
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float p = ex2(fmaf(s[x][mt][e], ck, nl[x][e & 1]));
              sum[mt][e >> 1] += key0 + 16 * mt + 8 * (e >> 1) + g < lim[x][e & 1] ? p : 0.f;
            }
      }
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          sum[mt][half] += __shfl_xor_sync(~0u, sum[mt][half], 1);
          sum[mt][half] += __shfl_xor_sync(~0u, sum[mt][half], 2);
        }
      const float mine_sum = t < 2 ? (t ? sum[0][1] : sum[0][0]) : (t & 1 ? sum[1][1] : sum[1][0]);
      if (key < n) a.out[place] = old + mine_sum;
    }
  }
}

}  // namespace
}  // namespace qv

using namespace qv;

extern "C" int qvggt_key_weights(const qvggt_key_weights_args* p, void* stream) {
  const char* name = "key_weights";
  if (!p) return set_error(QVGGT_ERR_INVALID, "%s: null arguments", name);
  if (p->num_blocks <= 0 || p->kv_heads <= 0 || p->q_heads <= 0 || p->Tq < 0 || p->requests < 0 || p->max_blocks < 0 ||
      p->max_q < 0 || p->max_kv < 0 || p->causal_chunk < 0)
    return set_error(QVGGT_ERR_INVALID, "%s: bad shape", name);
  if (p->q_heads % p->kv_heads)
    return set_error(QVGGT_ERR_INVALID, "%s: %lld query heads do not share %lld key heads evenly", name,
                     (long long)p->q_heads, (long long)p->kv_heads);
  if (p->block_size != 32 && p->block_size != 64 && p->block_size != 128)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: block_size must be 32, 64 or 128", name);
  if (p->head_dim != 64 && p->head_dim != 128)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128", name);
  if (p->dtype != QVGGT_DTYPE_F16 && p->dtype != QVGGT_DTYPE_BF16)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: dtype must be fp16 or bf16", name);
  if (!(p->scale > 1e-30) || p->scale > 1e30) return set_error(QVGGT_ERR_INVALID, "%s: scale must be positive", name);
  if (!(p->decay >= 0) || p->decay > 1) return set_error(QVGGT_ERR_INVALID, "%s: decay must be 0 to 1", name);
  if (p->q_heads > 65535 || p->Tq > 2147483647LL / p->q_heads || p->max_q > 2147483647LL / p->q_heads ||
      p->max_kv > 2147483647LL || p->requests > 1 << 24 || p->num_blocks > 2147483647LL / p->block_size ||
      p->max_blocks > (2147483647LL - 127) / p->block_size)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: too many rows, requests or keys", name);
  if (p->requests == 0 || p->max_blocks == 0) return QVGGT_OK;
  if (!p->k_cache || !p->k_scale || !p->block_tables || !p->cu_q || !p->kv_lens || !p->weights || !p->out ||
      (p->Tq && (!p->q || !p->lse)))
    return set_error(QVGGT_ERR_INVALID, "%s: null tensor", name);
  if (!aligned16(p->k_cache) || p->block_stride % 16)
    return set_error(QVGGT_ERR_ALIGN, "%s: cache codes and their block stride must be 16-byte aligned", name);
  if (p->block_stride < p->kv_heads * p->block_size * p->head_dim)
    return set_error(QVGGT_ERR_INVALID, "%s: block stride smaller than a block", name);
  if (!aligned16(p->q) || p->q_tok % 8 || p->q_head % 8)
    return set_error(QVGGT_ERR_ALIGN, "%s: q rows must be 16-byte aligned", name);
  KeyWeightArgs a{};
  a.kc = p->k_cache;
  a.ks = p->k_scale;
  a.q = static_cast<const uint16_t*>(p->q);
  a.lse = p->lse;
  a.table = p->block_tables;
  a.cu_q = p->cu_q;
  a.kv_lens = p->kv_lens;
  a.fresh = p->fresh_from;
  a.w = p->weights;
  a.out = p->out;
  a.q_tok = p->q_tok;
  a.q_head = p->q_head;
  a.block_stride = p->block_stride;
  a.Tq = p->Tq;
  a.B = (int)p->requests;
  a.hq = (int)p->q_heads;
  a.hk = (int)p->kv_heads;
  a.group = a.hq / a.hk;
  a.wide = (int)p->max_blocks;
  a.num_blocks = (int)p->num_blocks;
  a.bs_log2 = p->block_size == 32 ? 5 : p->block_size == 64 ? 6 : 7;
  a.chunk = (int)std::min<int64_t>(p->causal_chunk, 1 << 30);
  a.max_q = (int)p->max_q;
  a.scale_log2 = (float)(p->scale * 1.4426950408889634);
  a.decay = (float)p->decay;
  a.ctl = make_ctl();
  const bool bf16 = p->dtype == QVGGT_DTYPE_BF16;
  const long long rows = (long long)a.max_q * a.group, pairs = (long long)a.hk * a.B;
  if (rows > ROWS_MAX && key_weight_tiles_can_read(a))
    return launch_key_weight_tiles(a, (int)p->head_dim, bf16, static_cast<cudaStream_t>(stream));
  const long long units = std::max<long long>(1, (p->max_kv + UNIT - 1) / UNIT);
  // about eight CTAs per SM and at most eight units a warp before a CTA takes more
  const long long per = std::max<long long>(1, std::min<long long>(8, units * pairs / (32LL * device_info().num_sms)));
  const long long ctas = (units + WARPS * per - 1) / (WARPS * per);
  if (ctas * pairs > 2147483647LL || ctas * WARPS * 32 > 2147483647LL / UNIT)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: too many requests and keys", name);
  using Kfn = void (*)(KeyWeightArgs, int);
  static const Kfn fns[2][2][3] = {{{key_weights_rows_kernel<false, 64, 1>, key_weights_rows_kernel<false, 64, 2>,
                                     key_weights_rows_kernel<false, 64, 4>},
                                    {key_weights_rows_kernel<false, 128, 1>, key_weights_rows_kernel<false, 128, 2>,
                                     key_weights_rows_kernel<false, 128, 4>}},
                                   {{key_weights_rows_kernel<true, 64, 1>, key_weights_rows_kernel<true, 64, 2>,
                                     key_weights_rows_kernel<true, 64, 4>},
                                    {key_weights_rows_kernel<true, 128, 1>, key_weights_rows_kernel<true, 128, 2>,
                                     key_weights_rows_kernel<true, 128, 4>}}};
  const Kfn fn = fns[bf16][p->head_dim == 128][rows <= 8 ? 0 : rows <= 16 ? 1 : 2];
  int rc = check_cuda(launch_pdl(fn, dim3((unsigned)(ctas * pairs)), dim3(THREADS), 0, static_cast<cudaStream_t>(stream),
                                 1u, a, (int)ctas),
                      "key_weights launch");
  if (!rc) count_launch(1);
  return rc;
}
