// Attention over a paged K/V cache in 8 bits, few query rows
// (the mathematics is in attn_cache.cuh).
#include "attn_cache.cuh"
#include "attn_common.cuh"
#include "host.hpp"

namespace qv {
namespace {

constexpr int TOK_WARPS = 4;
constexpr int TOK_ROWS = 16;             // (query, head) rows of a tile: the M of mma.m16n8k16
constexpr int UNIT = 32;                 // keys a warp takes at a time: never across two blocks
constexpr int MAX_SPLITS = 64;

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

// One CTA per (16 rows, kv head, request, split of the keys); its warps take
// every fourth 32-key unit and merge at the end.
template <bool BF16, int D>
__global__ void __launch_bounds__(TOK_WARPS * 32) attn_cache_rows_kernel(CacheAttnArgs a) {
  constexpr int KC = D / 64;              // 64-dim chunks
  __shared__ float sm_o[TOK_WARPS][TOK_ROWS][D];
  __shared__ float sm_m[TOK_WARPS][TOK_ROWS], sm_l[TOK_WARPS][TOK_ROWS];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int kvh = blockIdx.y % a.hk, b = blockIdx.y / a.hk, sp = blockIdx.z;
  const int q0 = a.cu_q[b], ql = a.cu_q[b + 1] - q0;
  int n = a.kv_lens[b];
  if (q0 < 0 || ql < 0 || ql > a.max_q || (long long)q0 + ql > a.Tq || n < 0 || n > (a.wide << a.bs_log2)) {
    if (threadIdx.x == 0) report_status(a.ctl, ST_BAD_LENGTH);
    return;
  }
  const int rows = ql * a.group, row0 = blockIdx.x * TOK_ROWS;
  if (row0 >= rows) return;

  // rows g and g + 8 of the tile
  int lim[2];
  const uint16_t* qp[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = min(row0 + g + 8 * r, rows - 1);
    const int i = row / a.group, h = kvh * a.group + row % a.group;
    lim[r] = row0 + g + 8 * r < rows ? key_limit(i, ql, n, a.chunk) : 0;
    qp[r] = a.q + (long long)(q0 + i) * a.q_tok + (long long)h * a.q_head;
  }
  // A fragments: step s of chunk c takes dims 64c + 16t + 4s + {0, 1} as k
  // columns 2t, 2t+1 and {2, 3} as 2t+8, 2t+9 (any order of the dims will do,
  // as K's fragments use the same)
  uint32_t qa[KC][4][4];
#pragma unroll
  for (int c = 0; c < KC; ++c)
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint2 w = *reinterpret_cast<const uint2*>(qp[r] + 64 * c + 16 * t + 4 * s);
        qa[c][s][r] = w.x;
        qa[c][s][2 + r] = w.y;
      }
  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  // keys any row of the tile sees, cut into the splits
  const int last_lim = key_limit((min(rows, row0 + TOK_ROWS) - 1) / a.group, ql, n, a.chunk);
  const int units = (last_lim + UNIT - 1) / UNIT;
  const int u0 = (int)((long long)sp * units / a.splits), u1 = (int)((long long)(sp + 1) * units / a.splits);
  const int bs = 1 << a.bs_log2;
  for (int u = u0 + warp; u < u1; u += TOK_WARPS) {
    const int key0 = u * UNIT;
    const int blk = a.table[(long long)b * a.wide + (key0 >> a.bs_log2)];
    if (blk < 0 || blk >= a.num_blocks) {
      if (lane == 0) report_bad_block(a.ctl);
      continue;
    }
    const long long off = blk * a.block_stride + ((long long)kvh * bs + (key0 & (bs - 1))) * D;
    const float ck = a.ks[(long long)blk * a.hk + kvh] * a.scale_log2;
    const float vs = a.vs[(long long)blk * a.hk + kvh];
    const float lv = log2f(vs), inv_vs = 1.f / vs;
    const int8_t* kp = a.kc + off;
    const int8_t* vp = a.vc + off;
    float s[4][4];
#pragma unroll
    for (int nt = 0; nt < 4; ++nt) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const uint4 w = *reinterpret_cast<const uint4*>(kp + (nt * 8 + g) * D + 64 * c + 16 * t);
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int st = 0; st < 4; ++st)
          mma16816<BF16>(s[nt], qa[c][st], codes2<BF16, false>(ww[st]), codes2<BF16, true>(ww[st]));
      }
    }
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int nt = 0; nt < 4; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = key0 + nt * 8 + 2 * t + (e & 1);
        s[nt][e] = key < lim[e >> 1] ? s[nt][e] * ck + lv : -INFINITY;
        mx[e >> 1] = fmaxf(mx[e >> 1], s[nt][e]);
      }
    float base[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(~0u, mx[r], 1));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(~0u, mx[r], 2));
      const float mn = fmaxf(m[r], mx[r]);
      base[r] = mn == -INFINITY ? 0.f : mn;
      const float alpha = ex2(m[r] - base[r]);        // 0 while the row has seen no key
      m[r] = mn;
      l[r] *= alpha;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        o[i][2 * r] *= alpha;
        o[i][2 * r + 1] *= alpha;
      }
    }
    float ps[2] = {0.f, 0.f};
#pragma unroll
    for (int nt = 0; nt < 4; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[nt][e] = ex2(s[nt][e] - base[e >> 1]);
        ps[e >> 1] += s[nt][e];
      }
    // (a row that sees none of these keys takes nothing from their scale either)
    if (ps[0] != 0.f) l[0] += ps[0] * inv_vs;
    if (ps[1] != 0.f) l[1] += ps[1] * inv_vs;
    // O += P V: 16 keys a step; column n of dim tile i is dim 8n + i of a
    // 64-dim chunk, so lane g's operands are 8 consecutive bytes of a row
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const uint32_t pa[4] = {pack_half2(s[2 * st][0], s[2 * st][1]), pack_half2(s[2 * st][2], s[2 * st][3]),
                              pack_half2(s[2 * st + 1][0], s[2 * st + 1][1]),
                              pack_half2(s[2 * st + 1][2], s[2 * st + 1][3])};
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        uint2 w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w[k] = *reinterpret_cast<const uint2*>(vp + (16 * st + 2 * t + (k & 1) + 8 * (k >> 1)) * D + 64 * c + 8 * g);
#pragma unroll
        for (int hw = 0; hw < 2; ++hw) {
          const uint32_t x0 = (hw ? w[0].y : w[0].x) ^ 0x80808080u, x1 = (hw ? w[1].y : w[1].x) ^ 0x80808080u;
          const uint32_t y0 = (hw ? w[2].y : w[2].x) ^ 0x80808080u, y1 = (hw ? w[3].y : w[3].x) ^ 0x80808080u;
          const uint32_t xl = __byte_perm(x0, x1, 0x5140), xh = __byte_perm(x0, x1, 0x7362);
          const uint32_t yl = __byte_perm(y0, y1, 0x5140), yh = __byte_perm(y0, y1, 0x7362);
          float(*oc)[4] = &o[8 * c + 4 * hw];
          mma16816<false>(oc[0], pa, codes_f16<false>(xl), codes_f16<false>(yl));
          mma16816<false>(oc[1], pa, codes_f16<true>(xl), codes_f16<true>(yl));
          mma16816<false>(oc[2], pa, codes_f16<false>(xh), codes_f16<false>(yh));
          mma16816<false>(oc[3], pa, codes_f16<true>(xh), codes_f16<true>(yh));
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(~0u, l[r], 1);
    l[r] += __shfl_xor_sync(~0u, l[r], 2);
    if (t == 0) {
      sm_m[warp][g + 8 * r] = m[r];
      sm_l[warp][g + 8 * r] = l[r];
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        sm_o[warp][g + 8 * r][64 * (i / 8) + 8 * (2 * t + e) + i % 8] = o[i][2 * r + e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < TOK_ROWS * D / 2; i += TOK_WARPS * 32) {
    const int r = i / (D / 2), d = 2 * (i % (D / 2)), row = row0 + r;
    if (row >= rows) continue;
    float mt = -INFINITY;
#pragma unroll
    for (int w = 0; w < TOK_WARPS; ++w) mt = fmaxf(mt, sm_m[w][r]);
    const float base = mt == -INFINITY ? 0.f : mt;
    float lt = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < TOK_WARPS; ++w) {
      const float f = ex2(sm_m[w][r] - base);
      lt += f * sm_l[w][r];
      x += f * sm_o[w][r][d];
      y += f * sm_o[w][r][d + 1];
    }
    const float inv = lt == 0.f ? 0.f : 1.f / lt;
    const float lse2 = lt == 0.f ? -INFINITY : base + log2f(lt);
    const long long tok = q0 + row / a.group;
    const int h = kvh * a.group + row % a.group;
    if (a.splits > 1) {
      const long long part = (long long)sp * a.Tq * a.hq + tok * a.hq + h;
      *reinterpret_cast<float2*>(a.part_o + part * D + d) = make_float2(x * inv, y * inv);
      if (d == 0) a.part_lse[part] = lse2;
    } else {
      const uint32_t v = BF16 ? pack_bf162(x * inv, y * inv) : pack_half2(x * inv, y * inv);
      *reinterpret_cast<uint32_t*>(a.out + tok * a.o_tok + h * a.o_head + d) = v;
      if (d == 0 && a.lse) a.lse[h * a.Tq + tok] = lse2 * 0.6931471805599453f;
    }
  }
}

// Joins the splits' normalised rows, weighted by their sums: one warp per row.
template <bool BF16, int D>
__global__ void __launch_bounds__(256) attn_cache_join_kernel(CacheAttnArgs a) {
  pdl_wait();
  pdl_trigger();
  const long long row = (long long)blockIdx.x * 8 + threadIdx.x / 32, rows = a.Tq * a.hq;
  const int lane = threadIdx.x % 32;
  if (row >= rows) return;
  float mx = -INFINITY;
  for (int s = lane; s < a.splits; s += 32) mx = fmaxf(mx, a.part_lse[s * rows + row]);
  mx = warp_max(mx);
  const float base = mx == -INFINITY ? 0.f : mx;
  float l = 0.f, acc[D / 32];
#pragma unroll
  for (int e = 0; e < D / 32; ++e) acc[e] = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float w = ex2(a.part_lse[s * rows + row] - base);
    if (w == 0.f) continue;
    l += w;
    const float* p = a.part_o + (s * rows + row) * D + lane * (D / 32);
#pragma unroll
    for (int e = 0; e < D / 32; ++e) acc[e] += w * p[e];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const long long tok = row / a.hq;
  const int h = (int)(row - tok * a.hq);
  uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + tok * a.o_tok + h * a.o_head + lane * (D / 32));
#pragma unroll
  for (int e = 0; e < D / 64; ++e)
    dst[e] = BF16 ? pack_bf162(acc[2 * e] * inv, acc[2 * e + 1] * inv) : pack_half2(acc[2 * e] * inv, acc[2 * e + 1] * inv);
  if (lane == 0 && a.lse) a.lse[h * a.Tq + tok] = l == 0.f ? -INFINITY : (base + log2f(l)) * 0.6931471805599453f;
}

// How a call is laid out, by its sizes alone.
struct Plan {
  bool tiles;                            // attn_cache_sm100.cu's kernel
  int row_blocks, splits;                // 16-row tiles or Q blocks of a request, parts of the keys (row kernel)
  int64_t scratch;
};

// Few rows: splits so that the grid covers the SMs a few times over, each
// split keeping at least 4 units for each warp.
int row_splits(long long tiles, long long max_kv) {
  const long long sms = device_info().num_sms;
  const long long units = (max_kv + UNIT - 1) / UNIT;
  long long s = (4 * sms + tiles - 1) / std::max<long long>(1, tiles);
  s = std::min(s, units / (4 * TOK_WARPS));
  return (int)std::max<long long>(1, std::min<long long>(s, MAX_SPLITS));
}

Plan make_plan(long long Tq, int group, int kv_heads, int requests, int max_q, long long max_kv, int head_dim) {
  Plan p{};
  const long long rows = (long long)max_q * group;
  p.tiles = rows > TOK_ROWS && group <= 128;
  if (p.tiles) {
    const int tokens = 2 * (128 / group);
    p.row_blocks = (int)(((long long)max_q + tokens - 1) / tokens);
    p.splits = 1;
    p.scratch = tiles_scratch((long long)p.row_blocks * kv_heads * requests, max_kv, head_dim);
  } else {
    p.row_blocks = (int)((rows + TOK_ROWS - 1) / TOK_ROWS);
    p.splits = row_splits((long long)p.row_blocks * kv_heads * requests, max_kv);
    p.scratch = p.splits > 1 ? (int64_t)p.splits * Tq * kv_heads * group * (head_dim + 1) * 4 : 0;
  }
  return p;
}

int check_shape(const char* name, int64_t Tq, int32_t q_heads, int32_t kv_heads, int32_t requests, int32_t max_q,
                int64_t max_kv, int32_t head_dim) {
  if (Tq < 0 || requests < 0 || max_q < 0 || max_kv < 0 || q_heads <= 0 || kv_heads <= 0)
    return set_error(QVGGT_ERR_INVALID, "%s: bad shape", name);
  if (q_heads % kv_heads)
    return set_error(QVGGT_ERR_INVALID, "%s: %d query heads do not share %d key heads evenly", name, q_heads, kv_heads);
  if (head_dim != 64 && head_dim != 128)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128", name);
  if (Tq > 2147483647LL / q_heads || (int64_t)requests * kv_heads > 65535 || max_kv > 2147483647LL)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: too many rows, requests or keys", name);
  return QVGGT_OK;
}

}  // namespace
}  // namespace qv

using namespace qv;

extern "C" int qvggt_cached_attention_scratch(int64_t Tq, int32_t q_heads, int32_t kv_heads, int32_t requests,
                                              int32_t max_q, int64_t max_kv, int32_t head_dim, int64_t* bytes) {
  if (int rc = check_shape("cached_attention_scratch", Tq, q_heads, kv_heads, requests, max_q, max_kv, head_dim))
    return rc;
  if (!bytes) return set_error(QVGGT_ERR_INVALID, "cached_attention_scratch: null pointer");
  *bytes = make_plan(Tq, q_heads / kv_heads, kv_heads, requests, max_q, max_kv, head_dim).scratch;
  return QVGGT_OK;
}

extern "C" int qvggt_cached_attention(const void* q, int64_t q_tok, int64_t q_head, void* out, int64_t o_tok,
                                      int64_t o_head, float* lse, int64_t Tq, int32_t q_heads, int32_t dtype,
                                      const int8_t* k_cache, const int8_t* v_cache, int64_t block_stride,
                                      const float* k_scale, const float* v_scale, int32_t num_blocks,
                                      int32_t kv_heads, int32_t block_size, int32_t head_dim,
                                      const int32_t* block_tables, int32_t max_blocks, const int32_t* cu_q,
                                      const int32_t* kv_lens, int32_t requests, int32_t max_q, int64_t max_kv,
                                      int32_t causal_chunk, float scale, void* scratch, int64_t scratch_bytes,
                                      void* stream) {
  const char* name = "cached_attention";
  if (int rc = check_shape(name, Tq, q_heads, kv_heads, requests, max_q, max_kv, head_dim)) return rc;
  if (int rc = check_cache(name, k_cache, v_cache, k_scale, v_scale, block_stride, num_blocks, kv_heads, block_size,
                           head_dim))
    return rc;
  if (dtype != QVGGT_DTYPE_F16 && dtype != QVGGT_DTYPE_BF16)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: dtype must be fp16 or bf16", name);
  if (causal_chunk < 0 || max_blocks < 0) return set_error(QVGGT_ERR_INVALID, "%s: bad causal_chunk or table", name);
  if (!(scale > 0.f) || scale > 3.0e38f) return set_error(QVGGT_ERR_INVALID, "%s: scale must be positive", name);
  if ((int64_t)max_blocks * block_size > 2147483647LL)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: block tables hold more than 2^31 keys", name);
  if (Tq == 0 || requests == 0 || max_q == 0) return QVGGT_OK;
  if (!q || !out || !cu_q || !kv_lens || (!block_tables && max_blocks))
    return set_error(QVGGT_ERR_INVALID, "%s: null tensor", name);
  if (!aligned16(q) || !aligned16(out) || q_tok % 8 || q_head % 8 || o_tok % 8 || o_head % 8)
    return set_error(QVGGT_ERR_ALIGN, "%s: q and out rows must be 16-byte aligned", name);
  CacheAttnArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  a.kc = k_cache;
  a.vc = v_cache;
  a.ks = k_scale;
  a.vs = v_scale;
  a.table = block_tables;
  a.cu_q = cu_q;
  a.kv_lens = kv_lens;
  a.q_tok = q_tok;
  a.q_head = q_head;
  a.o_tok = o_tok;
  a.o_head = o_head;
  a.block_stride = block_stride;
  a.Tq = Tq;
  a.B = requests;
  a.hq = q_heads;
  a.hk = kv_heads;
  a.group = q_heads / kv_heads;
  a.wide = max_blocks;
  a.num_blocks = num_blocks;
  a.bs_log2 = block_size == 32 ? 5 : block_size == 64 ? 6 : 7;
  a.chunk = causal_chunk;
  a.max_q = max_q;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.ctl = make_ctl();
  Plan p = make_plan(Tq, a.group, kv_heads, requests, max_q, max_kv, head_dim);
  if (p.tiles && !tiles_can_read(a)) {
    // strides no TMA map takes (a broadcast or reversed query): the row kernel, unsplit
    p.tiles = false;
    p.row_blocks = (int)(((long long)max_q * a.group + TOK_ROWS - 1) / TOK_ROWS);
    p.splits = 1;
    p.scratch = 0;
  }
  const int64_t need = p.scratch;
  if (need && (!scratch || scratch_bytes < need || !aligned16(scratch)))
    return set_error(QVGGT_ERR_INVALID, "%s: needs %lld bytes of 16-byte aligned scratch, got %lld", name,
                     (long long)need, (long long)scratch_bytes);
  a.row_blocks = p.row_blocks;
  a.splits = p.splits;
  const bool bf16 = dtype == QVGGT_DTYPE_BF16;
  using Kfn = void (*)(CacheAttnArgs);
  static const Kfn rows_fns[2][2] = {{attn_cache_rows_kernel<false, 64>, attn_cache_rows_kernel<false, 128>},
                                     {attn_cache_rows_kernel<true, 64>, attn_cache_rows_kernel<true, 128>}};
  static const Kfn join_fns[2][2] = {{attn_cache_join_kernel<false, 64>, attn_cache_join_kernel<false, 128>},
                                     {attn_cache_join_kernel<true, 64>, attn_cache_join_kernel<true, 128>}};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p.tiles) return launch_tiles(a, head_dim, bf16, max_kv, scratch, st);
  a.part_o = static_cast<float*>(scratch);
  a.part_lse = need ? a.part_o + (long long)p.splits * Tq * q_heads * head_dim : nullptr;
  if (int rc = check_cuda(launch_pdl(rows_fns[bf16][head_dim == 128],
                                     dim3((unsigned)p.row_blocks, (unsigned)(kv_heads * requests), (unsigned)p.splits),
                                     dim3(TOK_WARPS * 32), 0, st, 1u, a),
                          "cached_attention launch"))
    return rc;
  count_launch(1);
  if (p.splits > 1) {
    if (int rc = check_cuda(launch_pdl(join_fns[bf16][head_dim == 128], dim3((unsigned)((Tq * q_heads + 7) / 8)),
                                       dim3(256), 0, st, 1u, a),
                            "cached_attention join launch"))
      return rc;
    count_launch(1);
  }
  return QVGGT_OK;
}
