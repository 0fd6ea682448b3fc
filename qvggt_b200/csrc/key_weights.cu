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
// More rows of a key head than this go to key_weights_sm100.cu.  Eight streams, 16
// heads, us here / there: head_dim 64 over 10,000 to 20,000 keys at 28 rows 62 / 127,
// at 40 (the codes unpacked twice) 158 / 127; head_dim 128 96 / 187 and 231 / 187;
// over 500 to 1,000 keys at 28 rows 15 / 15 and 20 / 18.
constexpr int ROWS_MAX = 32;

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

__device__ __forceinline__ float lds32(uint32_t at) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
// Copies that a lane makes for itself and awaits in groups.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int D>
struct RowLay {
  static constexpr int CODES = UNIT * D;                   // of a unit; its old weights follow
  static constexpr int STAGE = CODES + UNIT * 4;
  static constexpr int STAGES = D == 64 ? 3 : 2;         // units under way, a warp: more cost CTAs their room
  static constexpr int TOTAL = WARPS * STAGES * STAGE;
};

// The codes are the M operand of mma.m16n8k16 and the rows its N: a lane reads
// 16 codes of one key at once into the fragments (any order of the dims will do,
// as the queries' fragments use the same), and the sum over rows is over a lane's
// registers and four lanes.  A lane copies what it will read, some units ahead,
// into a ring of its own: no barrier.  Eight tokens over 26,000 to 44,000 keys of
// 16 heads x 64 (355 MB) take 72 us, 4.9 TB/s, with three units under way, 77 with
// six, 77 with one ahead in registers, 106 with nothing ahead, and 97 through a
// ring of bulk copies with mbarriers (small ones take an SM about 90 cycles each).
// More than 8 NT rows are taken 8 NT at a time.
template <bool BF16, int D, int NT>
__global__ void __launch_bounds__(THREADS, D == 64 ? (NT < 4 ? 4 : 3) : 4 - NT < 1 ? 1 : 4 - NT) key_weights_rows_kernel(KeyWeightArgs a, int ctas) {
  using L = RowLay<D>;
  constexpr int KC = D / 64;             // 64-dim chunks
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const uint32_t ring = smem_u32(smem) + warp * L::STAGES * L::STAGE + lane * 16, old_ring = ring + L::CODES - lane * 12;
  pdl_wait();
  pdl_trigger();
  const int pair = blockIdx.x / ctas, kvh = pair % a.hk, b = pair / a.hk;
  const int q0 = a.cu_q[b], ql = a.cu_q[b + 1] - q0, n = a.kv_lens[b];
  if (q0 < 0 || ql < 0 || ql > a.max_q || (long long)q0 + ql > a.Tq || n < 0 || n > (a.wide << a.bs_log2)) {
    if (threadIdx.x == 0) report_status(a.ctl, ST_BAD_LENGTH);
    return;
  }
  const int fresh = a.fresh ? a.fresh[b] : n;
  const int bs = 1 << a.bs_log2, rows = ql * a.group;
  const int32_t* table = a.table + (long long)b * a.wide;
  // this warp's units: first + i stride
  const int units = (int)(((long long)n + UNIT - 1) / UNIT), stride = ctas * WARPS, first = blockIdx.x % ctas * WARPS + warp;
  const int count = first < units ? (units - first + stride - 1) / stride : 0;
  // lane x holds the block of unit base + x and its scale, and those of the 32 units after
  auto fetch = [&](int i, int& id, float& ks) {
    id = -1;
    ks = 0.f;
    if (i >= count) return;
    id = table[((first + i * stride) * UNIT) >> a.bs_log2];
    if (id < 0 || id >= a.num_blocks) {
      report_bad_block(a.ctl);
      id = -1;
    } else {
      ks = a.ks[(long long)id * a.hk + kvh];
    }
  };
  int id, id2;
  float ks, ks2;
  fetch(lane, id, ks);
  fetch(32 + lane, id2, ks2);
  // the key whose weight this lane writes, in its unit
  const int mine = 16 * (t / 2) + 8 * (t % 2) + g;
  // starts the copies of unit i, in block blk (none where it is outside the cache), into stage x
  auto issue = [&](int i, int blk, int x) {
    if (i < count && blk >= 0) {
      const int key0 = (first + i * stride) * UNIT;
      const int8_t* kp = a.kc + blk * a.block_stride + ((long long)kvh * bs + (key0 & (bs - 1)) + g) * D + 16 * t;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < KC; ++c) copy16(ring + x * L::STAGE + (r * KC + c) * 512, kp + 8 * r * D + 64 * c);
      if (key0 + mine < min(n, fresh))
        copy4(old_ring + x * L::STAGE, a.w + (((long long)blk * a.hk + kvh) << a.bs_log2) + (key0 & (bs - 1)) + mine);
    }
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i < L::STAGES; ++i) issue(i, __shfl_sync(~0u, id, i), i);

  // B fragments of the queries (row g of each tile): step s of chunk c takes dims
  // 64 c + 16 t + 4 s + {0, 1} as k rows 2t, 2t + 1 and {2, 3} as 2t + 8, 2t + 9.
  // bf16 queries become fp16 times a power of two per row (its largest element near
  // 2^13; what fp16 then cannot hold exactly is below 2^-37 of that), because codes
  // unpack to fp16 in five instructions a word and to bf16 in eight.
  uint2 qb[NT][KC][4];
  float nl[NT][2];                       // -lse log2e of rows 2t, 2t + 1 of each tile
  float back[NT][2];                     // what undoes their powers of two
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
      float undo = 1.f;
      if (BF16) {
        float mx = 0.f;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const float2 p = unpack_bf162(qb[x][c][s].x), q = unpack_bf162(qb[x][c][s].y);
            mx = fmaxf(mx, fmaxf(fmaxf(fabsf(p.x), fabsf(p.y)), fmaxf(fabsf(q.x), fabsf(q.y))));
          }
        mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 2));
        // exponents of 2^up and 2^-up, kept in the normal range
        const int up = max(-115, min(110, 13 - ((int)(__float_as_uint(mx) >> 23) - 127)));
        const float f = __int_as_float((127 + up) << 23);
        undo = __int_as_float((127 - up) << 23);
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const float2 p = unpack_bf162(qb[x][c][s].x), q = unpack_bf162(qb[x][c][s].y);
            qb[x][c][s] = make_uint2(pack_half2(p.x * f, p.y * f), pack_half2(q.x * f, q.y * f));
          }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = row0 + 8 * x + 2 * t + e;
        const float l = r < rows ? a.lse[(long long)(kvh * a.group + r % a.group) * a.Tq + q0 + r / a.group] : INFINITY;
        nl[x][e] = -l * LOG2E;
        lim[x][e] = isfinite(l) ? key_limit(r / a.group, ql, n, a.chunk) : 0;
        back[x][e] = __shfl_sync(~0u, undo, (2 * t + e) * 4);
      }
    }
  };
  const bool once = rows <= 8 * NT;
  if (once && rows > 0) load_rows(0);

  int st = 0;                            // the ring's next stage
  for (int i = 0; i < count; ++i) {
    if (i && (i & 31) == 0) {
      id = id2;
      ks = ks2;
      fetch(i + 32 + lane, id2, ks2);
    }
    const int blk = __shfl_sync(~0u, id, i & 31);
    const float ck = __shfl_sync(~0u, ks, i & 31) * a.scale_log2;
    const int key0 = (first + i * stride) * UNIT, key = key0 + mine;
    copies_wait<L::STAGES - 1>();
    uint4 w[2][2][KC];                   // keys 16 mt + 8 half + g
    const uint32_t at = ring + st * L::STAGE;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int c = 0; c < KC; ++c) w[mt][half][c] = lds128(at + ((2 * mt + half) * KC + c) * 512);
    const float old = key < min(n, fresh) ? lds32(old_ring + st * L::STAGE) : 0.f;
    // the stage is read: the next unit that uses it
    const int j = i + L::STAGES;
    issue(j, __shfl_sync(~0u, j >> 5 == i >> 5 ? id : id2, j & 31), st);
    if (++st == L::STAGES) st = 0;
    if (blk < 0) continue;
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
            const uint32_t ka[4] = {codes2<false, false>(x0[sp]), codes2<false, false>(x1[sp]),
                                    codes2<false, true>(x0[sp]), codes2<false, true>(x1[sp])};
#pragma unroll
            for (int x = 0; x < NT; ++x) mma16816(s[x][mt], ka, qb[x][c][sp].x, qb[x][c][sp].y);
          }
        }
      }
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        const float cx[2] = {BF16 ? ck * back[x][0] : ck, BF16 ? ck * back[x][1] : ck};
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = ex2(fmaf(s[x][mt][e], cx[e & 1], nl[x][e & 1]));
            sum[mt][e >> 1] += key0 + 16 * mt + 8 * (e >> 1) + g < lim[x][e & 1] ? p : 0.f;
          }
      }
    }
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        sum[mt][half] += __shfl_xor_sync(~0u, sum[mt][half], 1);
        sum[mt][half] += __shfl_xor_sync(~0u, sum[mt][half], 2);
      }
    const float got = t < 2 ? (t ? sum[0][1] : sum[0][0]) : (t & 1 ? sum[1][1] : sum[1][0]);
    if (key < n) a.out[(((long long)blk * a.hk + kvh) << a.bs_log2) + (key & (bs - 1))] = fmaf(old, a.decay, got);
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
  if (!aligned16(p->q) || (p->Tq > 1 && p->q_tok % 8) || (p->q_heads > 1 && p->q_head % 8))
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
  if (rows > ROWS_MAX && a.Tq > 0 && key_weight_tiles_can_read(a))
    return launch_key_weight_tiles(a, (int)p->head_dim, bf16, static_cast<cudaStream_t>(stream));
  const long long units = std::max<long long>(1, (p->max_kv + UNIT - 1) / UNIT);
  // Units of a warp: up to 16, and fewer where there would be less than about six
  // CTAs for each SM (lengths differ, so CTAs do)
  const long long per = std::max<long long>(1, std::min<long long>(16, units * pairs / (24 * device_info().num_sms)));
  const long long ctas = (units + WARPS * per - 1) / (WARPS * per);
  if (ctas * pairs > 2147483647LL)
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
  const int d = p->head_dim == 128, nt = rows <= 8 ? 0 : rows <= 16 ? 1 : 2, smem = d ? RowLay<128>::TOTAL : RowLay<64>::TOTAL;
  static DeviceFlags attr[2][2][3];
  if (int rc = ensure_smem(attr[bf16][d][nt], fns[bf16][d][nt], smem, "cudaFuncSetAttribute(key_weights)")) return rc;
  int rc = check_cuda(launch_pdl(fns[bf16][d][nt], dim3((unsigned)(ctas * pairs)), dim3(THREADS), (size_t)smem,
                                 static_cast<cudaStream_t>(stream), 1u, a, (int)ctas),
                      "key_weights launch");
  if (!rc) count_launch(1);
  return rc;
}
