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
  int B, hq, hk, group, wide, num_blocks, bs_log2, chunk, max_q;
  int row_blocks;                        // Q blocks (16-row tiles) of the longest request
  int can_split;                         // items may be cut, a join follows
  float scale_log2;
  uint32_t wait_tries;                   // bound of every wait
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

// A score's factor (scales times a power of two) kept from rounding to 0: a
// hidden key's -inf times 0 would be NaN.  What it is raised to leaves a score
// 0 all the same (|q . c| is under 2^30 for fp16 queries).  NaN stays.
__device__ __forceinline__ float nonzero_factor(float x) { return x < 1.17549435e-38f ? 1.17549435e-38f : x; }

__device__ __forceinline__ bool lengths_ok(const CacheAttnArgs& a, int q0, int ql, int n) {
  if (q0 >= 0 && ql >= 0 && ql <= a.max_q && (long long)q0 + ql <= a.Tq && n >= 0 && n <= (a.wide << a.bs_log2)) return true;
  report_status(a.ctl, ST_BAD_LENGTH);
  return false;
}

// cp.async.bulk of contiguous bytes, completion on an mbarrier of this CTA.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// Bounded wait for the phase with parity `parity`: up to `tries` try_waits,
// each of which the hardware suspends for about 1.4 us if nothing arrives.
// Nothing but the loop, as it is inlined at every hand-off: the roles of an SM
// run from one instruction cache, and its misses cost this kernel 12 % when
// each wait carried its own time-out code.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, uint32_t tries) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\t"
      "mov.u32 n, %3;\n\t"
      "QV_TRY:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra QV_DONE;\n\t"
      "sub.u32 n, n, 1;\n\t"
      "setp.ne.u32 q, n, 0;\n\t"
      "@q bra QV_TRY;\n\t"
      "QV_DONE:\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(tries)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool wait(const uint64_t* bar, uint32_t parity, uint32_t tries) {
  return wait(smem_u32(bar), parity, tries);
}
// Whether the phase is complete, without waiting.
__device__ __forceinline__ bool test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

// A wait of a whole warp that then stays converged.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, uint32_t tries) {
  return __all_sync(0xffffffffu, wait(bar, parity, tries));
}
__device__ __forceinline__ bool warp_wait(const uint64_t* bar, uint32_t parity, uint32_t tries) {
  return warp_wait(smem_u32(bar), parity, tries);
}

// ------------------------------------------------------------------ pieces
// What a CTA does with one item (request, block of rows, kv head): key tiles
// [t0, t0 + nt).
struct __align__(16) Segment {
  int b, kvh, tok0, q0;                  // tok0: first token (tile kernel) or row (row kernel) of the block
  int ql, n, nqt, t0;
  int nt;                                // -1: no more segments
  int slot;                              // where the part is parked; -1: the item is whole
  int pad[2];
};

// Where a cut lies, for the join: written by the CTA after it.
struct __align__(16) Cut {
  int first, last;                       // CTAs that hold parts of the item (first < 0: the cut is between items)
  int kvh, tok0, q0, ql, pad[2];
};

// Running sums of the blocks' costs in shared memory, cum[0 .. THREADS]: entry
// x starts at block x * g.  All THREADS threads call it; ends with a barrier.
template <int THREADS, class Blk>
__device__ __forceinline__ void scan_blocks(const CacheAttnArgs& a, long long* cum, int blocks, int g) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  long long sum = 0;
  for (int p = threadIdx.x * g; p < min(blocks, ((int)threadIdx.x + 1) * g); ++p)
    sum += Blk(a, p / a.row_blocks, p % a.row_blocks).cost;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const long long o = __shfl_up_sync(~0u, sum, d);
    if (lane >= d) sum += o;
  }
  cum[threadIdx.x + 1] = sum;
  __syncthreads();
  if (warp == 0) {
    // sums of the warps before, added to every warp's
    long long s = lane < THREADS / 32 ? cum[lane * 32 + 32] : 0;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const long long o = __shfl_up_sync(~0u, s, d);
      if (lane >= d) s += o;
    }
    cum[0] = 0;
    __syncwarp();
    for (int w = 1; w < THREADS / 32; ++w) {
      const long long before = __shfl_sync(~0u, s, w - 1);
      cum[w * 32 + lane + 1] += before;
    }
  }
  __syncthreads();
}

// The items laid out as one line of cost (block after block, in a block one kv
// head after another), cut into equal pieces of at least Blk::MIN; CTA x walks
// piece x.  Tile t of an item belongs to the piece that holds its place on the
// line, so every CTA finds the others' parts by arithmetic alone.  An item's
// part that starts at tile 0 is parked in slot 2x + 1, any other in 2x: a CTA
// has at most one of each.
template <int THREADS, class Blk>
struct PieceWalk {
  long long W, begin, end, s;            // length of a piece, this one's ends, where block p starts
  int p, h, g;
  Blk blk;
  Cut cut;

  __device__ __forceinline__ PieceWalk(const CacheAttnArgs& a, const long long* cum, int blocks, int g_) : g(g_) {
    const long long total = cum[THREADS] * a.hk;
    const int grid = gridDim.x;
    W = (total + grid - 1) / grid;
    if (a.can_split && W < Blk::MIN) W = Blk::MIN;
    begin = blockIdx.x * W;
    end = min(total, begin + W);
    cut.first = -1;
    int e = 0;                           // entry that holds `begin`
    for (int len = THREADS; len > 1;) {
      const int half = len / 2;
      if (cum[e + half] * a.hk <= begin) e += half;
      len -= half;
    }
    p = e * g;
    s = cum[e] * a.hk;
    h = 0;
    if (begin < end) load(a, blocks);
    else p = blocks;
  }

  __device__ __forceinline__ void load(const CacheAttnArgs& a, int blocks) {
    for (; p < blocks; ++p) {
      blk = Blk(a, p / a.row_blocks, p % a.row_blocks);
      if (blk.cost > 0 && s + blk.cost * a.hk > begin) {
        h = begin > s ? (int)((begin - s) / blk.cost) : 0;
        return;
      }
      s += blk.cost * a.hk;
    }
  }

  // The next segment; false at the end of the piece.
  __device__ __forceinline__ bool next(const CacheAttnArgs& a, int blocks, Segment& sg) {
    const int grid = gridDim.x, x = blockIdx.x;
    while (p < blocks) {
      if (h == a.hk) {
        s += blk.cost * a.hk;
        ++p;
        load(a, blocks);
        continue;
      }
      const long long s0 = s + h * blk.cost, k0 = s0 + Blk::START;        // the item, its first tile
      if (s0 >= end) return false;
      const int head = h++;
      const int c = blk.tile_cost();
      int t_lo = 0, t_hi = blk.tiles, slot = -1;
      if (a.can_split && blk.tiles > 0) {
        auto at = [&](long long pos) { return pos <= k0 ? 0 : (int)min((long long)blk.tiles, (pos - k0 + c - 1) / c); };
        t_lo = at(begin);
        t_hi = x == grid - 1 ? blk.tiles : at(begin + W);
        if (t_lo >= t_hi) continue;
        const int first = (int)min(k0 / W, (long long)grid - 1);
        const int last = (int)min((k0 + (long long)(blk.tiles - 1) * c) / W, (long long)grid - 1);
        if (first != last) {
          slot = 2 * x + (t_lo == 0 ? 1 : 0);
          if (t_lo > 0) cut = Cut{first, last, head, blk.tok0, blk.q0, blk.ql, {0, 0}};
        }
      } else if (s0 < begin) {
        continue;                        // whole items: the CTA that holds the start
      }
      sg = Segment{p / a.row_blocks, head, blk.tok0, blk.q0, blk.ql, blk.n, blk.nqt, t_lo, t_hi - t_lo, slot, {0, 0}};
      return true;
    }
    return false;
  }
};

// Row `row` of a cut item, joined from its parts (rows_per_slot rows a slot) by
// D / 4 threads, four columns each: the parts' normalised rows weighted by
// their sums, in the pieces' order.
template <bool BF16, int D>
__device__ __forceinline__ void join_parts(const CacheAttnArgs& a, const Cut& cut, int rows_per_slot, int row, int col4,
                                           long long tok, int h) {
  auto at = [&](int k) { return (long long)(2 * k + (k == cut.first)) * rows_per_slot + row; };
  float mx = -INFINITY;
#pragma unroll 4
  for (int k = cut.first; k <= cut.last; ++k) mx = fmaxf(mx, a.part_lse[at(k)]);
  const float base = mx == -INFINITY ? 0.f : mx;
  float l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = cut.first; k <= cut.last; ++k) {
    const float w = exp2f(a.part_lse[at(k)] - base);
    const float4 v = *reinterpret_cast<const float4*>(a.part_o + at(k) * D + col4 * 4);
    l += w;
    acc.x += w * v.x;
    acc.y += w * v.y;
    acc.z += w * v.z;
    acc.w += w * v.w;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  acc = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(a.out + tok * a.o_tok + h * a.o_head + col4 * 4) =
      BF16 ? make_uint2(pack_bf162(acc.x, acc.y), pack_bf162(acc.z, acc.w))
           : make_uint2(pack_half2(acc.x, acc.y), pack_half2(acc.z, acc.w));
  if (col4 == 0 && a.lse) a.lse[h * a.Tq + tok] = l == 0.f ? -INFINITY : (base + log2f(l)) * 0.6931471805599453f;
}

// attn_cache_sm100.cu (many rows): whether its TMA map can read these queries;
// the scratch for `items` (request, Q block, kv head) triples; the launches.
bool tiles_can_read(const CacheAttnArgs& a);
int64_t tiles_scratch(long long items, long long max_kv, int D);
int launch_tiles(CacheAttnArgs& a, int D, bool bf16, long long max_kv, void* scratch, cudaStream_t stream);

}  // namespace qv
