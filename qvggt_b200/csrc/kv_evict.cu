// Making room in the paged 8-bit K/V cache: which keys of a request stay, and
// their move into the places of those that go.
//
// Keys may lie in any order in the cache (their positions are in the rotated
// rows), so only survivors past the new length move, each into the place of an
// evicted key below it; what stays where it is is not rounded again.
#include "host.hpp"
#include "kv_cache.cuh"

namespace qv {
namespace {

// ------------------------------------------------------------------- choice
constexpr int CHOOSE_THREADS = 512, CHOOSE_WARPS = CHOOSE_THREADS / 32;
constexpr int SPAN = 128;                // positions a warp takes at a time, four a lane
// Digits of the 32-bit keys, from the top: 12, 10 and 10 bits.  The first one
// holds the exponent and three bits more, which spreads weights of any size
// over enough bins that few lanes meet in one.
constexpr int BINS1 = 4096, BINS2 = 1024;

struct ChooseArgs {
  const float* w;                        // [layers][num_blocks][heads][bs]
  const int32_t *table, *lens, *keep;
  int32_t *src, *dst, *counts;           // [layers][B][heads][max_moves], counts without the last
  int B, heads, wide, num_blocks, bs_log2, sink, recent, max_moves;
  int room;                              // positions of a CTA that shared memory holds
  Ctl ctl;
};

// Weights as integers in their order: NaN and what is below every finite float
// count as the lowest, infinity as the largest finite one, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float w) {
  const float big = 3.4028234663852886e38f;
  const float x = (w != w ? -big : fminf(fmaxf(w, -big), big)) + 0.f;
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint4 ld_cluster_u4(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}

// One (layer, request, head) per cluster of up to eight CTAs.  The `keep`-th
// largest key is found digit by digit: each CTA counts its positions' digits in
// shared memory, after a cluster barrier each adds up all CTAs' counts.  The
// positions of a warp are consecutive, so ranks in order come from running sums
// over warps and CTAs, and the result does not depend on any order of arrival.
// Weights are read from memory once and kept as keys in shared memory where
// they fit (`room`), else read again for each digit.
__global__ void __launch_bounds__(CHOOSE_THREADS) evict_plan_kernel(ChooseArgs a) {
  extern __shared__ __align__(16) uint32_t keys[];
  __shared__ __align__(16) uint32_t hist[BINS1 + 2 * BINS2];
  __shared__ uint32_t warp_sum[CHOOSE_WARPS];
  __shared__ uint32_t found[3];          // the digit, how many of its keys stay, how many there are
  __shared__ int cnt[3][CHOOSE_WARPS];   // per warp: ties, holes, late survivors
  __shared__ __align__(16) int total[4]; // of this CTA
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  for (int i = tid; i < BINS1 + 2 * BINS2; i += CHOOSE_THREADS) hist[i] = 0;
  pdl_wait();
  pdl_trigger();
  const int C = (int)cluster_size(), rank = (int)cluster_ctarank();
  const int row = blockIdx.x / C, h = row % a.heads, b = row / a.heads % a.B, layer = row / a.heads / a.B;
  int n = a.lens[b], keep = a.keep[b];
  if (n < 0 || keep < 0 || n > (a.wide << a.bs_log2)) {
    if (tid == 0) report_status(a.ctl, ST_BAD_LENGTH);
    n = keep = 0;
  }
  int32_t* src = a.src + (long long)row * a.max_moves;
  int32_t* dst = a.dst + (long long)row * a.max_moves;
  auto pad_from = [&](int from) {
    for (int i = from + rank * CHOOSE_THREADS + tid; i < a.max_moves; i += C * CHOOSE_THREADS) src[i] = dst[i] = -1;
  };
  if (keep >= n) {                       // nothing goes (the same for the whole cluster)
    if (rank == 0 && tid == 0) a.counts[row] = 0;
    pad_from(0);
    return;
  }
  const int sink = min(a.sink, keep), recent = min(a.recent, keep - sink);
  const int middle = n - sink - recent;  // positions [sink, sink + middle) compete for the rest
  int want = keep - sink - recent;
  const int per_warp = (int)(((long long)n + C * CHOOSE_WARPS * SPAN - 1) / (C * CHOOSE_WARPS * SPAN)) * SPAN;
  const int start = (int)min((long long)n, (long long)(rank * CHOOSE_WARPS + warp) * per_warp);
  const int end = (int)min((long long)n, (long long)start + per_warp);
  const bool held = (long long)per_warp * CHOOSE_WARPS <= a.room;
  const float* w = a.w + (long long)layer * a.num_blocks * ((long long)a.heads << a.bs_log2);
  const int32_t* table = a.table + (long long)b * a.wide;
  const int bs = 1 << a.bs_log2;
  // the keys of positions i .. i + 3 (of one block) from memory
  auto fetch = [&](int i) {
    const int blk = table[i >> a.bs_log2];
    if (blk < 0 || blk >= a.num_blocks) {
      report_bad_block(a.ctl);
      return make_uint4(0, 0, 0, 0);
    }
    const float4 x = __ldg(reinterpret_cast<const float4*>(w + (((long long)blk * a.heads + h) << a.bs_log2) + (i & (bs - 1))));
    return make_uint4(order_of(x.x), order_of(x.y), order_of(x.z), order_of(x.w));
  };
  auto keys_of = [&](int i) {
    return held ? *reinterpret_cast<const uint4*>(keys + warp * per_warp + i - start) : fetch(i);
  };
  // f(position, key, valid) for this warp's positions, four a lane, in their order
  auto each = [&](auto load, auto f) {
#pragma unroll 4
    for (int base = start; base < end; base += SPAN) {
      const int i = base + lane * 4;
      uint4 k = make_uint4(0, 0, 0, 0);
      if (i < end) k = load(i);
      f(i, k);
    }
  };
  auto competes = [&](int i) { return (unsigned)(i - sink) < (unsigned)middle; };
  auto count = [&](uint32_t* bins, uint32_t bin, bool in) {
    // a whole warp in one bin (weights that are all 0, say) adds once
    const uint32_t first = __shfl_sync(~0u, bin, 0);
    if (__all_sync(~0u, in && bin == first)) {
      if (lane == 0) atomicAdd(&bins[first], 32u);
    } else if (in) {
      atomicAdd(&bins[bin], 1u);
    }
  };
  // The bin that holds the `want`-th key from the top, over all CTAs.
  auto find = [&](const uint32_t* bins, int size) {
    if (C > 1) cluster_sync();
    else __syncthreads();
    const int mine = size / CHOOSE_THREADS;                // 8 or 2 bins a thread, from the top
    const int lo = size - (tid + 1) * mine;
    uint32_t v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int r = 0; r < C; ++r) {
      const uint32_t at = mapa_shared(bins + (mine == 8 ? lo : lo & ~3), r);
      const uint4 x = ld_cluster_u4(at);
      if (mine == 8) {
        const uint4 y = ld_cluster_u4(at + 16);
        v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
        v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
      } else {
        v[6] += lo & 2 ? x.z : x.x;
        v[7] += lo & 2 ? x.w : x.y;
      }
    }
    uint32_t sum = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += v[e];
    uint32_t inc = sum;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const uint32_t o = __shfl_up_sync(~0u, inc, d);
      if (lane >= d) inc += o;
    }
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    uint32_t before = inc - sum;
    for (int x = 0; x < warp; ++x) before += warp_sum[x];
    if (before < (uint32_t)want && (uint32_t)want <= before + sum) {
      uint32_t c = before;
#pragma unroll
      for (int e = 7; e >= 0; --e) {                       // v[7] is the top one
        if (c < (uint32_t)want && (uint32_t)want <= c + v[e]) {
          found[0] = (uint32_t)(lo + e - (8 - mine));
          found[1] = (uint32_t)want - c;
          found[2] = v[e];
        }
        c += v[e];
      }
    }
    __syncthreads();
  };

  uint32_t border = 0xffffffffu, ties = 0, ties_kept = 0;  // no key is above this border
  if (held) {
    each(fetch, [&](int i, uint4 k) {
      if (i < end) *reinterpret_cast<uint4*>(keys + warp * per_warp + i - start) = k;
    });
    __syncwarp();
  }
  __syncthreads();
  if (want > 0) {
    const uint32_t* k1 = hist;
    each(keys_of, [&](int i, uint4 k) {
      const uint32_t x[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) count(hist, x[e] >> 20, i < end && competes(i + e));
    });
    find(k1, BINS1);
    border = found[0] << 20;
    want = (int)found[1];
    __syncthreads();
    each(keys_of, [&](int i, uint4 k) {
      const uint32_t x[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i < end && competes(i + e) && x[e] >> 20 == border >> 20) atomicAdd(&hist[BINS1 + (x[e] >> 10 & 1023)], 1u);
    });
    find(hist + BINS1, BINS2);
    border |= found[0] << 10;
    want = (int)found[1];
    __syncthreads();
    each(keys_of, [&](int i, uint4 k) {
      const uint32_t x[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i < end && competes(i + e) && x[e] >> 10 == border >> 10) atomicAdd(&hist[BINS1 + BINS2 + (x[e] & 1023)], 1u);
    });
    find(hist + BINS1 + BINS2, BINS2);
    border |= found[0];
    ties_kept = found[1];
    ties = found[2];
  }

  // Running sums over the CTAs and warps before this one of what `cnt[x]` holds.
  auto before_this = [&](int x) {
    __syncthreads();
    int in_cta = 0, all = 0;
    for (int y = 0; y < CHOOSE_WARPS; ++y) {
      if (y == warp) in_cta = all;
      all += cnt[x][y];
    }
    if (C == 1) return in_cta;
    if (tid == 0) total[x] = all;
    cluster_sync();
    for (int r = 0; r < rank; ++r) {
      int v;
      asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(&total[x], r)) : "memory");
      in_cta += v;
    }
    return in_cta;
  };
  const unsigned below = (1u << lane) - 1;
  // how many marks in lanes before this one, and in all, of four flags a lane
  auto rank4 = [&](const bool (&f)[4], int& all) {
    int mine = 0;
    all = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const unsigned m = __ballot_sync(~0u, f[e]);
      mine += __popc(m & below);
      all += __popc(m);
    }
    return mine;
  };
  // Of keys equal to the border the first `ties_kept` stay.
  const bool some_ties = ties != ties_kept;
  int tie0 = 0;
  if (some_ties) {
    int c = 0;
    each(keys_of, [&](int i, uint4 k) {
      const uint32_t x[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) c += i < end && competes(i + e) && x[e] == border;
    });
    c = __reduce_add_sync(~0u, c);
    if (lane == 0) cnt[0][warp] = c;
    tie0 = before_this(0);
  }
  // f(position, hole flags, late flags) in order
  auto marks = [&](auto f) {
    int tie = tie0;
    each(keys_of, [&](int i, uint4 k) {
      const uint32_t x[4] = {k.x, k.y, k.z, k.w};
      bool eq[4], hole[4], late[4];
      int rank_eq = 0, all = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) eq[e] = i < end && competes(i + e) && x[e] == border;
      if (some_ties) rank_eq = tie + rank4(eq, all);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int p = i + e;
        bool stays = !competes(p) || x[e] > border;
        if (eq[e]) stays = !some_ties ? ties > 0 : rank_eq < (int)ties_kept;
        rank_eq += eq[e];
        hole[e] = p < keep && !stays && i < end;
        late[e] = p >= keep && p < n && stays && i < end;
      }
      tie += all;
      f(i, hole, late);
    });
  };
  int holes = 0, lates = 0;
  marks([&](int, const bool (&hole)[4], const bool (&late)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      holes += hole[e];
      lates += late[e];
    }
  });
  holes = __reduce_add_sync(~0u, holes);
  lates = __reduce_add_sync(~0u, lates);
  if (lane == 0) {
    cnt[1][warp] = holes;
    cnt[2][warp] = lates;
  }
  int hole_at = before_this(1), late_at = before_this(2);
  bool over = false;
  marks([&](int i, const bool (&hole)[4], const bool (&late)[4]) {
    int all_h, all_l;
    int x = hole_at + rank4(hole, all_h), y = late_at + rank4(late, all_l);
    hole_at += all_h;
    late_at += all_l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (hole[e]) {
        if (x < a.max_moves) dst[x] = i + e;
        else over = true;
        ++x;
      }
      if (late[e]) {
        if (y < a.max_moves) src[y] = i + e;
        ++y;
      }
    }
  });
  if (over) report_status(a.ctl, ST_BAD_LENGTH);
  // the last warp's running sum is the number of moves; every CTA pads its share
  if (rank == C - 1 && warp == CHOOSE_WARPS - 1 && lane == 0) total[3] = hole_at;
  if (C > 1) cluster_sync();
  else __syncthreads();
  int moves;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(moves) : "r"(mapa_shared(&total[3], C - 1)) : "memory");
  moves = min(moves, a.max_moves);
  if (rank == 0 && tid == 0) a.counts[row] = moves;
  pad_from(moves);
  if (C > 1) cluster_sync();             // nobody leaves while others read its shared memory
}

// --------------------------------------------------------------------- move
constexpr int MOVE_THREADS = 256, MOVE_WARPS = MOVE_THREADS / 32;
constexpr int MOVE_BLOCKS = 256;         // blocks whose moves a CTA looks up at a time

struct MoveArgs {
  int8_t* codes[2];
  float* scales[2];                      // [layers][num_blocks][heads]
  float* w;                              // [layers][num_blocks][heads][bs] or null
  const int32_t *table, *keep, *src, *dst, *counts;
  long long layer_stride, block_stride;
  int B, heads, wide, num_blocks, bs_log2, max_moves;
  Ctl ctl;
};

// First i in [0, n) with a[i] >= x (n if none), a whole warp looking at 32
// places at a time; in [0, n] whatever a holds.
__device__ __forceinline__ int warp_lower_bound(const int32_t* a, int n, int x) {
  const int lane = threadIdx.x % 32;
  int lo = 0;
  while (n > 0) {
    const int step = (n + 31) / 32, at = lane * step;
    const int less = __popc(__ballot_sync(~0u, at < n && a[lo + at] < x));
    if (less == 0) return lo;
    // a[lo + (less - 1) step] < x
    const int skip = (less - 1) * step + 1;
    lo += skip;
    n = min(step - 1, n - skip);
  }
  return lo;
}

// One (layer, request, head) per cluster; a warp takes K or V of one block that
// receives rows: the rows' largest magnitude, the block's scale (it only grows,
// as when rows are appended), the rows' codes, and, where the scale grew, the
// block's other codes.  Rows leave places from the new length on and enter
// places below it, so the only block that is both read for others and written
// is the one that the new length falls into: it waits until the whole cluster
// is done with the others.
template <int D>
__global__ void __launch_bounds__(MOVE_THREADS) kv_evict_kernel(MoveArgs a) {
  constexpr int PARTS = D / 16;          // 16-byte pieces of a row
  __shared__ int2 range[MOVE_BLOCKS];    // a block's moves
  __shared__ int bounds[2];
  __shared__ int row_slot[MOVE_WARPS][128];                // where an incoming row is, -1: nowhere
  __shared__ uint8_t row_dst[MOVE_WARPS][128];
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int C = (int)cluster_size(), rank = (int)cluster_ctarank();
  const int row = blockIdx.x / C, h = row % a.heads, b = row / a.heads % a.B, layer = row / a.heads / a.B;
  const int bs = 1 << a.bs_log2;
  const int keep = a.keep[b];
  int moves = a.counts[row];
  if (keep < 0 || keep > (a.wide << a.bs_log2) || moves < 0 || moves > a.max_moves) {
    if (tid == 0) report_status(a.ctl, ST_BAD_LENGTH);
    moves = 0;
  }
  const int32_t* src = a.src + (long long)row * a.max_moves;
  const int32_t* dst = a.dst + (long long)row * a.max_moves;
  const int32_t* table = a.table + (long long)b * a.wide;
  const long long cell0 = (long long)layer * a.num_blocks * a.heads + h;
  auto cell = [&](int blk) { return cell0 + (long long)blk * a.heads; };
  auto in_pool = [&](int blk) { return blk >= 0 && blk < a.num_blocks; };

  // K (side 0) or V of block j, which receives moves [m0, m1)
  auto receive = [&](int j, int m0, int m1, int side) {
    const int blk = table[j], rows = min(m1 - m0, bs);
    if (!in_pool(blk)) {
      if (lane == 0) report_bad_block(a.ctl);
      return;
    }
    unsigned taken[4] = {0, 0, 0, 0};    // the block's rows that are written
    for (int r0 = 0; r0 < rows; r0 += 32) {
      const int r = r0 + lane;
      int slot = -1, to = 0;
      if (r < rows) {
        const int s = src[m0 + r];
        to = dst[m0 + r] - (j << a.bs_log2);
        const bool fits = s >= keep && s < (a.wide << a.bs_log2) && to >= 0 && to < bs && to + (j << a.bs_log2) < keep;
        const int from = fits ? table[s >> a.bs_log2] : 0;
        if (fits && in_pool(from)) slot = (from << a.bs_log2) + (s & (bs - 1));
        else report_status(a.ctl, fits ? ST_BAD_BLOCK : ST_BAD_LENGTH);
        row_slot[warp][r] = slot;
        row_dst[warp][r] = (uint8_t)to;
        if (side == 0 && a.w && slot >= 0)
          a.w[(cell(blk) << a.bs_log2) + to] = a.w[(cell(slot >> a.bs_log2) << a.bs_log2) + (slot & (bs - 1))];
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) taken[x] |= __reduce_or_sync(~0u, slot >= 0 && to / 32 == x ? 1u << (to & 31) : 0u);
    }
    __syncwarp();
    int8_t* codes = (side ? a.codes[1] : a.codes[0]) + layer * a.layer_stride + ((long long)h << a.bs_log2) * D;
    float* scales = side ? a.scales[1] : a.scales[0];
    const float before = scales[cell(blk)];
    auto at = [&](int slot, int part) {
      return reinterpret_cast<uint4*>(codes + (long long)(slot >> a.bs_log2) * a.block_stride + (slot & (bs - 1)) * D + part * 16);
    };
    float most = 0.f;
    for (int p = lane; p < rows * PARTS; p += 32) {
      const int slot = row_slot[warp][p / PARTS];
      if (slot < 0) continue;
      const uint4 c = *at(slot, p % PARTS);
      const uint32_t m = __vmaxu4(__vmaxu4(__vabs4(c.x), __vabs4(c.y)), __vmaxu4(__vabs4(c.z), __vabs4(c.w)));
      const uint32_t m1 = max(max(m & 0xffu, m >> 8 & 0xffu), max(m >> 16 & 0xffu, m >> 24));
      most = fmaxf(most, __fmul_rn((float)m1, scales[cell(slot >> a.bs_log2)]));
    }
    most = warp_max(most);
    const float s = fmaxf(fmaxf(before, __fdiv_rn(most, 127.f)), KV_SCALE_MIN);
    const float inv = __frcp_rn(s);
    auto round4 = [&](uint32_t c, float f, float g) {      // codes of c f g
      auto one = [&](int x) { return (uint32_t)(uint8_t)kv_code(__fmul_rn(__fmul_rn((float)x, f), g)); };
      return one((int8_t)c) | one((int8_t)(c >> 8)) << 8 | one((int8_t)(c >> 16)) << 16 | one((int8_t)(c >> 24)) << 24;
    };
    for (int p = lane; p < rows * PARTS; p += 32) {
      const int slot = row_slot[warp][p / PARTS];
      if (slot < 0) continue;
      const uint4 c = *at(slot, p % PARTS);
      const float f = scales[cell(slot >> a.bs_log2)];
      *at((blk << a.bs_log2) + row_dst[warp][p / PARTS], p % PARTS) =
          make_uint4(round4(c.x, f, inv), round4(c.y, f, inv), round4(c.z, f, inv), round4(c.w, f, inv));
    }
    __syncwarp();
    if (s == before) return;
    const float f = __fmul_rn(before, inv);
    for (int p = lane; p < bs * PARTS; p += 32) {
      const int to = p / PARTS;
      const unsigned word = to < 64 ? (to < 32 ? taken[0] : taken[1]) : (to < 96 ? taken[2] : taken[3]);
      if (word >> (to & 31) & 1) continue;
      uint4* q = at((blk << a.bs_log2) + to, p % PARTS);
      const uint4 c = *q;
      *q = make_uint4(round4(c.x, f, 1.f), round4(c.y, f, 1.f), round4(c.z, f, 1.f), round4(c.w, f, 1.f));
    }
    if (lane == 0) scales[cell(blk)] = s;
  };

  const int blocks = (int)(((long long)keep + bs - 1) >> a.bs_log2);
  const int edge = keep & (bs - 1) ? keep >> a.bs_log2 : -1;
  const int per = (blocks + C - 1) / C, last = min(blocks, (rank + 1) * per);
  int2 at_edge = make_int2(0, 0);
  if (moves > 0) {                       // (the same for the whole cluster)
    for (int j0 = rank * per; j0 < last; j0 += MOVE_BLOCKS) {
      const int j1 = min(last, j0 + MOVE_BLOCKS);
      __syncthreads();
      for (int j = tid; j < j1 - j0; j += MOVE_THREADS) range[j] = make_int2(0, 0);
      if (warp < 2) {
        const int x = warp_lower_bound(dst, moves, (warp == 0 ? j0 : j1) << a.bs_log2);
        if (lane == 0) bounds[warp] = x;
      }
      __syncthreads();
      // `dst` ascends: a block's moves are consecutive
      for (int i = bounds[0] + tid; i < bounds[1]; i += MOVE_THREADS) {
        const int j = dst[i] >> a.bs_log2;
        if (j < j0 || j >= j1) continue;
        if (i == bounds[0] || dst[i - 1] >> a.bs_log2 != j) range[j - j0].x = i;
        if (i + 1 == bounds[1] || dst[i + 1] >> a.bs_log2 != j) range[j - j0].y = i + 1;
      }
      __syncthreads();
      for (int u = warp; u < 2 * (j1 - j0); u += MOVE_WARPS) {
        const int j = j0 + u / 2;
        const int2 m = range[u / 2];
        if (m.x >= m.y) continue;
        if (j != edge) receive(j, m.x, m.y, u & 1);
      }
      if (edge >= j0 && edge < j1) at_edge = range[edge - j0];
    }
    if (C > 1) cluster_sync();
    else __syncthreads();
    if (at_edge.x < at_edge.y && warp < 2) receive(edge, at_edge.x, at_edge.y, warp);
  }
}

int log2_of(int64_t bs) { return bs == 32 ? 5 : bs == 64 ? 6 : 7; }

}  // namespace
}  // namespace qv

using namespace qv;

extern "C" int qvggt_evict_plan(const qvggt_evict_plan_args* p, void* stream) {
  const char* name = "evict_plan";
  if (!p || p->layers < 0 || p->num_blocks <= 0 || p->kv_heads <= 0 || p->requests < 0 || p->max_blocks < 0 ||
      p->sink < 0 || p->recent < 0 || p->max_moves < 0 || p->max_len < 0)
    return set_error(QVGGT_ERR_INVALID, "%s: bad shape", name);
  if (p->block_size != 32 && p->block_size != 64 && p->block_size != 128)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: block_size must be 32, 64 or 128", name);
  if (p->num_blocks > 2147483647LL / p->block_size || p->max_blocks > (1LL << 30) / p->block_size ||
      p->max_moves > 1LL << 30)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: more than 2^31 slots or 2^30 tokens a request", name);
  if (p->layers == 0 || p->requests == 0) return QVGGT_OK;
  // (each bound alone first, so that their product fits 64 bits)
  if (p->layers > 1 << 20 || p->requests > 1 << 24 || p->kv_heads > 65535 ||
      p->layers * p->kv_heads > 268435455LL / p->requests)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: too many layers, requests and heads", name);
  if (!p->weights || !p->block_tables || !p->lens || !p->keep || !p->counts || (p->max_moves && (!p->src || !p->dst)))
    return set_error(QVGGT_ERR_INVALID, "%s: null tensor", name);
  if (!aligned16(p->weights)) return set_error(QVGGT_ERR_ALIGN, "%s: weights must be 16-byte aligned", name);
  const int64_t rows = p->layers * p->requests * p->kv_heads;
  const int64_t longest = p->max_len ? std::min(p->max_len, p->max_blocks * p->block_size) : p->max_blocks * p->block_size;
  int C = 1;
  while (C < 8 && rows * C < 2 * device_info().num_sms && longest > 2048LL * C) C *= 2;
  const int64_t part = (longest + C * CHOOSE_WARPS * SPAN - 1) / (C * CHOOSE_WARPS * SPAN) * (CHOOSE_WARPS * SPAN);
  constexpr int ROOM_MAX = 48 * 1024;    // 192 KB of keys beside 25 KB of counts
  const int room = part <= ROOM_MAX ? (int)part : 0;
  ChooseArgs a{p->weights, p->block_tables, p->lens, p->keep, p->src, p->dst, p->counts, (int)p->requests,
               (int)p->kv_heads, (int)p->max_blocks, (int)p->num_blocks, log2_of(p->block_size),
               (int)std::min<int64_t>(p->sink, 2147483647LL), (int)std::min<int64_t>(p->recent, 2147483647LL),
               (int)p->max_moves, room, make_ctl()};
  static DeviceFlags attr;
  if (int rc = ensure_smem(attr, evict_plan_kernel, ROOM_MAX * 4, "cudaFuncSetAttribute(evict_plan)")) return rc;
  int rc = check_cuda(launch_pdl(evict_plan_kernel, dim3((unsigned)(rows * C)), dim3(CHOOSE_THREADS), (size_t)room * 4,
                                 static_cast<cudaStream_t>(stream), (unsigned)C, a),
                      "evict_plan launch");
  if (!rc) count_launch(1);
  return rc;
}

extern "C" int qvggt_kv_evict(const qvggt_kv_evict_args* p, void* stream) {
  const char* name = "kv_evict";
  if (!p) return set_error(QVGGT_ERR_INVALID, "%s: null arguments", name);
  const qvggt_kv_cache& c = p->cache;
  if (int rc = check_cache(name, c)) return rc;
  if (p->layers < 0 || p->requests < 0 || p->max_blocks < 0 || p->max_moves < 0)
    return set_error(QVGGT_ERR_INVALID, "%s: bad shape", name);
  if (p->max_blocks > (1LL << 30) / c.block_size || p->max_moves > 1LL << 30)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: more than 2^30 tokens a request", name);
  if (p->layers == 0 || p->requests == 0 || p->max_moves == 0) return QVGGT_OK;
  if (p->layers > 1 << 20 || p->requests > 1 << 24 || p->layers * c.kv_heads > 268435455LL / p->requests)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: too many layers, requests and heads", name);
  if (!p->block_tables || !p->keep || !p->src || !p->dst || !p->counts)
    return set_error(QVGGT_ERR_INVALID, "%s: null tensor", name);
  if (p->layer_stride % 16) return set_error(QVGGT_ERR_ALIGN, "%s: the layers must be 16-byte aligned", name);
  if (p->layers > 1 && p->layer_stride < (c.num_blocks - 1) * c.block_stride + c.kv_heads * c.block_size * c.head_dim)
    return set_error(QVGGT_ERR_INVALID, "%s: layer stride smaller than a layer", name);
  MoveArgs a{{c.k_cache, c.v_cache}, {c.k_scale, c.v_scale}, p->weights, p->block_tables, p->keep, p->src, p->dst,
             p->counts, p->layer_stride, c.block_stride, (int)p->requests, (int)c.kv_heads, (int)p->max_blocks,
             (int)c.num_blocks, log2_of(c.block_size), (int)p->max_moves, make_ctl()};
  const int64_t rows = p->layers * p->requests * c.kv_heads;
  int C = 1;
  while (C < 8 && rows * C < 8 * device_info().num_sms && p->max_blocks > 4LL * C) C *= 2;
  const auto fn = c.head_dim == 64 ? kv_evict_kernel<64> : kv_evict_kernel<128>;
  int rc = check_cuda(launch_pdl(fn, dim3((unsigned)(rows * C)), dim3(MOVE_THREADS), 0, static_cast<cudaStream_t>(stream),
                                 (unsigned)C, a),
                      "kv_evict launch");
  if (!rc) count_launch(1);
  return rc;
}
