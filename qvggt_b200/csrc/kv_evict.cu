// Making room in the paged 8-bit K/V cache: which keys of a request stay, and
// their move into the places of those that go.
//
// Keys may lie in any order in the cache (their positions are in the rotated
// rows), so only survivors past the new length move, each into the place of an
// evicted key below it; what stays where it is is not rounded again.
#include <type_traits>

#include "host.hpp"
#include "kv_cache.cuh"

namespace qv {
namespace {

// ------------------------------------------------------------------- choice
constexpr int CHOOSE_THREADS = 1024, CHOOSE_WARPS = CHOOSE_THREADS / 32;
constexpr int SPAN = 128;                // positions a warp takes at a time, four a lane
constexpr int ROOM_MAX = 48 * 1024;      // keys a CTA holds: 192 KB beside 25 KB of counts
// Digits of the 32-bit keys, from the top: 12, 10 and 10 bits.  The first one
// holds the exponent and three bits more, which spreads weights of any size
// over enough bins that few lanes meet in one.
constexpr int BINS1 = 4096, BINS2 = 1024;
static_assert(BINS1 == 4 * CHOOSE_THREADS && BINS2 == CHOOSE_THREADS, "a thread sums four bins, or one");

struct ChooseArgs {
  const float* w;                        // [layers][num_blocks][heads][bs]
  const int32_t *table, *lens, *keep;
  int32_t *src, *dst, *counts;           // [layers][B][heads][max_moves], counts without the last
  int B, heads, wide, num_blocks, bs_log2, sink, recent, max_moves;
  int room;                              // positions of a CTA that shared memory holds
  Ctl ctl;
};

// Weights as integers in their order: NaN and what is below every finite float
// count as the lowest (the maximum takes its other operand), infinity as the
// largest finite one, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float w) {
  const float big = 3.4028234663852886e38f;
  const int u = __float_as_int(fminf(fmaxf(w, -big), big) + 0.f);
  return (uint32_t)u ^ (uint32_t)(u >> 31 | 0x80000000);
}

__device__ __forceinline__ uint4 ld_cluster_u4(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}

// How many times four positions a thread has, of n over C CTAs with room for
// `room` keys each.  A multiple of four would put eight lanes' 16-byte reads into
// at most half of the banks: one more then, where it fits.
__host__ __device__ inline int quads_of(long long n, int C, int room) {
  const int q = (int)((n + 4LL * C * CHOOSE_THREADS - 1) / (4LL * C * CHOOSE_THREADS));
  return q % 4 == 0 && (q + 1) * 4LL * CHOOSE_THREADS <= room ? q + 1 : q;
}

// One (layer, request, head) per cluster of one to four CTAs.  The `keep`-th
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
  __shared__ uint32_t cnt[CHOOSE_WARPS]; // per warp: ties, then holes
  __shared__ uint32_t late_cnt[CHOOSE_WARPS];              // and late survivors
  __shared__ uint32_t total[3];          // of this CTA: ties, holes, late survivors
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
  uint32_t want = keep - sink - recent;
  const int run = 4 * quads_of(n, C, a.room), per_warp = 32 * run;
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
  auto competes = [&](int i) { return (unsigned)(i - sink) < (unsigned)middle; };
  // From the second pass on a lane looks at `run` positions in a row, which gives
  // ranks by sums alone (with four of each 128 it took votes: 83 us against 57,
  // 24 layers of 43,968).  Where all of a warp's runs lie among the competing
  // positions none is looked at alone.
  const int my = min((long long)n, (long long)start + lane * run), my_end = min((long long)n, (long long)my + run);
  const bool inside = __all_sync(~0u, my >= sink && my_end == my + run && my_end <= sink + middle);
  // f(position, key) of this lane's in their order
  auto own = [&](auto f) {
#pragma unroll 2
    for (int i = my; i < my_end; i += 4) {
      const uint4 k = keys_of(i);
      f(i, k.x);
      f(i + 1, k.y);
      f(i + 2, k.z);
      f(i + 3, k.w);
    }
  };
  // The bin that holds the `want`-th key from the top, over all CTAs.  PER: bins a thread sums.
  auto find = [&](const uint32_t* bins, auto PER) {
    if (C > 1) cluster_sync();
    else __syncthreads();
    const int lo = (CHOOSE_THREADS - 1 - tid) * PER;       // the first thread takes the top ones
    uint4 v = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (r >= C) continue;
      const uint32_t at = mapa_shared(bins + lo, r);
      if constexpr (PER == 4) {
        const uint4 x = ld_cluster_u4(at);
        v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
      } else {
        v.w += ld_cluster_u32(at);
      }
    }
    const uint32_t sum = v.x + v.y + v.z + v.w;
    uint32_t inc = sum;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const uint32_t o = __shfl_up_sync(~0u, inc, d);
      if (lane >= d) inc += o;
    }
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    const uint32_t others = lane < warp ? warp_sum[lane] : 0u;
    uint32_t c = __reduce_add_sync(~0u, others) + inc - sum;
    if (c < want && want <= c + sum) {
      const uint32_t x[4] = {v.w, v.z, v.y, v.x};          // from the top
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        if (c < want && want <= c + x[e]) {
          found[0] = (uint32_t)(lo + PER - 1 - e);
          found[1] = want - c;
          found[2] = x[e];
        }
        c += x[e];
      }
    }
    __syncthreads();
  };

  uint32_t border = 0xffffffffu, ties = 0, ties_kept = 0;  // no key is above this border
  __syncthreads();
  // the first digit is counted as the keys come in
#pragma unroll 2
  for (int base = start; base < end; base += SPAN) {
    const int i = base + lane * 4;
    uint4 k = make_uint4(0, 0, 0, 0);
    if (i < end) k = fetch(i);
    if (held && i < end) *reinterpret_cast<uint4*>(keys + warp * per_warp + i - start) = k;
    const uint32_t x[4] = {k.x >> 20, k.y >> 20, k.z >> 20, k.w >> 20};
    if (base >= sink && base + SPAN <= min(end, sink + middle)) {
      // all in one bin (weights that are all 0, say) add once: else they would queue
      const uint32_t first = __shfl_sync(~0u, x[0], 0);
      if (__all_sync(~0u, ((x[0] ^ first) | (x[1] ^ first) | (x[2] ^ first) | (x[3] ^ first)) == 0)) {
        if (lane == 0) atomicAdd(&hist[first], (uint32_t)SPAN);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) atomicAdd(&hist[x[e]], 1u);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i < end && competes(i + e)) atomicAdd(&hist[x[e]], 1u);
    }
  }
  __syncwarp();                          // the lanes read each other's keys from here on
  if (want > 0) {
    find(hist, std::integral_constant<int, 4>());
    border = found[0] << 20;
    want = found[1];
    __syncthreads();
    uint32_t* bins = hist + BINS1;
    own([&](int p, uint32_t x) {
      const uint32_t d = x - border;
      if (d < 1u << 20 && (inside || competes(p))) atomicAdd(&bins[d >> 10], 1u);
    });
    find(bins, std::integral_constant<int, 1>());
    border |= found[0] << 10;
    want = found[1];
    __syncthreads();
    bins += BINS2;
    if (inside) {
      // few keys have the border's first two digits: one branch for four
#pragma unroll 2
      for (int i = my; i < my_end; i += 4) {
        const uint4 k = keys_of(i);
        const uint32_t d[4] = {k.x - border, k.y - border, k.z - border, k.w - border};
        if (min(min(d[0], d[1]), min(d[2], d[3])) < 1024) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (d[e] < 1024) atomicAdd(&bins[d[e]], 1u);
        }
      }
    } else {
      own([&](int p, uint32_t x) {
        const uint32_t d = x - border;
        if (d < 1024 && competes(p)) atomicAdd(&bins[d], 1u);
      });
    }
    find(bins, std::integral_constant<int, 1>());
    border |= found[0];
    ties_kept = found[1];
    ties = found[2];
  }

  // The sum of the warps' counts before this one, and of all.
  auto warps_before = [&](const uint32_t* c, uint32_t& all) {
    const uint32_t v = c[lane];
    all = __reduce_add_sync(~0u, v);
    return __reduce_add_sync(~0u, lane < warp ? v : 0u);
  };
  static_assert(CHOOSE_WARPS == 32, "a lane per warp");
  // The sum over the lanes before this one.
  auto lanes_before = [&](int v) {
    int inc = v;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(~0u, inc, d);
      if (lane >= d) inc += o;
    }
    return inc - v;
  };
  // Of keys equal to the border the first `ties_kept` stay.
  const bool some_ties = ties != ties_kept;
  int tie0 = 0;
  if (some_ties) {
    int c = 0;
    own([&](int p, uint32_t x) { c += x == border && competes(p); });
    tie0 = lanes_before(c);
    c = __reduce_add_sync(~0u, c);
    if (lane == 0) cnt[warp] = c;
    __syncthreads();
    uint32_t all;
    tie0 += warps_before(cnt, all);
    if (tid == 0) total[0] = all;
    if (C > 1) {
      cluster_sync();
      const uint32_t v = lane < rank ? ld_cluster_u32(mapa_shared(&total[0], lane)) : 0u;
      tie0 += __reduce_add_sync(~0u, v);
    }
    __syncthreads();                     // everyone has read cnt
  }
  // Marks among the competing positions: below `keep` what goes (a hole), from there on
  // what stays (a late survivor), which has to move.  The last `tail` positions, which
  // all stay, are the last to move.
  const int tail = min(recent, n - keep);
  const bool among = my >= sink && my_end <= sink + middle, apart = my_end <= sink || my >= sink + middle;
  const bool plain = __all_sync(~0u, apart || (among && !some_ties && (my_end <= keep || my >= keep) && my_end % 4 == 0));
  const int last = apart ? my : my_end;
  // marks of positions i .. i + 3, the first one's in bit 3
  auto marks = [&](int i, int& tie, auto PLAIN) {
    const uint4 k = keys_of(i);
    const bool alike = PLAIN || (!some_ties && competes(i) && competes(i + 3) && (i >= keep) == (i + 3 >= keep));
    if (alike) {
      const uint32_t stay = (k.x >= border ? 8 : 0) | (k.y >= border ? 4 : 0) | (k.z >= border ? 2 : 0) | (k.w >= border ? 1 : 0);
      return stay ^ ((PLAIN ? my : i) >= keep ? 0u : 15u);
    }
    const uint32_t x[4] = {k.x, k.y, k.z, k.w};
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int p = i + e;
      const bool in = competes(p), stays = x[e] > border || (x[e] == border && in && (!some_ties || tie++ < (int)ties_kept));
      if (in && stays == (p >= keep)) bits |= 8 >> e;
    }
    return bits;
  };
  const std::true_type PLAIN;
  const std::false_type MIXED;
  int holes = 0, lates = 0, tie = tie0;
  uint64_t mark = 0;                     // of this lane's positions, the first one's in the highest bit
  static_assert(ROOM_MAX / CHOOSE_THREADS <= 64, "a mask of a lane's positions");
  if (held) {
    if (plain) {
#pragma unroll 2
      for (int i = my; i < last; i += 4) mark = mark << 4 | marks(i, tie, PLAIN);
    } else {
#pragma unroll 1
      for (int i = my; i < last; i += 4) mark = mark << 4 | marks(i, tie, MIXED);
    }
    if (last > my) mark <<= 64 - (last - my + 3) / 4 * 4;
    const int before_keep = max(0, keep - my);             // positions, 0 to all
    holes = __popcll(before_keep >= 64 ? mark : mark & ~(~0ull >> before_keep));
    lates = __popcll(mark) - holes;
  } else {
    for (int i = my; i < last; i += 4) {
      const uint32_t b = marks(i, tie, MIXED), h = i >= keep ? 0 : keep - i >= 4 ? b : b & ~(15u >> (keep - i));
      holes += __popc(h);
      lates += __popc(b ^ h);
    }
  }
  const int holes0 = lanes_before(holes), lates0 = lanes_before(lates);
  const int warp_holes = __reduce_add_sync(~0u, holes), warp_lates = __reduce_add_sync(~0u, lates);
  if (lane == 0) {
    cnt[warp] = warp_holes;
    late_cnt[warp] = warp_lates;
  }
  __syncthreads();
  uint32_t all_holes, all_lates;
  int hole_at = warps_before(cnt, all_holes), late_at = warps_before(late_cnt, all_lates);    // of this warp
  int moves = (int)all_holes;
  if (C > 1) {
    if (tid == 0) {
      total[1] = all_holes;
      total[2] = all_lates;
    }
    cluster_sync();
    const uint32_t vh = lane < C ? ld_cluster_u32(mapa_shared(&total[1], lane)) : 0u;
    const uint32_t vl = lane < rank ? ld_cluster_u32(mapa_shared(&total[2], lane)) : 0u;
    moves = __reduce_add_sync(~0u, vh);
    hole_at += __reduce_add_sync(~0u, lane < rank ? vh : 0u);
    late_at += __reduce_add_sync(~0u, vl);
  }
  if (held) {
    // through shared memory, in the place of this warp's keys: each lane's own are
    // scattered (16 % slower with 60,000 keys)
    int32_t* list = reinterpret_cast<int32_t*>(keys + warp * per_warp);
    const int to_late = warp_holes + lates0 - holes;       // a lane's holes come before its late survivors
    int c = 0;
    __syncwarp();
    for (uint64_t m = mark; m; ++c) {
      const int x = __clzll((long long)m);
      list[c + (c < holes ? holes0 : to_late)] = my + x;
      m &= ~(1ull << 63 >> x);
    }
    __syncwarp();
    for (int x = lane; x < warp_holes; x += 32)
      if (hole_at + x < a.max_moves) dst[hole_at + x] = list[x];
    for (int x = lane; x < warp_lates; x += 32)
      if (late_at + x < a.max_moves) src[late_at + x] = list[warp_holes + x];
  } else {
    hole_at += holes0;
    late_at += lates0;
    tie = tie0;
    for (int i = my; i < last; i += 4) {
      const uint32_t b = marks(i, tie, MIXED);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool on = b >> (3 - e) & 1, late = i + e >= keep;
        const int at = late ? late_at : hole_at;
        if (on && at < a.max_moves) (late ? src : dst)[at] = i + e;
        late_at += late && on;
        hole_at += !late && on;
      }
    }
  }
  for (int x = rank * CHOOSE_THREADS + tid; x < tail; x += C * CHOOSE_THREADS)
    if (moves - tail + x < a.max_moves) src[moves - tail + x] = n - tail + x;
  if (rank == 0 && tid == 0) {
    if (moves > a.max_moves) report_status(a.ctl, ST_BAD_LENGTH);
    a.counts[row] = min(moves, a.max_moves);
  }
  pad_from(moves);
  if (C > 1) cluster_sync();             // nobody leaves while others read its shared memory
}

// --------------------------------------------------------------------- move
constexpr int MOVE_THREADS = 256;
constexpr int MOVE_BLOCKS = 256;         // blocks of a CTA at most
constexpr int MOVE_ROWS = 2048;          // rows they receive at most
constexpr uint32_t NOWHERE = 0xffffffffu;
constexpr int MOVE_LOADS = 8;            // 16-byte pieces a lane has under way

struct MoveArgs {
  int8_t* codes[2];
  float* scales[2];                      // [layers][num_blocks][heads]
  float* w;                              // [layers][num_blocks][heads][bs] or null
  const int32_t *table, *keep, *src, *dst, *counts;
  long long layer_stride, block_stride;
  int B, heads, wide, num_blocks, bs_log2, max_moves;
  int parts, span;                       // CTAs of a (layer, request, head), blocks of each
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

// Four codes c rounded anew: rint(c f g).  A byte with its sign bit flipped under
// the exponent of 2^23 is the float 2^23 + 128 + c, and adding 1.5 * 2^23 rounds to
// the nearest integer, ties to even, into the low byte: a conversion each way goes
// through the 16-a-clock pipe, which then bounds the kernel.  (The products stay
// between -128 and 127 because the scale covers them.)
template <bool TWO>
__device__ __forceinline__ uint32_t recode4(uint32_t c, float f, float g) {
  const uint32_t u = c ^ 0x80808080u;
  const uint64_t B = f2_pack(-8388736.f, -8388736.f), M = f2_pack(12582912.f, 12582912.f), F = f2_pack(f, f);
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; e += 2) {
    uint64_t x = f2_add(f2_pack(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 | e)),
                                __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441 | e))), B);
    if (TWO) x = f2_mul(x, F);
    // the last product alone: a paired one is compiled into one rounding with the addition
    const float z = TWO ? g : f;
    f2_unpack(x, y[e], y[e + 1]);
    f2_unpack(f2_add(f2_pack(__fmul_rn(y[e], z), __fmul_rn(y[e + 1], z)), M), y[e], y[e + 1]);
  }
  return __byte_perm(__byte_perm(__float_as_uint(y[0]), __float_as_uint(y[1]), 0x0040),
                     __byte_perm(__float_as_uint(y[2]), __float_as_uint(y[3]), 0x0040), 0x5410);
}
template <bool TWO>
__device__ __forceinline__ uint4 recode16(uint4 c, float f, float g) {
  return make_uint4(recode4<TWO>(c.x, f, g), recode4<TWO>(c.y, f, g), recode4<TWO>(c.z, f, g), recode4<TWO>(c.w, f, g));
}
// The largest magnitude of 16 codes.
__device__ __forceinline__ float largest16(uint4 c) {
  const uint32_t m = __vmaxu4(__vmaxu4(__vabs4(c.x), __vabs4(c.y)), __vmaxu4(__vabs4(c.z), __vabs4(c.w)));
  return (float)max(max(m & 0xffu, m >> 8 & 0xffu), max(m >> 16 & 0xffu, m >> 24));
}

// A CTA takes up to MOVE_BLOCKS blocks of one (layer, request, head).  It looks up
// where all their incoming rows are and at what scales (a chain of four loads that
// each block would wait for alone), and moves their weights.  Then a warp takes K
// or V of one block that receives rows: the rows' largest magnitude, the block's
// scale (it only grows, as when rows are appended), the rows' codes, and, where
// the scale grew, the block's other codes.  Rows leave places from the new length
// on and enter places below it, so the only block that is both read for others
// and written is the one that the new length falls into: a second launch (EDGE)
// does that one, when all others are done.
template <int D, bool EDGE>
__global__ void __launch_bounds__(MOVE_THREADS, 3) kv_evict_kernel(MoveArgs a) {
  constexpr int PARTS = D / 16;          // 16-byte pieces of a row
  __shared__ int2 range[MOVE_BLOCKS];    // a block's moves, from the CTA's first on
  __shared__ int block_id[MOVE_BLOCKS];  // -1: outside the cache
  __shared__ float block_scale[2][MOVE_BLOCKS];
  __shared__ int bounds[2];
  __shared__ uint32_t row_at[MOVE_ROWS];   // where an incoming row's codes are, in 16-byte pieces, NOWHERE: nowhere
  __shared__ float row_scale[2][MOVE_ROWS];
  __shared__ uint8_t row_to[MOVE_ROWS];
  pdl_wait();
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const int h = row % a.heads, b = row / a.heads % a.B, layer = row / a.heads / a.B;
  const int bs = 1 << a.bs_log2;
  const int keep = a.keep[b];
  const int moves = a.counts[row];
  if (moves == 0) return;                // whatever `keep` says: a request that holds no more stays
  if (keep < 0 || keep > (a.wide << a.bs_log2) || moves < 0 || moves > a.max_moves) {
    if (tid == 0) report_status(a.ctl, ST_BAD_LENGTH);
    return;
  }
  const int blocks = (int)(((long long)keep + bs - 1) >> a.bs_log2);
  const int edge = keep & (bs - 1) ? keep >> a.bs_log2 : -1;
  const int j0 = EDGE ? edge : part * a.span, j1 = EDGE ? edge + 1 : min(blocks, j0 + a.span);
  const int32_t* src = a.src + (long long)row * a.max_moves;
  const int32_t* dst = a.dst + (long long)row * a.max_moves;
  // (places that lie in no block below `keep`, at either end as they ascend, come to no CTA's list)
  if (!EDGE && part == 0 && tid == 0 && (dst[0] < 0 || dst[moves - 1] >= keep)) report_status(a.ctl, ST_BAD_LENGTH);
  if (j0 < 0 || j0 >= j1) return;
  const int32_t* table = a.table + (long long)b * a.wide;
  const long long cell0 = (long long)layer * a.num_blocks * a.heads + h;
  auto cell = [&](int blk) { return cell0 + (long long)blk * a.heads; };
  auto in_pool = [&](int blk) { return blk >= 0 && blk < a.num_blocks; };
  auto piece_of = [&](int blk) { return (uint32_t)(blk * (a.block_stride / 16)) + (uint32_t)(h << a.bs_log2) * PARTS; };

  for (int j = tid; j < j1 - j0; j += blockDim.x) {
    const int blk = table[j0 + j];
    range[j] = make_int2(0, 0);
    block_id[j] = in_pool(blk) ? blk : -1;
    if (in_pool(blk)) {
      block_scale[0][j] = a.scales[0][cell(blk)];
      block_scale[1][j] = a.scales[1][cell(blk)];
    }
  }
  if (warp < 2) {
    const int x = warp_lower_bound(dst, moves, (warp == 0 ? j0 : j1) << a.bs_log2);
    if (lane == 0) bounds[warp] = x;
  }
  __syncthreads();
  // `dst` ascends: a block's moves are consecutive, and no more than its rows
  const int m0 = bounds[0], m1 = min(bounds[1], m0 + MOVE_ROWS);
  for (int m = m0 + tid; m < m1; m += blockDim.x) {
    const int to = dst[m], s = src[m], j = to >> a.bs_log2;
    row_at[m - m0] = NOWHERE;
    if (j < j0 || j >= j1) continue;
    if (m == m0 || dst[m - 1] >> a.bs_log2 != j) range[j - j0].x = m - m0;
    if (m + 1 == m1 || dst[m + 1] >> a.bs_log2 != j) range[j - j0].y = m + 1 - m0;
    if (!EDGE && j == edge) continue;    // the second launch's
    const bool fits = s >= keep && s < (a.wide << a.bs_log2) && to < keep;
    const int from = fits ? table[s >> a.bs_log2] : -1, at = block_id[j - j0];
    if (in_pool(from) && at >= 0) {
      row_at[m - m0] = piece_of(from) + (s & (bs - 1)) * PARTS;
      row_to[m - m0] = (uint8_t)(to & (bs - 1));
      row_scale[0][m - m0] = a.scales[0][cell(from)];
      row_scale[1][m - m0] = a.scales[1][cell(from)];
      if (a.w) a.w[(cell(at) << a.bs_log2) + (to & (bs - 1))] = a.w[(cell(from) << a.bs_log2) + (s & (bs - 1))];
    } else {
      report_status(a.ctl, fits ? ST_BAD_BLOCK : ST_BAD_LENGTH);
    }
  }
  __syncthreads();
  // A group of lanes for each side of a block: a warp, or eight lanes where the
  // blocks receive few rows.  A step that makes room for one frame in 32 moves two
  // rows into a block: 24 layers of 43,968 keys, scales that hold what comes in, 124
  // us, 368 with a warp each.  (464 the first time, when the scales of a quarter of
  // all blocks grow and their other rows are rounded anew, by eight lanes a block.)
  const auto units = [&](auto GROUP) {
    constexpr int G = GROUP, AT_ONCE = G * MOVE_LOADS;     // pieces under way
    const int gl = tid % G;
    const unsigned mask = G == 32 ? ~0u : ((1u << (G & 31)) - 1) << (lane & ~(G - 1));
    for (int u = tid / G; u < 2 * (j1 - j0); u += blockDim.x / G) {
      const int j = u / 2, side = u & 1, blk = block_id[j];
      const int2 m = range[j];
      const int rows = min(m.y - m.x, bs);
      if (rows <= 0 || blk < 0 || (!EDGE && j0 + j == edge)) continue;
      const uint32_t* from = row_at + m.x;
      const float* from_scale = row_scale[side] + m.x;
      const uint8_t* to = row_to + m.x;
      uint4* codes = reinterpret_cast<uint4*>((side ? a.codes[1] : a.codes[0]) + layer * a.layer_stride);
      uint4* mine = codes + piece_of(blk);
      const float before = block_scale[side][j];
      const int pieces = rows * PARTS;
      uint4 c[MOVE_LOADS];
      auto load = [&](int p0) {
#pragma unroll
        for (int x = 0; x < MOVE_LOADS; ++x) {
          const int p = p0 + G * x + gl;
          c[x] = make_uint4(0, 0, 0, 0);
          if (p < pieces && from[p / PARTS] != NOWHERE) c[x] = codes[from[p / PARTS] + p % PARTS];
        }
      };
      // where all rows fit the registers (`once`) they are read once, else again for their codes
      const bool once = pieces <= AT_ONCE;
      float most = 0.f;
      for (int p0 = 0; p0 < pieces; p0 += AT_ONCE) {
        load(p0);
#pragma unroll
        for (int x = 0; x < MOVE_LOADS; ++x) {
          const int p = p0 + G * x + gl;
          if (p < pieces && from[p / PARTS] != NOWHERE) most = fmaxf(most, __fmul_rn(largest16(c[x]), from_scale[p / PARTS]));
        }
      }
#pragma unroll
      for (int d = G / 2; d > 0; d /= 2) most = fmaxf(most, __shfl_xor_sync(mask, most, d));
      const float s = fmaxf(fmaxf(before, __fdiv_rn(most, 127.f)), KV_SCALE_MIN);
      const float inv = __frcp_rn(s);
      for (int p0 = 0; p0 < pieces; p0 += AT_ONCE) {
        if (!once) load(p0);
#pragma unroll
        for (int x = 0; x < MOVE_LOADS; ++x) {
          const int p = p0 + G * x + gl, r = p / PARTS;
          if (p < pieces && from[r] != NOWHERE) mine[to[r] * PARTS + p % PARTS] = recode16<true>(c[x], from_scale[r], inv);
        }
      }
      if (s == before) continue;
      // (in the block that the new length falls into these rows are incoming ones' sources too: all lanes' reads first)
      __syncwarp(mask);
      unsigned taken[4] = {0, 0, 0, 0};  // the block's rows that were written
      for (int r0 = 0; r0 < rows; r0 += G) {
        const int r = r0 + gl;
        const int at = r < rows && from[r] != NOWHERE ? to[r] : 128;
#pragma unroll
        for (int x = 0; x < 4; ++x) taken[x] |= __reduce_or_sync(mask, at / 32 == x ? 1u << (at & 31) : 0u);
      }
      const float f = __fmul_rn(before, inv);
      for (int p0 = 0; p0 < bs * PARTS; p0 += AT_ONCE) {
        auto stays = [&](int x) {
          const int r = (p0 + G * x + gl) / PARTS;
          const unsigned word = r < 64 ? (r < 32 ? taken[0] : taken[1]) : (r < 96 ? taken[2] : taken[3]);
          return r < bs && !(word >> (r & 31) & 1);
        };
#pragma unroll
        for (int x = 0; x < MOVE_LOADS; ++x)
          if (stays(x)) c[x] = mine[p0 + G * x + gl];
#pragma unroll
        for (int x = 0; x < MOVE_LOADS; ++x)
          if (stays(x)) mine[p0 + G * x + gl] = recode16<false>(c[x], f, 0.f);
      }
      if (gl == 0) (side ? a.scales[1] : a.scales[0])[cell(blk)] = s;
    }
  };
  if (EDGE || (m1 - m0) * PARTS > 32 * (j1 - j0)) units(std::integral_constant<int, 32>());
  else units(std::integral_constant<int, 8>());
  // at the end: CTAs of the next kernel that wait beside this one's slow it (four
  // layers and their reading, no scale grows: 213 us with the call at the start, 198 here)
  pdl_trigger();
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
  // Clusters where the rows alone leave SMs idle and each CTA still has 8192 keys:
  // a cluster's barriers cost about 8 us (16 rows of 44,000 keys: 45 us as one CTA
  // each, 21 as four; 128 rows of 8,000: 11.5 and 24).  Eight CTAs to a cluster
  // only halve how many run at once (16 rows: 40 us).  The rule looks at the rows
  // alone.  Where the longest passes ROOM_MAX nothing is held with one CTA a row, and
  // two CTAs for each row, which hold it, would take 107 us against 145 (384 rows of
  // 49,464 keys), 161 against 211 (of 60,456), 43 against 64 (128 of 49,464); for one
  // such row of 24 beside short ones (16 heads) 66 against 55.
  while (C < 4 && 2 * rows * C <= device_info().num_sms && longest > 8192LL * C) C *= 2;
  const int64_t part = quads_of(longest, C, ROOM_MAX) * 4LL * CHOOSE_THREADS;
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
  // (places are 32-bit numbers of 16-byte pieces)
  if (c.num_blocks * c.block_stride / 16 >= NOWHERE)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: a layer of more than 2^36 bytes", name);
  if (p->layers > 1 && p->layer_stride % 16) return set_error(QVGGT_ERR_ALIGN, "%s: the layers must be 16-byte aligned", name);
  if (p->layers > 1 && p->layer_stride < (c.num_blocks - 1) * c.block_stride + c.kv_heads * c.block_size * c.head_dim)
    return set_error(QVGGT_ERR_INVALID, "%s: layer stride smaller than a layer", name);
  const int64_t rows = p->layers * p->requests * c.kv_heads;
  // as many blocks a CTA as leave every SM some CTAs, and as its lists hold: all rows
  // of the blocks, or all moves there can be
  const int64_t most = p->max_moves <= MOVE_ROWS ? MOVE_BLOCKS : std::min<int64_t>(MOVE_BLOCKS, MOVE_ROWS / c.block_size);
  const int64_t span = std::max<int64_t>(4, std::min<int64_t>(most, rows * p->max_blocks / (16 * device_info().num_sms)));
  const int64_t parts = std::max<int64_t>(1, (p->max_blocks + span - 1) / span);
  if (rows * parts > 2147483647LL) return set_error(QVGGT_ERR_UNSUPPORTED, "%s: too many blocks", name);
  MoveArgs a{{c.k_cache, c.v_cache}, {c.k_scale, c.v_scale}, p->weights, p->block_tables, p->keep, p->src, p->dst,
             p->counts, p->layers > 1 ? p->layer_stride : 0, c.block_stride, (int)p->requests, (int)c.kv_heads, (int)p->max_blocks,
             (int)c.num_blocks, log2_of(c.block_size), (int)p->max_moves, (int)parts, (int)span, make_ctl()};
  using Kfn = void (*)(MoveArgs);
  static const Kfn fns[2][2] = {{kv_evict_kernel<64, false>, kv_evict_kernel<64, true>},
                                {kv_evict_kernel<128, false>, kv_evict_kernel<128, true>}};
  for (int edge = 0; edge < 2; ++edge) {
    if (edge) a.parts = 1;
    if (int rc = check_cuda(launch_pdl(fns[c.head_dim == 128][edge], dim3((unsigned)(rows * a.parts)),
                                       dim3(edge ? 64 : MOVE_THREADS), 0, static_cast<cudaStream_t>(stream), 1u, a),
                            "kv_evict launch"))
      return rc;
    count_launch(1);
  }
  return QVGGT_OK;
}
