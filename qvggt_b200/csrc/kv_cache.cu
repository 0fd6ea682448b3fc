// A paged K/V cache in 8 bits: block tables and slot maps, the quantising
// write, and the read-back.
//
// Layout: codes int8 [blocks][kv heads][block_size][head_dim] (one tensor for
// K, one for V) and one fp32 scale per (block, kv head): a (block, head) tile
// is contiguous, so attention fetches it with one bulk copy.  Token j of
// request b is at offset j % block_size of block table[b][j / block_size].
#include "host.hpp"
#include "kv_cache.cuh"

namespace qv {
namespace {

// ------------------------------------------------------------ block tables
constexpr int PLAN_THREADS = 512;
constexpr int PLAN_MAX_REQUESTS = 8192;   // 4 prefix arrays of it fit shared memory

enum : int32_t {
  PLAN_OK = 0, PLAN_NO_BLOCKS = 1, PLAN_TABLE_FULL = 2, PLAN_BAD_LENGTH = 3, PLAN_MORE_TOKENS = 4, PLAN_BAD_POOL = 5
};

struct PlanArgs {
  const int32_t *cached, *target;
  int32_t* table;
  int32_t* ring;
  const long long* free_range;
  int32_t *slots, *cu_new, *cu_blocks, *lens, *status;
  long long* free_out;
  int B, wide, bs, num_blocks, most;
  Ctl ctl;
};

// New tokens and blocks given back add up to at most 2^32 - 1 and stay there:
// 8192 requests' can be more than 32 bits hold, and no sum that large is served.
// (The other two counts are not above the new tokens.)
__device__ __forceinline__ unsigned add_sat(unsigned a, unsigned b) { return a + b < a ? ~0u : a + b; }
struct Quad {
  unsigned new_tok, grow, drop, touched;
  __device__ Quad operator+(const Quad& o) const {
    return {add_sat(new_tok, o.new_tok), grow + o.grow, add_sat(drop, o.drop), touched + o.touched};
  }
};
__device__ __forceinline__ Quad shfl_up(const Quad& v, int d) {
  return {__shfl_up_sync(~0u, v.new_tok, d), __shfl_up_sync(~0u, v.grow, d), __shfl_up_sync(~0u, v.drop, d),
          __shfl_up_sync(~0u, v.touched, d)};
}

// What request i contributes when it goes from `c` to `t` tokens.
__device__ __forceinline__ Quad plan_counts(int c, int t, int bs) {
  const int have = (int)(((long long)c + bs - 1) / bs), need = (int)(((long long)t + bs - 1) / bs);
  return {(unsigned)max(t - c, 0), (unsigned)max(need - have, 0), (unsigned)max(have - need, 0),
          t > c ? (unsigned)((t - 1) / bs - c / bs + 1) : 0u};
}

// Largest i in [0, n) with a[i] <= x (a[0] = 0 <= x, a non-decreasing).
__device__ __forceinline__ int last_le(const int* a, int n, int x) {
  int lo = 0;
  while (n > 1) {
    const int half = n / 2;
    if (a[lo + half] <= x) lo += half;
    n -= half;
  }
  return lo;
}

// One launch, no CTA waits for another: every CTA repeats the scan over the
// requests (a few KB out of L2) and then writes its share of the slots and
// table entries.  The call changes all requests or, when it cannot serve one
// of them, none.
__global__ void __launch_bounds__(PLAN_THREADS) block_plan_kernel(PlanArgs a) {
  extern __shared__ int sm[];
  int* cu_new = sm;                          // [B + 1] exclusive prefix sums
  int* first = cu_new + a.B + 1;             // blocks taken by the requests before
  int* freed = first + a.B + 1;              // blocks given back by the requests before
  int* cu_blk = freed + a.B + 1;             // blocks written by the requests before
  __shared__ Quad warp_sum_[PLAN_THREADS / 32];
  __shared__ int bad;
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int per = (a.B + PLAN_THREADS - 1) / PLAN_THREADS;
  const int i0 = min(a.B, tid * per), i1 = min(a.B, i0 + per);
  if (tid == 0) bad = 0;
  __syncthreads();
  Quad sum{0, 0, 0, 0};
  int my_bad = 0;
  for (int i = i0; i < i1; ++i) {
    const int c = a.cached[i], t = a.target[i];
    if (c < 0 || t < 0) {
      my_bad |= 1 << PLAN_BAD_LENGTH;
      continue;
    }
    if (((long long)t + a.bs - 1) / a.bs > a.wide || ((long long)c + a.bs - 1) / a.bs > a.wide)
      my_bad |= 1 << PLAN_TABLE_FULL;
    sum = sum + plan_counts(c, t, a.bs);
  }
  if (my_bad) atomicOr(&bad, my_bad);
  Quad inc = sum;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const Quad o = shfl_up(inc, d);
    if (lane >= d) inc = inc + o;
  }
  if (lane == 31) warp_sum_[warp] = inc;
  __syncthreads();
  Quad base{0, 0, 0, 0}, total{0, 0, 0, 0};
  for (int w = 0; w < PLAN_THREADS / 32; ++w) {
    if (w == warp) base = total;
    total = total + warp_sum_[w];
  }
  const long long head = a.free_range[0], tail = a.free_range[1];
  int flags = bad;
  if (total.new_tok > (unsigned)a.most) flags |= 1 << PLAN_MORE_TOKENS;
  if ((long long)total.grow > tail - head) flags |= 1 << PLAN_NO_BLOCKS;
  // The free blocks and those given back have to fit the ring: then no place of
  // it is written that holds a free block, nor one outside it.
  if (head < 0 || tail < head || tail - head > a.num_blocks ||
      (long long)total.drop > a.num_blocks - (tail - head))
    flags |= 1 << PLAN_BAD_POOL;
  // the first reason in this order is reported
  const int status = flags & (1 << PLAN_BAD_LENGTH)    ? PLAN_BAD_LENGTH
                     : flags & (1 << PLAN_TABLE_FULL)  ? PLAN_TABLE_FULL
                     : flags & (1 << PLAN_MORE_TOKENS) ? PLAN_MORE_TOKENS
                     : flags & (1 << PLAN_BAD_POOL)    ? PLAN_BAD_POOL
                     : flags & (1 << PLAN_NO_BLOCKS)   ? PLAN_NO_BLOCKS
                                                       : PLAN_OK;
  const bool ok = status == PLAN_OK;
  if (!ok) total = Quad{0, 0, 0, 0};
  const int new_tok = (int)total.new_tok, grow = (int)total.grow, drop = (int)total.drop;
  Quad run = base + Quad{inc.new_tok - sum.new_tok, inc.grow - sum.grow, inc.drop - sum.drop,
                         inc.touched - sum.touched};
  for (int i = i0; i < i1; ++i) {
    cu_new[i] = ok ? run.new_tok : 0;
    first[i] = run.grow;
    freed[i] = run.drop;
    cu_blk[i] = ok ? run.touched : 0;
    const int c = a.cached[i], t = a.target[i];
    if (blockIdx.x == 0) a.lens[i] = ok ? t : c;
    if (ok) run = run + plan_counts(c, t, a.bs);
  }
  if (tid == 0) {
    cu_new[a.B] = new_tok;
    first[a.B] = grow;
    freed[a.B] = drop;
    cu_blk[a.B] = total.touched;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int i = tid; i <= a.B; i += PLAN_THREADS) {
      a.cu_new[i] = cu_new[i];
      a.cu_blocks[i] = cu_blk[i];
    }
    if (tid == 0) {
      a.free_out[0] = head + grow;
      a.free_out[1] = tail + drop;
      a.status[0] = status;
    }
  }
  const int gtid = blockIdx.x * PLAN_THREADS + tid, gsize = gridDim.x * PLAN_THREADS;
  const int head_m = (int)(head % a.num_blocks), tail_m = (int)(tail % a.num_blocks);
  auto ring_at = [&](int from, int off) {    // off < num_blocks
    const int x = from + off;
    return x >= a.num_blocks ? x - a.num_blocks : x;
  };
  // Block ids are handed on as they stand; one outside the cache is reported,
  // and its tokens get no slot (a product of it could look like one).
  auto in_cache = [&](int blk) {
    if (blk >= 0 && blk < a.num_blocks) return true;
    report_bad_block(a.ctl);
    return false;
  };
  for (int n = gtid; n < a.most; n += gsize) {
    int slot = -1;
    if (n < new_tok) {
      const int b = last_le(cu_new, a.B, n);
      const int c = a.cached[b], pos = c + (n - cu_new[b]);
      const int have = (c + a.bs - 1) / a.bs, j = pos / a.bs;
      const int blk = j < have ? a.table[(long long)b * a.wide + j] : a.ring[ring_at(head_m, first[b] + j - have)];
      if (in_cache(blk)) slot = blk * a.bs + pos - j * a.bs;
    }
    a.slots[n] = slot;
  }
  for (int n = gtid; n < grow; n += gsize) {
    const int b = last_le(first, a.B, n);
    const int have = (a.cached[b] + a.bs - 1) / a.bs;
    const int blk = a.ring[ring_at(head_m, n)];
    in_cache(blk);
    a.table[(long long)b * a.wide + have + n - first[b]] = blk;
  }
  for (int n = gtid; n < drop; n += gsize) {
    const int b = last_le(freed, a.B, n);
    const int need = (a.target[b] + a.bs - 1) / a.bs;
    const int blk = a.table[(long long)b * a.wide + need + n - freed[b]];
    in_cache(blk);
    a.ring[ring_at(tail_m, n)] = blk;
  }
}

// ------------------------------------------------------------------ append
constexpr int APPEND_SIDE = 128;          // threads for K, and as many for V
constexpr int APPEND_THREADS = 2 * APPEND_SIDE;

struct AppendArgs {
  const uint16_t* x[2];                  // K, V: [tokens][heads][D], unit stride in D
  long long tok_stride[2], head_stride[2];
  int8_t* codes[2];
  float* scales[2];
  const int32_t *table, *cached, *cu_new, *cu_blocks;
  long long block_stride;                // codes between blocks
  long long tokens;
  int B, wide, bs, num_blocks, heads, D, max_units;
  Ctl ctl;
};

// Largest i in [0, n) with a[i] <= x, a whole warp looking at 32 places at a
// time; a place in [0, n) whatever a holds.
__device__ __forceinline__ int warp_last_le(const int32_t* a, int n, int x) {
  const int lane = threadIdx.x % 32;
  int lo = 0;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int at = lane * step;
    const unsigned le = __ballot_sync(~0u, at < n && a[lo + at] <= x);
    const int k = 31 - __clz(le | 1);    // a[lo] <= x, if a is what it should be
    lo += k * step;
    n = min(step, n - k * step);
  }
  return lo;
}

// Four codes of x * inv.  Adding 1.5 * 2^23 rounds to the nearest integer,
// ties to even, and leaves it in the low byte: two instructions an element
// where a conversion would go through the 16-a-clock pipe.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float inv) {
  const float M = 12582912.f;
  const uint32_t x = __byte_perm(__float_as_uint(__fadd_rn(__fmul_rn(a, inv), M)),
                                 __float_as_uint(__fadd_rn(__fmul_rn(b, inv), M)), 0x0040);
  const uint32_t y = __byte_perm(__float_as_uint(__fadd_rn(__fmul_rn(c, inv), M)),
                                 __float_as_uint(__fadd_rn(__fmul_rn(d, inv), M)), 0x0040);
  return __byte_perm(x, y, 0x5410);
}
__device__ __forceinline__ uint32_t codes4_any(float a, float b, float c, float d, float inv) {
  return (uint32_t)(uint8_t)kv_code(a * inv) | (uint32_t)(uint8_t)kv_code(b * inv) << 8 |
         (uint32_t)(uint8_t)kv_code(c * inv) << 16 | (uint32_t)(uint8_t)kv_code(d * inv) << 24;
}

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t u) {
  return BF16 ? unpack_bf162(u) : unpack_half2(u);
}

// One CTA per (written block, head): half the threads for K, half for V.  The
// new rows are read once, all loads of a thread at once, and stay in registers
// (NV 16-byte pieces a thread) while the largest magnitude is found; then the
// scale, the codes.  Bound by memory: 2 bytes in and 1 out per element.
template <bool BF16, int NV>
__global__ void __launch_bounds__(APPEND_THREADS) kv_append_kernel(AppendArgs a) {
  __shared__ uint32_t red[APPEND_THREADS / 32];
  constexpr uint32_t INF = BF16 ? 0x7f80u : 0x7c00u;
  pdl_wait();
  pdl_trigger();
  // heads fastest: neighbouring CTAs then read neighbouring pieces of the same rows
  const int unit = blockIdx.x / a.heads, h = blockIdx.x - unit * a.heads;
  const int side = threadIdx.x / APPEND_SIDE, th = threadIdx.x % APPEND_SIDE;
  const int units = a.cu_blocks[a.B];
  if (units > a.max_units && blockIdx.x == 0 && threadIdx.x == 0) report_status(a.ctl, ST_BAD_LENGTH);   // some have no CTA
  if (unit >= units) return;
  const int b = warp_last_le(a.cu_blocks, a.B, unit);
  const int c = a.cached[b], n0 = a.cu_new[b], n1 = a.cu_new[b + 1];
  // the block's place in the request's row of the table; outside it where a
  // length is negative or too large or the running sums are out of order
  const int j = (int)((unsigned)(c / a.bs) + (unsigned)unit - (unsigned)a.cu_blocks[b]);
  const bool in_row = (unsigned)j < (unsigned)a.wide;
  const int blk = in_row ? a.table[(long long)b * a.wide + j] : -1;
  const int start = in_row ? j * a.bs : 0;
  const int lo = max(c, start), hi = (int)min((long long)c + n1 - n0, (long long)start + a.bs);  // new tokens of the block
  const bool lengths = in_row && c >= 0 && n0 >= 0 && n1 <= a.tokens && hi > lo;
  // 8 or 16 16-byte pieces to a row; a thread's pieces are 16 or 8 rows apart
  const int row_log2 = a.D == 64 ? 3 : 4, pieces = lengths ? (hi - lo) << row_log2 : 0;
  const long long stride = side ? a.tok_stride[1] : a.tok_stride[0];
  const uint16_t* x = (side ? a.x[1] + h * a.head_stride[1] : a.x[0] + h * a.head_stride[0]) +
                      ((long long)(n0 + lo - c) + (th >> row_log2)) * stride + (th & ((1 << row_log2) - 1)) * 8;
  const long long step = stride * (APPEND_SIDE >> row_log2);
  uint4 v[NV];
  uint32_t m = 0;                        // magnitudes of two elements, as integers
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = th + i * APPEND_SIDE;
    v[i] = make_uint4(0, 0, 0, 0);
    if (p < pieces) v[i] = __ldg(reinterpret_cast<const uint4*>(x + i * step));
  }
  if (!lengths || blk < 0 || blk >= a.num_blocks) {
    if (threadIdx.x == 0) report_status(a.ctl, lengths ? ST_BAD_BLOCK : ST_BAD_LENGTH);
    return;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) m = __vmaxu2(m, w[e] & 0x7fff7fffu);
  }
  const int older = lo - start;                                        // earlier tokens of the block
  int8_t* codes = (side ? a.codes[1] : a.codes[0]) + blk * a.block_stride + (long long)h * a.bs * a.D;
  float* scale = (side ? a.scales[1] : a.scales[0]) + (long long)blk * a.heads + h;
  const float before = older > 0 ? *scale : 0.f;
  m = __reduce_max_sync(~0u, max(m & 0xffffu, m >> 16));
  if (th % 32 == 0) red[threadIdx.x / 32] = m;
  __syncthreads();
  const uint32_t* r4 = red + side * (APPEND_SIDE / 32);
  m = max(max(r4[0], r4[1]), max(r4[2], r4[3]));
  const bool odd = m >= INF;             // an infinity or NaN among them
  if (odd) {
    // the largest finite magnitude instead (both halves of the CTA pass this barrier or neither)
    m = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t l = w[e] & 0x7fffu, u = (w[e] >> 16) & 0x7fffu;
        m = max(m, max(l < INF ? l : 0u, u < INF ? u : 0u));
      }
    }
    m = __reduce_max_sync(~0u, m);
  }
  if (__syncthreads_or(odd)) {
    if (odd && th % 32 == 0) red[threadIdx.x / 32] = m;
    __syncthreads();
    if (odd) m = max(max(r4[0], r4[1]), max(r4[2], r4[3]));
  }
  const float s = fmaxf(fmaxf(before, __fdiv_rn(half_bits_to_f32<BF16>((uint16_t)m), 127.f)), KV_SCALE_MIN);
  const float inv = __frcp_rn(s);
  if (th == 0) *scale = s;               // (everyone read the old one before the barriers)
  if (older > 0 && s != before) {
    const float f = before * inv;
    uint4* old = reinterpret_cast<uint4*>(codes);
    for (int i = th; i < older * a.D / 16; i += APPEND_SIDE) {
      uint4 q = old[i];
      uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = codes4_any((float)(int8_t)w[e], (float)(int8_t)(w[e] >> 8), (float)(int8_t)(w[e] >> 16),
                          (float)(int8_t)(w[e] >> 24), f);
      old[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  uint2* out = reinterpret_cast<uint2*>(codes + older * a.D);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = th + i * APPEND_SIDE;
    if (p >= pieces) continue;
    const float2 p0 = unpack2<BF16>(v[i].x), p1 = unpack2<BF16>(v[i].y), p2 = unpack2<BF16>(v[i].z),
                 p3 = unpack2<BF16>(v[i].w);
    out[p] = odd ? make_uint2(codes4_any(p0.x, p0.y, p1.x, p1.y, inv), codes4_any(p2.x, p2.y, p3.x, p3.y, inv))
                 : make_uint2(codes4(p0.x, p0.y, p1.x, p1.y, inv), codes4(p2.x, p2.y, p3.x, p3.y, inv));
  }
}

// ------------------------------------------------------------------ gather
constexpr int GATHER_THREADS = 256;

struct GatherArgs {
  const int8_t* codes[2];
  const float* scales[2];
  const int32_t* slots;
  uint16_t* out;                         // [n][2][heads][D], rows of out_stride
  long long out_stride, block_stride, n;
  int bs, bs_log2, num_blocks, heads, D;
  Ctl ctl;
};

// 16 codes per thread and step; the grid sweeps the rows' pieces in order.  A
// slot of -1 gives a row of zeros.  Bound by memory latency at full occupancy:
// 5.3 TB/s read and written at 43,968 rows of 2 x 16 x 64 (8 codes a thread:
// 61 us against 51; several rows a thread in flight, which costs occupancy: 62).
template <bool BF16>
__global__ void __launch_bounds__(GATHER_THREADS, 8) kv_gather_kernel(GatherArgs a) {
  pdl_wait();
  pdl_trigger();
  const int head_log2 = a.D == 64 ? 2 : 3, per_side = a.heads << head_log2, per_row = 2 * per_side;
  const int t = blockIdx.x * GATHER_THREADS + threadIdx.x, threads = gridDim.x * GATHER_THREADS;
  const int d_row = threads / per_row, d_rem = threads - d_row * per_row;   // a step of the sweep
  int rem = t % per_row;
  for (long long row = t / per_row; row < a.n;) {
    const int side = rem >= per_side, hp = rem - side * per_side, h = hp >> head_log2;
    const int slot = a.slots[row], blk = slot >> a.bs_log2;
    uint4 c = make_uint4(0, 0, 0, 0);
    float s = 0.f;
    if (slot >= 0 && blk < a.num_blocks) {
      c = __ldg(reinterpret_cast<const uint4*>((side ? a.codes[1] : a.codes[0]) + blk * a.block_stride +
                                               ((long long)h * a.bs + (slot & (a.bs - 1))) * a.D +
                                               (hp - (h << head_log2)) * 16));
      s = (side ? a.scales[1] : a.scales[0])[(long long)blk * a.heads + h];
    } else if (slot >= 0 && rem == 0) {
      report_bad_block(a.ctl);
    }
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    uint32_t o[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      // the code as a float: its byte, sign bit flipped, under the exponent of 2^23
      const uint32_t f = w[k / 2] ^ 0x80808080u;
      const float x0 = __uint_as_float(__byte_perm(f, 0x4b000000u, k & 1 ? 0x7442 : 0x7440)) - 8388736.f;
      const float x1 = __uint_as_float(__byte_perm(f, 0x4b000000u, k & 1 ? 0x7443 : 0x7441)) - 8388736.f;
      o[k] = BF16 ? pack_bf162(x0 * s, x1 * s) : pack_half2(x0 * s, x1 * s);
    }
    uint4* dst = reinterpret_cast<uint4*>(a.out + row * a.out_stride + rem * 16);
    dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
    dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
    row += d_row;
    rem += d_rem;
    if (rem >= per_row) {
      rem -= per_row;
      ++row;
    }
  }
}

}  // namespace

int check_cache(const char* name, const qvggt_kv_cache& c) {
  if (c.num_blocks <= 0 || c.kv_heads <= 0 || c.kv_heads > 65535)
    return set_error(QVGGT_ERR_INVALID, "%s: bad cache shape", name);
  if (c.block_size != 32 && c.block_size != 64 && c.block_size != 128)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: block_size must be 32, 64 or 128", name);
  if (c.head_dim != 64 && c.head_dim != 128)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128", name);
  if (!c.k_cache || !c.v_cache || !c.k_scale || !c.v_scale)
    return set_error(QVGGT_ERR_INVALID, "%s: null cache tensor", name);
  if (!aligned16(c.k_cache) || !aligned16(c.v_cache) || c.block_stride % 16)
    return set_error(QVGGT_ERR_ALIGN, "%s: cache codes and their block stride must be 16-byte aligned", name);
  if (c.block_stride < c.kv_heads * c.block_size * c.head_dim)
    return set_error(QVGGT_ERR_INVALID, "%s: block stride smaller than a block", name);
  if (c.num_blocks > 2147483647LL / c.block_size)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: more than 2^31 slots", name);
  return QVGGT_OK;
}

}  // namespace qv

using namespace qv;

extern "C" int qvggt_block_plan(const qvggt_block_plan_args* p, void* stream) {
  if (!p || p->requests < 0 || p->max_blocks < 0 || p->num_blocks <= 0 || p->max_new < 0)
    return set_error(QVGGT_ERR_INVALID, "block_plan: bad shape");
  if (p->requests > PLAN_MAX_REQUESTS)
    return set_error(QVGGT_ERR_UNSUPPORTED, "block_plan: at most %d requests", PLAN_MAX_REQUESTS);
  if (p->block_size <= 0 || (p->block_size & (p->block_size - 1)))
    return set_error(QVGGT_ERR_INVALID, "block_plan: block_size must be a power of two");
  if (p->num_blocks > 2147483647LL / p->block_size || p->max_blocks > 2147483647LL / p->block_size ||
      p->max_new > 2147483647LL)
    return set_error(QVGGT_ERR_UNSUPPORTED, "block_plan: more than 2^31 slots");
  if (!p->free_ring || !p->free_range || !p->cu_new || !p->cu_blocks || !p->free_range_out || !p->status ||
      (p->max_new && !p->slots) || (p->requests && (!p->cached_lens || !p->target_lens || !p->lens_out)) ||
      (p->requests && p->max_blocks && !p->block_tables))
    return set_error(QVGGT_ERR_INVALID, "block_plan: null tensor");
  if ((p->requests && (p->lens_out == p->cached_lens || p->lens_out == p->target_lens)) ||
      p->free_range_out == p->free_range)
    return set_error(QVGGT_ERR_INVALID, "block_plan: the outputs must not be the inputs");
  PlanArgs a{p->cached_lens, p->target_lens, p->block_tables, p->free_ring,
             reinterpret_cast<const long long*>(p->free_range), p->slots, p->cu_new, p->cu_blocks, p->lens_out,
             p->status, reinterpret_cast<long long*>(p->free_range_out), (int)p->requests, (int)p->max_blocks,
             (int)p->block_size, (int)p->num_blocks, (int)p->max_new, make_ctl()};
  const int smem = 4 * (a.B + 1) * (int)sizeof(int);
  static DeviceFlags attr;
  if (int rc = ensure_smem(attr, block_plan_kernel, 4 * (PLAN_MAX_REQUESTS + 1) * (int)sizeof(int),
                           "cudaFuncSetAttribute(block_plan)"))
    return rc;
  const int sms = device_info().num_sms;
  const int grid = (int)std::min<int64_t>(sms, std::max<int64_t>(1, (p->max_new + PLAN_THREADS - 1) / PLAN_THREADS));
  int rc = check_cuda(launch_pdl(block_plan_kernel, dim3(grid), dim3(PLAN_THREADS), (size_t)smem,
                                 static_cast<cudaStream_t>(stream), 1u, a),
                      "block_plan launch");
  if (!rc) count_launch(1);
  return rc;
}

extern "C" int qvggt_kv_append(const qvggt_kv_append_args* p, void* stream) {
  if (!p) return set_error(QVGGT_ERR_INVALID, "kv_append: null arguments");
  if (int rc = check_cache("kv_append", p->cache)) return rc;
  if (p->dtype != QVGGT_DTYPE_F16 && p->dtype != QVGGT_DTYPE_BF16)
    return set_error(QVGGT_ERR_UNSUPPORTED, "kv_append: dtype must be fp16 or bf16");
  if (p->tokens < 0 || p->requests < 0 || p->max_blocks < 0 || p->max_units < 0 || p->requests > 2147483646LL ||
      p->max_blocks > 2147483647LL / p->cache.block_size || p->max_units > 2147483647LL / p->cache.kv_heads)
    return set_error(QVGGT_ERR_INVALID, "kv_append: bad shape");
  if (p->tokens == 0 || p->requests == 0 || p->max_units == 0) return QVGGT_OK;
  if (!p->k || !p->v || !p->block_tables || !p->cached_lens || !p->cu_new || !p->cu_blocks)
    return set_error(QVGGT_ERR_INVALID, "kv_append: null tensor");
  if (!aligned16(p->k) || !aligned16(p->v) || p->k_tok % 8 || p->k_head % 8 || p->v_tok % 8 || p->v_head % 8)
    return set_error(QVGGT_ERR_ALIGN, "kv_append: k and v rows must be 16-byte aligned");
  AppendArgs a{};
  a.x[0] = static_cast<const uint16_t*>(p->k);
  a.x[1] = static_cast<const uint16_t*>(p->v);
  a.tok_stride[0] = p->k_tok;
  a.tok_stride[1] = p->v_tok;
  a.head_stride[0] = p->k_head;
  a.head_stride[1] = p->v_head;
  a.codes[0] = p->cache.k_cache;
  a.codes[1] = p->cache.v_cache;
  a.scales[0] = p->cache.k_scale;
  a.scales[1] = p->cache.v_scale;
  a.table = p->block_tables;
  a.cached = p->cached_lens;
  a.cu_new = p->cu_new;
  a.cu_blocks = p->cu_blocks;
  a.block_stride = p->cache.block_stride;
  a.tokens = p->tokens;
  a.B = (int)p->requests;
  a.wide = (int)p->max_blocks;
  a.bs = (int)p->cache.block_size;
  a.num_blocks = (int)p->cache.num_blocks;
  a.heads = (int)p->cache.kv_heads;
  a.D = (int)p->cache.head_dim;
  a.max_units = (int)p->max_units;
  a.ctl = make_ctl();
  using Kfn = void (*)(AppendArgs);
  static const Kfn fns[2][4] = {
      {kv_append_kernel<false, 2>, kv_append_kernel<false, 4>, kv_append_kernel<false, 8>, kv_append_kernel<false, 16>},
      {kv_append_kernel<true, 2>, kv_append_kernel<true, 4>, kv_append_kernel<true, 8>, kv_append_kernel<true, 16>}};
  const int nv = a.bs * a.D / 8 / APPEND_SIDE;             // 2, 4, 8 or 16 pieces a thread
  int rc = check_cuda(launch_pdl(fns[p->dtype == QVGGT_DTYPE_BF16][nv == 2 ? 0 : nv == 4 ? 1 : nv == 8 ? 2 : 3],
                                 dim3((unsigned)(p->max_units * a.heads)), dim3(APPEND_THREADS), 0,
                                 static_cast<cudaStream_t>(stream), 1u, a),
                      "kv_append launch");
  if (!rc) count_launch(1);
  return rc;
}

extern "C" int qvggt_kv_gather(const qvggt_kv_gather_args* p, void* stream) {
  if (!p) return set_error(QVGGT_ERR_INVALID, "kv_gather: null arguments");
  if (int rc = check_cache("kv_gather", p->cache)) return rc;
  if (p->dtype != QVGGT_DTYPE_F16 && p->dtype != QVGGT_DTYPE_BF16)
    return set_error(QVGGT_ERR_UNSUPPORTED, "kv_gather: dtype must be fp16 or bf16");
  if (p->n < 0) return set_error(QVGGT_ERR_INVALID, "kv_gather: bad shape");
  if (p->n == 0) return QVGGT_OK;
  if (!p->slots || !p->out) return set_error(QVGGT_ERR_INVALID, "kv_gather: null tensor");
  const qvggt_kv_cache& c = p->cache;
  if (!aligned16(p->out) || p->out_stride % 8 || p->out_stride < 2 * c.kv_heads * c.head_dim)
    return set_error(QVGGT_ERR_ALIGN, "kv_gather: out rows must be 16-byte aligned and hold K and V");
  GatherArgs a{{c.k_cache, c.v_cache}, {c.k_scale, c.v_scale}, p->slots, static_cast<uint16_t*>(p->out),
               p->out_stride, c.block_stride, p->n, (int)c.block_size,
               c.block_size == 32 ? 5 : c.block_size == 64 ? 6 : 7, (int)c.num_blocks, (int)c.kv_heads,
               (int)c.head_dim, make_ctl()};
  // up to 16 CTAs per SM (8 at a time)
  const long long want = (p->n * 2 * a.heads * (a.D / 16) + GATHER_THREADS - 1) / GATHER_THREADS;
  const long long grid = std::min<long long>(want, 16LL * device_info().num_sms);
  const auto fn = p->dtype == QVGGT_DTYPE_BF16 ? kv_gather_kernel<true> : kv_gather_kernel<false>;
  int rc = check_cuda(launch_pdl(fn, dim3((unsigned)grid), dim3(GATHER_THREADS), 0,
                                 static_cast<cudaStream_t>(stream), 1u, a),
                      "kv_gather launch");
  if (!rc) count_launch(1);
  return rc;
}
