// Attention over a paged K/V cache in 8 bits, few query rows
// (the mathematics is in attn_cache.cuh).
#include <new>

#include "attn_cache.cuh"
#include "attn_common.cuh"
#include "host.hpp"

namespace qv {
namespace {

constexpr int UNIT = 32;                 // keys a warp takes at a time: never across two blocks

// NT: 8-row tiles of an item, a row being a (token, query head of the group) pair.
template <int D, int NT>
struct RowLay {
  static constexpr int ROWS = 8 * NT;
  static constexpr int WARPS = D == 128 ? 6 : NT < 4 ? 8 : 4;
  static constexpr int THREADS = WARPS * 32;
  static constexpr int STAGES = 96 * 1024 / (WARPS * 2 * UNIT * D);   // units in flight per warp: 3, 6 or 2
  static constexpr int SIDE = UNIT * D;                    // K or V codes of a unit
  static constexpr int RING = 0;                           // [warp][stage][K, V]
  static constexpr int RING_BYTES = WARPS * STAGES * 2 * SIDE;
  static constexpr int BAR = RING + RING_BYTES;            // [warp][stage]
  static constexpr int CUM = BAR + WARPS * STAGES * 8;     // long long [THREADS + 1]
  static constexpr int SEG = CUM + (THREADS + 2) * 8;      // Segment [2]
  static constexpr int ML = SEG + 2 * (int)sizeof(Segment);   // float [warp][row] maxima, then sums
  static constexpr int WALK = ML + 2 * WARPS * ROWS * 4;   // PieceWalk, one thread's
  static constexpr int Q = WALK + 256;                     // q's fragments, where they do not fit registers
  static constexpr bool Q_SHARED = D == 128 && NT == 2;
  static constexpr int TOTAL = Q + (Q_SHARED ? NT * (D / 16) * 32 * 8 : 0);
  // the warps' O, merged at the end of a segment, lie in the drained ring
  static_assert(WARPS * ROWS * D * 4 <= RING_BYTES, "O does not fit the ring");
};

// The rows of an item, their keys in units.
template <int D, int NT>
struct RowBlock {
  // A segment's start and merge cost about as much as two units on each warp;
  // a piece is not cut below four units for each (a join costs about that).
  static constexpr int START = 2 * RowLay<D, NT>::WARPS, MIN = START + 4 * RowLay<D, NT>::WARPS;
  int q0, ql, n, tok0, nqt, tiles;       // tok0: first row (token * group + head)
  long long cost;
  __device__ __forceinline__ int tile_cost() const { return 1; }
  __device__ __forceinline__ RowBlock() {}
  __device__ __forceinline__ RowBlock(const CacheAttnArgs& a, int b, int qb) {
    q0 = a.cu_q[b];
    ql = a.cu_q[b + 1] - q0;
    n = a.kv_lens[b];
    tok0 = qb * RowLay<D, NT>::ROWS;
    nqt = 1;
    tiles = 0;
    cost = 0;
    // (a negative number of queries is for lengths_ok to report)
    if ((ql >= 0 && tok0 >= (long long)ql * a.group) || !lengths_ok(a, q0, ql, n)) return;
    const int last = (min(ql * a.group, tok0 + RowLay<D, NT>::ROWS) - 1) / a.group;
    tiles = (key_limit(last, ql, n, a.chunk) + UNIT - 1) / UNIT;
    cost = START + (long long)tiles;
  }
};

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
__device__ __forceinline__ uint2 lds64(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
  return v;
}

// 8 x 8 transpose of 16-bit elements across the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// A CTA walks its piece of the items' line (attn_cache.cuh); the
// units of a segment go round its warps.  Each warp streams its own units
// through a ring of bulk copies that only it fills and reads, so nothing but
// its own mbarriers holds it up: up to 192 KB in flight per SM, well over what
// the memory's latency needs.  Two CTAs share an SM, so one streams while the
// other starts or merges.  The warps' softmax states merge at the segment's end.
//
// The codes are the M operand of mma.m16n8k16 and the rows its N: S^T = K q^T,
// O^T += V^T P^T.  The instructions that unpack a code are then paid once for
// all rows (they bound the kernel: with the rows as M, 668 instructions a unit
// against 450 now, 150 us against 113 at 8 x 16 heads x 37,000 keys, 632 MB), and each
// of up to 8 rows costs what one does.
template <bool BF16, int D, int NT>
__global__ void __launch_bounds__(RowLay<D, NT>::THREADS, 2) attn_cache_rows_kernel(CacheAttnArgs a) {
  using L = RowLay<D, NT>;
  constexpr int KC = D / 64;              // 64-dim chunks
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR) + warp * L::STAGES;
  Segment* segs = reinterpret_cast<Segment*>(smem + L::SEG);
  float* sm_m = reinterpret_cast<float*>(smem + L::ML);
  float* sm_l = sm_m + L::WARPS * L::ROWS;
  float* sm_o = reinterpret_cast<float*>(smem + L::RING);
  const uint32_t ring = sbase + L::RING + warp * L::STAGES * 2 * L::SIDE;
  if (lane == 0) {
    for (int s = 0; s < L::STAGES; ++s) mbar_init(&bars[s], 1);
    fence_mbar_init();
  }
  __syncwarp();
  pdl_wait();
  pdl_trigger();
  const int blocks = a.B * a.row_blocks, bg = (blocks + L::THREADS - 1) / L::THREADS;
  long long* cum = reinterpret_cast<long long*>(smem + L::CUM);
  scan_blocks<L::THREADS, RowBlock<D, NT>>(a, cum, blocks, bg);
  // one thread walks (its state in shared memory, not in every thread's
  // registers); it finds the next segment before it starts on this one's units
  using Walk = PieceWalk<L::THREADS, RowBlock<D, NT>>;
  static_assert(sizeof(Walk) <= 256, "no room for the walk");
  Walk* walk = reinterpret_cast<Walk*>(smem + L::WALK);
  auto advance = [&](int slot) {
    Segment sg;
    if (!walk->next(a, blocks, sg)) sg.nt = -1;
    segs[slot] = sg;
  };
  if (threadIdx.x == L::THREADS - 32) {
    new (walk) Walk(a, cum, blocks, bg);
    advance(0);
  }
  __syncthreads();
  const int bs = 1 << a.bs_log2;
  int st = 0;                             // the ring's next stage and its phase
  uint32_t phase = 0;
  bool ok = true;
  for (int seg = 0;; ++seg) {
    const Segment sg = segs[seg & 1];
    if (sg.nt < 0) break;
    if (threadIdx.x == L::THREADS - 32) advance((seg + 1) & 1);
    __syncwarp();
    const int kvh = sg.kvh, ql = sg.ql, n = sg.n, rows = ql * a.group, row0 = sg.tok0;

    // this warp's units: t0 + warp + WARPS i.  Lane x holds the block of unit
    // i = base + x and its scales; the next 32 ids are fetched while these are used
    const int first = sg.t0 + warp, last = sg.t0 + sg.nt;
    const int count = first < last ? (last - first + L::WARPS - 1) / L::WARPS : 0;
    const int32_t* table = a.table + (long long)sg.b * a.wide;
    auto fetch_id = [&](int i) {
      return i < count ? table[((first + i * L::WARPS) * UNIT) >> a.bs_log2] : -1;
    };
    // the constants of the lane's unit: the score's factor, log2 and inverse of the V scale
    float ck, lv, inv_vs;
    auto constants = [&](int id) {
      const bool good = id >= 0 && id < a.num_blocks;
      const float vs = good ? a.vs[(long long)id * a.hk + kvh] : 1.f;
      ck = good ? a.ks[(long long)id * a.hk + kvh] * a.scale_log2 : 1.f;
      if (!BF16) ck = nonzero_factor(ck);   // (bf16: with the row's own factor, below)
      lv = log2f(vs);
      inv_vs = 1.f / vs;
    };
    int id = fetch_id(lane), id2 = fetch_id(32 + lane);
    bool bad = false;
    // starts the copies of unit i into stage x (a block outside the cache: none)
    auto issue = [&](int i, int block, int x) {
      const int key0 = (first + i * L::WARPS) * UNIT;
      if (lane == 0) {
        const bool good = block >= 0 && block < a.num_blocks;
        bad |= !good;
        mbar_arrive_expect_tx(&bars[x], good ? 2 * L::SIDE : 0);
        if (good) {
          const long long off = block * a.block_stride + ((long long)kvh * bs + (key0 & (bs - 1))) * D;
          const uint32_t dst = ring + x * 2 * L::SIDE;
          bulk_load(dst, a.kc + off, L::SIDE, smem_u32(&bars[x]));
          bulk_load(dst + L::SIDE, a.vc + off, L::SIDE, smem_u32(&bars[x]));
        }
      }
    };
    for (int i = 0; i < L::STAGES && i < count; ++i) issue(i, __shfl_sync(~0u, id, i), (st + i) % L::STAGES);
    constants(id);

    // rows 2t and 2t + 1 of each 8-row tile
    int lim[NT][2];
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = row0 + 8 * x + 2 * t + e;
        lim[x][e] = row < rows ? key_limit(row / a.group, ql, n, a.chunk) : 0;
      }
    const int all = key_limit(row0 / a.group, ql, n, a.chunk);   // keys that every row sees
    // B fragments of q (row g of each tile): step s of chunk c takes dims
    // 64c + 16t + 4s + {0, 1} as k rows 2t, 2t+1 and {2, 3} as 2t+8, 2t+9 (any
    // order of the dims will do, as K's fragments use the same).  bf16 queries
    // become fp16 times a power of two per row (its largest element near 2^13;
    // what fp16 then cannot hold exactly is below 2^-37 of that), because codes
    // unpack to fp16 in five instructions a word and to bf16 in eight: 63 us
    // against 56 at 16 ragged requests x 8 heads x 128, 177 MB.
    uint32_t qb[L::Q_SHARED ? 1 : NT][KC][4][2];
    float row_ck[NT][2];                  // what undoes it, of rows 2t and 2t + 1
    if (L::Q_SHARED) __syncthreads();     // the segment before is done with the shared fragments
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const int row = min(row0 + 8 * x + g, rows - 1);
      const uint16_t* qp = a.q + (long long)(sg.q0 + row / a.group) * a.q_tok +
                           (long long)(kvh * a.group + row % a.group) * a.q_head;
      uint2 w[KC][4];
#pragma unroll
      for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int s = 0; s < 4; ++s) w[c][s] = *reinterpret_cast<const uint2*>(qp + 64 * c + 16 * t + 4 * s);
      float back = 1.f;
      if (BF16) {
        float mx = 0.f;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const float2 p = unpack_bf162(w[c][s].x), q = unpack_bf162(w[c][s].y);
            mx = fmaxf(mx, fmaxf(fmaxf(fabsf(p.x), fabsf(p.y)), fmaxf(fabsf(q.x), fabsf(q.y))));
          }
        mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 2));
        // exponents of 2^up and 2^-up; rows of zeros, infinities or NaN (and
        // magnitudes whose factor would leave the normal range) stay within it
        const int up = max(-115, min(110, 13 - ((int)(__float_as_uint(mx) >> 23) - 127)));
        const float f = __int_as_float((127 + up) << 23);
        back = __int_as_float((127 - up) << 23);
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const float2 p = unpack_bf162(w[c][s].x), q = unpack_bf162(w[c][s].y);
            w[c][s] = make_uint2(pack_half2(p.x * f, p.y * f), pack_half2(q.x * f, q.y * f));
          }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) row_ck[x][e] = __shfl_sync(~0u, back, (2 * t + e) * 4);
#pragma unroll
      for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          if constexpr (L::Q_SHARED) {
            if (warp == 0) reinterpret_cast<uint2*>(smem + L::Q)[((x * KC + c) * 4 + s) * 32 + lane] = w[c][s];
          } else {
            qb[x][c][s][0] = w[c][s].x;
            qb[x][c][s][1] = w[c][s].y;
          }
        }
    }
    if (L::Q_SHARED) __syncthreads();
    float o[NT][D / 16][4];               // O^T: tile 4c + 2w + j, slots (dim, dim + 1) x rows (2t, 2t + 1)
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[x][d][e] = 0.f;
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[x][e] = -INFINITY;
        l[x][e] = 0.f;
      }
    // Slot g of 8 keys is key (g >> 1) + 4 (g & 1): the four t lanes, which
    // need slots 2t, 2t + 1 of V, then read rows in both halves of the
    // shared-memory banks.
    const int kappa = (g >> 1) + 4 * (g & 1);

    int i = 0;
    for (; i < count; ++i) {
      if (i && (i & 31) == 0) {
        id = id2;
        id2 = fetch_id(i + 32 + lane);
        constants(id);
      }
      const int blk = __shfl_sync(~0u, id, i & 31);
      const float uck = __shfl_sync(~0u, ck, i & 31), ulv = __shfl_sync(~0u, lv, i & 31);
      const float uinv = __shfl_sync(~0u, inv_vs, i & 31);
      if (!warp_wait(&bars[st], phase, a.wait_tries)) { ok = false; break; }
      const int key0 = (first + i * L::WARPS) * UNIT;
      const uint32_t kb = ring + st * 2 * L::SIDE, vb = kb + L::SIDE;
      if (blk >= 0 && blk < a.num_blocks) {
        float s[NT][2][4];                // S^T: 16 keys x 8 rows; keys kappa, kappa + 8 x rows 2t, 2t + 1
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
          for (int x = 0; x < NT; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[x][mt][e] = 0.f;
#pragma unroll
          for (int c = 0; c < KC; ++c) {
            const uint4 w0 = lds128(kb + (16 * mt + kappa) * D + 64 * c + 16 * t);
            const uint4 w1 = lds128(kb + (16 * mt + 8 + kappa) * D + 64 * c + 16 * t);
            const uint32_t x0[4] = {w0.x, w0.y, w0.z, w0.w}, x1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
            for (int sp = 0; sp < 4; ++sp) {
              const uint32_t ka[4] = {codes2<false, false>(x0[sp]), codes2<false, false>(x1[sp]),
                                      codes2<false, true>(x0[sp]), codes2<false, true>(x1[sp])};
#pragma unroll
              for (int x = 0; x < NT; ++x) {
                if constexpr (L::Q_SHARED) {
                  const uint2 q2 = lds64(sbase + L::Q + (((x * KC + c) * 4 + sp) * 32 + lane) * 8);
                  mma16816(s[x][mt], ka, q2.x, q2.y);
                } else {
                  mma16816(s[x][mt], ka, qb[x][c][sp][0], qb[x][c][sp][1]);
                }
              }
            }
          }
        }
        uint32_t pb[NT][2][2];
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          float cx[2] = {uck, uck}, ix[2] = {uinv, uinv}, lx[2] = {ulv, ulv};
          if (BF16) {                     // (small rows over small keys: 2^-110 times 2^-60 and less)
#pragma unroll
            for (int e = 0; e < 2; ++e) cx[e] = nonzero_factor(uck * row_ck[x][e]);
          }
          if (key0 + UNIT > all) {        // warp-uniform
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (key0 + 16 * mt + kappa + 8 * (e >> 1) >= lim[x][e & 1]) s[x][mt][e] = -INFINITY;
            // a row that sees none of these keys takes nothing from their scale either
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (key0 >= lim[x][e]) {
                cx[e] = 1.f;
                lx[e] = 0.f;
                ix[e] = 0.f;
              }
          }
          float alpha[2], nm[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(fmaxf(s[x][0][e], s[x][0][e + 2]), fmaxf(s[x][1][e], s[x][1][e + 2]));
#pragma unroll
            for (int d = 4; d < 32; d *= 2) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, d));
            const float mn = fmaxf(m[x][e], fmaf(mx, cx[e], lx[e]));
            const float base = mn == -INFINITY ? 0.f : mn;
            alpha[e] = ex2(m[x][e] - base);                // 0 while the row has seen no key
            m[x][e] = mn;
            nm[e] = lx[e] - base;
          }
          if (__any_sync(~0u, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              l[x][e] *= alpha[e];
#pragma unroll
              for (int d = 0; d < D / 16; ++d) {
                o[x][d][e] *= alpha[e];
                o[x][d][e + 2] *= alpha[e];
              }
            }
          }
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[x][mt][e] = ex2(fmaf(s[x][mt][e], cx[e & 1], nm[e & 1]));
            // P^T as the B operand: keys 2t, 2t + 1 (slots) x row g
            pb[x][mt][0] = transpose8(pack_half2(s[x][mt][0], s[x][mt][1]));
            pb[x][mt][1] = transpose8(pack_half2(s[x][mt][2], s[x][mt][3]));
          }
#pragma unroll
          for (int e = 0; e < 2; ++e)
            l[x][e] = fmaf((s[x][0][e] + s[x][0][e + 2]) + (s[x][1][e] + s[x][1][e + 2]), ix[e], l[x][e]);
        }
        // O^T += V^T P^T, 16 keys a step: lane t's rows of V are slots 2t, 2t + 1,
        // 2t + 8, 2t + 9 = keys t + {0, 4, 8, 12}, of which it takes 8 bytes
#pragma unroll
        for (int sp = 0; sp < 2; ++sp)
#pragma unroll
          for (int c = 0; c < KC; ++c) {
            uint2 w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = lds64(vb + (16 * sp + t + 4 * k) * D + 64 * c + 8 * g);
#pragma unroll
            for (int hw = 0; hw < 2; ++hw) {
              const uint32_t x0 = hw ? w[0].y : w[0].x, x1 = hw ? w[1].y : w[1].x;
              const uint32_t y0 = hw ? w[2].y : w[2].x, y1 = hw ? w[3].y : w[3].x;
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const uint32_t xx = __byte_perm(x0, x1, j ? 0x7362 : 0x5140) ^ 0x80808080u;
                const uint32_t yy = __byte_perm(y0, y1, j ? 0x7362 : 0x5140) ^ 0x80808080u;
                const uint32_t va[4] = {codes_f16<false>(xx), codes_f16<true>(xx), codes_f16<false>(yy),
                                        codes_f16<true>(yy)};
#pragma unroll
                for (int x = 0; x < NT; ++x) mma16816(o[x][4 * c + 2 * hw + j], va, pb[x][sp][0], pb[x][sp][1]);
              }
            }
          }
      }
      // refill the stage once every lane has read it (ordinary loads before the
      // copy's writes)
      const int nx = i + L::STAGES;
      const int nblk = __shfl_sync(~0u, (nx ^ i) & 32 ? id2 : id, nx & 31);
      if (nx < count) {
        fence_proxy_async_smem();
        __syncwarp();
        issue(nx, nblk, st);             // (STAGES units on: the same stage)
      }
      if (++st == L::STAGES) {
        st = 0;
        phase ^= 1;
      }
    }
    if (bad) report_bad_block(a.ctl);
    if (!ok) {
      if (lane == 0) {
        report_status(a.ctl, ST_TIMEOUT_FULL);
        for (int x = i; x < min(count, i + L::STAGES); ++x) {
          mbar_wait_drain(&bars[st], phase, 200000000ull);
          if (++st == L::STAGES) {
            st = 0;
            phase ^= 1;
          }
        }
      }
      __syncwarp();
    }
    // every warp is done with its ring before any writes O over it
    if (__syncthreads_or(!ok)) break;
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = 4; d < 32; d *= 2) l[x][e] += __shfl_xor_sync(~0u, l[x][e], d);
        const int r = 8 * x + 2 * t + e;
        if (g == 0) {
          sm_m[warp * L::ROWS + r] = m[x][e];
          sm_l[warp * L::ROWS + r] = l[x][e];
        }
        if (row0 + r < rows) {
          // dims 64c + 8g + 4w + 2j + (0, 1) of the row
          float* dst = sm_o + (warp * L::ROWS + r) * D + 8 * g;
#pragma unroll
          for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int hw = 0; hw < 2; ++hw) {
              const int d = 4 * c + 2 * hw;
              *reinterpret_cast<float4*>(dst + 64 * c + 4 * hw) =
                  make_float4(o[x][d][e], o[x][d][e + 2], o[x][d + 1][e], o[x][d + 1][e + 2]);
            }
        }
      }
    __syncthreads();
    const int live = min(L::ROWS, rows - row0);
    for (int x = threadIdx.x; x < live * (D / 2); x += L::THREADS) {
      const int r = x / (D / 2), d = 2 * (x % (D / 2)), row = row0 + r;
      float mt = -INFINITY;
#pragma unroll
      for (int w = 0; w < L::WARPS; ++w) mt = fmaxf(mt, sm_m[w * L::ROWS + r]);
      const float base = mt == -INFINITY ? 0.f : mt;
      float lt = 0.f, p = 0.f, q = 0.f;
#pragma unroll
      for (int w = 0; w < L::WARPS; ++w) {
        const float f = ex2(sm_m[w * L::ROWS + r] - base);
        const float2 v = *reinterpret_cast<const float2*>(sm_o + (w * L::ROWS + r) * D + d);
        lt += f * sm_l[w * L::ROWS + r];
        p += f * v.x;
        q += f * v.y;
      }
      const float inv = lt == 0.f ? 0.f : 1.f / lt;
      const float lse2 = lt == 0.f ? -INFINITY : base + log2f(lt);
      const long long tok = sg.q0 + row / a.group;
      const int h = kvh * a.group + row % a.group;
      if (sg.slot >= 0) {
        const long long part = (long long)sg.slot * L::ROWS + r;
        *reinterpret_cast<float2*>(a.part_o + part * D + d) = make_float2(p * inv, q * inv);
        if (d == 0) a.part_lse[part] = lse2;
      } else {
        *reinterpret_cast<uint32_t*>(a.out + tok * a.o_tok + h * a.o_head + d) =
            BF16 ? pack_bf162(p * inv, q * inv) : pack_half2(p * inv, q * inv);
        if (d == 0 && a.lse) a.lse[h * a.Tq + tok] = lse2 * 0.6931471805599453f;
      }
    }
    // the merge's reads of the ring before the next segment's copies into it
    fence_proxy_async_smem();
    __syncthreads();
  }
  if (threadIdx.x == L::THREADS - 32 && a.can_split)
    reinterpret_cast<Cut*>(a.part_lse + 2LL * gridDim.x * L::ROWS)[blockIdx.x] = walk->cut;
}

// Adds the parts of the items that a cut went through: CTA x looks at the cut
// before piece x + 1, and the item's first cut does the work.
template <bool BF16, int D, int NT>
__global__ void __launch_bounds__(NT * 2 * D) attn_cache_rows_join_kernel(CacheAttnArgs a, int grid) {
  pdl_wait();
  pdl_trigger();
  const int x = blockIdx.x + 1, r = threadIdx.x / (D / 4);
  const Cut cut = reinterpret_cast<const Cut*>(a.part_lse + 2LL * grid * 8 * NT)[x];
  if (cut.first != x - 1) return;
  const int row = cut.tok0 + r;
  if (row >= cut.ql * a.group) return;
  join_parts<BF16, D>(a, cut, 8 * NT, r, threadIdx.x % (D / 4), cut.q0 + row / a.group,
                      cut.kvh * a.group + row % a.group);
}

// Sizes and launch of the row kernel with NT 8-row tiles.
template <int D, int NT>
struct Rows {
  using L = RowLay<D, NT>;
  using B = RowBlock<D, NT>;
  // Whether items may be cut (a rule on the hint alone: the join is launched
  // by it): above four units for each warp.
  static bool split(long long max_kv) { return max_kv > 4 * UNIT * L::WARPS; }
  static int grid(long long items, long long max_kv) {
    const long long cost = items * (B::START + (max_kv + UNIT - 1) / UNIT);
    const long long pieces = split(max_kv) ? (cost + B::MIN - 1) / B::MIN : items;
    return (int)std::max<long long>(1, std::min<long long>(pieces, 2LL * device_info().num_sms));
  }
  static int64_t scratch(long long items, long long max_kv) {
    const int64_t n = grid(items, max_kv);
    return split(max_kv) && n > 1 ? n * (2 * L::ROWS * (D + 1) * (int64_t)sizeof(float) + (int64_t)sizeof(Cut)) : 0;
  }
  static int launch(CacheAttnArgs& a, bool bf16, long long max_kv, bool may_split, void* scratch, cudaStream_t stream) {
    if (L::TOTAL > device_info().max_smem_optin)
      return set_error(QVGGT_ERR_UNSUPPORTED, "cached_attention: shared memory %d > %d", L::TOTAL,
                       device_info().max_smem_optin);
    const int n = grid((long long)a.B * a.row_blocks * a.hk, max_kv);
    a.can_split = may_split && n > 1 && split(max_kv);
    a.part_o = static_cast<float*>(scratch);
    a.part_lse = a.can_split ? a.part_o + 2LL * n * L::ROWS * D : nullptr;
    static DeviceFlags attr[2];
    const auto fn = bf16 ? attn_cache_rows_kernel<true, D, NT> : attn_cache_rows_kernel<false, D, NT>;
    if (int rc = ensure_smem(attr[bf16], fn, L::TOTAL, "cudaFuncSetAttribute(cached_attention)")) return rc;
    if (int rc = check_cuda(launch_pdl(fn, dim3((unsigned)n), dim3(L::THREADS), L::TOTAL, stream, 1u, a),
                            "cached_attention launch"))
      return rc;
    count_launch(1);
    if (a.can_split) {
      const auto join = bf16 ? attn_cache_rows_join_kernel<true, D, NT> : attn_cache_rows_join_kernel<false, D, NT>;
      if (int rc = check_cuda(launch_pdl(join, dim3((unsigned)(n - 1)), dim3(NT * 2 * D), 0, stream, 1u, a, n),
                              "cached_attention join launch"))
        return rc;
      count_launch(1);
    }
    return QVGGT_OK;
  }
};

// Rows (of a kv head) up to which the row kernel serves a call.  It reads the
// cache once for each 8, 16 or 32 rows at up to memory speed; the tile kernel
// reads it once for up to 256, at a rate that its softmax sets.  Measured on 8
// requests of 37,000 keys, 16 heads x 64: 1 row 113 us, 16 rows 152, 17 to 32
// rows 267 here and 341 there (33 rows or 64).  With head_dim 128 a second pass
// over the keys for rows 17 to 32 takes what the tile kernel does (92 us at 20
// rows of 16 ragged requests, 58 at 16), and its registers do not hold 32 rows.
// Other lengths, on the device, here / there in us: 20 rows of one request, 16
// heads x 64, 300 keys 13.6 / 12.4, 4,000 26.7 / 29.2, 37,000 52 / 55; 40 rows
// 14.9 / 12.5, 31 / 29, 81 / 56; 8 heads x 128 at 16 rows 13.5 / 13.1, 29 / 27,
// 43 / 51, at 20 rows 14.0 / 13.1, 30 / 27, 50 / 51.  Short caches lose 1 us and
// at most 3 by the rule.
constexpr int ROWS_MAX_64 = 32, ROWS_MAX_128 = 16;

// How a call is laid out, by its sizes alone.
struct Plan {
  bool tiles;                            // attn_cache_sm100.cu's kernel
  int nt;                                // 8-row tiles of the row kernel's items
  int row_blocks;                        // blocks of rows of a request
  int64_t scratch;
};

// Calls f with the row kernel's sizes for head_dim and 8-row tiles.
template <class F>
auto with_rows(int head_dim, int nt, F f) {
  if (head_dim == 64) return nt == 1 ? f(Rows<64, 1>()) : nt == 2 ? f(Rows<64, 2>()) : f(Rows<64, 4>());
  return nt == 1 ? f(Rows<128, 1>()) : f(Rows<128, 2>());
}

Plan make_plan(int group, int kv_heads, int requests, int max_q, long long max_kv, int head_dim, bool force_rows) {
  Plan p{};
  const long long rows = (long long)max_q * group, pairs = (long long)kv_heads * requests;
  p.nt = rows <= 8 ? 1 : rows <= 16 || head_dim == 128 ? 2 : 4;
  p.tiles = rows > (head_dim == 64 ? ROWS_MAX_64 : ROWS_MAX_128) && group <= 128 && !force_rows;
  if (p.tiles) {
    const int tokens = 2 * (128 / group);
    p.row_blocks = (int)(((long long)max_q + tokens - 1) / tokens);
    p.scratch = tiles_scratch(p.row_blocks * pairs, max_kv, head_dim);
  } else {
    p.row_blocks = (int)((rows + 8 * p.nt - 1) / (8 * p.nt));
    p.scratch = with_rows(head_dim, p.nt, [&](auto k) { return k.scratch(p.row_blocks * pairs, max_kv); });
  }
  return p;
}

int check_shape(const char* name, int64_t Tq, int64_t q_heads, int64_t kv_heads, int64_t requests, int64_t max_q,
                int64_t max_kv, int64_t head_dim) {
  if (Tq < 0 || requests < 0 || max_q < 0 || max_kv < 0 || q_heads <= 0 || kv_heads <= 0)
    return set_error(QVGGT_ERR_INVALID, "%s: bad shape", name);
  if (q_heads % kv_heads)
    return set_error(QVGGT_ERR_INVALID, "%s: %lld query heads do not share %lld key heads evenly", name,
                     (long long)q_heads, (long long)kv_heads);
  if (head_dim != 64 && head_dim != 128)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128", name);
  if (q_heads > 65535 || Tq > 2147483647LL / q_heads || max_q > 2147483647LL / q_heads || max_kv > 2147483647LL ||
      requests > 1 << 24)
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
  *bytes = make_plan(q_heads / kv_heads, kv_heads, requests, max_q, max_kv, head_dim, false).scratch;
  return QVGGT_OK;
}

extern "C" int qvggt_cached_attention(const qvggt_cached_attention_args* p, void* stream) {
  const char* name = "cached_attention";
  if (!p) return set_error(QVGGT_ERR_INVALID, "%s: null arguments", name);
  const qvggt_kv_cache& c = p->cache;
  if (int rc = check_shape(name, p->Tq, p->q_heads, c.kv_heads, p->requests, p->max_q, p->max_kv, c.head_dim)) return rc;
  if (int rc = check_cache(name, c)) return rc;
  if (p->dtype != QVGGT_DTYPE_F16 && p->dtype != QVGGT_DTYPE_BF16)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: dtype must be fp16 or bf16", name);
  if (p->causal_chunk < 0 || p->max_blocks < 0)
    return set_error(QVGGT_ERR_INVALID, "%s: bad causal_chunk or table", name);
  if (!(p->scale > 1e-30) || p->scale > 1e30) return set_error(QVGGT_ERR_INVALID, "%s: scale must be positive", name);
  if (p->max_blocks > 2147483647LL / c.block_size)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: block tables hold more than 2^31 keys", name);
  if (p->Tq == 0 || p->requests == 0 || p->max_q == 0) return QVGGT_OK;
  if (!p->q || !p->out || !p->cu_q || !p->kv_lens || (!p->block_tables && p->max_blocks))
    return set_error(QVGGT_ERR_INVALID, "%s: null tensor", name);
  if (!aligned16(p->q) || !aligned16(p->out) || p->q_tok % 8 || p->q_head % 8 || p->o_tok % 8 || p->o_head % 8)
    return set_error(QVGGT_ERR_ALIGN, "%s: q and out rows must be 16-byte aligned", name);
  CacheAttnArgs a{};
  a.q = static_cast<const uint16_t*>(p->q);
  a.out = static_cast<uint16_t*>(p->out);
  a.lse = p->lse;
  a.kc = c.k_cache;
  a.vc = c.v_cache;
  a.ks = c.k_scale;
  a.vs = c.v_scale;
  a.table = p->block_tables;
  a.cu_q = p->cu_q;
  a.kv_lens = p->kv_lens;
  a.q_tok = p->q_tok;
  a.q_head = p->q_head;
  a.o_tok = p->o_tok;
  a.o_head = p->o_head;
  a.block_stride = c.block_stride;
  a.Tq = p->Tq;
  a.B = (int)p->requests;
  a.hq = (int)p->q_heads;
  a.hk = (int)c.kv_heads;
  a.group = a.hq / a.hk;
  a.wide = (int)p->max_blocks;
  a.num_blocks = (int)c.num_blocks;
  a.bs_log2 = c.block_size == 32 ? 5 : c.block_size == 64 ? 6 : 7;
  a.chunk = (int)std::min<int64_t>(p->causal_chunk, 1 << 30);
  a.max_q = (int)p->max_q;
  a.scale_log2 = (float)(p->scale * 1.4426950408889634);
  a.ctl = make_ctl();
  const int head_dim = (int)c.head_dim;
  // strides no TMA map takes (a broadcast or reversed query): the row kernel,
  // items whole where the scratch is laid out for the tile kernel
  const bool strided = !tiles_can_read(a);
  Plan plan = make_plan(a.group, a.hk, a.B, a.max_q, p->max_kv, head_dim, false);
  const bool fits = !(strided && plan.tiles);
  if (!fits) {
    plan = make_plan(a.group, a.hk, a.B, a.max_q, p->max_kv, head_dim, true);
    plan.scratch = 0;
  }
  if (plan.scratch && (!p->scratch || p->scratch_bytes < plan.scratch || !aligned16(p->scratch)))
    return set_error(QVGGT_ERR_INVALID, "%s: needs %lld bytes of 16-byte aligned scratch, got %lld", name,
                     (long long)plan.scratch, (long long)p->scratch_bytes);
  if ((long long)a.B * plan.row_blocks > 1 << 30)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: too many rows", name);
  a.row_blocks = plan.row_blocks;
  // a try_wait that fails takes about 1.4 us
  a.wait_tries = (uint32_t)std::min<unsigned long long>(1u << 26, a.ctl.timeout_ns / 1024 + 1);
  const bool bf16 = p->dtype == QVGGT_DTYPE_BF16;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (plan.tiles) return launch_tiles(a, head_dim, bf16, p->max_kv, p->scratch, st);
  return with_rows(head_dim, plan.nt, [&](auto k) { return k.launch(a, bf16, p->max_kv, fits, p->scratch, st); });
}
