// Attention over a paged K/V cache in 8 bits, few query rows
// (the mathematics is in attn_cache.cuh).
#include <new>

#include "attn_cache.cuh"
#include "attn_common.cuh"
#include "host.hpp"

namespace qv {
namespace {

constexpr int TOK_ROWS = 16;             // (query, head) rows of an item: the M of mma.m16n8k16
constexpr int UNIT = 32;                 // keys a warp takes at a time: never across two blocks

template <int D>
struct RowLay {
  static constexpr int WARPS = D == 64 ? 16 : 8;
  static constexpr int THREADS = WARPS * 32;
  static constexpr int STAGES = 3;                         // units in flight per warp
  static constexpr int SIDE = UNIT * D;                    // K or V codes of a unit
  static constexpr int RING = 0;                           // [warp][stage][K, V]
  static constexpr int RING_BYTES = WARPS * STAGES * 2 * SIDE;
  static constexpr int BAR = RING + RING_BYTES;            // [warp][stage]
  static constexpr int CUM = BAR + WARPS * STAGES * 8;     // long long [THREADS + 1]
  static constexpr int SEG = CUM + (THREADS + 2) * 8;      // Segment [2]
  static constexpr int ML = SEG + 2 * (int)sizeof(Segment);   // float [warp][row] maxima, then sums
  static constexpr int WALK = ML + 2 * WARPS * TOK_ROWS * 4;   // PieceWalk, one thread's
  static constexpr int TOTAL = WALK + 256;
  // the warps' O, merged at the end of a segment, lie in the drained ring
  static_assert(WARPS * TOK_ROWS * D * 4 <= RING_BYTES, "O does not fit the ring");
};

// 16 rows of a request, their keys in units.
template <int D>
struct RowBlock {
  // A segment's start and merge cost about as much as two units on each warp;
  // a piece is not cut below four units for each (a join costs about that).
  static constexpr int START = 2 * RowLay<D>::WARPS, MIN = START + 4 * RowLay<D>::WARPS;
  int q0, ql, n, tok0, nqt, tiles;       // tok0: first row (token * group + head)
  long long cost;
  __device__ __forceinline__ int tile_cost() const { return 1; }
  __device__ __forceinline__ RowBlock() {}
  __device__ __forceinline__ RowBlock(const CacheAttnArgs& a, int b, int qb) {
    q0 = a.cu_q[b];
    ql = a.cu_q[b + 1] - q0;
    n = a.kv_lens[b];
    tok0 = qb * TOK_ROWS;
    nqt = 1;
    tiles = 0;
    cost = 0;
    if (tok0 >= (long long)ql * a.group || !lengths_ok(a, q0, ql, n)) return;
    const int last = (min(ql * a.group, tok0 + TOK_ROWS) - 1) / a.group;
    tiles = (key_limit(last, ql, n, a.chunk) + UNIT - 1) / UNIT;
    cost = START + (long long)tiles;
  }
};

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

// One CTA per SM walks its piece of the items' line (attn_cache.cuh); the
// units of a segment go round its warps.  Each warp streams its own units
// through a ring of bulk copies that only it fills and reads, so nothing but
// its own mbarriers holds it up: up to 192 KB in flight per SM, well over what
// the memory's latency needs.  The warps' softmax states merge at the segment's end.
template <bool BF16, int D>
__global__ void __launch_bounds__(RowLay<D>::THREADS, 1) attn_cache_rows_kernel(CacheAttnArgs a) {
  using L = RowLay<D>;
  constexpr int KC = D / 64;              // 64-dim chunks
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR) + warp * L::STAGES;
  Segment* segs = reinterpret_cast<Segment*>(smem + L::SEG);
  float* sm_m = reinterpret_cast<float*>(smem + L::ML);
  float* sm_l = sm_m + L::WARPS * TOK_ROWS;
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
  scan_blocks<L::THREADS, RowBlock<D>>(a, cum, blocks, bg);
  // one thread walks (its state in shared memory, not in every thread's
  // registers); it finds the next segment before it starts on this one's units
  using Walk = PieceWalk<L::THREADS, RowBlock<D>>;
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
  uint32_t used = 0;                      // units this warp has taken from its ring
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
    auto fetch_scale = [&](const float* sc, int id) {
      return id >= 0 && id < a.num_blocks ? sc[(long long)id * a.hk + kvh] : 0.f;
    };
    int id = fetch_id(lane), id2 = fetch_id(32 + lane);
    float ks = fetch_scale(a.ks, id), vs = fetch_scale(a.vs, id);
    bool bad = false;
    // starts the copies of unit i (a block outside the cache: none)
    auto issue = [&](int i, int block) {
      const uint32_t u = used + i, st = u % L::STAGES;
      const int key0 = (first + i * L::WARPS) * UNIT;
      if (lane == 0) {
        const bool good = block >= 0 && block < a.num_blocks;
        bad |= !good;
        mbar_arrive_expect_tx(&bars[st], good ? 2 * L::SIDE : 0);
        if (good) {
          const long long off = block * a.block_stride + ((long long)kvh * bs + (key0 & (bs - 1))) * D;
          const uint32_t dst = ring + st * 2 * L::SIDE;
          bulk_load(dst, a.kc + off, L::SIDE, smem_u32(&bars[st]));
          bulk_load(dst + L::SIDE, a.vc + off, L::SIDE, smem_u32(&bars[st]));
        }
      }
    };
    for (int i = 0; i < L::STAGES && i < count; ++i) issue(i, __shfl_sync(~0u, id, i));

    // rows g and g + 8 of the tile
    int lim[2];
    const uint16_t* qp[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = min(row0 + g + 8 * r, rows - 1);
      const int i = row / a.group, h = kvh * a.group + row % a.group;
      lim[r] = row0 + g + 8 * r < rows ? key_limit(i, ql, n, a.chunk) : 0;
      qp[r] = a.q + (long long)(sg.q0 + i) * a.q_tok + (long long)h * a.q_head;
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

    int i = 0;
    for (; i < count; ++i) {
      if (i && (i & 31) == 0) {
        id = id2;
        id2 = fetch_id(i + 32 + lane);
        ks = fetch_scale(a.ks, id);
        vs = fetch_scale(a.vs, id);
      }
      const int blk = __shfl_sync(~0u, id, i & 31);
      const float uks = __shfl_sync(~0u, ks, i & 31), uvs = __shfl_sync(~0u, vs, i & 31);
      const uint32_t u = used + i, st = u % L::STAGES;
      if (!warp_wait(&bars[st], (u / L::STAGES) & 1, a.wait_tries)) { ok = false; break; }
      const int key0 = (first + i * L::WARPS) * UNIT;
      const uint32_t kb = ring + st * 2 * L::SIDE, vb = kb + L::SIDE;
      if (blk >= 0 && blk < a.num_blocks) {
        const float ck = uks * a.scale_log2, lv = log2f(uvs), inv_vs = 1.f / uvs;
        // column c of 8-key tile nt is key 8 nt + (c >> 1) + 4 (c & 1): with
        // this order the four t lanes' V rows below fall into both halves of
        // the shared-memory banks
        float s[4][4];
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
#pragma unroll
          for (int c = 0; c < KC; ++c) {
            const uint4 w = lds128(kb + (nt * 8 + (g >> 1) + 4 * (g & 1)) * D + 64 * c + 16 * t);
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int sp = 0; sp < 4; ++sp)
              mma16816<BF16>(s[nt], qa[c][sp], codes2<BF16, false>(ww[sp]), codes2<BF16, true>(ww[sp]));
          }
        }
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int nt = 0; nt < 4; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + nt * 8 + t + 4 * (e & 1);
            s[nt][e] = key < lim[e >> 1] ? s[nt][e] * ck + lv : -INFINITY;
            mx[e >> 1] = fmaxf(mx[e >> 1], s[nt][e]);
          }
        float base[2], alpha[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          mx[r] = fmaxf(mx[r], __shfl_xor_sync(~0u, mx[r], 1));
          mx[r] = fmaxf(mx[r], __shfl_xor_sync(~0u, mx[r], 2));
          const float mn = fmaxf(m[r], mx[r]);
          base[r] = mn == -INFINITY ? 0.f : mn;
          alpha[r] = ex2(m[r] - base[r]);                  // 0 while the row has seen no key
          m[r] = mn;
        }
        if (__any_sync(~0u, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            l[r] *= alpha[r];
#pragma unroll
            for (int d = 0; d < D / 8; ++d) {
              o[d][2 * r] *= alpha[r];
              o[d][2 * r + 1] *= alpha[r];
            }
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
        // O += P V: 16 keys a step, lane t's four are t + {0, 4, 8, 12}; column n
        // of dim tile d is dim 8n + d of a 64-dim chunk, so lane g's operands are
        // 8 consecutive bytes of a row
#pragma unroll
        for (int sp = 0; sp < 2; ++sp) {
          const uint32_t pa[4] = {pack_half2(s[2 * sp][0], s[2 * sp][1]), pack_half2(s[2 * sp][2], s[2 * sp][3]),
                                  pack_half2(s[2 * sp + 1][0], s[2 * sp + 1][1]),
                                  pack_half2(s[2 * sp + 1][2], s[2 * sp + 1][3])};
#pragma unroll
          for (int c = 0; c < KC; ++c) {
            uint2 w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = lds64(vb + (16 * sp + t + 4 * k) * D + 64 * c + 8 * g);
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
      // refill the stage once every lane has read it (ordinary loads before the
      // copy's writes)
      const int nx = i + L::STAGES;
      const int nblk = __shfl_sync(~0u, (nx ^ i) & 32 ? id2 : id, nx & 31);
      if (nx < count) {
        fence_proxy_async_smem();
        __syncwarp();
        issue(nx, nblk);
      }
    }
    used += count;
    if (bad) report_bad_block(a.ctl);
    if (!ok) {
      if (lane == 0) {
        report_status(a.ctl, ST_TIMEOUT_FULL);
        for (int x = i; x < min(count, i + L::STAGES); ++x)
          mbar_wait_drain(&bars[(used - count + x) % L::STAGES], ((used - count + x) / L::STAGES) & 1, 200000000ull);
      }
      __syncwarp();
    }
    // every warp is done with its ring before any writes O over it
    if (__syncthreads_or(!ok)) break;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(~0u, l[r], 1);
      l[r] += __shfl_xor_sync(~0u, l[r], 2);
      if (t == 0) {
        sm_m[warp * TOK_ROWS + g + 8 * r] = m[r];
        sm_l[warp * TOK_ROWS + g + 8 * r] = l[r];
      }
      if (row0 + g + 8 * r < rows) {
        // dims 64c + 16t + 8e + (0..7) of the row
        float* dst = sm_o + (warp * TOK_ROWS + g + 8 * r) * D;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int d = 0; d < 8; d += 4)
              *reinterpret_cast<float4*>(dst + 64 * c + 16 * t + 8 * e + d) =
                  make_float4(o[8 * c + d][2 * r + e], o[8 * c + d + 1][2 * r + e], o[8 * c + d + 2][2 * r + e],
                              o[8 * c + d + 3][2 * r + e]);
      }
    }
    __syncthreads();
    const int live = min(TOK_ROWS, rows - row0);
    for (int x = threadIdx.x; x < live * (D / 2); x += L::THREADS) {
      const int r = x / (D / 2), d = 2 * (x % (D / 2)), row = row0 + r;
      float mt = -INFINITY;
#pragma unroll
      for (int w = 0; w < L::WARPS; ++w) mt = fmaxf(mt, sm_m[w * TOK_ROWS + r]);
      const float base = mt == -INFINITY ? 0.f : mt;
      float lt = 0.f, p = 0.f, q = 0.f;
#pragma unroll
      for (int w = 0; w < L::WARPS; ++w) {
        const float f = ex2(sm_m[w * TOK_ROWS + r] - base);
        const float2 v = *reinterpret_cast<const float2*>(sm_o + (w * TOK_ROWS + r) * D + d);
        lt += f * sm_l[w * TOK_ROWS + r];
        p += f * v.x;
        q += f * v.y;
      }
      const float inv = lt == 0.f ? 0.f : 1.f / lt;
      const float lse2 = lt == 0.f ? -INFINITY : base + log2f(lt);
      const long long tok = sg.q0 + row / a.group;
      const int h = kvh * a.group + row % a.group;
      if (sg.slot >= 0) {
        const long long part = (long long)sg.slot * TOK_ROWS + r;
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
    reinterpret_cast<Cut*>(a.part_lse + 2LL * gridDim.x * TOK_ROWS)[blockIdx.x] = walk->cut;
}

// Adds the parts of the items that a cut went through: CTA x looks at the cut
// before piece x + 1, and the item's first cut does the work, a warp per row.
template <bool BF16, int D>
__global__ void __launch_bounds__(TOK_ROWS * 32) attn_cache_rows_join_kernel(CacheAttnArgs a, int grid) {
  pdl_wait();
  pdl_trigger();
  const int x = blockIdx.x + 1, lane = threadIdx.x % 32, r = threadIdx.x / 32;
  const Cut cut = reinterpret_cast<const Cut*>(a.part_lse + 2LL * grid * TOK_ROWS)[x];
  if (cut.first != x - 1) return;
  const int row = cut.tok0 + r;
  if (row >= cut.ql * a.group) return;
  join_parts<BF16, D>(a, cut, TOK_ROWS, r, lane, cut.q0 + row / a.group, cut.kvh * a.group + row % a.group);
}

// How a call is laid out, by its sizes alone.
struct Plan {
  bool tiles;                            // attn_cache_sm100.cu's kernel
  int row_blocks;                        // 16-row tiles or Q blocks of a request
  int64_t scratch;
};

// Rows served by the row kernel: it reads the cache at memory speed for each 16
// rows, the tile kernel at about a third of that for any number up to 256.
constexpr int ROWS_MAX = 16;

// Whether the row kernel's items may be cut (a rule on the hint alone: the join
// is launched by it): above four units for each warp.
bool rows_split(long long max_kv, int D) { return max_kv > 4 * UNIT * (D == 64 ? RowLay<64>::WARPS : RowLay<128>::WARPS); }

int rows_grid(long long items, long long max_kv, int D) {
  const long long start = D == 64 ? RowBlock<64>::START : RowBlock<128>::START;
  const long long least = D == 64 ? RowBlock<64>::MIN : RowBlock<128>::MIN;
  const long long cost = items * (start + (max_kv + UNIT - 1) / UNIT);
  const long long pieces = rows_split(max_kv, D) ? (cost + least - 1) / least : items;
  return (int)std::max<long long>(1, std::min<long long>(pieces, device_info().num_sms));
}

int64_t rows_scratch(long long items, long long max_kv, int D) {
  if (!rows_split(max_kv, D)) return 0;
  const int64_t grid = rows_grid(items, max_kv, D);
  return grid > 1 ? grid * (2 * TOK_ROWS * (D + 1) * (int64_t)sizeof(float) + (int64_t)sizeof(Cut)) : 0;
}

int launch_rows(CacheAttnArgs& a, int D, bool bf16, long long max_kv, bool split, void* scratch, cudaStream_t stream) {
  const int smem = D == 64 ? RowLay<64>::TOTAL : RowLay<128>::TOTAL;
  const int threads = D == 64 ? RowLay<64>::THREADS : RowLay<128>::THREADS;
  if (smem > device_info().max_smem_optin)
    return set_error(QVGGT_ERR_UNSUPPORTED, "cached_attention: shared memory %d > %d", smem,
                     device_info().max_smem_optin);
  const long long items = (long long)a.B * a.row_blocks * a.hk;
  const int grid = rows_grid(items, max_kv, D);
  a.can_split = split && grid > 1 && rows_split(max_kv, D);
  a.part_o = static_cast<float*>(scratch);
  a.part_lse = a.can_split ? a.part_o + 2LL * grid * TOK_ROWS * D : nullptr;
  using Kfn = void (*)(CacheAttnArgs);
  static const Kfn fns[2][2] = {{attn_cache_rows_kernel<false, 64>, attn_cache_rows_kernel<false, 128>},
                                {attn_cache_rows_kernel<true, 64>, attn_cache_rows_kernel<true, 128>}};
  using Jfn = void (*)(CacheAttnArgs, int);
  static const Jfn joins[2][2] = {{attn_cache_rows_join_kernel<false, 64>, attn_cache_rows_join_kernel<false, 128>},
                                  {attn_cache_rows_join_kernel<true, 64>, attn_cache_rows_join_kernel<true, 128>}};
  static DeviceFlags attr[2][2];
  if (int rc = ensure_smem(attr[bf16][D == 128], fns[bf16][D == 128], smem, "cudaFuncSetAttribute(cached_attention)"))
    return rc;
  if (int rc = check_cuda(launch_pdl(fns[bf16][D == 128], dim3((unsigned)grid), dim3(threads), smem, stream, 1u, a),
                          "cached_attention launch"))
    return rc;
  count_launch(1);
  if (a.can_split) {
    if (int rc = check_cuda(launch_pdl(joins[bf16][D == 128], dim3((unsigned)(grid - 1)), dim3(TOK_ROWS * 32), 0,
                                       stream, 1u, a, grid),
                            "cached_attention join launch"))
      return rc;
    count_launch(1);
  }
  return QVGGT_OK;
}

Plan make_plan(int group, int kv_heads, int requests, int max_q, long long max_kv, int head_dim) {
  Plan p{};
  const long long rows = (long long)max_q * group;
  p.tiles = rows > ROWS_MAX && group <= 128;
  if (p.tiles) {
    const int tokens = 2 * (128 / group);
    p.row_blocks = (int)(((long long)max_q + tokens - 1) / tokens);
    p.scratch = tiles_scratch((long long)p.row_blocks * kv_heads * requests, max_kv, head_dim);
  } else {
    p.row_blocks = (int)((rows + TOK_ROWS - 1) / TOK_ROWS);
    p.scratch = rows_scratch((long long)p.row_blocks * kv_heads * requests, max_kv, head_dim);
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
  *bytes = make_plan(q_heads / kv_heads, kv_heads, requests, max_q, max_kv, head_dim).scratch;
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
  Plan p = make_plan(a.group, kv_heads, requests, max_q, max_kv, head_dim);
  const bool strided = p.tiles && !tiles_can_read(a);
  if (strided) {
    // strides no TMA map takes (a broadcast or reversed query): the row kernel, items whole
    p.tiles = false;
    p.row_blocks = (int)(((long long)max_q * a.group + TOK_ROWS - 1) / TOK_ROWS);
    p.scratch = 0;
  }
  const int64_t need = p.scratch;
  if (need && (!scratch || scratch_bytes < need || !aligned16(scratch)))
    return set_error(QVGGT_ERR_INVALID, "%s: needs %lld bytes of 16-byte aligned scratch, got %lld", name,
                     (long long)need, (long long)scratch_bytes);
  a.row_blocks = p.row_blocks;
  // a try_wait that fails takes about 1.4 us
  a.wait_tries = (uint32_t)std::min<unsigned long long>(1u << 26, a.ctl.timeout_ns / 1024 + 1);
  const bool bf16 = dtype == QVGGT_DTYPE_BF16;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return p.tiles ? launch_tiles(a, head_dim, bf16, max_kv, scratch, st)
                 : launch_rows(a, head_dim, bf16, max_kv, !strided, scratch, st);
}
