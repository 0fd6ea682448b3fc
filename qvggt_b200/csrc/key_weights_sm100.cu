// What cached keys have gathered, many query rows: tcgen05 + TMEM.
//
// The mathematics is key_weights.cu's.  The keys are the product's M: S^T = K
// Q^T puts a key on a TMEM lane, so the thread that owns the lane sums over the
// rows in its registers; nothing is exchanged, nothing rounded below fp32.  An
// item is (request, block of 256 keys, kv head); items are dealt to the CTAs in
// turn (one CTA per SM), heads fastest, which mixes the blocks that a causal
// mask leaves many rows with those that it leaves few.  Per tile of 128 rows:
//   warp 0         the items, two ahead; TMA of the Q tile into a ring
//   warps 1, 2     S_i = K_i Q^T, a warp for each 128-key tile i (a wait costs an
//                  issuer 150 to 250 cycles: one warp for both held the rest up)
//   warp 3         -lse log2e of the rows of each Q tile, and how many keys they see
//   warps 4..7     codes of the next item -> fp16 / bf16 operand tiles (two
//                  items' worth), their scales and places; each warp takes 32
//                  keys of each key tile, which are in one block, and has their
//                  loads under way before it waits for room
//   warps 8..23    exponentials and sums: a thread has a key of each key tile;
//                  warpgroup w takes 32 of the tile's 128 rows, whose constants it
//                  reads once for both keys (a shared-memory read of four rows'
//                  costs as much as half a row's exponentials)
// All waits are bounded; on expiry every role leaves and the status word is set.
//
// TMEM columns: S_i of Q tile t at 256 (t % 2) + 128 i.
#include "key_weights.cuh"
#include "attn_cache.cuh"
#include "attn_common.cuh"
#include "host.hpp"

namespace qv {
namespace {

constexpr int THREADS = 768;
constexpr int KEYS = 256;       // keys of an item
constexpr int ITEMS = 4;        // items handed out ahead
// Sums being put together: a warp opens item x + 4 only when all have opened x
// (the items' ring), so it writes its sums of x + 5 after all others' of x are read.
constexpr int PARTS = ITEMS + 1;
constexpr int ITEM_READERS = 3 + 4 + 16;   // issuers and rows, keys, sums
constexpr uint32_t TMEM_COLS = 512;

// What a CTA does with one item: Q tiles [t0, t1) of request b.
struct __align__(16) Item {
  int b, kvh, key0, n;
  int q0, ql, t0, t1;
  int nkt;                               // key tiles; -1: no more items
  int fresh, pad[2];
};

template <int D>
struct Lay {
  static constexpr int PANELS = D / 64;
  static constexpr int PANEL = 128 * 128;                  // bytes: 128 rows x 64 dims
  static constexpr int QS = D == 64 ? 4 : 2;               // stages of Q tiles
  static constexpr int Q = 0;                              // [stage][panel]
  static constexpr int K = Q + QS * PANELS * PANEL;        // [item % 2][key tile][panel]
  static constexpr int KEY = K + 2 * 2 * PANELS * PANEL;   // [item % 2][256]: factor of the exponent, place
  static constexpr int ROW = KEY + 2 * KEYS * 8;           // [stage][128]: -lse log2e
  static constexpr int LIM = ROW + QS * 128 * 4;           // [stage][128]: keys the row sees
  static constexpr int SEEN = LIM + QS * 128 * 4;          // [stage][warpgroup]: the fewest and the most keys its rows see
  static constexpr int PART = SEEN + QS * 32;              // [item % PARTS][warpgroup][256]: sums of its rows
  static constexpr int BAR = PART + PARTS * 4 * KEYS * 4;
  // q_full[QS], q_empty[QS], k_full[2], k_empty[2], item_full[ITEMS], item_empty[ITEMS],
  // s_full[2], s_free[2], part_full[PARTS], drain[2]
  static constexpr int NUM_BARS = 2 * QS + 4 + 2 * ITEMS + 6 + PARTS;
  static constexpr int MISC = BAR + (NUM_BARS + 1) / 2 * 16;
  static constexpr int ITEM = MISC + 16;
  static constexpr int CUM = ITEM + ITEMS * (int)sizeof(Item);   // long long [THREADS + 1]
  static constexpr int TOTAL = CUM + (THREADS + 2) * 8 + 1024;
};

// The items of a request: blocks of 256 keys.
struct Request {
  using Args = KeyWeightArgs;
  long long cost;
  __device__ __forceinline__ Request(const KeyWeightArgs& a, int b, int) {
    const int q0 = a.cu_q[b], ql = a.cu_q[b + 1] - q0, n = a.kv_lens[b];
    cost = 0;
    if (q0 < 0 || ql < 0 || ql > a.max_q || (long long)q0 + ql > a.Tq || n < 0 || n > (a.wide << a.bs_log2)) {
      report_status(a.ctl, ST_BAD_LENGTH);
      return;
    }
    cost = ((long long)n + KEYS - 1) / KEYS;
  }
};

__device__ __forceinline__ uint64_t exp2_of(uint64_t x2) {
  float x0, x1;
  f2_unpack(x2, x0, x1);
  return f2_pack(ex2(x0), ex2(x1));
}

template <bool BF16, int D>
__global__ void __launch_bounds__(THREADS, 1)
    key_weights_tiles_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ KeyWeightArgs a) {
  using L = Lay<D>;
  constexpr int QS = L::QS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + L::BAR);
  uint64_t* q_empty = q_full + QS;
  uint64_t* k_full = q_empty + QS;
  uint64_t* k_empty = k_full + 2;
  uint64_t* item_full = k_empty + 2;
  uint64_t* item_empty = item_full + ITEMS;
  uint64_t* s_full = item_empty + ITEMS;       // [Q tile % 2]
  uint64_t* s_free = s_full + 2;
  uint64_t* part_full = s_free + 2;
  uint64_t* drain = part_full + PARTS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC);
  volatile Item* items = reinterpret_cast<volatile Item*>(smem + L::ITEM);
  float* key_ck = reinterpret_cast<float*>(smem + L::KEY);         // [item % 2][256]
  int* key_at = reinterpret_cast<int*>(key_ck + 2 * KEYS);         // block * block_size + offset, -1: none
  float* row_nl = reinterpret_cast<float*>(smem + L::ROW);
  int* row_lim = reinterpret_cast<int*>(smem + L::LIM);
  int2* row_seen = reinterpret_cast<int2*>(smem + L::SEEN);
  float* part = reinterpret_cast<float*>(smem + L::PART);
  long long* cum = reinterpret_cast<long long*>(smem + L::CUM);
  const uint32_t tries = a.wait_tries;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    for (int s = 0; s < QS; ++s) {
      mbar_init(&q_full[s], 2);                // the tile and its rows' constants
      mbar_init(&q_empty[s], 2 + 16);           // the products, and the warps that read the rows' constants
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], 4);
      mbar_init(&k_empty[s], 2 + 16);
      mbar_init(&s_full[s], 4);
      mbar_init(&s_free[s], 16);
    }
    for (int s = 0; s < ITEMS; ++s) {
      mbar_init(&item_full[s], 1);
      mbar_init(&item_empty[s], ITEM_READERS);
    }
    for (int s = 0; s < PARTS; ++s) mbar_init(&part_full[s], 16);
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) tma_prefetch_desc(&tmQ);
  pdl_wait();
  const int g = (a.B + THREADS - 1) / THREADS;
  tc_fence_before();
  scan_blocks<THREADS, Request>(a, cum, a.B, g);
  tc_fence_after();
  pdl_trigger();                                           // (this CTA has its TMEM by now)
  const uint32_t tmem = *tmem_slot;
  const int tpt = 128 / a.group;                           // tokens of a Q tile

  if (warp < 4) {
    if (warp == 0) {
      // ------------------------------------------------- items and Q tiles
      const long long total = cum[THREADS] * a.hk;
      int b = 0;                               // the request that holds an item's block, and the blocks before it
      long long s = 0;
      int have = -1, rq0 = 0, rql = 0, rn = 0;
      auto publish = [&](int it) {             // one lane; false if there was no room in time
        const int st = it % ITEMS;
        const long long x = blockIdx.x + (long long)it * gridDim.x;
        if (!wait(&item_empty[st], ((it / ITEMS) & 1) ^ 1, tries)) return false;
        items[st].nkt = -1;
        if (x < total) {
          const long long blk = x / a.hk;
          // skip whole groups of requests, then requests
          while (b / g + 1 < THREADS && cum[b / g + 1] <= blk) {
            b = (b / g + 1) * g;
            s = cum[b / g];
          }
          for (;; ++b) {
            const long long c = b == have ? ((long long)rn + KEYS - 1) / KEYS : Request(a, b, 0).cost;
            if (blk < s + c) break;
            s += c;
          }
          if (b != have) {
            have = b;
            rq0 = a.cu_q[b];
            rql = a.cu_q[b + 1] - rq0;
            rn = a.kv_lens[b];
          }
          const int key0 = (int)(blk - s) * KEYS;
          // the first row that sees key0
          long long first = 0;
          if (a.chunk) first = (long long)(key0 / a.chunk) * a.chunk - ((long long)rn - rql);
          const int t1 = (int)(((long long)rql + tpt - 1) / tpt);
          items[st].b = b;
          items[st].kvh = (int)(x % a.hk);
          items[st].key0 = key0;
          items[st].n = rn;
          items[st].q0 = rq0;
          items[st].ql = rql;
          items[st].t0 = first <= 0 ? 0 : first >= rql ? t1 : (int)first / tpt;
          items[st].t1 = t1;
          items[st].fresh = a.fresh ? a.fresh[b] : rn;
          items[st].nkt = rn - key0 > 128 ? 2 : 1;
        }
        mbar_arrive(&item_full[st]);
        return true;
      };
      // Two items ahead of the one whose tiles are loaded, so that its keys are
      // ready in time; a reader gives an item's slot back when it starts on it.
      bool ok = true;
      int tg = 0;                              // Q tiles so far
      int it = 0;
      if (lane == 0) ok = publish(0) && (blockIdx.x >= total || publish(1));
      ok = __shfl_sync(~0u, ok, 0);
      for (; ok && blockIdx.x + (long long)it * gridDim.x < total; ++it) {
        const int is = it % ITEMS;
        __syncwarp();
        const int t0 = items[is].t0, t1 = items[is].t1, kvh = items[is].kvh, q0 = items[is].q0;
        __syncwarp();
        // the slot after the last item's holds the end mark
        if (lane == 0 && blockIdx.x + (long long)(it + 1) * gridDim.x < total) ok = publish(it + 2);
        ok = __shfl_sync(~0u, ok, 0);
        for (int t = t0; ok && t < t1; ++t) {
          const int st = tg % QS;
          ok = warp_wait(&q_empty[st], ((tg / QS) & 1) ^ 1, tries);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&q_full[st], L::PANELS * tpt * a.group * 128);
            for (int p = 0; p < L::PANELS; ++p)
              tma_load_3d(smem + L::Q + (st * L::PANELS + p) * L::PANEL, &tmQ, &q_full[st], p * 64, kvh * a.group,
                          q0 + t * tpt);
          }
          ++tg;
        }
      }
      // gave up: the copies in flight have to land before the CTA exits, but their
      // barriers wait for the rows' constants too; 2 ms are far more than a copy takes
      if (!ok && lane == 0) {
        report_status(a.ctl, ST_TIMEOUT_TMA_EMPTY);
        for (int x = max(0, tg - QS); x < tg; ++x) mbar_wait_drain(&q_full[x % QS], (x / QS) & 1, 2000000ull);
      }
    } else if (warp < 3) {
      // ---------------------------------------------------------- S = K Q^T
      constexpr uint32_t idesc = idesc_f16(128, 128, false, false, BF16);
      const int i = warp - 1;
      uint32_t used = 0;                       // products so far
      int tg = 0;
      bool ok = true;
      for (int it = 0; ok; ++it) {
        const int is = it % ITEMS, kb = it & 1;
        if (!warp_wait(&item_full[is], (it / ITEMS) & 1, tries)) { ok = false; break; }
        const int nkt = items[is].nkt, t0 = items[is].t0, t1 = items[is].t1;
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[is]);
        if (nkt < 0) break;
        if (!warp_wait(&k_full[kb], (it / 2) & 1, tries)) { ok = false; break; }
        for (int t = t0; t < t1; ++t, ++tg) {
          const int st = tg % QS;
          if (!warp_wait(&q_full[st], (tg / QS) & 1, tries)) { ok = false; break; }
          const int x = used & 1;
          const uint32_t u = used++ >> 1;      // uses of these score tiles before
          if (u > 0 && !warp_wait(&s_free[x], (u - 1) & 1, tries)) { ok = false; break; }
          tc_fence_after();
          if (elect_one()) {
            if (i < nkt) {
#pragma unroll
              for (int p = 0; p < L::PANELS; ++p)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  mma_f16_ss(tmem + 256 * x + 128 * i,
                             sdesc_sw128(sbase + L::K + ((kb * 2 + i) * L::PANELS + p) * L::PANEL + k * 32),
                             sdesc_sw128(sbase + L::Q + (st * L::PANELS + p) * L::PANEL + k * 32), idesc,
                             (p | k) ? 1u : 0u);
            }
            tc_commit(&s_full[x]);
            mbar_arrive(&s_full[x]);           // hands on the rows' and keys' constants
            tc_commit(&q_empty[st]);
          }
          __syncwarp();
        }
        if (ok && elect_one()) tc_commit(&k_empty[kb]);
        __syncwarp();
      }
      if (!ok && elect_one()) {
        report_status(a.ctl, ST_TIMEOUT_FULL);
        tc_commit(&drain[i]);
        mbar_wait_drain(&drain[i], 0, 200000000ull);
      }
      __syncwarp();
    } else {
      // ---------------------------------------------------------- constants of rows
      const int most = tpt * a.group;          // rows of a tile
      // this lane's rows lane + 32 x: token of the tile, head of the group
      int tok[4], head[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        tok[x] = (lane + 32 * x) / a.group;
        head[x] = (lane + 32 * x) % a.group;
      }
      int tg = 0;
      bool ok = true;
      for (int it = 0; ok; ++it) {
        const int is = it % ITEMS;
        if (!warp_wait(&item_full[is], (it / ITEMS) & 1, tries)) break;
        const int nkt = items[is].nkt, t0 = items[is].t0, t1 = items[is].t1, kvh = items[is].kvh, q0 = items[is].q0;
        const int n = items[is].n, ql = items[is].ql;
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[is]);
        if (nkt < 0) break;
        float l[4];                            // rows lane + 32 x of the next tile
        auto fetch = [&](int t) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int i = t * tpt + tok[x];
            l[x] = lane + 32 * x < most && i < ql && t < t1 ? a.lse[(long long)(kvh * a.group + head[x]) * a.Tq + q0 + i] : INFINITY;
          }
        };
        fetch(t0);
        for (int t = t0; t < t1; ++t, ++tg) {
          const int st = tg % QS;
          float nl[4];
          int lim[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            nl[x] = -l[x] * LOG2E;
            // key_limit without its division
            int seen = n;
            if (a.chunk) {
              const int pos = n - ql + t * tpt + tok[x];
              const unsigned c = a.chunk == 1 ? (unsigned)pos : __umulhi((unsigned)pos, a.chunk_mul) >> a.chunk_shift;
              seen = pos < 0 ? 0 : (int)min((long long)n, (long long)(c + 1) * a.chunk);
            }
            lim[x] = isfinite(l[x]) ? seen : 0;
          }
          fetch(t + 1);
          if (!warp_wait(&q_empty[st], ((tg / QS) & 1) ^ 1, tries)) { ok = false; break; }
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            row_nl[st * 128 + lane + 32 * x] = nl[x];
            row_lim[st * 128 + lane + 32 * x] = lim[x];
            // (rows that no token has score 0 and weigh 0: they are no reason to look at each)
            const int fewest = __reduce_min_sync(~0u, lane + 32 * x < most ? lim[x] : n), largest = __reduce_max_sync(~0u, lim[x]);
            if (lane == 0) row_seen[st * 4 + x] = make_int2(fewest, largest);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&q_full[st]);
        }
      }
    }
  } else if (warp < 8) {
    // ------------------------------------------------------------ keys of an item
    const int bs = 1 << a.bs_log2;
    // rows that no token of a tile has (the group does not divide 128) score 0
    if (tpt * a.group < 128)
      for (int p = threadIdx.x - 128; p < QS * L::PANELS * L::PANEL / 16; p += 128)
        if (p / 8 % 128 >= tpt * a.group)
          asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(sbase + L::Q + p * 16), "r"(0) : "memory");
    constexpr int LOADS = 4;                   // 16-byte pieces a lane has under way: 32 keys with head_dim 64, 16 with 128
    constexpr int STEPS = D / 64;              // of a key tile
    bool bad = false;
    // An item, and the blocks and scales of this warp's keys in its key tiles.
    struct Keys {
      int nkt, kvh, key0, n, id[2];
      float ks[2];
    };
    auto open = [&](int it, Keys& x) {
      const int is = it % ITEMS;
      if (!warp_wait(&item_full[is], (it / ITEMS) & 1, tries)) return false;
      x.nkt = items[is].nkt;
      x.kvh = items[is].kvh;
      x.key0 = items[is].key0 + 32 * (warp - 4);
      x.n = items[is].n;
      const int b = items[is].b;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[is]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int k = x.key0 + 128 * i;        // this warp's first key
        x.id[i] = -1;
        x.ks[i] = 0.f;
        if (i < x.nkt && k < x.n) {
          x.id[i] = a.table[(long long)b * a.wide + (k >> a.bs_log2)];
          if (x.id[i] >= 0 && x.id[i] < a.num_blocks) {
            x.ks[i] = a.ks[(long long)x.id[i] * a.hk + x.kvh];
          } else {
            x.id[i] = -1;
            bad = true;
          }
        }
      }
      return true;
    };
    auto load = [&](const Keys& x, int u, uint4 (&w)[LOADS]) {
      const int i = u / STEPS, part = u % STEPS, blk = i ? x.id[1] : x.id[0];
      const int8_t* kp = a.kc + blk * a.block_stride + ((long long)x.kvh * bs + ((x.key0 + 128 * i) & (bs - 1))) * D;
#pragma unroll
      for (int y = 0; y < LOADS; ++y) {
        w[y] = make_uint4(0, 0, 0, 0);
        if (blk >= 0) w[y] = __ldg(reinterpret_cast<const uint4*>(kp) + (part * LOADS + y) * 32 + lane);
      }
    };
    Keys cur, next;
    uint4 w[LOADS], ahead[LOADS];
    bool ok = open(0, cur);
    if (ok && cur.nkt > 0) load(cur, 0, w);
    for (int it = 0; ok && cur.nkt > 0; ++it) {
      const int kb = it & 1;
      ok = open(it + 1, next);
      for (int u = 0; ok && u < cur.nkt * STEPS; ++u) {
        // the next step's codes are on their way while these are unpacked
        if (u + 1 < cur.nkt * STEPS) load(cur, u + 1, ahead);
        else if (next.nkt > 0) load(next, 0, ahead);
        if (u == 0 && it >= 2 && !warp_wait(&k_empty[kb], ((it - 2) / 2) & 1, tries)) { ok = false; break; }
        const int i = u / STEPS, part = u % STEPS;
        if (part == 0) {
          const int blk = i ? cur.id[1] : cur.id[0];
          const int key = cur.key0 + 128 * i + lane, at = kb * KEYS + 128 * i + 32 * (warp - 4) + lane;
          key_ck[at] = (i ? cur.ks[1] : cur.ks[0]) * a.scale_log2;
          key_at[at] = blk < 0 || key >= cur.n ? -1 : (blk << a.bs_log2) + (key & (bs - 1));
        }
#pragma unroll
        for (int x = 0; x < LOADS; ++x) {
          const int p = (part * LOADS + x) * 32 + lane;    // piece p % (D / 16) of row p / (D / 16)
          const int piece = p % (D / 16), r = 32 * (warp - 4) + p / (D / 16), panel = piece / 4;
          const uint32_t c[4] = {w[x].x, w[x].y, w[x].z, w[x].w};
          uint32_t y[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[2 * e] = codes2<BF16, false>(c[e]);
            y[2 * e + 1] = codes2<BF16, true>(c[e]);
          }
          // 16-byte chunks 2 piece and 2 piece + 1 of the row, at chunk ^ (row & 7)
          const uint32_t line = sbase + L::K + ((kb * 2 + i) * L::PANELS + panel) * L::PANEL + r * 128;
          const uint32_t c0 = ((2 * (piece & 3)) ^ (r & 7)) * 16, c1 = c0 ^ 16;
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(line + c0), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]) : "memory");
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(line + c1), "r"(y[4]), "r"(y[5]), "r"(y[6]), "r"(y[7]) : "memory");
        }
#pragma unroll
        for (int x = 0; x < LOADS; ++x) w[x] = ahead[x];
      }
      if (!ok) break;
      fence_proxy_async_smem();                // these stores before the products' reads
      __syncwarp();
      if (lane == 0) mbar_arrive(&k_full[kb]);
      cur = next;
    }
    if (bad && lane == 0) report_bad_block(a.ctl);
  } else {
    // ------------------------------------------------------------ exponentials and sums
    const int wg = (warp - 8) / 4, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t tS = tmem + ((uint32_t)(quarter * 32) << 16) + 32 * wg;
    uint32_t tg = 0;                           // Q tiles so far
    bool ok = true;
    for (int it = 0; ok; ++it) {
      const int is = it % ITEMS, kb = it & 1, pb = it % PARTS;
      if (!warp_wait(&item_full[is], (it / ITEMS) & 1, tries)) { ok = false; break; }
      const int nkt = items[is].nkt, nt = items[is].t1 - items[is].t0, kvh = items[is].kvh, key0 = items[is].key0;
      const int fresh = items[is].fresh;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[is]);
      if (nkt < 0) break;
      if (!warp_wait(&k_full[kb], (it / 2) & 1, tries)) { ok = false; break; }
      // this thread's keys, and the one whose sums it puts together (two warpgroups do)
      const float ck0 = key_ck[kb * KEYS + r], ck1 = nkt > 1 ? key_ck[kb * KEYS + 128 + r] : 0.f;
      const int at = wg < nkt ? key_at[kb * KEYS + 128 * wg + r] : -1;
      __syncwarp();
      if (lane == 0) mbar_arrive(&k_empty[kb]);            // (the products arrive too)
      const long long place = (((long long)(at >> a.bs_log2) * a.hk + kvh) << a.bs_log2) + (at & ((1 << a.bs_log2) - 1));
      float old = 0.f;
      if (at >= 0 && key0 + 128 * wg + r < fresh) old = a.w[place];
      uint64_t s0 = f2_pack(0.f, 0.f), s1 = s0;
      bool ready = false;
      for (int t = 0; t < nt; ++t, ++tg) {
        const int st = tg % QS, x = tg & 1;
        if (!__all_sync(~0u, ready) && !warp_wait(&s_full[x], (tg >> 1) & 1, tries)) { ok = false; break; }
        tc_fence_after();
        // whether every row sees every key of the item, and whether one sees any
        const int2 seen = row_seen[st * 4 + wg];
        const bool all = seen.x >= key0 + 128 * nkt, none = seen.y <= key0;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t v0[16], v1[16];
          tmem_ld16(tS + 256 * x + 16 * half, v0);
          if (nkt > 1) tmem_ld16(tS + 256 * x + 16 * half + 128, v1);
          const float4* nl = reinterpret_cast<const float4*>(row_nl + st * 128 + 32 * wg + 16 * half);
          const int4* lim = reinterpret_cast<const int4*>(row_lim + st * 128 + 32 * wg + 16 * half);
          tmem_ld_wait();
          reg_fence<0, 16>(v0);
          reg_fence<0, 16>(v1);
          if (half) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_free[x]);
            // asked ahead: an answer takes a while
            ready = t + 1 < nt && test(smem_u32(&s_full[x ^ 1]), ((tg + 1) >> 1) & 1);
          }
          if (none) continue;
          if (all) {
            const uint64_t c0 = f2_pack(ck0, ck0), c1 = f2_pack(ck1, ck1);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float4 z = nl[e];
              const uint64_t za = f2_pack(z.x, z.y), zb = f2_pack(z.z, z.w);
              s0 = f2_add(s0, exp2_of(f2_fma(f2_pack(__uint_as_float(v0[4 * e]), __uint_as_float(v0[4 * e + 1])), c0, za)));
              s0 = f2_add(s0, exp2_of(f2_fma(f2_pack(__uint_as_float(v0[4 * e + 2]), __uint_as_float(v0[4 * e + 3])), c0, zb)));
              if (nkt > 1) {
                s1 = f2_add(s1, exp2_of(f2_fma(f2_pack(__uint_as_float(v1[4 * e]), __uint_as_float(v1[4 * e + 1])), c1, za)));
                s1 = f2_add(s1, exp2_of(f2_fma(f2_pack(__uint_as_float(v1[4 * e + 2]), __uint_as_float(v1[4 * e + 3])), c1, zb)));
              }
            }
          } else {
            float t0 = 0.f, t1 = 0.f;
            const int k0 = key0 + r, k1 = nkt > 1 ? k0 + 128 : 0x7fffffff;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float z = reinterpret_cast<const float*>(nl)[e];
              const int m = reinterpret_cast<const int*>(lim)[e];
              const float p0 = ex2(fmaf(__uint_as_float(v0[e]), ck0, z)), p1 = ex2(fmaf(__uint_as_float(v1[e]), ck1, z));
              t0 += k0 < m ? p0 : 0.f;
              t1 += k1 < m ? p1 : 0.f;
            }
            s0 = f2_add(s0, f2_pack(t0, 0.f));
            s1 = f2_add(s1, f2_pack(t1, 0.f));
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_empty[st]);
      }
      if (!ok) break;
      // the warpgroups' sums join in their order
      float lo, hi;
      f2_unpack(s0, lo, hi);
      part[(pb * 4 + wg) * KEYS + r] = lo + hi;
      f2_unpack(s1, lo, hi);
      part[(pb * 4 + wg) * KEYS + 128 + r] = lo + hi;
      __syncwarp();
      if (lane == 0) mbar_arrive(&part_full[pb]);
      if (wg < 2) {
        if (!warp_wait(&part_full[pb], (it / PARTS) & 1, tries)) { ok = false; break; }
        const float* p = part + pb * 4 * KEYS + 128 * wg + r;
        if (at >= 0) a.out[place] = fmaf(old, a.decay, (p[0] + p[KEYS]) + (p[2 * KEYS] + p[3 * KEYS]));
      }
    }
    if (!ok && lane == 0) report_status(a.ctl, ST_TIMEOUT_SOFTMAX);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

}  // namespace

bool key_weight_tiles_can_read(const KeyWeightArgs& a) {
  return a.group <= 128 && (a.hq == 1 || a.q_head > 0) && (a.Tq == 1 || a.q_tok > 0);
}

int launch_key_weight_tiles(KeyWeightArgs& a, int D, bool bf16, cudaStream_t stream) {
  const int smem = D == 64 ? Lay<64>::TOTAL : Lay<128>::TOTAL;
  if (smem > device_info().max_smem_optin)
    return set_error(QVGGT_ERR_UNSUPPORTED, "key_weights: shared memory %d > %d", smem, device_info().max_smem_optin);
  CUtensorMap tmQ;
  const uint64_t dims[3] = {(uint64_t)D, (uint64_t)a.hq, (uint64_t)a.Tq};
  const uint64_t strides[2] = {(uint64_t)(a.hq == 1 ? D : a.q_head) * 2,
                               (uint64_t)(a.Tq == 1 ? a.hq * D : a.q_tok) * 2};
  const uint32_t box[3] = {64, (uint32_t)a.group, (uint32_t)(128 / a.group)};
  if (int rc = encode_tmap(&tmQ, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, a.q,
                           dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  a.row_blocks = 1;
  // a try_wait that fails takes about 1.4 us
  a.wait_tries = (uint32_t)std::min<unsigned long long>(1u << 26, a.ctl.timeout_ns / 1024 + 1);
  // p / chunk = (p mul) >> (31 + s) for p < 2^31: mul = 2^(31 + s) / chunk, rounded
  // up, with 2^s >= chunk (a chunk of 1 needs none of it)
  int s = 1;
  while (1LL << s < a.chunk) ++s;
  a.chunk_shift = s - 1;
  a.chunk_mul = a.chunk > 1 ? (uint32_t)((1ull << (31 + s)) / (unsigned)a.chunk + 1) : 0;
  const long long most = (long long)a.B * (((long long)a.wide << a.bs_log2) + KEYS - 1) / KEYS * a.hk;
  const int grid = (int)std::min<long long>(std::max<long long>(1, most), device_info().num_sms);
  using Kfn = void (*)(CUtensorMap, KeyWeightArgs);
  static const Kfn fns[2][2] = {{key_weights_tiles_kernel<false, 64>, key_weights_tiles_kernel<false, 128>},
                                {key_weights_tiles_kernel<true, 64>, key_weights_tiles_kernel<true, 128>}};
  static DeviceFlags attr[2][2];
  const Kfn fn = fns[bf16][D == 128];
  if (int rc = ensure_smem(attr[bf16][D == 128], fn, smem, "cudaFuncSetAttribute(key_weights)")) return rc;
  int rc = check_cuda(launch_pdl(fn, dim3((unsigned)grid), dim3(THREADS), smem, stream, 1u, tmQ, a), "key_weights launch");
  if (!rc) count_launch(1);
  return rc;
}

}  // namespace qv
