// What cached keys have gathered, many query rows: tcgen05 + TMEM.
//
// The mathematics is key_weights.cu's.  The keys are the product's M: S^T = K
// Q^T puts a key on a TMEM lane, so the thread that owns the lane sums over the
// rows in its registers; nothing is exchanged, nothing rounded below fp32.  An
// item is (request, block of 256 keys, kv head); items are dealt to the CTAs in
// turn (one CTA per SM), heads fastest, which mixes the blocks that a causal
// mask leaves many rows with those that it leaves few.  Per tile of 128 rows:
//   warp 0         TMA of the Q tile into a ring
//   warp 1         S_i = K_i Q^T for the two 128-key tiles i
//   warp 2         the items, a few ahead
//   warps 4..7     codes of the next item -> fp16 / bf16 operand tiles (two
//                  items' worth), their scales and places; -lse log2e of the
//                  rows of each Q tile, and how many keys they see
//   warps 8..23    exponentials and sums: warpgroup 2 + x takes key tile x % 2,
//                  every other Q tile (x / 2), so that TMEM holds a tile of
//                  scores being read and one being made for each key tile
// All waits are bounded; on expiry every role leaves and the status word is set.
//
// TMEM columns: S of key tile i, Q tile t at 128 (i + 2 (t % 2)).
#include "key_weights.cuh"
#include "attn_cache.cuh"
#include "attn_common.cuh"
#include "host.hpp"

namespace qv {
namespace {

constexpr int THREADS = 768;
constexpr int KEYS = 256;       // keys of an item
constexpr int ITEMS = 4;        // items handed out ahead
constexpr int ITEM_READERS = 2 + 4 + 16;
constexpr uint32_t TMEM_COLS = 512;

// What a CTA does with one item: Q tiles [t0, t1) of request b.
struct __align__(16) Item {
  int b, kvh, key0, n;
  int q0, ql, t0, t1;
  int nkt;                               // key tiles; -1: no more items
  int pad[3];
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
  static constexpr int LOW = LIM + QS * 128 * 4;           // [stage][4 warps]: the fewest any row sees
  static constexpr int PART = LOW + QS * 16;               // [key tile][128]: sums of the odd Q tiles
  static constexpr int BAR = PART + 2 * 128 * 4;
  // q_full[QS], q_empty[QS], row_full[QS], k_full[2], k_empty[2], item_full[ITEMS], item_empty[ITEMS],
  // s_full[4], s_free[4], part_full[2], part_free[2], drain
  static constexpr int NUM_BARS = 3 * QS + 4 + 2 * ITEMS + 8 + 4 + 1;
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
  uint64_t* row_full = q_empty + QS;
  uint64_t* k_full = row_full + QS;
  uint64_t* k_empty = k_full + 2;
  uint64_t* item_full = k_empty + 2;
  uint64_t* item_empty = item_full + ITEMS;
  uint64_t* s_full = item_empty + ITEMS;       // [key tile + 2 (Q tile % 2)]
  uint64_t* s_free = s_full + 4;
  uint64_t* part_full = s_free + 4;
  uint64_t* part_free = part_full + 2;
  uint64_t* drain = part_free + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC);
  volatile Item* items = reinterpret_cast<volatile Item*>(smem + L::ITEM);
  float* key_ck = reinterpret_cast<float*>(smem + L::KEY);         // [item % 2][256]
  int* key_at = reinterpret_cast<int*>(key_ck + 2 * KEYS);         // block * block_size + offset, -1: none
  float* row_nl = reinterpret_cast<float*>(smem + L::ROW);
  int* row_lim = reinterpret_cast<int*>(smem + L::LIM);
  int* low = reinterpret_cast<int*>(smem + L::LOW);
  float* part = reinterpret_cast<float*>(smem + L::PART);
  long long* cum = reinterpret_cast<long long*>(smem + L::CUM);
  const uint32_t tries = a.wait_tries;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    for (int s = 0; s < QS; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1 + 8);           // the product and the warps that the tile's parity belongs to
      mbar_init(&row_full[s], 4);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], 4);
      mbar_init(&k_empty[s], 1 + 16);
      mbar_init(&part_full[s], 4);
      mbar_init(&part_free[s], 4);
    }
    for (int s = 0; s < ITEMS; ++s) {
      mbar_init(&item_full[s], 1);
      mbar_init(&item_empty[s], ITEM_READERS);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&s_free[s], 4);
    }
    mbar_init(drain, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) tma_prefetch_desc(&tmQ);
  pdl_wait();
  pdl_trigger();
  const int g = (a.B + THREADS - 1) / THREADS;
  tc_fence_before();
  scan_blocks<THREADS, Request>(a, cum, a.B, g);
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int tpt = 128 / a.group;                           // tokens of a Q tile

  // Registers: launched at 80 each; 256 * 48 + 512 * 96 = 768 * 80.
  // Every warp of a warpgroup runs the same setmaxnreg.
  if (warp < 4) {
    regs_dec<48>();
    if (warp == 2) {
      // ------------------------------------------------------------- items
      if (lane == 0) {
        const long long total = cum[THREADS] * a.hk;
        int b = 0;                             // the request that holds block x / hk, and the blocks before it
        long long s = 0;
        int have = -1, q0 = 0, ql = 0, n = 0;
        for (int it = 0;; ++it) {
          const long long x = blockIdx.x + (long long)it * gridDim.x;
          const bool more = x < total;
          const int st = it % ITEMS;
          if (!wait(&item_empty[st], ((it / ITEMS) & 1) ^ 1, tries)) break;
          if (more) {
            const long long blk = x / a.hk;
            // skip whole groups of requests, then requests
            while (b / g + 1 < THREADS && cum[b / g + 1] <= blk) {
              b = (b / g + 1) * g;
              s = cum[b / g];
            }
            for (;; ++b) {
              const long long c = b == have ? ((long long)n + KEYS - 1) / KEYS : Request(a, b, 0).cost;
              if (blk < s + c) break;
              s += c;
            }
            if (b != have) {
              have = b;
              q0 = a.cu_q[b];
              ql = a.cu_q[b + 1] - q0;
              n = a.kv_lens[b];
            }
            const int key0 = (int)(blk - s) * KEYS;
            // the first row that sees key0
            long long first = 0;
            if (a.chunk) first = (long long)(key0 / a.chunk) * a.chunk - ((long long)n - ql);
            const int t1 = (int)(((long long)ql + tpt - 1) / tpt);
            items[st].b = b;
            items[st].kvh = (int)(x % a.hk);
            items[st].key0 = key0;
            items[st].n = n;
            items[st].q0 = q0;
            items[st].ql = ql;
            items[st].t0 = first <= 0 ? 0 : first >= ql ? t1 : (int)first / tpt;
            items[st].t1 = t1;
            items[st].nkt = n - key0 > 128 ? 2 : 1;
          } else {
            items[st].nkt = -1;
          }
          mbar_arrive(&item_full[st]);
          if (!more) break;
        }
      }
    } else if (warp == 0) {
      // ---------------------------------------------------------- Q tiles
      bool ok = true;
      int tg = 0;                              // Q tiles so far
      for (int it = 0;; ++it) {
        const int is = it % ITEMS;
        ok = warp_wait(&item_full[is], (it / ITEMS) & 1, tries);
        if (!ok) break;
        const int nkt = items[is].nkt, t0 = items[is].t0, t1 = items[is].t1, kvh = items[is].kvh, q0 = items[is].q0;
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[is]);
        if (nkt < 0) break;
        for (int t = t0; t < t1; ++t, ++tg) {
          const int st = tg % QS;
          ok = warp_wait(&q_empty[st], ((tg / QS) & 1) ^ 1, tries);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&q_full[st], L::PANELS * tpt * a.group * 128);
            for (int p = 0; p < L::PANELS; ++p)
              tma_load_3d(smem + L::Q + (st * L::PANELS + p) * L::PANEL, &tmQ, &q_full[st], p * 64, kvh * a.group,
                          q0 + t * tpt);
          }
        }
        if (!ok) break;
      }
      if (!ok && lane == 0) {
        // gave up: let the copies in flight land before the CTA exits
        report_status(a.ctl, ST_TIMEOUT_TMA_EMPTY);
        for (int x = max(0, tg - QS); x < tg; ++x) mbar_wait_drain(&q_full[x % QS], (x / QS) & 1, 200000000ull);
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------- S = K Q^T
      constexpr uint32_t idesc = idesc_f16(128, 128, false, false, BF16);
      uint32_t used[4] = {0, 0, 0, 0};         // products into each score tile so far
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
        for (int t = t0; ok && t < t1; ++t, ++tg) {
          const int st = tg % QS;
          if (!warp_wait(&q_full[st], (tg / QS) & 1, tries)) { ok = false; break; }
          const int odd = (t - t0) & 1;
          for (int i = 0; i < nkt; ++i) {
            const int x = i + 2 * odd;
            const uint32_t u = x == 0 ? used[0] : x == 1 ? used[1] : x == 2 ? used[2] : used[3];
            if (u > 0 && !warp_wait(&s_free[x], (u - 1) & 1, tries)) { ok = false; break; }
            if (x == 0) ++used[0];
            else if (x == 1) ++used[1];
            else if (x == 2) ++used[2];
            else ++used[3];
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int p = 0; p < L::PANELS; ++p)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  mma_f16_ss(tmem + 128 * x,
                             sdesc_sw128(sbase + L::K + ((kb * 2 + i) * L::PANELS + p) * L::PANEL + k * 32),
                             sdesc_sw128(sbase + L::Q + (st * L::PANELS + p) * L::PANEL + k * 32), idesc,
                             (p | k) ? 1u : 0u);
              tc_commit(&s_full[x]);
              if (i == nkt - 1) tc_commit(&q_empty[st]);
            }
            __syncwarp();
          }
        }
        if (ok && elect_one()) tc_commit(&k_empty[kb]);
        __syncwarp();
      }
      if (!ok && elect_one()) {
        report_status(a.ctl, ST_TIMEOUT_FULL);
        tc_commit(drain);
        mbar_wait_drain(drain, 0, 200000000ull);
      }
      __syncwarp();
    }
  } else if (warp < 8) {
    // ------------------------------------------------ keys of an item, constants of rows
    regs_dec<48>();
    const int th = threadIdx.x - 128;          // 0..127
    constexpr int PARTS = D / 16;              // 16-code pieces of a row
    const int bs = 1 << a.bs_log2;
    // rows that no token of a tile has (the group does not divide 128) score 0
    if (tpt * a.group < 128)
      for (int p = th; p < QS * L::PANELS * L::PANEL / 16; p += 128)
        if (p / 8 % 128 >= tpt * a.group)
          asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(sbase + L::Q + p * 16), "r"(0) : "memory");
    int tg = 0;
    bool ok = true, bad = false;
    for (int it = 0; ok; ++it) {
      const int is = it % ITEMS, kb = it & 1;
      if (!warp_wait(&item_full[is], (it / ITEMS) & 1, tries)) { ok = false; break; }
      const int nkt = items[is].nkt, t0 = items[is].t0, t1 = items[is].t1, kvh = items[is].kvh, q0 = items[is].q0;
      const int key0 = items[is].key0, n = items[is].n, ql = items[is].ql, b = items[is].b;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[is]);
      if (nkt < 0) break;
      if (it >= 2 && !warp_wait(&k_empty[kb], ((it - 2) / 2) & 1, tries)) { ok = false; break; }
      const int32_t* table = a.table + (long long)b * a.wide;
      for (int i = 0; i < nkt; ++i) {
        const int key = key0 + 128 * i + th;
        int id = key < n ? table[key >> a.bs_log2] : -1;
        if (key < n && (id < 0 || id >= a.num_blocks)) {
          id = -1;
          bad = true;
        }
        key_ck[kb * KEYS + 128 * i + th] = id < 0 ? 0.f : a.ks[(long long)id * a.hk + kvh] * a.scale_log2;
        key_at[kb * KEYS + 128 * i + th] = id < 0 ? -1 : (id << a.bs_log2) + (key & (bs - 1));
        // pieces of 16 codes: th / PARTS is the first row, 128 / PARTS rows apart
        const int piece = th % PARTS, panel = piece / 4;
#pragma unroll 4
        for (int r = th / PARTS; r < 128; r += 128 / PARTS) {
          const int k = key0 + 128 * i + r;
          uint4 w = make_uint4(0, 0, 0, 0);
          if (k < n) {
            const int blk = table[k >> a.bs_log2];
            if (blk >= 0 && blk < a.num_blocks)
              w = __ldg(reinterpret_cast<const uint4*>(a.kc + blk * a.block_stride + ((long long)kvh * bs + (k & (bs - 1))) * D + piece * 16));
          }
          const uint32_t x[4] = {w.x, w.y, w.z, w.w};
          uint32_t y[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[2 * e] = codes2<BF16, false>(x[e]);
            y[2 * e + 1] = codes2<BF16, true>(x[e]);
          }
          // 16-byte chunks 2 piece and 2 piece + 1 of the row, at chunk ^ (row & 7)
          const uint32_t line = sbase + L::K + ((kb * 2 + i) * L::PANELS + panel) * L::PANEL + r * 128;
          const uint32_t c0 = ((2 * (piece & 3)) ^ (r & 7)) * 16, c1 = c0 ^ 16;
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(line + c0), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]) : "memory");
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(line + c1), "r"(y[4]), "r"(y[5]), "r"(y[6]), "r"(y[7]) : "memory");
        }
      }
      fence_proxy_async_smem();                // these stores before the products' reads
      __syncwarp();
      if (lane == 0) mbar_arrive(&k_full[kb]);
      const int tok = th / a.group, head = kvh * a.group + th % a.group;
      for (int t = t0; t < t1; ++t, ++tg) {
        const int st = tg % QS;
        const int i = t * tpt + tok;           // the row's token
        const bool row = th < tpt * a.group && i < ql;
        const float l = row ? a.lse[(long long)head * a.Tq + q0 + i] : INFINITY;
        const int lim = isfinite(l) ? key_limit(i, ql, n, a.chunk) : 0;
        if (!warp_wait(&q_empty[st], ((tg / QS) & 1) ^ 1, tries)) { ok = false; break; }
        row_nl[st * 128 + th] = -l * LOG2E;
        row_lim[st * 128 + th] = lim;
        const int fewest = __reduce_min_sync(~0u, th < tpt * a.group ? lim : n);
        if (lane == 0) low[st * 4 + warp - 4] = fewest;
        __syncwarp();
        if (lane == 0) mbar_arrive(&row_full[st]);
      }
    }
    if (bad) report_bad_block(a.ctl);
  } else {
    // ------------------------------------------------------------ exponentials and sums
    regs_inc<96>();
    const int wg = (warp - 8) / 4, i = wg & 1, odd = wg >> 1, x = wg;   // score tile i + 2 odd
    const int quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t tS = tmem + ((uint32_t)(quarter * 32) << 16) + 128 * x;
    uint32_t cnt = 0;                          // tiles of this warpgroup so far
    uint32_t parts = 0;                        // items of this key tile so far
    int tg = 0;                                // Q tiles of the CTA so far
    bool ok = true;
    for (int it = 0; ok; ++it) {
      const int is = it % ITEMS, kb = it & 1;
      if (!warp_wait(&item_full[is], (it / ITEMS) & 1, tries)) break;
      const int nkt = items[is].nkt, nt = items[is].t1 - items[is].t0, kvh = items[is].kvh, key0 = items[is].key0;
      const int fresh = nkt < 0 || !a.fresh ? 0x7fffffff : a.fresh[items[is].b];
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[is]);
      if (nkt < 0) break;
      if (!warp_wait(&k_full[kb], (it / 2) & 1, tries)) break;
      const int key = key0 + 128 * i + r;
      const float ck = i < nkt ? key_ck[kb * KEYS + 128 * i + r] : 0.f;
      const int at = i < nkt ? key_at[kb * KEYS + 128 * i + r] : -1;
      const long long place = (((long long)(at >> a.bs_log2) * a.hk + kvh) << a.bs_log2) + (at & ((1 << a.bs_log2) - 1));
      float old = 0.f;
      if (!odd && at >= 0 && key < fresh) old = a.w[place];
      __syncwarp();
      if (lane == 0) mbar_arrive(&k_empty[kb]);            // (its product arrives too)
      const uint64_t ck2 = f2_pack(ck, ck);
      uint64_t sa = f2_pack(0.f, 0.f), sb = sa;
      for (int t = 0; t < nt; ++t, ++tg) {
        const int st = tg % QS;
        if ((t & 1) != odd) continue;
        if (!warp_wait(&row_full[st], (tg / QS) & 1, tries)) { ok = false; break; }
        if (i >= nkt) {                        // no such key tile
          if (lane == 0) mbar_arrive(&q_empty[st]);
          continue;
        }
        if (!warp_wait(&s_full[x], cnt & 1, tries)) { ok = false; break; }
        ++cnt;
        tc_fence_after();
        const int fewest = min(min(low[st * 4], low[st * 4 + 1]), min(low[st * 4 + 2], low[st * 4 + 3]));
        const bool all = fewest > key0 + 128 * i + 127;    // every row sees every key of the tile
        const float4* nl = reinterpret_cast<const float4*>(row_nl + st * 128);
        const int4* lim = reinterpret_cast<const int4*>(row_lim + st * 128);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t s[32];
          tmem_ld32(tS + 32 * c, s);
          tmem_ld_wait();
          reg_fence<0, 32>(s);
          if (c == 3) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_free[x]);
          }
          if (all) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float4 z = nl[8 * c + e];
              const uint64_t xa = f2_fma(f2_pack(__uint_as_float(s[4 * e]), __uint_as_float(s[4 * e + 1])), ck2, f2_pack(z.x, z.y));
              const uint64_t xb = f2_fma(f2_pack(__uint_as_float(s[4 * e + 2]), __uint_as_float(s[4 * e + 3])), ck2, f2_pack(z.z, z.w));
              float p0, p1;
              f2_unpack(xa, p0, p1);
              sa = f2_add(sa, f2_pack(ex2(p0), ex2(p1)));
              f2_unpack(xb, p0, p1);
              sb = f2_add(sb, f2_pack(ex2(p0), ex2(p1)));
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float4 z = nl[8 * c + e];
              const int4 m = lim[8 * c + e];
              const float p0 = ex2(fmaf(__uint_as_float(s[4 * e]), ck, z.x)), p1 = ex2(fmaf(__uint_as_float(s[4 * e + 1]), ck, z.y));
              const float p2 = ex2(fmaf(__uint_as_float(s[4 * e + 2]), ck, z.z)), p3 = ex2(fmaf(__uint_as_float(s[4 * e + 3]), ck, z.w));
              sa = f2_add(sa, f2_pack(key < m.x ? p0 : 0.f, key < m.y ? p1 : 0.f));
              sb = f2_add(sb, f2_pack(key < m.z ? p2 : 0.f, key < m.w ? p3 : 0.f));
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_empty[st]);
      }
      if (!ok) break;
      if (i >= nkt) continue;
      float s0, s1;
      f2_unpack(f2_add(sa, sb), s0, s1);
      const float sum = s0 + s1;
      // the odd Q tiles' sums join the even ones'
      if (odd) {
        if (parts > 0 && !warp_wait(&part_free[i], (parts - 1) & 1, tries)) { ok = false; break; }
        part[i * 128 + r] = sum;
        __syncwarp();
        if (lane == 0) mbar_arrive(&part_full[i]);
      } else {
        if (!warp_wait(&part_full[i], parts & 1, tries)) { ok = false; break; }
        const float other = part[i * 128 + r];
        __syncwarp();
        if (lane == 0) mbar_arrive(&part_free[i]);
        if (at >= 0) a.out[place] = fmaf(old, a.decay, sum + other);
      }
      ++parts;
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
