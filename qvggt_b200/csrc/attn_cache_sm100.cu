// Attention over the paged 8-bit K/V cache, many query rows: tcgen05 + TMEM.
//
// The mathematics is attn_cache.cuh's: the codes are the products' operands
// and both scales live in the softmax, per 32 keys (never across two blocks)
//   x = ck S + lv,  ck = scale log2e ks_B, lv = log2 vs_B,  P = 2^(x - m),
//   O += P c_v,  l += (1 / vs_B) sum P,  out = O / l.
// An item is (request, block of two 128-row Q tiles, kv head); a row is a
// (token, query head of the group) pair, so the heads that share K/V share its
// tiles.  Lengths are ragged and known on the GPU only, and a causal mask gives
// late blocks many times the keys of early ones, so the items' key tiles are
// laid out as one line of cost and cut into equal pieces, one per SM: each CTA
// scans the requests (a few KB), finds its piece and walks it.  Where a cut
// falls inside an item, both sides park normalised rows and their log-sum-exp,
// and the join kernel adds them; at most two parts per CTA, so the scratch does
// not grow with the problem.  Per key tile of KT keys (128 for head_dim 64, 64
// for 128):
//   warp 0         block ids and scales, cp.async.bulk of the raw codes (RAW
//                  stages of 16 KB), constants of the tile into a small ring
//   warps 4..7     codes -> fp16 (bf16 for K with bf16 queries) into the
//                  128-byte-swizzled operand tiles (two stages each of K, V)
//   warp 1         S_i = Q_i K^T        warp 3   O_i += P_i V
//   warps 8..15    softmax, one thread per row of Q tile i = 0, 1
//   warp 2         the segments (an item, or the part of it that falls to this
//                  CTA), a few ahead; every other role reads them from a ring
// The next segment's loads and first S products run under the end of the one before.
// The running maximum is raised lazily (2^8), as in attention_sm100.cu.  All
// waits are bounded; on expiry every role leaves and the status word is set.
//
// TMEM columns: S_i at i KT, P_i at 2 KT + i KT / 2, O_i at 512 - (2 - i) D.
#include "attn_cache.cuh"
#include "attn_common.cuh"
#include "host.hpp"

namespace qv {
namespace {

constexpr int THREADS = 512;
constexpr int RAW = 4;          // stages of raw codes
constexpr int KV = 2;           // operand stages of K and of V
constexpr int CRING = 8;        // constants: more than RAW + KV tiles back nothing reads them
constexpr int SEGS = 4;         // segments handed out ahead
constexpr int SEG_READERS = 15; // producer, two issuers, 4 + 8 warps
constexpr int Q_ROWS = 256;     // rows of an item
// Cost of an item on the line: a start-up (loads, first products, epilogue)
// and its key tiles; with one Q tile a softmax warpgroup idles, but the other's
// chain per tile is nearly as long.
constexpr int COST_START = 30, COST_TILE2 = 10, COST_TILE1 = 8;
// No piece is cut shorter than this (8 tiles): a join costs about as much.
constexpr int COST_MIN = COST_START + 8 * COST_TILE2;
constexpr int RAW_BYTES = 8192; // K or V codes of a tile
constexpr int OP_BYTES = 16384; // the same as fp16
constexpr uint32_t TMEM_COLS = 512;

template <int D>
struct Lay {
  static constexpr int KT = D == 64 ? 128 : 64;
  static constexpr int PANELS = D / 64;                    // 64-dim (128-byte) panels of Q and K / V rows
  static constexpr int Q_PANEL = 128 * 128;                // bytes: 128 rows x 64 dims
  static constexpr int Q = 0;                              // [tile][panel]
  static constexpr int K = Q + 2 * PANELS * Q_PANEL;       // [stage][panel] KT rows of 128 bytes
  static constexpr int V = K + KV * OP_BYTES;
  static constexpr int RK = V + KV * OP_BYTES;             // raw codes [stage]
  static constexpr int RV = RK + RAW * RAW_BYTES;
  static constexpr int CONST = RV + RAW * RAW_BYTES;       // float4 [CRING][KT / 32]
  static constexpr int BAR = CONST + CRING * (KT / 32) * 16;
  // q_full, q_empty, raw_full[RAW], raw_empty[RAW], k_full[KV], k_empty[KV], v_full[KV],
  // v_empty[KV], seg_full[SEGS], seg_empty[SEGS], s_full[2], s_free[2], p_full[2], o_done[2], drain, drain2
  static constexpr int NUM_BARS = 2 + 2 * RAW + 4 * KV + 2 * SEGS + 8 + 2;
  static constexpr int MISC = BAR + NUM_BARS * 8;          // TMEM base
  static constexpr int SEG = MISC + 32;                    // Segment [SEGS]
  static constexpr int CUM = SEG + SEGS * 64;              // long long [THREADS + 1]
  static constexpr int ROWS = CUM + (THREADS + 2) * 8;     // int2 [256]: token and head of each row
  static constexpr int TOTAL = ROWS + 256 * 8 + 1024;
};

// One lane of a converged warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(p));
  return p != 0;
}

// K-major or MN-major operand with 128-byte swizzle; lead: bytes between the
// 64-element panels of an MN-major operand (unused by K-major ones).
__device__ __forceinline__ uint64_t sdesc_panels(uint32_t saddr, uint32_t lead) {
  return (sdesc_sw128(saddr) & ~(0x3fffull << 16)) | ((uint64_t)(lead >> 4) << 16);
}

// Constants of a 32-key chunk.
struct Chunk {
  float ck, lv, inv_vs;
};

// A tile that the row sees in part (valid < KT keys, may be <= 0): hidden
// scores become -inf, and a chunk without a visible key gets neutral constants
// (whatever its block's scales are, the row takes nothing from them).
template <int KT>
__device__ __forceinline__ void hide_keys(uint32_t (&s)[KT], Chunk (&k)[KT / 32], int valid) {
#pragma unroll
  for (int e = 0; e < KT; ++e)
    if (e >= valid) s[e] = 0xff800000u;
#pragma unroll
  for (int c = 0; c < KT / 32; ++c)
    if (32 * c >= valid) k[c] = {1.f, 0.f, 0.f};
}

// Max over the row of ck S + lv: each chunk's largest score first, four chains.
template <int KT>
__device__ __forceinline__ float tile_max(const uint32_t (&s)[KT], const Chunk (&k)[KT / 32], float mx) {
#pragma unroll
  for (int c = 0; c < KT / 32; ++c) {
    float m[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const uint32_t* v = &s[32 * c + 8 * x];
      m[x] = max3f(max3f(__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2])), __uint_as_float(v[3]),
                   __uint_as_float(v[4]));
      m[x] = max3f(m[x], __uint_as_float(v[5]), fmaxf(__uint_as_float(v[6]), __uint_as_float(v[7])));
    }
    mx = fmaxf(mx, fmaf(max3f(fmaxf(m[0], m[1]), m[2], m[3]), k[c].ck, k[c].lv));
  }
  return mx;
}

// P of chunk C as fp16 pairs into s[16 C..16 C + 16) (no earlier chunk wrote
// the scores it reads), its sum over 1 / vs into l.  POLY of 8 pairs take the
// FMA-pipe exponential.
template <int POLY, int C, int KT>
__device__ __forceinline__ void exp_chunk(uint32_t (&s)[KT], const Chunk& k, float neg_m, float& l) {
  const uint64_t c2 = f2_pack(k.ck, k.ck), nm2 = f2_pack(k.lv + neg_m, k.lv + neg_m);
  uint64_t la = f2_pack(0.f, 0.f), lb = f2_pack(0.f, 0.f);
#pragma unroll
  for (int e = 16 * C; e < 16 * C + 16; ++e) {
    const uint64_t x2 = f2_fma(f2_pack(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), c2, nm2);
    float p0, p1;
    if ((e & 7) < POLY) {
      exp2_poly_pair(x2, p0, p1);
    } else {
      float x0, x1;
      f2_unpack(x2, x0, x1);
      p0 = ex2(x0);
      p1 = ex2(x1);
    }
    if (e & 1) lb = f2_add(lb, f2_pack(p0, p1));
    else la = f2_add(la, f2_pack(p0, p1));
    s[e] = pack_half2(p0, p1);
  }
  float l0, l1;
  f2_unpack(f2_add(la, lb), l0, l1);
  l = fmaf(l0 + l1, k.inv_vs, l);
}

// P of the tile to TMEM, a chunk at a time (the stores overlap the
// exponentials still to come).  P may be written once the PV product of the
// tile before has read the previous one: that wait (unless `first`) comes
// just before the first store.  False if it gave up.
template <int POLY, int KT>
__device__ __forceinline__ bool exp_store(uint32_t (&s)[KT], const Chunk (&k)[KT / 32], float neg_m, float& l,
                                          uint32_t tP, bool first, uint32_t o_done, uint32_t o_parity, uint32_t tries) {
  // asked before the first exponentials: a test's answer takes about 100 cycles
  const bool ready = first || test(o_done, o_parity);
  exp_chunk<POLY, 0>(s, k[0], neg_m, l);
  if (!__all_sync(~0u, ready) && !warp_wait(o_done, o_parity, tries)) return false;
  tc_fence_after();
  tmem_st16(tP, *reinterpret_cast<const uint32_t(*)[16]>(&s[0]));
  exp_chunk<POLY, 1>(s, k[1], neg_m, l);
  tmem_st16(tP + 16, *reinterpret_cast<const uint32_t(*)[16]>(&s[16]));
  if constexpr (KT == 128) {
    exp_chunk<POLY, 2>(s, k[2], neg_m, l);
    tmem_st16(tP + 32, *reinterpret_cast<const uint32_t(*)[16]>(&s[32]));
    exp_chunk<POLY, 3>(s, k[3], neg_m, l);
    tmem_st16(tP + 48, *reinterpret_cast<const uint32_t(*)[16]>(&s[48]));
  }
  tmem_st_wait();
  return true;
}

// Q block `qb` of request b: its rows and keys.
template <int KT>
struct Block {
  static constexpr int START = COST_START, MIN = COST_MIN;
  int q0, ql, n, tok0, nqt, tiles;
  long long cost;                        // of one kv head; 0: no such block
  __device__ __forceinline__ int tile_cost() const { return nqt == 2 ? COST_TILE2 : COST_TILE1; }
  __device__ __forceinline__ Block() {}
  __device__ __forceinline__ Block(const CacheAttnArgs& a, int b, int qb) {
    q0 = a.cu_q[b];
    ql = a.cu_q[b + 1] - q0;
    n = a.kv_lens[b];
    const int tpt = 128 / a.group;       // tokens of a Q tile
    tok0 = qb * 2 * tpt;
    nqt = tok0 + tpt < ql ? 2 : 1;
    tiles = 0;
    cost = 0;
    // (a negative number of queries is for lengths_ok to report)
    if ((ql >= 0 && tok0 >= ql) || !lengths_ok(a, q0, ql, n)) return;
    tiles = (key_limit(min(ql, tok0 + 2 * tpt) - 1, ql, n, a.chunk) + KT - 1) / KT;
    cost = COST_START + (long long)tiles * tile_cost();
  }
};

template <bool BF16, int D>
__global__ void __launch_bounds__(THREADS, 1)
    attn_cache_tiles_kernel(const __grid_constant__ CUtensorMap tmQ, CacheAttnArgs a) {
  using L = Lay<D>;
  constexpr int KT = L::KT, CH = KT / 32;
  constexpr uint32_t COL_S = 0, COL_P = 2 * KT, COL_O = 512 - 2 * D;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + L::BAR);
  uint64_t* q_empty = q_full + 1;
  uint64_t* raw_full = q_empty + 1;
  uint64_t* raw_empty = raw_full + RAW;
  uint64_t* k_full = raw_empty + RAW;
  uint64_t* k_empty = k_full + KV;
  uint64_t* v_full = k_empty + KV;
  uint64_t* v_empty = v_full + KV;
  uint64_t* seg_full = v_empty + KV;
  uint64_t* seg_empty = seg_full + SEGS;
  // the softmax warps address the next four [2] arrays from s_full[i] at byte offsets 16, 32, 48
  uint64_t* s_full = seg_empty + SEGS;
  uint64_t* s_free = s_full + 2;
  uint64_t* p_full = s_free + 2;
  uint64_t* o_done = p_full + 2;
  uint64_t* drain = o_done + 2;
  uint64_t* drain2 = drain + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC);
  volatile Segment* segs = reinterpret_cast<volatile Segment*>(smem + L::SEG);
  long long* cum = reinterpret_cast<long long*>(smem + L::CUM);
  const uint32_t tries = a.wait_tries;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int s = 0; s < RAW; ++s) {
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_empty[s], 4);
    }
    for (int s = 0; s < KV; ++s) {
      mbar_init(&k_full[s], 4);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 4);
      mbar_init(&v_empty[s], 1);
    }
    for (int s = 0; s < SEGS; ++s) {
      mbar_init(&seg_full[s], 1);
      mbar_init(&seg_empty[s], SEG_READERS);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 2);
      mbar_init(&s_free[i], 4);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(drain, 1);
    mbar_init(drain2, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) tma_prefetch_desc(&tmQ);
  pdl_wait();
  pdl_trigger();
  const int blocks = a.B * a.row_blocks, g = (blocks + THREADS - 1) / THREADS;
  tc_fence_before();
  scan_blocks<THREADS, Block<KT>>(a, cum, blocks, g);
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int tpt = 128 / a.group;                           // tokens of a Q tile

  // Registers: launched at 128 each; 128 (56 + 56 + 2 * 200) = 128 * 512.
  // Every warp of a warpgroup runs the same setmaxnreg.
  if (warp < 4) {
    regs_dec<56>();
    if (warp == 2) {
      // ---------------------------------------------------------- segments
      if (lane == 0) {
        PieceWalk<THREADS, Block<KT>> walk(a, cum, blocks, g);
        Segment sg;
        for (int seg = 0;; ++seg) {
          const bool more = walk.next(a, blocks, sg);
          const int st = seg % SEGS;
          if (!wait(&seg_empty[st], ((seg / SEGS) & 1) ^ 1, tries)) break;
          segs[st].b = sg.b;
          segs[st].kvh = sg.kvh;
          segs[st].tok0 = sg.tok0;
          segs[st].q0 = sg.q0;
          segs[st].ql = sg.ql;
          segs[st].n = sg.n;
          segs[st].nqt = sg.nqt;
          segs[st].t0 = sg.t0;
          segs[st].nt = more ? sg.nt : -1;
          segs[st].slot = sg.slot;
          mbar_arrive(&seg_full[st]);
          if (!more) break;
        }
        if (a.can_split) reinterpret_cast<Cut*>(a.part_lse + 2LL * gridDim.x * Q_ROWS)[blockIdx.x] = walk.cut;
      }
    } else if (warp == 0) {
      // ---------------------------------------------------------- producer
      const int bs = 1 << a.bs_log2;
      const int piece = min(bs, KT);                       // keys of one copy
      const int pieces = KT / piece;
      bool bad = false, ok = true;
      int jg = 0, it = 0;                                  // key tiles and Q blocks loaded so far
      for (int seg = 0;; ++seg) {
        const int ss = seg % SEGS;
        ok = warp_wait(&seg_full[ss], (seg / SEGS) & 1, tries);
        if (!ok) break;
        const int b = segs[ss].b, kvh = segs[ss].kvh, n = segs[ss].n, t0 = segs[ss].t0, nt = segs[ss].nt;
        const int q_tok = segs[ss].q0 + segs[ss].tok0, nqt = segs[ss].nqt;
        __syncwarp();
        if (lane == 0) mbar_arrive(&seg_empty[ss]);
        if (nt < 0) break;
        if (nt == 0) continue;
        const int32_t* row = a.table + (long long)b * a.wide;
        // lane i holds the id and scales of block base + i; the next 32 are
        // fetched while these are used
        int base = (t0 * KT) >> a.bs_log2;
        const int last = (min((t0 + nt) * KT, n) - 1) >> a.bs_log2;
        auto fetch_id = [&](int j) { return j <= last ? row[j] : -1; };
        auto fetch_scales = [&](int id, float& ks, float& vs) {
          const bool good = id >= 0 && id < a.num_blocks;
          ks = good ? a.ks[(long long)id * a.hk + kvh] : 0.f;
          vs = good ? a.vs[(long long)id * a.hk + kvh] : 0.f;
        };
        int id = fetch_id(base + lane);
        float ks, vs;
        fetch_scales(id, ks, vs);
        int id2 = fetch_id(base + 32 + lane);
        bool q_loaded = false;
        for (int j = 0; j < nt; ++j, ++jg) {
          const int key0 = (t0 + j) * KT;
          if (((key0 + KT - 1) >> a.bs_log2) >= base + 32) {
            // blocks and tiles nest, so a tile starts on the batch's boundary
            base += 32;
            id = id2;
            fetch_scales(id, ks, vs);
            id2 = fetch_id(base + 32 + lane);
          }
          // constants of the tile's 32-key chunks: seen by the softmax through
          // raw_full, k_full and the S issuer's own arrival on s_full
          const int cj = min(((key0 + 32 * lane) >> a.bs_log2) - base, 31);
          const int cid = __shfl_sync(~0u, id, cj);
          const float cks = __shfl_sync(~0u, ks, cj), cvs = __shfl_sync(~0u, vs, cj);
          // the copy of lane's piece
          const int pkey = key0 + lane * piece;
          const int pid = __shfl_sync(~0u, id, min((pkey >> a.bs_log2) - base, 31));
          const bool mine = lane < pieces && pkey < n;
          const bool good = mine && pid >= 0 && pid < a.num_blocks;
          bad |= mine && !good;
          const int st = jg % RAW;
          ok = warp_wait(&raw_empty[st], ((jg / RAW) & 1) ^ 1, tries);
          if (!ok) break;
          if (lane < CH) {
            const bool have = cid >= 0 && cid < a.num_blocks && key0 + 32 * lane < n;
            // a skipped block: every score -inf
            const float4 k = have ? make_float4(nonzero_factor(cks * a.scale_log2), log2f(cvs), 1.f / cvs, 0.f)
                                  : make_float4(1.f, -INFINITY, 0.f, 0.f);
            reinterpret_cast<float4*>(smem + L::CONST)[(jg % CRING) * CH + lane] = k;
          }
          const uint32_t count = __popc(__ballot_sync(~0u, good));
          __syncwarp();
          if (lane == 0) {
            mbar_arrive_expect_tx(&raw_full[st], count * 2 * piece * D);
          }
          __syncwarp();
          if (good) {
            const long long off = pid * a.block_stride + ((long long)kvh * bs + (pkey & (bs - 1))) * D;
            const uint32_t at = st * RAW_BYTES + lane * piece * D, bar = smem_u32(&raw_full[st]);
            bulk_load(sbase + L::RK + at, a.kc + off, piece * D, bar);
            bulk_load(sbase + L::RV + at, a.vc + off, piece * D, bar);
          }
          if (!q_loaded && (j == min(nt, 2) - 1)) {
            // Q is free once the S products of the item before are done; by
            // then this item's first codes are on their way
            q_loaded = true;
            ok = it == 0 || warp_wait(q_empty, (it - 1) & 1, tries);
            if (!ok) { ++jg; break; }
            if (lane == 0) {
              mbar_arrive_expect_tx(q_full, nqt * L::PANELS * tpt * a.group * 128);
              for (int i = 0; i < nqt; ++i)
                for (int p = 0; p < L::PANELS; ++p)
                  tma_load_3d(smem + L::Q + (i * L::PANELS + p) * L::Q_PANEL, &tmQ, q_full, p * 64, kvh * a.group,
                              q_tok + i * tpt);
            }
            ++it;
          }
        }
        if (!ok) break;
      }
      if (bad) report_bad_block(a.ctl);
      if (!ok && lane == 0) {
        // gave up: let the copies in flight land before the CTA exits
        report_status(a.ctl, ST_TIMEOUT_TMA_EMPTY);
        if (it > 0) mbar_wait_drain(q_full, (it - 1) & 1, 200000000ull);
        for (int jj = max(0, jg - RAW); jj < jg; ++jj)
          mbar_wait_drain(&raw_full[jj % RAW], (jj / RAW) & 1, 200000000ull);
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------- S = Q K^T
      // The issuers walk their loops as whole warps and elect a lane for each
      // group of MMAs: from inside a one-lane branch the same MMAs issue a
      // third slower (their descriptors are then not warp-uniform).
      constexpr uint32_t idesc = idesc_f16(128, KT, false, false, BF16);
      uint32_t cs[2] = {0, 0};                             // S_i products issued so far
      int jg = 0, it = 0;
      bool ok = true;
      for (int seg = 0; ok; ++seg) {
        const int ss = seg % SEGS;
        if (!warp_wait(&seg_full[ss], (seg / SEGS) & 1, tries)) { ok = false; break; }
        const int nt = segs[ss].nt, nqt = segs[ss].nqt;
        __syncwarp();
        if (lane == 0) mbar_arrive(&seg_empty[ss]);
        if (nt < 0) break;
        if (nt == 0) continue;
        if (!warp_wait(q_full, it & 1, tries)) { ok = false; break; }
        ++it;
        for (int j = 0; j < nt; ++j, ++jg) {
          const int st = jg % KV;
          if (!warp_wait(&k_full[st], (jg / KV) & 1, tries)) { ok = false; break; }
          for (int i = 0; i < nqt; ++i) {
            if (cs[i] > 0 && !warp_wait(&s_free[i], (cs[i] - 1) & 1, tries)) { ok = false; break; }
            ++cs[i];
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int p = 0; p < L::PANELS; ++p)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  mma_f16_ss(tmem + COL_S + i * KT,
                             sdesc_sw128(sbase + L::Q + (i * L::PANELS + p) * L::Q_PANEL + k * 32),
                             sdesc_sw128(sbase + L::K + st * OP_BYTES + p * KT * 128 + k * 32), idesc,
                             (p | k) ? 1u : 0u);
              tc_commit(&s_full[i]);
              mbar_arrive(&s_full[i]);
              if (i == nqt - 1) {
                tc_commit(&k_empty[st]);
                if (j == nt - 1) tc_commit(q_empty);
              }
            }
            __syncwarp();
          }
          if (!ok) break;
        }
      }
      if (!ok && elect_one()) {
        report_status(a.ctl, ST_TIMEOUT_FULL);
        tc_commit(drain);
        mbar_wait_drain(drain, 0, 200000000ull);
      }
      __syncwarp();
    } else if (warp == 3) {
      // ---------------------------------------------------------- O += P V
      constexpr uint32_t idesc = idesc_f16(128, D, false, true);
      uint32_t cp[2] = {0, 0};                             // PV_i products issued so far
      int jg = 0;
      bool ok = true;
      for (int seg = 0; ok; ++seg) {
        const int ss = seg % SEGS;
        if (!warp_wait(&seg_full[ss], (seg / SEGS) & 1, tries)) { ok = false; break; }
        const int nt = segs[ss].nt, nqt = segs[ss].nqt;
        __syncwarp();
        if (lane == 0) mbar_arrive(&seg_empty[ss]);
        if (nt < 0) break;
        for (int j = 0; j < nt; ++j, ++jg) {
          const int st = jg % KV;
          if (!warp_wait(&v_full[st], (jg / KV) & 1, tries)) { ok = false; break; }
          for (int i = 0; i < nqt; ++i) {
            if (!warp_wait(&p_full[i], cp[i] & 1, tries)) { ok = false; break; }
            ++cp[i];
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < KT / 16; ++k)
                mma_f16_ts(tmem + COL_O + i * D, tmem + COL_P + i * (KT / 2) + k * 8,
                           sdesc_panels(sbase + L::V + st * OP_BYTES + k * 2048, KT * 128), idesc,
                           (j > 0 || k > 0) ? 1u : 0u);
              tc_commit(&o_done[i]);
              if (i == nqt - 1) tc_commit(&v_empty[st]);
            }
            __syncwarp();
          }
          if (!ok) break;
        }
      }
      if (!ok && elect_one()) {
        report_status(a.ctl, ST_TIMEOUT_SOFTMAX);
        tc_commit(drain2);
        mbar_wait_drain(drain2, 0, 200000000ull);
      }
      __syncwarp();
    }
  } else if (warp < 8) {
    // ------------------------------------------------------------ codes -> fp16 / bf16
    regs_dec<56>();
    const int th = threadIdx.x - 128;                      // 0..127
    constexpr int PARTS = D / 16;                          // 16-code pieces of a row
    constexpr int IT = KT * PARTS / 128;                   // pieces per thread
    const int part = th % PARTS, row0 = th / PARTS, panel = part / 4;
    bool ok = true;
    int jg = 0;
    for (int seg = 0; ok; ++seg) {
      const int ss = seg % SEGS;
      if (!warp_wait(&seg_full[ss], (seg / SEGS) & 1, tries)) { ok = false; break; }
      const int nt = segs[ss].nt;
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[ss]);
      if (nt < 0) break;
      for (int j = 0; ok && j < nt; ++j, ++jg) {
        const int rs = jg % RAW, st = jg % KV;
        if (!warp_wait(&raw_full[rs], (jg / RAW) & 1, tries)) { ok = false; break; }
#pragma unroll(BF16 ? 2 : 1)
        for (int side = 0; side < 2; ++side) {
          const uint32_t src = sbase + (side ? L::RV : L::RK) + rs * RAW_BYTES;
          const uint32_t dst = sbase + (side ? L::V : L::K) + st * OP_BYTES + panel * KT * 128;
          uint4 w[IT];
#pragma unroll
          for (int it = 0; it < IT; ++it)
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[it].x), "=r"(w[it].y), "=r"(w[it].z), "=r"(w[it].w)
                         : "r"(src + (row0 + it * (128 / PARTS)) * D + part * 16)
                         : "memory");
          uint64_t* empty = side ? &v_empty[st] : &k_empty[st];
          if (!warp_wait(empty, ((jg / KV) & 1) ^ 1, tries)) { ok = false; break; }
#pragma unroll
          for (int it = 0; it < IT; ++it) {
            const int r = row0 + it * (128 / PARTS);
            const uint32_t x[4] = {w[it].x, w[it].y, w[it].z, w[it].w};
            uint32_t y[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (side || !BF16) {
                y[2 * e] = codes2<false, false>(x[e]);
                y[2 * e + 1] = codes2<false, true>(x[e]);
              } else {
                y[2 * e] = codes2<true, false>(x[e]);
                y[2 * e + 1] = codes2<true, true>(x[e]);
              }
            }
            // 16-byte chunks 2 part and 2 part + 1 of the row, at chunk ^ (row & 7);
            // lanes of the second panel write them in the other order, which
            // keeps the banks of a quarter warp apart
            const uint32_t line = dst + r * 128;
            const uint32_t c0 = ((2 * (part & 3)) ^ (r & 7)) * 16, c1 = c0 ^ 16;
            const bool swap = panel != 0;
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(line + (swap ? c1 : c0)),
                         "r"(swap ? y[4] : y[0]), "r"(swap ? y[5] : y[1]), "r"(swap ? y[6] : y[2]),
                         "r"(swap ? y[7] : y[3])
                         : "memory");
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(line + (swap ? c0 : c1)),
                         "r"(swap ? y[0] : y[4]), "r"(swap ? y[1] : y[5]), "r"(swap ? y[2] : y[6]),
                         "r"(swap ? y[3] : y[7])
                         : "memory");
          }
          // orders these stores before the MMA's reads, and the loads of the raw
          // stage before the copy that refills it
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(side ? &v_full[st] : &k_full[st]);
            if (side) mbar_arrive(&raw_empty[rs]);
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------ softmax of Q tile i
    regs_inc<200>();
    const int i = (warp - 8) / 4;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem + lane_base + COL_S + i * KT;
    const uint32_t tP = tmem + lane_base + COL_P + i * (KT / 2);
    const uint32_t tO = tmem + lane_base + COL_O + i * D;
    const uint32_t bar_s_full = smem_u32(&s_full[i]);
    const uint32_t bar_s_free = bar_s_full + 16, bar_p_full = bar_s_full + 32, bar_o_done = bar_s_full + 48;
    const float4* consts = reinterpret_cast<const float4*>(smem + L::CONST);
    // the row's token in the block (past any block's for a row that holds none)
    // and head in the group: kept in shared memory, as registers held through
    // the tile loop push scores to local memory
    volatile int2* row_at = reinterpret_cast<volatile int2*>(smem + L::ROWS) + (threadIdx.x - 256);
    row_at->x = r < tpt * a.group ? i * tpt + r / a.group : 1 << 30;
    row_at->y = r % a.group;
    bool ok = true;
    uint32_t cnt = 0;                                      // tiles of this warpgroup so far
    int jg = 0;                                            // tiles of the CTA so far
    for (int seg = 0; ok; ++seg) {
      const int ss = seg % SEGS;
      if (!warp_wait(&seg_full[ss], (seg / SEGS) & 1, tries)) break;
      const int nt = segs[ss].nt;
      if (nt < 0) break;
      const int ntr = i < segs[ss].nqt ? nt : 0;
      // keys the row sees, from the segment's first tile on; rows past the end
      // compute on whatever their tile holds and are not stored
      int left;
      {
        const int ql = segs[ss].ql, in_block = ql - segs[ss].tok0, x = row_at->x;
        left = (x < in_block ? key_limit(segs[ss].tok0 + x, ql, segs[ss].n, a.chunk) : segs[ss].n) - segs[ss].t0 * KT;
      }
      float m_used = -INFINITY, l = 0.f;
      bool ready = false;
      for (int j = 0; j < ntr; ++j, ++cnt) {
        if (!__all_sync(~0u, ready) && !warp_wait(bar_s_full, cnt & 1, tries)) { ok = false; break; }
        const int cj = (jg + j) % CRING;
        tc_fence_after();
        uint32_t s[KT];
#pragma unroll
        for (int c = 0; c < CH; ++c) tmem_ld32(tS + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&s[32 * c]));
        tmem_ld_wait();
        reg_fence<0, KT>(s);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive(bar_s_free);
        Chunk k[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const float4* at = &consts[cj * CH + c];
          k[c] = {at->x, at->y, at->z};
        }
        const int valid = left - j * KT;                   // keys of the tile that the row sees (may be <= 0)
        if (__any_sync(~0u, valid < KT)) hide_keys(s, k, valid);
        const float mx = tile_max(s, k, m_used);
        const bool need = mx > m_used + 8.0f;
        float alpha = 1.f;
        bool rescale = false;
        if (__any_sync(~0u, need)) {
          const float m_target = need ? mx : m_used;
          alpha = m_target == m_used ? 1.f : ex2(m_used - m_target);
          rescale = j > 0;
          m_used = m_target;
        }
        const float neg_m = m_used == -INFINITY ? 0.f : -m_used;
        float lj = 0.f;
        // (the previous item's epilogue has waited for its last PV product)
        if (!exp_store<1>(s, k, neg_m, lj, tP, j == 0, bar_o_done, (cnt - 1) & 1, tries)) { ok = false; break; }
        ready = j + 1 < ntr && test(bar_s_full, (cnt + 1) & 1);
        l = l * alpha + lj;
        if (rescale) {
#pragma unroll 1
          for (int cc = 0; cc < D / 16; ++cc) {
            uint32_t v[16];
            tmem_ld16(tO + cc * 16, v);
            tmem_ld_wait();
            reg_fence<0, 16>(v);
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * alpha);
            tmem_st16(tO + cc * 16, v);
          }
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive(bar_p_full);
      }
      jg += nt;
      // ---------------------------------------------------------- epilogue
      if (ok && ntr > 0) {
        ok = warp_wait(bar_o_done, (cnt - 1) & 1, tries);
        tc_fence_after();
      }
      if (ok) {                                            // warp-uniform
        const int x = row_at->x, tok = segs[ss].tok0 + x, slot = segs[ss].slot;
        const bool row_ok = x < segs[ss].ql - segs[ss].tok0;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const float lse2 = l == 0.f ? -INFINITY : m_used + log2f(l);
        const long long gtok = segs[ss].q0 + tok;
        const int h = segs[ss].kvh * a.group + row_at->y;
        const long long part = (long long)slot * Q_ROWS + i * 128 + r;
        float4* part_dst = reinterpret_cast<float4*>(a.part_o + part * D);
        uint4* dst = reinterpret_cast<uint4*>(a.out + gtok * a.o_tok + h * a.o_head);
        // 16 columns at a time where the score row is 128 wide: more would cost
        // the tile loop registers
        constexpr int W = D == 64 ? 16 : 32;
#pragma unroll 1
        for (int cc = 0; cc < D; cc += W) {
          uint32_t v[W];
          if (ntr > 0) {
            if constexpr (W == 16) tmem_ld16(tO + cc, v);
            else tmem_ld32(tO + cc, v);
            tmem_ld_wait();
            reg_fence<0, W>(v);
          }
          if (!row_ok) continue;
#pragma unroll
          for (int e = 0; e < W; ++e) v[e] = l == 0.f ? 0u : __float_as_uint(__uint_as_float(v[e]) * inv);
          if (slot >= 0) {
#pragma unroll
            for (int e = 0; e < W / 4; ++e)
              part_dst[cc / 4 + e] = make_float4(__uint_as_float(v[4 * e]), __uint_as_float(v[4 * e + 1]),
                                                 __uint_as_float(v[4 * e + 2]), __uint_as_float(v[4 * e + 3]));
          } else {
#pragma unroll
            for (int e = 0; e < W / 8; ++e) {
              uint32_t o[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const float p = __uint_as_float(v[8 * e + 2 * x]), q = __uint_as_float(v[8 * e + 2 * x + 1]);
                o[x] = BF16 ? pack_bf162(p, q) : pack_half2(p, q);
              }
              dst[cc / 8 + e] = make_uint4(o[0], o[1], o[2], o[3]);
            }
          }
        }
        if (row_ok) {
          if (slot >= 0) a.part_lse[part] = lse2;
          else if (a.lse) a.lse[h * a.Tq + gtok] = lse2 * 0.6931471805599453f;
        }
      }
      tc_fence_before();                                   // O_i read before the next item's products
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[ss]);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// Adds the parts of the items that a cut went through.  CTA (x, y) looks at
// the cut before piece x + 1; the item's first cut does the work, 256 / (D / 4)
// rows a CTA.
template <bool BF16, int D>
__global__ void __launch_bounds__(256) attn_cache_tiles_join_kernel(CacheAttnArgs a, int grid) {
  pdl_wait();
  pdl_trigger();
  const int x = blockIdx.x + 1;
  const Cut cut = reinterpret_cast<const Cut*>(a.part_lse + 2LL * grid * Q_ROWS)[x];
  if (cut.first != x - 1) return;
  const int row = blockIdx.y * (1024 / D) + threadIdx.x / (D / 4), r = row & 127;
  const int tpt = 128 / a.group, tok = cut.tok0 + (row >> 7) * tpt + r / a.group;
  if (r >= tpt * a.group || tok >= cut.ql) return;
  join_parts<BF16, D>(a, cut, Q_ROWS, row, threadIdx.x % (D / 4), cut.q0 + tok, cut.kvh * a.group + r % a.group);
}

}  // namespace

bool tiles_can_read(const CacheAttnArgs& a) {
  return a.group <= 128 && (a.hq == 1 || a.q_head > 0) && (a.Tq == 1 || a.q_tok > 0);
}

// Whether items may be cut (a rule on the hint alone: the join is launched by it).
static bool tiles_split(long long max_kv, int D) { return max_kv > 8 * (D == 64 ? 128 : 64); }

// One CTA per SM at most, and no more than there can be pieces.
static int tiles_grid(long long items, long long max_kv, int D) {
  const int kt = D == 64 ? 128 : 64;
  const long long cost = items * (COST_START + (max_kv + kt - 1) / kt * COST_TILE2);
  const long long pieces = tiles_split(max_kv, D) ? (cost + COST_MIN - 1) / COST_MIN : items;
  return (int)std::max<long long>(1, std::min<long long>(pieces, device_info().num_sms));
}

int64_t tiles_scratch(long long items, long long max_kv, int D) {
  if (!tiles_split(max_kv, D)) return 0;
  const int64_t grid = tiles_grid(items, max_kv, D);
  return grid > 1 ? grid * (2 * Q_ROWS * (D + 1) * (int64_t)sizeof(float) + (int64_t)sizeof(Cut)) : 0;
}

int launch_tiles(CacheAttnArgs& a, int D, bool bf16, long long max_kv, void* scratch, cudaStream_t stream) {
  const int smem = D == 64 ? Lay<64>::TOTAL : Lay<128>::TOTAL;
  if (smem > device_info().max_smem_optin)
    return set_error(QVGGT_ERR_UNSUPPORTED, "cached_attention: shared memory %d > %d", smem,
                     device_info().max_smem_optin);
  CUtensorMap tmQ;
  const uint64_t dims[3] = {(uint64_t)D, (uint64_t)a.hq, (uint64_t)a.Tq};
  const uint64_t strides[2] = {(uint64_t)(a.hq == 1 ? D : a.q_head) * 2,
                               (uint64_t)(a.Tq == 1 ? a.hq * D : a.q_tok) * 2};
  const uint32_t box[3] = {64, (uint32_t)a.group, (uint32_t)(128 / a.group)};
  if (int rc = encode_tmap(&tmQ, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, a.q,
                           dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  const long long items = (long long)a.B * a.row_blocks * a.hk;
  const int grid = tiles_grid(items, max_kv, D);
  a.can_split = grid > 1 && tiles_split(max_kv, D);
  a.part_o = static_cast<float*>(scratch);
  a.part_lse = a.can_split ? a.part_o + 2LL * grid * Q_ROWS * D : nullptr;
  using Kfn = void (*)(CUtensorMap, CacheAttnArgs);
  static const Kfn fns[2][2] = {{attn_cache_tiles_kernel<false, 64>, attn_cache_tiles_kernel<false, 128>},
                                {attn_cache_tiles_kernel<true, 64>, attn_cache_tiles_kernel<true, 128>}};
  using Jfn = void (*)(CacheAttnArgs, int);
  static const Jfn joins[2][2] = {{attn_cache_tiles_join_kernel<false, 64>, attn_cache_tiles_join_kernel<false, 128>},
                                  {attn_cache_tiles_join_kernel<true, 64>, attn_cache_tiles_join_kernel<true, 128>}};
  static DeviceFlags attr[2][2];
  const Kfn fn = fns[bf16][D == 128];
  if (int rc = ensure_smem(attr[bf16][D == 128], fn, smem, "cudaFuncSetAttribute(cached_attention)")) return rc;
  if (int rc = check_cuda(launch_pdl(fn, dim3((unsigned)grid), dim3(THREADS), smem, stream, 1u, tmQ, a),
                          "cached_attention launch"))
    return rc;
  count_launch(1);
  if (a.can_split) {
    if (int rc = check_cuda(launch_pdl(joins[bf16][D == 128], dim3((unsigned)(grid - 1), Q_ROWS * D / 1024), dim3(256), 0,
                                       stream, 1u, a, grid),
                            "cached_attention join launch"))
      return rc;
    count_launch(1);
  }
  return QVGGT_OK;
}

}  // namespace qv
