// Attention over whole sequences packed one after another: tcgen05 + TMEM.
//
//   x = (scale log2e) q.k,  P = 2^(x - m),  O += P v,  l += sum P,  out = O / l
// over the keys a row sees.  An item is (sequence, block of two 128-row Q tiles,
// kv head); a row is a (token, query head of the group) pair, so the heads that
// share K/V share its tiles.  Lengths are known on the GPU only and a causal mask
// gives late blocks many times the keys of early ones: the items' key tiles are
// laid out as one line of cost and cut into equal pieces, one per SM
// (attn_cache.cuh); what a cut separates is joined by a second launch.
// Per key tile of KT keys (128; 64 where no sequence is longer):
//   warp 0         TMA of K, V and Q tiles, K and V through rings of KV stages
//   warp 1         S_i = Q_i K^T        warp 3   O_i += P_i V
//   warp 2         the segments (an item, or the part of it that falls to this
//                  CTA), two ahead, read by every role from a ring; cleans V tiles
//                  that some row of the block does not see whole
//   warps 4..11    softmax, one thread per row of Q tile i = 0, 1
// The running maximum is raised lazily (2^8).  All waits are bounded; on expiry
// every role leaves and the status word is set.
//
// What a row does not see must not reach it.  Its scores become -inf and its
// weights exactly 0, which is all that keeps finite V out, the next sequence's in
// the last tile among it.  But 0 times an infinity or NaN of V would still be NaN.
// So the tiles that the block's first row does not see to their end are looked
// through, and where one holds such an element, these and its rows past the
// sequence become 0; the rows that do see the element add it at the end (add_odd).
//
// TMEM columns: S_i at i KT, P_i at 2 KT + i KT / 2, O_i at 512 - (2 - i) D.  With
// head_dim 128 and 128-key tiles that is 128 columns too many: S_0 and S_1 take
// turns at column 0 (a score tile is read into registers at once, so its place is
// free again long before the exponentials are done), and P_i is at KT + i KT / 2.
// 64-key tiles with places of their own cost half as many waits and TMEM reads
// again for each key: 1,234 us against 1,020 when this was chosen (two sequences of
// 8,192, 16 heads; 940 to 980 now).
#include "attn_cache.cuh"
#include "attn_common.cuh"
#include "host.hpp"

namespace qv {
namespace {

constexpr int THREADS = 384;
constexpr int SEGS = 4;         // segments handed out ahead
constexpr int SEG_READERS = 12; // producer, two issuers, the V tiles' warp, 8 warps
constexpr int Q_ROWS = 256;     // rows of an item
// Cost of an item on the line, in tenths of a tile with two Q tiles: a start-up
// (loads, first products, epilogue), its key tiles, and again those that its first
// row does not see to their end (their V is looked through, their scores hidden).
// By fits of equal items: 2 to 2.5 tiles, and 0.5 to 1 for each such tile.  Against a
// start of 50 for all items, in short runs at full clock: nine causal sequences to
// 4,099, 32 / 8 heads x 128 540 -> 525 us, four streams of one to six frames, 16 x 128
// 666 -> 632, 16 x 64 the same.
constexpr int COST_START = 20, COST_TILE2 = 10, COST_TILE1 = 9, COST_MASKED = 10;
// No piece is cut shorter than this (8 tiles): a join costs about as much.
constexpr int COST_MIN = COST_START + 8 * COST_TILE2;
constexpr uint32_t TMEM_COLS = 512;

struct PromptArgs {
  const uint16_t* v;                     // read again where it is not finite
  uint16_t* out;
  float* lse;                            // [heads][Tq] or null
  const int32_t* cu;
  float *part_o, *part_lse;              // parts of rows, and their log2-sum-exp
  long long v_tok, v_head, o_tok, o_head, Tq;
  int B, hq, hk, group, chunk, max_len;
  int row_blocks;                        // Q blocks of the longest sequence
  int can_split;                         // items may be cut, a join follows
  float scale_log2;
  uint32_t wait_tries;                   // bound of every wait
  Ctl ctl;
};

template <int D, int KT>
struct Lay {
  static constexpr int OP_BYTES = KT * D * 2;              // K or V of a tile
  static constexpr int KV = OP_BYTES > 16384 ? 2 : 4;      // stages of each
  static constexpr int PANELS = D / 64;                    // 64-dim (128-byte) panels of Q and K / V rows
  static constexpr int Q_PANEL = 128 * 128;                // bytes: 128 rows x 64 dims
  static constexpr int Q = 0;                              // [tile][panel]
  static constexpr int K = Q + 2 * PANELS * Q_PANEL;       // [stage][panel] KT rows of 128 bytes
  static constexpr int V = K + KV * OP_BYTES;
  static constexpr int BAR = V + KV * OP_BYTES;
  // q_full, q_empty, k_full[KV], k_empty[KV], v_full[KV], v_clean[KV], v_empty[KV], seg_full[SEGS],
  // seg_empty[SEGS], s_full[2], s_free[2], p_full[2], o_done[2], drain, drain2
  static constexpr int NUM_BARS = 2 + 5 * KV + 2 * SEGS + 8 + 2;
  static constexpr int MISC = BAR + NUM_BARS * 8;          // TMEM base
  static constexpr int SEG = MISC + 32;                    // Segment [SEGS]
  static constexpr int CUM = SEG + SEGS * 64;              // long long [THREADS + 1]
  static constexpr int ROWS = CUM + (THREADS + 2) * 8;     // int2 [256]: token and head of each row
  static constexpr int TOTAL = ROWS + 256 * 8 + 1024;
};

// Hides the scores of keys from `valid` (may be <= 0) on.
template <int KT>
__device__ __forceinline__ void hide_keys(uint32_t (&s)[KT], int valid) {
#pragma unroll
  for (int e = 0; e < KT; ++e)
    if (e >= valid) s[e] = 0xff800000u;
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Max over the row, four chains; NaN if there is one.
template <int KT>
__device__ __forceinline__ float tile_max(const uint32_t (&s)[KT]) {
  auto f = [&](int e) { return __uint_as_float(s[e]); };
  float m[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) m[x] = max3_nan(f(x), f(4 + x), f(8 + x));
#pragma unroll
  for (int e = 12; e + 8 <= KT; e += 8)
#pragma unroll
    for (int x = 0; x < 4; ++x) m[x] = max3_nan(m[x], f(e + x), f(e + 4 + x));
  // KT = 12 + 8 k + 4: four are left
  m[0] = max3_nan(m[0], f(KT - 4), f(KT - 3));
  m[1] = max3_nan(m[1], f(KT - 2), f(KT - 1));
  return max3_nan(max3_nan(m[0], m[1], m[2]), m[3], m[3]);
}

// P of 32 keys as fp16 / bf16 pairs into s[16 C..16 C + 16) (no earlier chunk wrote
// the scores it reads), its sum into l.  POLY of 8 pairs take the FMA-pipe exponential.
template <bool BF16, int POLY, int C, int KT>
__device__ __forceinline__ void exp_chunk(uint32_t (&s)[KT], uint64_t c2, uint64_t nm2, uint64_t& la, uint64_t& lb) {
#pragma unroll
  for (int e = 16 * C; e < 16 * C + 16; ++e) {
    const uint64_t x2 = f2_fma(f2_pack(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), c2, nm2);
    float p0, p1;
    if ((e & 7) < POLY) {
      exp2_poly_pair<BF16>(x2, p0, p1);                    // (bf16 holds the 2^-125 of hidden keys)
    } else {
      float x0, x1;
      f2_unpack(x2, x0, x1);
      p0 = ex2(x0);
      p1 = ex2(x1);
    }
    if (e & 1) lb = f2_add(lb, f2_pack(p0, p1));
    else la = f2_add(la, f2_pack(p0, p1));
    s[e] = BF16 ? pack_bf162(p0, p1) : pack_half2(p0, p1);
  }
}

// P of the tile to TMEM, a chunk at a time (the stores overlap the
// exponentials still to come).  P may be written once the PV product of the
// tile before has read the previous one: that wait (unless `first`) comes
// just before the first store.  False if it gave up.
template <bool BF16, int POLY, int KT>
__device__ __forceinline__ bool exp_store(uint32_t (&s)[KT], float c, float neg_m, float& l, uint32_t tP, bool first,
                                          uint32_t o_done, uint32_t o_parity, uint32_t tries) {
  // asked before the first exponentials: a test's answer takes about 100 cycles
  const bool ready = first || test(o_done, o_parity);
  const uint64_t c2 = f2_pack(c, c), nm2 = f2_pack(neg_m, neg_m);
  uint64_t la = f2_pack(0.f, 0.f), lb = f2_pack(0.f, 0.f);
  exp_chunk<BF16, POLY, 0>(s, c2, nm2, la, lb);
  if (!__all_sync(~0u, ready) && !warp_wait(o_done, o_parity, tries)) return false;
  tc_fence_after();
  tmem_st16(tP, *reinterpret_cast<const uint32_t(*)[16]>(&s[0]));
  exp_chunk<BF16, POLY, 1>(s, c2, nm2, la, lb);
  tmem_st16(tP + 16, *reinterpret_cast<const uint32_t(*)[16]>(&s[16]));
  if constexpr (KT == 128) {
    exp_chunk<BF16, POLY, 2>(s, c2, nm2, la, lb);
    tmem_st16(tP + 32, *reinterpret_cast<const uint32_t(*)[16]>(&s[32]));
    exp_chunk<BF16, POLY, 3>(s, c2, nm2, la, lb);
    tmem_st16(tP + 48, *reinterpret_cast<const uint32_t(*)[16]>(&s[48]));
  }
  float l0, l1;
  f2_unpack(f2_add(la, lb), l0, l1);
  l += l0 + l1;
  tmem_st_wait();
  return true;
}

__device__ __forceinline__ bool sequence_ok(const PromptArgs& a, int q0, int ql) {
  if (q0 >= 0 && ql >= 0 && ql <= a.max_len && (long long)q0 + ql <= a.Tq) return true;
  report_status(a.ctl, ST_BAD_LENGTH);
  return false;
}

// Q block `qb` of sequence b: its rows and keys.
template <int KT>
struct Block {
  using Args = PromptArgs;
  static constexpr int MIN = COST_MIN;
  int q0, ql, n, tok0, nqt, tiles, masked;
  long long cost;                        // of one kv head; 0: no such block
  __device__ __forceinline__ int tile_cost() const { return nqt == 2 ? COST_TILE2 : COST_TILE1; }
  __device__ __forceinline__ int start() const { return COST_START + masked * COST_MASKED; }
  __device__ __forceinline__ Block() {}
  __device__ __forceinline__ Block(const PromptArgs& a, int b, int qb) {
    q0 = a.cu[b];
    n = ql = a.cu[b + 1] - q0;
    const int tpt = 128 / a.group;       // tokens of a Q tile
    tok0 = qb * 2 * tpt;
    nqt = tok0 + tpt < ql ? 2 : 1;
    tiles = masked = 0;
    cost = 0;
    // (a negative length is for sequence_ok to report)
    if ((ql >= 0 && tok0 >= ql) || !sequence_ok(a, q0, ql)) return;
    tiles = (key_limit(min(ql, tok0 + 2 * tpt) - 1, ql, n, a.chunk) + KT - 1) / KT;
    masked = tiles - key_limit(tok0, ql, n, a.chunk) / KT;
    cost = start() + (long long)tiles * tile_cost();
  }
};

// Bits 15 and 31: whether the word's halves are infinities or NaN (adding one to
// the exponent carries into the sign's place only then).
template <bool BF16>
__device__ __forceinline__ uint32_t odd_bits(uint32_t w) {
  return (w & 0x7fff7fffu) + (BF16 ? 0x00800080u : 0x04000400u);
}

// 0 w + sum in both halves: NaN once w was an infinity or NaN, else +-0.
template <bool BF16>
__device__ __forceinline__ uint32_t add_zero_times(uint32_t w, uint32_t sum) {
  uint32_t r;
  if (BF16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0), "r"(sum));
  else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0), "r"(sum));
  return r;
}

// Adds what was taken out of the V tiles to columns cc.. of a row that sees
// keys [from, to): elements that are not finite.  Any weight of theirs gives
// the same sum, an infinity or NaN.
template <bool BF16, int W>
__device__ __forceinline__ void add_odd(const PromptArgs& a, uint32_t (&acc)[W], int q0, int kvh, int cc, int from, int to) {
#pragma unroll 1
  for (int j = from; j < to; ++j) {
    const uint16_t* p = a.v + (long long)(q0 + j) * a.v_tok + (long long)kvh * a.v_head + cc;
#pragma unroll
    for (int e = 0; e < W; ++e)
      if (odd_bits<BF16>(p[e]) & 0x8000u) acc[e] = __float_as_uint(__uint_as_float(acc[e]) + half_bits_to_f32<BF16>(p[e]));
  }
}

template <bool BF16, int D, int KT>
__global__ void __launch_bounds__(THREADS, 1)
    prompt_attention_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                            const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PromptArgs a) {
  using L = Lay<D, KT>;
  constexpr int KV = L::KV, OP_BYTES = L::OP_BYTES;
  constexpr bool ONE_S = 3 * KT + 2 * D > 512;           // both Q tiles' scores take turns in one place
  constexpr uint32_t COL_S = 0, COL_P = ONE_S ? KT : 2 * KT, COL_O = 512 - 2 * D;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + L::BAR);
  uint64_t* q_empty = q_full + 1;
  uint64_t* k_full = q_empty + 1;
  uint64_t* k_empty = k_full + KV;
  uint64_t* v_full = k_empty + KV;
  uint64_t* v_clean = v_full + KV;
  uint64_t* v_empty = v_clean + KV;
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
  volatile Segment* segs = reinterpret_cast<volatile Segment*>(smem + L::SEG);   // pad[0]: V had odd elements
  long long* cum = reinterpret_cast<long long*>(smem + L::CUM);
  const uint32_t tries = a.wait_tries;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int s = 0; s < KV; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_clean[s], 1);
      mbar_init(&v_empty[s], 2);     // the product, and the warp that has seen to the tile
    }
    for (int s = 0; s < SEGS; ++s) {
      mbar_init(&seg_full[s], 1);
      mbar_init(&seg_empty[s], SEG_READERS);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 2);
    }
    mbar_init(drain, 1);
    mbar_init(drain2, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  pdl_wait();
  const int blocks = a.B * a.row_blocks, g = (blocks + THREADS - 1) / THREADS;
  tc_fence_before();
  scan_blocks<THREADS, Block<KT>>(a, cum, blocks, g);
  tc_fence_after();
  pdl_trigger();                                           // (this CTA has its TMEM by now)
  const uint32_t tmem = *tmem_slot;
  const int tpt = 128 / a.group;                           // tokens of a Q tile

  // Registers: launched at 168 each; 128 (64 + 2 * 216) <= 168 * 384.
  // Every warp of a warpgroup runs the same setmaxnreg.
  if (warp < 4) {
    regs_dec<64>();
    if (warp == 2) {
      // ------------------------------------------------- segments and V tiles
      PieceWalk<THREADS, Block<KT>> walk(a, cum, blocks, g);               // (lane 0's is used)
      auto publish = [&](int seg) {            // lane 0; whether there was room in time, and one to hand out
        const int st = seg % SEGS;
        Segment sg;
        const bool more = walk.next(a, blocks, sg);
        if (!wait(&seg_empty[st], ((seg / SEGS) & 1) ^ 1, tries)) return -1;
        segs[st].b = sg.b;
        segs[st].kvh = sg.kvh;
        segs[st].tok0 = sg.tok0;
        segs[st].q0 = sg.q0;
        segs[st].ql = sg.ql;
        segs[st].nqt = sg.nqt;
        segs[st].t0 = sg.t0;
        segs[st].nt = more ? sg.nt : -1;
        segs[st].slot = sg.slot;
        segs[st].pad[0] = 0;
        mbar_arrive(&seg_full[st]);
        return more ? 1 : 0;
      };
      int left = 2;                            // 1: the last segment is out, 0: its end mark too, -1: gave up
      auto hand_out = [&](int seg) {
        int more = 0;
        if (lane == 0) more = publish(seg);
        return __shfl_sync(~0u, more, 0);
      };
      int jg = 0, ahead = 0;                   // tiles so far; segments handed out
      for (; left > 0 && ahead < 2; ++ahead) left = hand_out(ahead);
      for (int seg = 0; left >= 0; ++seg) {
        if (left > 0) {
          left = hand_out(ahead);
          ++ahead;
          if (left < 0) break;
        }
        const int ss = seg % SEGS;
        __syncwarp();
        const int nt = segs[ss].nt, t0 = segs[ss].t0, n = segs[ss].ql, tok0 = segs[ss].tok0;
        if (nt < 0) {
          if (lane == 0) mbar_arrive(&seg_empty[ss]);
          break;
        }
        const int seen = key_limit(tok0, n, n, a.chunk);   // keys that every row sees
        bool ok = true;
        for (int j = 0; j < nt; ++j, ++jg) {
          const int st = jg % KV, key0 = (t0 + j) * KT;
          ok = warp_wait(&v_full[st], (jg / KV) & 1, tries);
          if (!ok) break;
          if (key0 + KT > seen) {
            // 16-byte pieces (the swizzle moves them within their row only): is there
            // an odd one?  P V may wait for this, so one product per word looks first
            // (222 causal sequences of 256, 16 heads x 128: 232 us; 258 with a test of
            // the exponents, 196 with no look at all), and the rest works on what is found.
            const int first = max(0, seen - key0);         // the tile's first row that some row does not see
            uint32_t sum[4] = {0, 0, 0, 0};                // of 0 times each: 0, or NaN
#pragma unroll 1
            for (int panel = 0; panel < L::PANELS; ++panel) {
              const uint32_t at = sbase + L::V + st * OP_BYTES + panel * KT * 128;
#pragma unroll 4
              for (int p = first * 8 + lane; p < KT * 8; p += 32) {
                uint32_t w[4];
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at + p * 16) : "memory");
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] = add_zero_times<BF16>(w[e], sum[e]);
              }
            }
            if (__any_sync(~0u, ((sum[0] | sum[1] | sum[2] | sum[3]) & 0x7fff7fffu) != 0)) {
              bool odd = false;
#pragma unroll 1
              for (int p = lane; p < OP_BYTES / 16; p += 32) {
                const int key = key0 + p / 8 % KT;
                const uint32_t at = sbase + L::V + st * OP_BYTES + p * 16;
                if (key < seen) continue;
                uint32_t w[4];
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const uint32_t o = odd_bits<BF16>(w[e]);
                  odd |= key < n && (o & 0x80008000u);
                  if (key >= n || o & 0x8000u) w[e] &= 0xffff0000u;
                  if (key >= n || o & 0x80000000u) w[e] &= 0xffffu;
                }
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
              }
              if (odd) segs[ss].pad[0] = 1;
            }
            fence_proxy_async_smem();          // these stores before the product's reads
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_clean[st]);
          }
          if (lane == 0) mbar_arrive(&v_empty[st]);
        }
        if (!ok) break;
        __syncwarp();
        if (lane == 0) mbar_arrive(&seg_empty[ss]);
      }
      if (lane == 0 && a.can_split) reinterpret_cast<Cut*>(a.part_lse + 2LL * gridDim.x * Q_ROWS)[blockIdx.x] = walk.cut;
    } else if (warp == 0) {
      // ---------------------------------------------------------- producer
      bool ok = true;
      int jg = 0, it = 0;                                  // key tiles and Q blocks loaded so far
      int vg = 0;                                          // V tiles
      for (int seg = 0;; ++seg) {
        const int ss = seg % SEGS;
        ok = warp_wait(&seg_full[ss], (seg / SEGS) & 1, tries);
        if (!ok) break;
        const int kvh = segs[ss].kvh, q0 = segs[ss].q0, t0 = segs[ss].t0, nt = segs[ss].nt;
        const int q_tok = q0 + segs[ss].tok0, nqt = segs[ss].nqt;
        __syncwarp();
        if (lane == 0) mbar_arrive(&seg_empty[ss]);
        if (nt < 0) break;
        for (int j = 0; j < nt; ++j, ++jg) {
          const int st = jg % KV, row = q0 + (t0 + j) * KT;
          ok = warp_wait(&k_empty[st], ((jg / KV) & 1) ^ 1, tries);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&k_full[st], OP_BYTES);
            for (int p = 0; p < L::PANELS; ++p)
              tma_load_3d(smem + L::K + st * OP_BYTES + p * KT * 128, &tmK, &k_full[st], p * 64, kvh, row);
          }
          if (j == 0) {
            // Q is free once the S products of the item before are done
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
          ok = warp_wait(&v_empty[st], ((vg / KV) & 1) ^ 1, tries);
          if (!ok) { ++jg; break; }
          if (lane == 0) {
            mbar_arrive_expect_tx(&v_full[st], OP_BYTES);
            for (int p = 0; p < L::PANELS; ++p)
              tma_load_3d(smem + L::V + st * OP_BYTES + p * KT * 128, &tmV, &v_full[st], p * 64, kvh, row);
          }
          ++vg;
        }
        if (!ok) break;
      }
      if (!ok && lane == 0) {
        // gave up: let the copies in flight land before the CTA exits
        report_status(a.ctl, ST_TIMEOUT_TMA_EMPTY);
        if (it > 0) mbar_wait_drain(q_full, (it - 1) & 1, 200000000ull);
        for (int jj = max(0, jg - KV); jj < jg; ++jj)
          mbar_wait_drain(&k_full[jj % KV], (jj / KV) & 1, 200000000ull);
        for (int jj = max(0, vg - KV); jj < vg; ++jj)
          mbar_wait_drain(&v_full[jj % KV], (jj / KV) & 1, 200000000ull);
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------- S = Q K^T
      // The issuers walk their loops as whole warps and elect a lane for each
      // group of MMAs: from inside a one-lane branch the same MMAs issue a
      // third slower (their descriptors are then not warp-uniform).
      constexpr uint32_t idesc = idesc_f16(128, KT, false, false, BF16);
      uint32_t cs[2] = {0, 0};                             // products issued so far into each place of scores
      int jg = 0, it = 0;
      bool ok = true;
      for (int seg = 0; ok; ++seg) {
        const int ss = seg % SEGS;
        if (!warp_wait(&seg_full[ss], (seg / SEGS) & 1, tries)) { ok = false; break; }
        const int nt = segs[ss].nt, nqt = segs[ss].nqt;
        __syncwarp();
        if (lane == 0) mbar_arrive(&seg_empty[ss]);
        if (nt < 0) break;
        if (!warp_wait(q_full, it & 1, tries)) { ok = false; break; }
        ++it;
        for (int j = 0; j < nt; ++j, ++jg) {
          const int st = jg % KV;
          if (!warp_wait(&k_full[st], (jg / KV) & 1, tries)) { ok = false; break; }
          for (int i = 0; i < nqt; ++i) {
            const int x = ONE_S ? 0 : i;
            if (cs[x] > 0 && !warp_wait(&s_free[x], (cs[x] - 1) & 1, tries)) { ok = false; break; }
            ++cs[x];
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int p = 0; p < L::PANELS; ++p)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  mma_f16_ss(tmem + COL_S + x * KT,
                             sdesc_sw128(sbase + L::Q + (i * L::PANELS + p) * L::Q_PANEL + k * 32),
                             sdesc_sw128(sbase + L::K + st * OP_BYTES + p * KT * 128 + k * 32), idesc,
                             (p | k) ? 1u : 0u);
              tc_commit(&s_full[i]);
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
      constexpr uint32_t idesc = idesc_f16(128, D, false, true, BF16);
      uint32_t cp[2] = {0, 0};                             // PV_i products issued so far
      int jg = 0;
      uint32_t cleaned = 0;                                // bit st: phase of v_clean[st], completed by cleaned tiles alone
      bool ok = true;
      for (int seg = 0; ok; ++seg) {
        const int ss = seg % SEGS;
        if (!warp_wait(&seg_full[ss], (seg / SEGS) & 1, tries)) { ok = false; break; }
        const int nt = segs[ss].nt, nqt = segs[ss].nqt, t0 = segs[ss].t0, n = segs[ss].ql;
        const int seen = nt < 0 ? 0 : key_limit(segs[ss].tok0, n, n, a.chunk);
        __syncwarp();
        if (lane == 0) mbar_arrive(&seg_empty[ss]);
        if (nt < 0) break;
        for (int j = 0; j < nt; ++j, ++jg) {
          const int st = jg % KV;
          if ((t0 + j + 1) * KT > seen) {
            if (!warp_wait(&v_clean[st], cleaned >> st & 1, tries)) { ok = false; break; }
            cleaned ^= 1u << st;
          } else if (!warp_wait(&v_full[st], (jg / KV) & 1, tries)) { ok = false; break; }
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
              mbar_arrive(&o_done[i]);                     // hands on what the warps that clean V wrote
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
  } else {
    // ------------------------------------------------------------ softmax of Q tile i
    regs_inc<216>();
    const int i = (warp - 4) / 4;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem + lane_base + COL_S + (ONE_S ? 0 : i * KT);
    const uint32_t tP = tmem + lane_base + COL_P + i * (KT / 2);
    const uint32_t tO = tmem + lane_base + COL_O + i * D;
    const uint32_t bar_s_full = smem_u32(&s_full[i]);
    const uint32_t bar_s_free = ONE_S ? smem_u32(s_free) : bar_s_full + 16, bar_p_full = bar_s_full + 32, bar_o_done = bar_s_full + 48;
    const float c = a.scale_log2;
    // the row's token in the block (past any block's for a row that holds none)
    // and head in the group: kept in shared memory, as registers held through
    // the tile loop push scores to local memory
    volatile int2* row_at = reinterpret_cast<volatile int2*>(smem + L::ROWS) + (threadIdx.x - 128);
    row_at->x = r < tpt * a.group ? i * tpt + r / a.group : 1 << 30;
    row_at->y = r % a.group;
    bool ok = true;
    uint32_t cnt = 0;                                      // tiles of this warpgroup so far
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
        left = (x < in_block ? key_limit(segs[ss].tok0 + x, ql, ql, a.chunk) : ql) - segs[ss].t0 * KT;
      }
      float m_used = -INFINITY, l = 0.f;
      bool ready = false;
      for (int j = 0; j < ntr; ++j, ++cnt) {
        if (!__all_sync(~0u, ready) && !warp_wait(bar_s_full, cnt & 1, tries)) { ok = false; break; }
        tc_fence_after();
        uint32_t s[KT];
#pragma unroll
        for (int x = 0; x < KT / 32; ++x) tmem_ld32(tS + 32 * x, *reinterpret_cast<uint32_t(*)[32]>(&s[32 * x]));
        tmem_ld_wait();
        reg_fence<0, KT>(s);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive(bar_s_free);
        const int valid = left - j * KT;                   // keys of the tile that the row sees (may be <= 0)
        if (__any_sync(~0u, valid < KT)) hide_keys(s, valid);
        const float top = tile_max(s) * c;
        // A score that is NaN makes the row NaN (the exponentials alone would not: the
        // polynomial's clamp drops NaN).  So does one past 2^27 or 2^31: the maximum m is
        // rounded, so x - m of the largest score is off by up to m 2^-25, and 2^4 beside
        // the lazy maximum's 2^8, or 2^64, is what P's type holds either way (past that
        // a row would become 0 in silence).
        if (!(top <= (BF16 ? 2147483648.f : 134217728.f))) l = __int_as_float(0x7fffffff);
        const float mx = fmaxf(m_used, top);
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
        // (the previous item's epilogue has waited for its last PV product.)  Two of 16
        // exponentials on the FMA pipe with head_dim 64, whose limit the others are; with
        // 128 none (two sequences of 8,192: 955 us, 990 with two).  With bf16 they pay for
        // the select to 0 too (four streams of one to six frames, 16 x 64: 483 us, 491
        // with none, 470 with fp16, which needs no select)
        if (!exp_store<BF16, D == 64 ? 1 : 0>(s, c, neg_m, lj, tP, j == 0, bar_o_done, (cnt - 1) & 1, tries)) { ok = false; break; }
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
      // ---------------------------------------------------------- epilogue
      if (ok && ntr > 0) {
        ok = warp_wait(bar_o_done, (cnt - 1) & 1, tries);
        tc_fence_after();
      }
      if (ok && ntr > 0) {                                 // warp-uniform
        const int x = row_at->x, tok = segs[ss].tok0 + x, slot = segs[ss].slot;
        const bool row_ok = x < segs[ss].ql - segs[ss].tok0;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const float lse2 = l == 0.f ? -INFINITY : m_used + log2f(l);
        const long long gtok = segs[ss].q0 + tok;
        const int h = segs[ss].kvh * a.group + row_at->y;
        const long long part = (long long)slot * Q_ROWS + i * 128 + r;
        float4* part_dst = reinterpret_cast<float4*>(a.part_o + part * D);
        uint4* dst = reinterpret_cast<uint4*>(a.out + gtok * a.o_tok + h * a.o_head);
        const bool odd = segs[ss].pad[0] != 0;
        // 16 columns at a time where the score row is 128 wide: more would cost
        // the tile loop registers
        constexpr int W = KT == 128 ? 16 : 32;
#pragma unroll 1
        for (int cc = 0; cc < D; cc += W) {
          uint32_t v[W];
          if constexpr (W == 16) tmem_ld16(tO + cc, v);
          else tmem_ld32(tO + cc, v);
          tmem_ld_wait();
          reg_fence<0, W>(v);
          if (!row_ok) continue;
          if (odd) {
            // keys of the tiles that were cleaned: from what every row sees to what this one does
            const int ql = segs[ss].ql, t0 = segs[ss].t0 * KT;
            const int from = max(t0, key_limit(segs[ss].tok0, ql, ql, a.chunk));
            add_odd<BF16, W>(a, v, segs[ss].q0, segs[ss].kvh, cc, from, min(t0 + nt * KT, t0 + left));
          }
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
__global__ void __launch_bounds__(256) prompt_attention_join_kernel(PromptArgs a, int grid) {
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

// Whether items may be cut (a rule on the longest length alone: the join is launched by it).
bool can_cut(long long max_len) { return max_len > 8 * 128; }

// 64-key tiles where one holds the longest sequence (400 sequences of 20 to 40
// causal tokens, 16 heads x 128: 143 us, 203 with 128-key tiles; five: 9.5 and
// 11.4), else 128 (80 of 100 to 200 tokens: 87, 85 with 64-key tiles; five of up to
// 256: 17 and 21).
int tile_keys(long long max_len) { return max_len <= 64 ? 64 : 128; }

// One CTA per SM at most, and no more than there can be pieces.
int grid_of(long long items, long long max_len) {
  const int kt = tile_keys(max_len);
  const long long cost = items * (COST_START + (max_len + kt - 1) / kt * COST_TILE2);
  const long long pieces = can_cut(max_len) ? (cost + COST_MIN - 1) / COST_MIN : items;
  return (int)std::max<long long>(1, std::min<long long>(pieces, device_info().num_sms));
}

int64_t row_blocks_of(int64_t max_len, int group) { return (max_len + 2 * (128 / group) - 1) / (2 * (128 / group)); }

int64_t scratch_of(long long items, long long max_len, int D) {
  if (!can_cut(max_len)) return 0;
  const int64_t grid = grid_of(items, max_len);
  return grid > 1 ? grid * (2 * Q_ROWS * (D + 1) * (int64_t)sizeof(float) + (int64_t)sizeof(Cut)) : 0;
}

int check_shape(const char* name, int64_t T, int64_t q_heads, int64_t kv_heads, int64_t sequences, int64_t max_len,
                int64_t head_dim) {
  if (T < 0 || sequences < 0 || max_len < 0 || q_heads <= 0 || kv_heads <= 0)
    return set_error(QVGGT_ERR_INVALID, "%s: bad shape", name);
  if (q_heads % kv_heads)
    return set_error(QVGGT_ERR_INVALID, "%s: %lld query heads do not share %lld key heads evenly", name,
                     (long long)q_heads, (long long)kv_heads);
  if (head_dim != 64 && head_dim != 128)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128", name);
  if (q_heads / kv_heads > 128)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: more than 128 query heads to a key head", name);
  if (q_heads > 65535 || T > 2147483647LL / q_heads || sequences > 1 << 24)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: too many rows or sequences", name);
  if (sequences * row_blocks_of(std::min(max_len, T), (int)(q_heads / kv_heads)) > 1 << 30)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: too many sequences of this length", name);
  return QVGGT_OK;
}

// Tile map of rows [T][heads][D].
int rows_map(CUtensorMap* map, bool bf16, const void* base, int64_t D, int64_t heads, int64_t T, int64_t head, int64_t tok,
             uint32_t box_heads, uint32_t box_rows) {
  const uint64_t dims[3] = {(uint64_t)D, (uint64_t)heads, (uint64_t)T};
  const uint64_t strides[2] = {(uint64_t)(heads == 1 ? D : head) * 2, (uint64_t)(T == 1 ? heads * D : tok) * 2};
  const uint32_t box[3] = {64, box_heads, box_rows};
  return encode_tmap(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, base, dims,
                     strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace
}  // namespace qv

using namespace qv;

extern "C" int qvggt_prompt_attention_scratch(int64_t T, int32_t q_heads, int32_t kv_heads, int32_t sequences,
                                              int64_t max_len, int32_t head_dim, int64_t* bytes) {
  if (int rc = check_shape("prompt_attention_scratch", T, q_heads, kv_heads, sequences, max_len, head_dim)) return rc;
  if (!bytes) return set_error(QVGGT_ERR_INVALID, "prompt_attention_scratch: null pointer");
  max_len = std::min(max_len, T);
  *bytes = scratch_of(sequences * row_blocks_of(max_len, q_heads / kv_heads) * kv_heads, max_len, head_dim);
  return QVGGT_OK;
}

extern "C" int qvggt_prompt_attention(const qvggt_prompt_attention_args* p, void* stream) {
  const char* name = "prompt_attention";
  if (!p) return set_error(QVGGT_ERR_INVALID, "%s: null arguments", name);
  if (int rc = check_shape(name, p->T, p->q_heads, p->kv_heads, p->sequences, p->max_len, p->head_dim)) return rc;
  if (p->dtype != QVGGT_DTYPE_F16 && p->dtype != QVGGT_DTYPE_BF16)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: dtype must be fp16 or bf16", name);
  if (p->causal_chunk < 0) return set_error(QVGGT_ERR_INVALID, "%s: bad causal_chunk", name);
  if (!(p->scale > 1e-30) || p->scale > 1e30) return set_error(QVGGT_ERR_INVALID, "%s: scale must be positive", name);
  if (p->T == 0 || p->sequences == 0 || p->max_len == 0) return QVGGT_OK;
  if (!p->q || !p->k || !p->v || !p->out || !p->cu) return set_error(QVGGT_ERR_INVALID, "%s: null tensor", name);
  const int64_t T = p->T, D = p->head_dim, max_len = std::min(p->max_len, T);
  if (!aligned16(p->q) || !aligned16(p->k) || !aligned16(p->v) || !aligned16(p->out) ||
      ((T > 1 ? p->q_tok | p->k_tok | p->v_tok | p->o_tok : 0) | (p->q_heads > 1 ? p->q_head | p->o_head : 0) |
       (p->kv_heads > 1 ? p->k_head | p->v_head : 0)) % 8)
    return set_error(QVGGT_ERR_ALIGN, "%s: q, k, v and out rows must be 16-byte aligned", name);
  const auto positive = [&](int64_t tok, int64_t head, int64_t heads) {
    return (T == 1 || (tok > 0 && tok < 1LL << 38)) && (heads == 1 || (head > 0 && head < 1LL << 38));
  };
  if (!positive(p->q_tok, p->q_head, p->q_heads) || !positive(p->k_tok, p->k_head, p->kv_heads) ||
      !positive(p->v_tok, p->v_head, p->kv_heads) || !positive(p->o_tok, p->o_head, p->q_heads))
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: token and head strides must be positive and below 2^38", name);
  PromptArgs a{};
  a.v = static_cast<const uint16_t*>(p->v);
  a.out = static_cast<uint16_t*>(p->out);
  a.lse = p->lse;
  a.cu = p->cu;
  a.v_tok = p->v_tok;
  a.v_head = p->v_head;
  a.o_tok = p->o_tok;
  a.o_head = p->o_head;
  a.Tq = T;
  a.B = (int)p->sequences;
  a.hq = (int)p->q_heads;
  a.hk = (int)p->kv_heads;
  a.group = a.hq / a.hk;
  a.chunk = (int)std::min<int64_t>(p->causal_chunk, 1 << 30);
  a.max_len = (int)max_len;
  a.row_blocks = (int)row_blocks_of(max_len, a.group);
  a.scale_log2 = (float)(p->scale * 1.4426950408889634);
  a.ctl = make_ctl();
  // a try_wait that fails takes about 1.4 us
  a.wait_tries = (uint32_t)std::min<unsigned long long>(1u << 26, a.ctl.timeout_ns / 1024 + 1);
  const long long items = (long long)a.B * a.row_blocks * a.hk;
  const int64_t need = scratch_of(items, max_len, (int)D);
  if (need && (!p->scratch || p->scratch_bytes < need || !aligned16(p->scratch)))
    return set_error(QVGGT_ERR_INVALID, "%s: needs %lld bytes of 16-byte aligned scratch, got %lld", name, (long long)need,
                     (long long)p->scratch_bytes);
  const int kt = tile_keys(max_len);
  const int smem = D == 64 ? (kt == 64 ? Lay<64, 64>::TOTAL : Lay<64, 128>::TOTAL)
                           : (kt == 64 ? Lay<128, 64>::TOTAL : Lay<128, 128>::TOTAL);
  if (smem > device_info().max_smem_optin)
    return set_error(QVGGT_ERR_UNSUPPORTED, "%s: shared memory %d > %d", name, smem, device_info().max_smem_optin);
  const bool bf16 = p->dtype == QVGGT_DTYPE_BF16;
  CUtensorMap tmQ, tmK, tmV;
  if (int rc = rows_map(&tmQ, bf16, p->q, D, a.hq, T, p->q_head, p->q_tok, (uint32_t)a.group, (uint32_t)(128 / a.group)))
    return rc;
  if (int rc = rows_map(&tmK, bf16, p->k, D, a.hk, T, p->k_head, p->k_tok, 1, (uint32_t)kt)) return rc;
  if (int rc = rows_map(&tmV, bf16, p->v, D, a.hk, T, p->v_head, p->v_tok, 1, (uint32_t)kt)) return rc;
  const int grid = grid_of(items, max_len);
  a.can_split = need > 0;
  a.part_o = static_cast<float*>(p->scratch);
  a.part_lse = a.can_split ? a.part_o + 2LL * grid * Q_ROWS * D : nullptr;
  using Kfn = void (*)(CUtensorMap, CUtensorMap, CUtensorMap, PromptArgs);
  static const Kfn fns[2][2][2] = {
      {{prompt_attention_kernel<false, 64, 64>, prompt_attention_kernel<false, 64, 128>},
       {prompt_attention_kernel<false, 128, 64>, prompt_attention_kernel<false, 128, 128>}},
      {{prompt_attention_kernel<true, 64, 64>, prompt_attention_kernel<true, 64, 128>},
       {prompt_attention_kernel<true, 128, 64>, prompt_attention_kernel<true, 128, 128>}}};
  using Jfn = void (*)(PromptArgs, int);
  static const Jfn joins[2][2] = {{prompt_attention_join_kernel<false, 64>, prompt_attention_join_kernel<false, 128>},
                                  {prompt_attention_join_kernel<true, 64>, prompt_attention_join_kernel<true, 128>}};
  static DeviceFlags attr[2][2][2];
  const Kfn fn = fns[bf16][D == 128][kt == 128];
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int rc = ensure_smem(attr[bf16][D == 128][kt == 128], fn, smem, "cudaFuncSetAttribute(prompt_attention)")) return rc;
  if (int rc = check_cuda(launch_pdl(fn, dim3((unsigned)grid), dim3(THREADS), smem, st, 1u, tmQ, tmK, tmV, a),
                          "prompt_attention launch"))
    return rc;
  count_launch(1);
  if (a.can_split) {
    if (int rc = check_cuda(launch_pdl(joins[bf16][D == 128], dim3((unsigned)(grid - 1), (unsigned)(Q_ROWS * D / 1024)), dim3(256), 0,
                                       st, 1u, a, grid),
                            "prompt_attention join launch"))
      return rc;
    count_launch(1);
  }
  return QVGGT_OK;
}
