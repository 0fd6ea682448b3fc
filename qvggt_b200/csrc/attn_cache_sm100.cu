// Attention over the paged 8-bit K/V cache, many query rows: tcgen05 + TMEM.
//
// The mathematics is attn_cache.cuh's: the codes are the products' operands
// and both scales live in the softmax, per 32 keys (never across two blocks)
//   x = ck S + lv,  ck = scale log2e ks_B, lv = log2 vs_B,  P = 2^(x - m),
//   O += P c_v,  l += (1 / vs_B) sum P,  out = O / l.
// One CTA per (request, kv head, two 128-row Q tiles, split of the keys); a
// row is a (token, query head of the group) pair, so the heads that share K/V
// share its tiles.  Per key tile of KT keys (128 for head_dim 64, 64 for 128):
//   warp 0         block ids and scales, cp.async.bulk of the raw codes (RAW
//                  stages of 16 KB), constants of the tile into a small ring
//   warps 4..7     codes -> fp16 (bf16 for K with bf16 queries) into the
//                  128-byte-swizzled operand tiles (two stages each of K, V)
//   warp 1         S_i = Q_i K^T        warp 3   O_i += P_i V
//   warps 8..15    softmax, one thread per row of Q tile i = 0, 1
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
  // q_full, raw_full[RAW], raw_empty[RAW], c_full[CRING], k_full[KV], k_empty[KV], v_full[KV], v_empty[KV],
  // s_full[2], s_free[2], p_full[2], o_done[2], drain, drain2
  static constexpr int NUM_BARS = 1 + 2 * RAW + CRING + 4 * KV + 8 + 2;
  static constexpr int MISC = BAR + NUM_BARS * 8;          // TMEM base, abort flag, status pointer, timeout
  static constexpr int TOTAL = MISC + 32 + 1024;
};

// cp.async.bulk of contiguous bytes, completion on an mbarrier of this CTA.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// K-major or MN-major operand with 128-byte swizzle; lead: bytes between the
// 64-element panels of an MN-major operand (unused by K-major ones).
__device__ __forceinline__ uint64_t sdesc_panels(uint32_t saddr, uint32_t lead) {
  return (sdesc_sw128(saddr) & ~(0x3fffull << 16)) | ((uint64_t)(lead >> 4) << 16);
}

// Max over the 32 scores of a chunk, of the first `valid` with PARTIAL.
template <bool PARTIAL, int E0, int N>
__device__ __forceinline__ float chunk_max(const uint32_t (&s)[N], int valid) {
  float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
  for (int e = E0; e < E0 + 32; e += 4) {
    if (!PARTIAL) {
      m0 = max3f(m0, __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
      m1 = max3f(m1, __uint_as_float(s[e + 2]), __uint_as_float(s[e + 3]));
    } else {
      if (e + 0 < valid) m0 = fmaxf(m0, __uint_as_float(s[e + 0]));
      if (e + 1 < valid) m1 = fmaxf(m1, __uint_as_float(s[e + 1]));
      if (e + 2 < valid) m0 = fmaxf(m0, __uint_as_float(s[e + 2]));
      if (e + 3 < valid) m1 = fmaxf(m1, __uint_as_float(s[e + 3]));
    }
  }
  return fmaxf(m0, m1);
}

__device__ __forceinline__ float4 lds_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// P of chunk E0 / 16 (pairs E0..E0+15) as fp16 pairs into s[E0..), its sum
// over 1 / vs into l.  POLY of 8 pairs take the FMA-pipe exponential.
template <bool PARTIAL, int POLY, int E0, int N>
__device__ __forceinline__ void exp_chunk(uint32_t (&s)[N], const float4& k, float neg_m, float& l, int valid) {
  const uint64_t c2 = f2_pack(k.x, k.x), nm2 = f2_pack(k.y + neg_m, k.y + neg_m);
  uint64_t la = f2_pack(0.f, 0.f), lb = f2_pack(0.f, 0.f);
#pragma unroll
  for (int e = E0; e < E0 + 16; ++e) {
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
    if (PARTIAL) {
      if (2 * e >= valid) p0 = 0.f;
      if (2 * e + 1 >= valid) p1 = 0.f;
    }
    if (e & 1) lb = f2_add(lb, f2_pack(p0, p1));
    else la = f2_add(la, f2_pack(p0, p1));
    s[e] = pack_half2(p0, p1);
  }
  float l0, l1;
  f2_unpack(f2_add(la, lb), l0, l1);
  const float sum = l0 + l1;
  if (!PARTIAL || sum != 0.f) l += sum * k.z;   // a row that sees none of the keys takes nothing from their scale
}

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
  uint64_t* raw_full = q_full + 1;
  uint64_t* raw_empty = raw_full + RAW;
  uint64_t* c_full = raw_empty + RAW;
  uint64_t* k_full = c_full + CRING;
  uint64_t* k_empty = k_full + KV;
  uint64_t* v_full = k_empty + KV;
  uint64_t* v_empty = v_full + KV;
  // the softmax warps address the next four [2] arrays from s_full[i] at byte offsets 16, 32, 48
  uint64_t* s_full = v_empty + KV;
  uint64_t* s_free = s_full + 2;
  uint64_t* p_full = s_free + 2;
  uint64_t* o_done = p_full + 2;
  uint64_t* drain = o_done + 2;
  uint64_t* drain2 = drain + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC);
  const uint32_t misc = sbase + L::MISC;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < RAW; ++s) {
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_empty[s], 4);
    }
    for (int s = 0; s < CRING; ++s) mbar_init(&c_full[s], 1);
    for (int s = 0; s < KV; ++s) {
      mbar_init(&k_full[s], 4);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 4);
      mbar_init(&v_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(drain, 1);
    mbar_init(drain2, 1);
    *reinterpret_cast<int*>(smem + L::MISC + 4) = 0;
    *reinterpret_cast<uint32_t**>(smem + L::MISC + 8) = a.ctl.status;
    *reinterpret_cast<unsigned long long*>(smem + L::MISC + 16) = a.ctl.timeout_ns;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) tma_prefetch_desc(&tmQ);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  pdl_trigger();
  const uint32_t tmem = *tmem_slot;

  // The item.  Blocks of later tokens first: under a causal mask they see the
  // most keys, and the longest CTAs should not start last.
  const int sp = blockIdx.x % a.splits;
  const int bh = (blockIdx.x / a.splits) % (a.B * a.hk);
  const int qb = a.row_blocks - 1 - blockIdx.x / (a.splits * a.B * a.hk);
  const int b = bh / a.hk, kvh = bh % a.hk;
  const int q0 = a.cu_q[b], ql = a.cu_q[b + 1] - q0, n = a.kv_lens[b];
  const int tpt = 128 / a.group;                           // tokens of a Q tile
  const int tok0 = qb * 2 * tpt;
  bool live = tok0 < ql;
  if (q0 < 0 || ql < 0 || ql > a.max_q || (long long)q0 + ql > a.Tq || n < 0 || n > (a.wide << a.bs_log2)) {
    if (threadIdx.x == 0) report_status(a.ctl, ST_BAD_LENGTH);
    live = false;
  }
  const int nqt = tok0 + tpt < ql ? 2 : 1;                 // Q tiles that hold rows
  int t0 = 0, nt = 0;                                      // key tiles of this CTA
  if (live) {
    const int lim = key_limit(min(ql, tok0 + 2 * tpt) - 1, ql, n, a.chunk);
    const int tiles = (lim + KT - 1) / KT;
    t0 = (int)((long long)sp * tiles / a.splits);
    nt = (int)((long long)(sp + 1) * tiles / a.splits) - t0;
  }

  // Registers: launched at 128 each; 128 (48 + 80 + 2 * 192) = 128 * 512.
  // Every warp of a warpgroup runs the same setmaxnreg.
  if (warp < 4) {
    regs_dec<48>();
    if (warp == 0 && nt > 0) {
      // ---------------------------------------------------------- producer
      if (lane == 0) {
        const int rows = tpt * a.group;
        mbar_arrive_expect_tx(q_full, nqt * L::PANELS * rows * 128);
        for (int i = 0; i < nqt; ++i)
          for (int p = 0; p < L::PANELS; ++p)
            tma_load_3d(smem + L::Q + (i * L::PANELS + p) * L::Q_PANEL, &tmQ, q_full, p * 64, kvh * a.group,
                        q0 + tok0 + i * tpt);
      }
      const int bs = 1 << a.bs_log2;
      const int piece = min(bs, KT);                       // keys of one copy
      const int pieces = KT / piece;
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
      bool bad = false, ok = true;
      int j = 0;
      for (; j < nt; ++j) {
        const int key0 = (t0 + j) * KT;
        if (((key0 + KT - 1) >> a.bs_log2) >= base + 32) {
          // blocks and tiles nest, so a tile starts on the batch's boundary
          base += 32;
          id = id2;
          fetch_scales(id, ks, vs);
          id2 = fetch_id(base + 32 + lane);
        }
        // constants of the tile's 32-key chunks
        const int cj = min(((key0 + 32 * lane) >> a.bs_log2) - base, 31);
        const int cid = __shfl_sync(~0u, id, cj);
        const float cks = __shfl_sync(~0u, ks, cj), cvs = __shfl_sync(~0u, vs, cj);
        // the copy of lane's piece
        const int pkey = key0 + lane * piece;
        const int pid = __shfl_sync(~0u, id, min((pkey >> a.bs_log2) - base, 31));
        const bool mine = lane < pieces && pkey < n;
        const bool good = mine && pid >= 0 && pid < a.num_blocks;
        bad |= mine && !good;
        const int st = j % RAW;
        ok = __all_sync(~0u, wait(&raw_empty[st], ((j / RAW) & 1) ^ 1, misc, ST_TIMEOUT_TMA_EMPTY));
        if (!ok) break;
        if (lane < CH) {
          const bool have = cid >= 0 && cid < a.num_blocks && key0 + 32 * lane < n;
          // a skipped block: every score -inf
          const float4 k = have ? make_float4(cks * a.scale_log2, log2f(cvs), 1.f / cvs, 0.f)
                                : make_float4(0.f, -INFINITY, 0.f, 0.f);
          reinterpret_cast<float4*>(smem + L::CONST)[(j % CRING) * CH + lane] = k;
        }
        const uint32_t count = __popc(__ballot_sync(~0u, good));
        if (lane == 0) {
          mbar_arrive(&c_full[j % CRING]);
          mbar_arrive_expect_tx(&raw_full[st], count * 2 * piece * D);
        }
        __syncwarp();
        if (good) {
          const long long off = pid * a.block_stride + ((long long)kvh * bs + (pkey & (bs - 1))) * D;
          const uint32_t at = st * RAW_BYTES + lane * piece * D, bar = smem_u32(&raw_full[st]);
          bulk_load(sbase + L::RK + at, a.kc + off, piece * D, bar);
          bulk_load(sbase + L::RV + at, a.vc + off, piece * D, bar);
        }
      }
      if (bad) report_bad_block(a.ctl);
      if (!ok && lane == 0) {
        // aborted: let the copies in flight land before the CTA exits
        mbar_wait_drain(q_full, 0, 200000000ull);
        for (int jj = max(0, j - RAW); jj < j; ++jj)
          mbar_wait_drain(&raw_full[jj % RAW], (jj / RAW) & 1, 200000000ull);
      }
    } else if (warp == 1 && nt > 0) {
      // ---------------------------------------------------------- S = Q K^T
      if (lane == 0) {
        constexpr uint32_t idesc = idesc_f16(128, KT, false, false, BF16);
        bool ok = wait(q_full, 0, misc, ST_TIMEOUT_FULL);
        for (int j = 0; ok && j < nt; ++j) {
          const int st = j % KV;
          if (!wait(&k_full[st], (j / KV) & 1, misc, ST_TIMEOUT_DEQ)) { ok = false; break; }
          for (int i = 0; i < nqt; ++i) {
            if (j > 0 && !wait(&s_free[i], (j - 1) & 1, misc, ST_TIMEOUT_SOFTMAX)) { ok = false; break; }
            tc_fence_after();
#pragma unroll
            for (int p = 0; p < L::PANELS; ++p)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                mma_f16_ss(tmem + COL_S + i * KT,
                           sdesc_sw128(sbase + L::Q + (i * L::PANELS + p) * L::Q_PANEL + k * 32),
                           sdesc_sw128(sbase + L::K + st * OP_BYTES + p * KT * 128 + k * 32), idesc,
                           (p | k) ? 1u : 0u);
            tc_commit(&s_full[i]);
          }
          if (!ok) break;
          tc_commit(&k_empty[st]);
        }
        if (!ok) {
          tc_commit(drain);
          mbar_wait_drain(drain, 0, 200000000ull);
        }
      }
    } else if (warp == 3 && nt > 0) {
      // ---------------------------------------------------------- O += P V
      if (lane == 0) {
        constexpr uint32_t idesc = idesc_f16(128, D, false, true);
        bool ok = true;
        for (int j = 0; ok && j < nt; ++j) {
          const int st = j % KV;
          for (int i = 0; i < nqt; ++i) {
            if (!wait(&p_full[i], j & 1, misc, ST_TIMEOUT_SOFTMAX)) { ok = false; break; }
            if (i == 0 && !wait(&v_full[st], (j / KV) & 1, misc, ST_TIMEOUT_DEQ)) { ok = false; break; }
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < KT / 16; ++k)
              mma_f16_ts(tmem + COL_O + i * D, tmem + COL_P + i * (KT / 2) + k * 8,
                         sdesc_panels(sbase + L::V + st * OP_BYTES + k * 2048, KT * 128), idesc,
                         (j > 0 || k > 0) ? 1u : 0u);
            tc_commit(&o_done[i]);
          }
          if (!ok) break;
          tc_commit(&v_empty[st]);
        }
        if (!ok) {
          tc_commit(drain2);
          mbar_wait_drain(drain2, 0, 200000000ull);
        }
      }
    }
  } else if (warp < 8) {
    // ------------------------------------------------------------ codes -> fp16 / bf16
    regs_dec<80>();
    const int th = threadIdx.x - 128;                      // 0..127
    constexpr int PARTS = D / 16;                          // 16-code pieces of a row
    constexpr int IT = KT * PARTS / 128;                   // pieces per thread
    const int part = th % PARTS, row0 = th / PARTS, panel = part / 4;
    bool ok = nt > 0;
    for (int j = 0; ok && j < nt; ++j) {
      const int rs = j % RAW, st = j % KV;
      if (!__all_sync(~0u, wait(&raw_full[rs], (j / RAW) & 1, misc, ST_TIMEOUT_FULL))) { ok = false; break; }
#pragma unroll
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
        if (!__all_sync(~0u, wait(empty, ((j / KV) & 1) ^ 1, misc, ST_TIMEOUT_DEQ))) { ok = false; break; }
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
  } else {
    // ------------------------------------------------------------ softmax of Q tile i
    regs_inc<192>();
    const int i = (warp - 8) / 4;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem + lane_base + COL_S + i * KT;
    const uint32_t tP = tmem + lane_base + COL_P + i * (KT / 2);
    const uint32_t tO = tmem + lane_base + COL_O + i * D;
    const uint32_t bar_s_full = smem_u32(&s_full[i]);
    const uint32_t bar_s_free = bar_s_full + 16, bar_p_full = bar_s_full + 32, bar_o_done = bar_s_full + 48;
    const uint32_t consts = sbase + L::CONST;
    const int tok = tok0 + i * tpt + r / a.group;          // within the request
    const bool row_ok = live && r < tpt * a.group && tok < ql;
    // rows past the end compute on whatever their tile holds and are not stored
    const int lim = row_ok ? key_limit(tok, ql, n, a.chunk) : n;
    float m_used = -INFINITY, l = 0.f;
    bool ok = live;
    const int ntr = (live && i < nqt) ? nt : 0;
    for (int j = 0; j < ntr; ++j) {
      if (!softmax_wait(bar_s_full, j & 1, misc)) { ok = false; break; }
      if (!softmax_wait(smem_u32(&c_full[j % CRING]), (j / CRING) & 1, misc)) { ok = false; break; }
      tc_fence_after();
      uint32_t s[KT];
#pragma unroll
      for (int c = 0; c < CH; ++c) tmem_ld32(tS + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&s[32 * c]));
      tmem_ld_wait();
      reg_fence<0, KT>(s);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive(bar_s_free);
      const uint32_t cb = consts + (j % CRING) * (CH * 16);
      const int valid = lim - (t0 + j) * KT;               // keys of the tile that the row sees (may be <= 0)
      const bool full = __all_sync(~0u, valid >= KT);
      float mx = m_used;
#define QV_MAX(C)                                                                                            \
  if (C < CH) {                                                                                              \
    const float4 k = lds_f4(cb + 16 * C);                                                                    \
    const float v = full ? chunk_max<false, 32 * (C % CH)>(s, valid) : chunk_max<true, 32 * (C % CH)>(s, valid); \
    mx = fmaxf(mx, fmaf(v, k.x, k.y));                                                                       \
  }
      QV_MAX(0) QV_MAX(1) QV_MAX(2) QV_MAX(3)
#undef QV_MAX
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
      bool stored = true;
      // P_i may be written once PV_i(j-1) has read the one before
#define QV_EXP(C)                                                                                \
  if (C < CH) {                                                                                  \
    const float4 k = lds_f4(cb + 16 * C);                                                        \
    if (full) exp_chunk<false, 1, 16 * (C % CH)>(s, k, neg_m, lj, valid);                        \
    else exp_chunk<true, 1, 16 * (C % CH)>(s, k, neg_m, lj, valid);                              \
    if (C == 0 && j > 0) {                                                                       \
      stored = softmax_wait(bar_o_done, (j - 1) & 1, misc);                                      \
      tc_fence_after();                                                                          \
    }                                                                                            \
    if (stored) tmem_st16(tP + 16 * C, *reinterpret_cast<const uint32_t(*)[16]>(&s[16 * (C % CH)])); \
  }
      QV_EXP(0) QV_EXP(1) QV_EXP(2) QV_EXP(3)
#undef QV_EXP
      if (!stored) { ok = false; break; }
      tmem_st_wait();
      l = l * alpha + lj;
      if (rescale) {
#pragma unroll 1
        for (int cc = 0; cc < D / 16; ++cc) {
          uint32_t v[16];
          tmem_ld16(tO + cc * 16, v);
          tmem_ld_wait();
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
    // ------------------------------------------------------------ epilogue
    if (ok && ntr > 0) {
      ok = softmax_wait(bar_o_done, (ntr - 1) & 1, misc);
      tc_fence_after();
    }
    if (ok) {                                              // warp-uniform
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const float lse2 = l == 0.f ? -INFINITY : m_used + log2f(l);
      const long long gtok = q0 + tok;
      const int h = kvh * a.group + r % a.group;
      const long long part = (long long)sp * a.Tq * a.hq + gtok * a.hq + h;
#pragma unroll 1
      for (int cc = 0; cc < D / 16; ++cc) {
        uint32_t v[16];
        if (ntr > 0) {
          tmem_ld16(tO + cc * 16, v);
          tmem_ld_wait();
          reg_fence<0, 16>(v);
        }
        if (!row_ok) continue;
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = l == 0.f ? 0u : __float_as_uint(__uint_as_float(v[e]) * inv);
        if (a.splits > 1) {
          float4* dst = reinterpret_cast<float4*>(a.part_o + part * D + cc * 16);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            dst[e] = make_float4(__uint_as_float(v[4 * e]), __uint_as_float(v[4 * e + 1]),
                                 __uint_as_float(v[4 * e + 2]), __uint_as_float(v[4 * e + 3]));
        } else {
          uint32_t o[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x = __uint_as_float(v[2 * e]), y = __uint_as_float(v[2 * e + 1]);
            o[e] = BF16 ? pack_bf162(x, y) : pack_half2(x, y);
          }
          uint4* dst = reinterpret_cast<uint4*>(a.out + gtok * a.o_tok + h * a.o_head + cc * 16);
          dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
          dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
        }
      }
      if (row_ok) {
        if (a.splits > 1) a.part_lse[part] = lse2;
        else if (a.lse) a.lse[h * a.Tq + gtok] = lse2 * 0.6931471805599453f;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

}  // namespace

bool tiles_can_read(const CacheAttnArgs& a) {
  return a.group <= 128 && (a.hq == 1 || a.q_head > 0) && (a.Tq == 1 || a.q_tok > 0);
}

int launch_tiles(const CacheAttnArgs& a, int D, bool bf16, cudaStream_t stream) {
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
  using Kfn = void (*)(CUtensorMap, CacheAttnArgs);
  static const Kfn fns[2][2] = {{attn_cache_tiles_kernel<false, 64>, attn_cache_tiles_kernel<false, 128>},
                                {attn_cache_tiles_kernel<true, 64>, attn_cache_tiles_kernel<true, 128>}};
  static DeviceFlags attr[2][2];
  const Kfn fn = fns[bf16][D == 128];
  if (int rc = ensure_smem(attr[bf16][D == 128], fn, smem, "cudaFuncSetAttribute(cached_attention)")) return rc;
  const long long grid = (long long)a.row_blocks * a.B * a.hk * a.splits;
  if (grid > 2147483647LL) return set_error(QVGGT_ERR_UNSUPPORTED, "cached_attention: grid too large");
  return check_cuda(launch_pdl(fn, dim3((unsigned)grid), dim3(THREADS), smem, stream, 1u, tmQ, a),
                    "cached_attention launch");
}

}  // namespace qv
