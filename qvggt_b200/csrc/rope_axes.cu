// Rotary positions with several axes (time, height, width): q and k rotated in
// one pass, positions and frequencies given.
//
// Pair j of a head (j < R/2) is rotated by the angle t_j = pos[axis_j] * f_j:
//   y[lo] = x[lo] cos t - x[hi] sin t,   y[hi] = x[hi] cos t + x[lo] sin t
// (the inverse, which is also the gradient, turns by -t); dims >= R pass
// through.  A token's angles are shared by all its heads, so a CTA first
// computes the sines and cosines of its tokens into shared memory and then
// streams the heads through registers: 2 bytes in and 2 out per element, HBM
// bound.
#include "host.hpp"

namespace qv {
namespace {

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_MAX_PAIRS = 128;     // head_dim <= 256
constexpr int ROPE_MAX_TOK = 8;         // tokens of one CTA
constexpr int ROPE_AXES = 4;

enum RopeLayout : int32_t { ROPE_AXIAL = 0, ROPE_SPLIT = 1, ROPE_INTERLEAVED = 2 };

struct RopeSide {                        // q or k: element strides of tokens and heads
  const uint16_t* in;
  uint16_t* out;
  long long in_ts, in_hs, out_ts, out_hs;
  int heads;
};

struct RopeArgs {
  RopeSide s[2];
  const int32_t* pos;                    // [axes][T], row stride pos_stride
  const float* inv_freq;                 // [pairs]
  long long pos_stride, T;
  int D, pairs, tok, layout;
  int sect_end[ROPE_AXES];               // pair index one past each axis' last (unused axes: pairs)
  float sign;
};

template <int V>
struct VecBits;
template <> struct VecBits<8> { using T = uint4; };
template <> struct VecBits<4> { using T = uint2; };
template <> struct VecBits<2> { using T = uint32_t; };
template <> struct VecBits<1> { using T = uint16_t; };

template <bool BF16>
__device__ __forceinline__ float to_f32(uint16_t u) {
  if (BF16) return __uint_as_float((uint32_t)u << 16);
  return __half2float(__ushort_as_half(u));
}
template <bool BF16>
__device__ __forceinline__ uint16_t from_f32(float x) {
  if (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(x));
  return __half_as_ushort(__float2half_rn(x));
}

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t u) {
  return BF16 ? unpack_bf162(u) : unpack_half2(u);
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  return BF16 ? pack_bf162(x, y) : pack_half2(x, y);
}

// V pairs per item: two V-element vectors in, two out.
template <bool BF16, int V>
__global__ void __launch_bounds__(ROPE_THREADS, 8) rope_axes_kernel(RopeArgs a) {
  using Vec = typename VecBits<V>::T;
  union Pack {
    Vec v;
    uint16_t e[V];
    uint32_t w[(V + 1) / 2];
  };
  // [tok][pairs] cosines, then sines: apart, so that the 16-byte reads of a
  // warp's items lie 32 bytes apart, not 64 (half the bank conflicts)
  extern __shared__ __align__(16) float cosines[];
  float* sines = cosines + a.tok * a.pairs;
  pdl_wait();
  pdl_trigger();
  const long long t0 = (long long)blockIdx.x * a.tok;
  const int nt = (int)min((long long)a.tok, a.T - t0);
  // The angle is reduced modulo 2 pi in double: a float product of a large
  // position and its frequency would already be off by the angle's ulp.
  for (int i = threadIdx.x; i < nt * a.pairs; i += ROPE_THREADS) {
    const int tt = i / a.pairs, j = i - tt * a.pairs;
    int ax = 0;
#pragma unroll
    for (int x = 0; x < ROPE_AXES - 1; ++x) ax += j >= a.sect_end[x];
    const double t = (double)a.pos[ax * a.pos_stride + t0 + tt] * (double)a.inv_freq[j];
    const double r = t - rint(t * 0.15915494309189533577) * 6.28318530717958647693;
    float sn, cn;
    sincosf((float)r, &sn, &cn);
    cosines[i] = cn;
    sines[i] = sn * a.sign;
  }
  __syncthreads();
  const int rot = a.pairs / V;                            // rotation items of a head
  const int copy = (a.D - 2 * a.pairs) / V;               // pass-through items
  const int per_head = rot + copy;
  const int heads = a.s[0].heads + a.s[1].heads;
  const int per_tok = heads * per_head;
  // a thread's items are ROPE_THREADS apart: token, head and item advance by
  // fixed amounts with carries, so nothing is divided in the loop
  const int d_tok = ROPE_THREADS / per_tok, d_rem = ROPE_THREADS - d_tok * per_tok;
  const int d_head = d_rem / per_head, d_item = d_rem - d_head * per_head;
  int tt = threadIdx.x / per_tok, hh = (threadIdx.x - tt * per_tok) / per_head;
  int item = threadIdx.x - tt * per_tok - hh * per_head;
  auto advance = [&] {
    item += d_item;
    hh += d_head;
    tt += d_tok;
    if (item >= per_head) {
      item -= per_head;
      ++hh;
    }
    if (hh >= heads) {
      hh -= heads;
      ++tt;
    }
  };
  for (; tt < nt; advance()) {
    const bool side = hh >= a.s[0].heads;
    const int h = side ? hh - a.s[0].heads : hh;
    const uint16_t* in = side ? a.s[1].in + (t0 + tt) * a.s[1].in_ts + h * a.s[1].in_hs
                              : a.s[0].in + (t0 + tt) * a.s[0].in_ts + h * a.s[0].in_hs;
    uint16_t* out = side ? a.s[1].out + (t0 + tt) * a.s[1].out_ts + h * a.s[1].out_hs
                         : a.s[0].out + (t0 + tt) * a.s[0].out_ts + h * a.s[0].out_hs;
    if (item >= rot) {
      const int d = 2 * a.pairs + (item - rot) * V;
      *reinterpret_cast<Vec*>(out + d) = *reinterpret_cast<const Vec*>(in + d);
      continue;
    }
    const int j = item * V;
    int lo, hi;
    if (a.layout == ROPE_SPLIT) {
      lo = j;
      hi = j + a.pairs;
    } else if (a.layout == ROPE_INTERLEAVED) {
      lo = 2 * j;
      hi = lo + V;
    } else {
      int base = 0, end = a.sect_end[0];
#pragma unroll
      for (int x = 0; x < ROPE_AXES - 1; ++x)
        if (j >= a.sect_end[x]) {
          base = a.sect_end[x];
          end = a.sect_end[x + 1];
        }
      lo = base + j;
      hi = lo + (end - base);
    }
    Pack x, y;
    x.v = *reinterpret_cast<const Vec*>(in + lo);
    y.v = *reinterpret_cast<const Vec*>(in + hi);
    const float* c = cosines + tt * a.pairs + j;
    const float* s = sines + tt * a.pairs + j;
    if constexpr (V == 1) {
      const float p = to_f32<BF16>(x.e[0]), q = to_f32<BF16>(y.e[0]);
      x.e[0] = from_f32<BF16>(p * c[0] - q * s[0]);
      y.e[0] = from_f32<BF16>(q * c[0] + p * s[0]);
    } else if (a.layout == ROPE_INTERLEAVED) {
      // each word of the 2V consecutive elements (x | y) is a pair
#pragma unroll
      for (int e = 0; e < V / 2; ++e) {
        const float2 u = unpack2<BF16>(x.w[e]), w = unpack2<BF16>(y.w[e]);
        const float c0 = c[e], s0 = s[e], c1 = c[V / 2 + e], s1 = s[V / 2 + e];
        x.w[e] = pack2<BF16>(u.x * c0 - u.y * s0, u.y * c0 + u.x * s0);
        y.w[e] = pack2<BF16>(w.x * c1 - w.y * s1, w.y * c1 + w.x * s1);
      }
    } else {
      // two pairs to a word of x and y
#pragma unroll
      for (int e = 0; e < V / 2; ++e) {
        const float2 p = unpack2<BF16>(x.w[e]), q = unpack2<BF16>(y.w[e]);
        const float2 cc = *reinterpret_cast<const float2*>(c + 2 * e), ss = *reinterpret_cast<const float2*>(s + 2 * e);
        x.w[e] = pack2<BF16>(p.x * cc.x - q.x * ss.x, p.y * cc.y - q.y * ss.y);
        y.w[e] = pack2<BF16>(q.x * cc.x + p.x * ss.x, q.y * cc.y + p.y * ss.y);
      }
    }
    *reinterpret_cast<Vec*>(out + lo) = x.v;
    *reinterpret_cast<Vec*>(out + hi) = y.v;
  }
}

}  // namespace
}  // namespace qv

using namespace qv;

extern "C" int qvggt_rope_axes(const qvggt_rope_axes_args* p, void* stream) {
  if (!p) return set_error(QVGGT_ERR_INVALID, "rope_axes: null arguments");
  if (p->T < 0 || p->q_heads < 0 || p->k_heads < 0 || p->q_heads + p->k_heads == 0 || p->q_heads > 65535 ||
      p->k_heads > 65535)
    return set_error(QVGGT_ERR_INVALID, "rope_axes: bad shape");
  if (p->dtype != QVGGT_DTYPE_F16 && p->dtype != QVGGT_DTYPE_BF16)
    return set_error(QVGGT_ERR_UNSUPPORTED, "rope_axes: dtype must be fp16 or bf16");
  if (p->layout < 0 || p->layout > 2) return set_error(QVGGT_ERR_INVALID, "rope_axes: layout must be 0, 1 or 2");
  if (p->n_axes < 1 || p->n_axes > ROPE_AXES)
    return set_error(QVGGT_ERR_INVALID, "rope_axes: 1 to %d axes", ROPE_AXES);
  const int n_axes = (int)p->n_axes, layout = (int)p->layout;
  const int64_t T = p->T, head_dim = p->head_dim, *sections = p->sections;
  RopeArgs a{};
  int pairs = 0;
  for (int x = 0; x < n_axes; ++x) {
    if (sections[x] <= 0) return set_error(QVGGT_ERR_INVALID, "rope_axes: section sizes must be positive");
    pairs += sections[x] > ROPE_MAX_PAIRS ? ROPE_MAX_PAIRS + 1 : (int)sections[x];
    a.sect_end[x] = pairs;
  }
  for (int x = n_axes; x < ROPE_AXES; ++x) a.sect_end[x] = pairs;
  if (pairs > ROPE_MAX_PAIRS || head_dim > 2 * ROPE_MAX_PAIRS)
    return set_error(QVGGT_ERR_UNSUPPORTED, "rope_axes: head_dim up to %d", 2 * ROPE_MAX_PAIRS);
  if (2 * pairs > head_dim)
    return set_error(QVGGT_ERR_INVALID, "rope_axes: %d rotated pairs do not fit head_dim %d", pairs, (int)head_dim);
  if (T == 0) return QVGGT_OK;
  if (!p->positions || !p->inv_freq || (p->q_heads && (!p->q || !p->q_out)) || (p->k_heads && (!p->k || !p->k_out)))
    return set_error(QVGGT_ERR_INVALID, "rope_axes: null tensor");
  a.s[0] = {static_cast<const uint16_t*>(p->q), static_cast<uint16_t*>(p->q_out), p->q_tok, p->q_head, p->qo_tok,
            p->qo_head, (int)p->q_heads};
  a.s[1] = {static_cast<const uint16_t*>(p->k), static_cast<uint16_t*>(p->k_out), p->k_tok, p->k_head, p->ko_tok,
            p->ko_head, (int)p->k_heads};
  a.pos = p->positions;
  a.inv_freq = p->inv_freq;
  a.pos_stride = p->pos_stride;
  a.T = T;
  a.D = (int)head_dim;
  a.pairs = pairs;
  a.layout = layout;
  a.sign = p->inverse ? -1.f : 1.f;
  // Widest vector that divides every run of pairs, the pass-through tail, the
  // strides and the addresses.
  long long align = 8;
  auto limit = [&](long long v) {
    while (v % align) align /= 2;
  };
  if (layout == ROPE_AXIAL)
    for (int x = 0; x < n_axes; ++x) limit(sections[x]);
  limit(pairs);
  limit(head_dim - 2 * pairs);
  for (const RopeSide& s : a.s) {
    if (!s.heads) continue;
    const long long strides[4] = {s.in_ts, s.in_hs, s.out_ts, s.out_hs};
    for (long long v : strides) limit(v < 0 ? -v : v);
    if ((reinterpret_cast<uintptr_t>(s.in) | reinterpret_cast<uintptr_t>(s.out)) & 1)
      return set_error(QVGGT_ERR_ALIGN, "rope_axes: tensors must be aligned to their element");
    limit((long long)(reinterpret_cast<uintptr_t>(s.in) / 2 % 8));
    limit((long long)(reinterpret_cast<uintptr_t>(s.out) / 2 % 8));
  }
  // Tokens per CTA: few enough that every SM has several CTAs, up to 8 so that
  // the per-CTA start-up is paid for several rows (16: 94 us against 80 at
  // 20,000 tokens x 32 heads x 128, as the angles' phase then stands alone).
  const long long want = 4LL * device_info().num_sms;
  a.tok = 1;
  while (a.tok < ROPE_MAX_TOK && T / (2 * a.tok) >= want) a.tok *= 2;
  const long long grid = (T + a.tok - 1) / a.tok;
  if (grid > 2147483647LL) return set_error(QVGGT_ERR_UNSUPPORTED, "rope_axes: too many tokens");
  using Kfn = void (*)(RopeArgs);
  static const Kfn fns[2][4] = {
      {rope_axes_kernel<false, 1>, rope_axes_kernel<false, 2>, rope_axes_kernel<false, 4>, rope_axes_kernel<false, 8>},
      {rope_axes_kernel<true, 1>, rope_axes_kernel<true, 2>, rope_axes_kernel<true, 4>, rope_axes_kernel<true, 8>}};
  const int vi = align == 8 ? 3 : align == 4 ? 2 : align == 2 ? 1 : 0;
  int rc = check_cuda(launch_pdl(fns[p->dtype == QVGGT_DTYPE_BF16][vi], dim3((unsigned)grid), dim3(ROPE_THREADS),
                                 (size_t)a.tok * pairs * 2 * sizeof(float), static_cast<cudaStream_t>(stream), 1u, a),
                      "rope_axes launch");
  if (!rc) count_launch(1);
  return rc;
}
