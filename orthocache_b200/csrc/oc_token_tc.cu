// Token-level attention on the 5th-generation tensor cores (bfloat16, head_dim
// 64, 128 or 256): drafted trees and query chunks with enough rows per KV head to
// fill 128-row tiles.
//
// Mathematics and masks: oc_token.cuh.  Per row and key 4 D multiply-adds and one
// exponential (with a cap, a polynomial more); per 128-row tile and key 4 D bytes
// of keys and values.  At D = 128 the products of two row tiles and a key tile
// take 2,048 cycles and their exponentials as many on the MUFU unit; a pair takes
// about 3,200.  Measured: 4 x 2048 rows x 32 heads on 8K keys without a mask 0.92
// ms = 1,200 TFLOP/s (0.72 of the measured bf16 burst peak), causal on 32K 1,160,
// capped 925-1,000; D = 64 690; D = 256 705; few rows on a long cache read it at 5
// to 5.4 TB/s.
//
// Layout (one persistent CTA of 384 threads per SM):
//   * a row tile is 128 rows of one KV head: Gp neighbouring heads (the largest
//     power of two that divides G = Hq / Hkv) x 128 / Gp query positions, so
//     that few drafted tokens of many heads still fill a tile; a work unit is two
//     row tiles that share every key tile (at D = 256, where O alone takes 256
//     columns of tensor memory, one), over all keys that its rows may see or a run
//     of them.  When there is one row tile in all (dual), both halves of the CTA
//     work on it, on the even and the odd key tiles, as if on two tiles;
//   * warp 8 loads by TMA (128-byte swizzle): the query tiles, then K and V tiles
//     of 128 tokens into a ring; from the cache, its pages, or the drafted
//     tokens.  The key tiles come nearest first;
//   * warp 9 issues the tcgen05.mma: per key tile j and row tile t PV_t(j-1), then
//     S_t(j) (S_t = Q_t K^T into tensor memory, O_t += P_t V with P_t from tensor
//     memory over the scores), so that one tile's softmax runs under the other's
//     products, and the next unit's first S under the output of the last.  Two
//     threads, one per tile, fell into step and were slower (1,380 us against 1,075
//     on the 8K case above);
//   * warp 10 overwrites V of tokens that nobody may see (behind the sequence,
//     padding) with zeros before the tile is multiplied: their weights are zero,
//     but zero times whatever memory holds may not be;
//   * warps 0-3 / 4-7 are the softmax of tile 0 / 1, a thread per row (setmaxnreg
//     moves registers to them from the other warps): 128 scores from tensor
//     memory, scale, 2^x, sum, pack.  No maximum is sought (kRefMax below).  P is
//     rounded to bfloat16 (half a step, 2^-8 of each weight); row sums are float32,
//     taken before the rounding.  Sixteen warps with half a row each were slower
//     without a cap (1,065 us against 935) and no faster with one;
//   * only key tiles that some row's limit, a document border or the drafted tree
//     cuts are masked, by a bit per key; tiles without a visible key are never
//     loaded (causal limits; with documents, the span of tiles that hold a unit's
//     documents, found by two small kernels beforehand).
// Every wait is bounded; one that gives up sets a status and an abort flag, and
// the CTA frees its tensor memory and returns.
#include <cuda.h>

#include "oc_mma.cuh"
#include "oc_tcgen05.cuh"
#include "oc_token.cuh"

namespace oc {

__device__ int g_token_status = 0;

namespace {

constexpr int kRows = 128;  // rows of a tile (UMMA M)
constexpr int kTok = 128;   // keys of a tile
constexpr int kThreads = 384;
constexpr int kProducerWarp = 8, kMmaWarp = 9, kCleanWarp = 10;
constexpr int kTmemCols = 512;

template <int D> struct TcCfg {
  static constexpr int kTileBytes = kRows * D * 2;
  static constexpr int kBox = kRows * 128;               // one 128-row x 64-channel box
  static constexpr int kPerUnit = D == 256 ? 1 : 2;      // row tiles of a unit
  static constexpr int kSlots = D == 256 ? 2 : D == 128 ? 5 : 10;
  static constexpr int kKeyTiles = D == 256 ? 1 : 2;     // column sums: key tiles of a unit
  static constexpr int kQuerySlots = D == 256 ? 2 : 4;   // column sums: ring of query tiles
};

template <int D>
struct TcSmem {
  unsigned char q[TcCfg<D>::kPerUnit][TcCfg<D>::kTileBytes];
  unsigned char kv[TcCfg<D>::kSlots][TcCfg<D>::kTileBytes];
  uint64_t kv_full[TcCfg<D>::kSlots + 1], kv_empty[TcCfg<D>::kSlots + 1];
  uint64_t q_full, q_empty;
  uint64_t v_clean[TcCfg<D>::kSlots + 1];
  uint64_t s_full[2], p_full[2], o_full[2], o_free[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
  int pre[kMaxEvenBatch + 1];
};

struct TcArgs {
  TokArgs t;
  int Gp, nhs, P, tiles;  // row tiles per (b, h): nhs head groups x position tiles of P
  int per_unit, upb, units;  // row tiles of a unit, units per (b, h), in all
  const uint4* tree_bits;   // [(b, node)][2] ancestor bits; row T of each batch row: seen by any node
  const int2* key_docs;     // [(b, key tile)] least and largest document
  const int4* query_docs;   // [(b, position tile)] least, largest document; first key tile, last + 1
  int nkt, npt;
  float k_in;               // scale / cap
};

struct TcUnit {
  int b, h, bh, len;
  int part;            // -1: all of its keys
  int ntile;
  int p0[2], hs[2], min_hi[2];
  int jt0, ncache, n;  // first cache tile, cache tiles, all tiles
  int d0;              // first drafted tile
  bool dual;           // both halves of the CTA on one row tile, key tiles in turn
};

// The k-th unit of this CTA.  Units are ordered by falling work and dealt out
// in a snake (0 .. n-1, n-1 .. 0, ...), which evens out a linear fall.
__device__ __forceinline__ int tc_deal(int k) {
  return k * gridDim.x + (k & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

__device__ __forceinline__ TcUnit tc_unit(const TcArgs& x, const TokSeg& seg) {
  const TokArgs& a = x.t;
  TcUnit w;
  const int first_tile = x.upb == 1 ? 0 : seg.unit % x.upb * x.per_unit;
  w.b = seg.b;
  w.h = x.upb == 1 ? seg.unit : seg.unit / x.upb;
  w.bh = w.b * a.Hkv + w.h;
  w.part = seg.part;
  w.len = tok_len(a, w.b);
  w.ntile = x.per_unit == 2 && first_tile + 1 < x.tiles ? 2 : 1;
  int first = INT32_MAX, last = 0, top = 0;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int r = first_tile + t, pt = x.nhs == 1 ? r : r / x.nhs;
    w.hs[t] = r - pt * x.nhs;
    w.p0[t] = pt * x.P;
    w.min_hi[t] = 0;
    if (t >= w.ntile) continue;
    int hi = w.len, lo = w.len;
    if (!a.dk) {
      const int pos0 = w.len - a.Sq + w.p0[t], pos1 = w.len - a.Sq + min(w.p0[t] + x.P, a.Sq) - 1;
      if (a.causal) {
        const int pre = a.prefix ? a.prefix[w.b] : 0;
        hi = min(w.len, max(pos1 + 1, pre));
        lo = min(w.len, max(pos0 + 1, pre));
      }
      if (pos0 < 0) lo = 0;
      if (pos1 < 0) hi = 0;
    }
    w.min_hi[t] = lo;
    int t0 = 0, t1 = (hi + kTok - 1) / kTok;
    if (a.docs) {
      const int4 q = x.query_docs[(size_t)w.b * x.npt + pt];
      t0 = q.z;
      t1 = min(t1, q.w);
    }
    if (t0 < t1) {
      first = min(first, t0);
      last = max(last, t1);
    }
    top = max(top, hi);
  }
  const int nct = (w.len + kTok - 1) / kTok;  // tiles of the cache; drafted tokens follow
  if (first == INT32_MAX) first = last = 0;
  w.jt0 = max(first, min(seg.t0, nct));
  w.ncache = max(0, min(last, seg.t1) - w.jt0);
  w.d0 = max(seg.t0 - nct, 0);
  w.n = w.ncache + (a.dk && seg.t1 > nct ? min(seg.t1 - nct, (a.Sq + kTok - 1) / kTok) - w.d0 : 0);
  w.dual = x.per_unit == 2 && x.tiles == 1 && seg.part >= 0;
  return w;
}

// Tile j of a unit: cache tiles from the last to the first, so that a row's
// reference point comes from its nearest keys, then drafted tiles.
__device__ __forceinline__ int tc_tile(const TcUnit& w, int j) {
  return j < w.ncache ? w.jt0 + w.ncache - 1 - j : w.d0 + j - w.ncache;
}

// This CTA's units in order: its run of the even cut, or whole units.
struct TcWalk {
  TokWalk even;
  int k;
  __device__ __forceinline__ TcWalk(const TcArgs& x, const int* pre) : even(x.t, pre, blockIdx.x), k(0) {}
  __device__ __forceinline__ bool next(const TcArgs& x, const int* pre, TcUnit& w) {
    TokSeg seg;
    if (x.t.even) {
      if (!even.next(x.t, pre, blockIdx.x, seg)) return false;
    } else {
      int u = x.units;
      while (u >= x.units) {
        if (k * (int)gridDim.x >= x.units) return false;
        u = tc_deal(k++);
      }
      const int BH = x.t.B * x.t.Hkv, bh = u % BH;  // the rows with most keys first
      seg = TokSeg{bh / x.t.Hkv, bh % x.t.Hkv * x.upb + x.upb - 1 - u / BH, 0, INT32_MAX, -1};
    }
    w = tc_unit(x, seg);
    return true;
  }
};

// First key row of cache tile jt in the (rows, Hkv, D) view; -1: no such page.
__device__ __forceinline__ int tc_key_row(const TokArgs& a, int b, int jt) { return (int)tok_kv_row(a, b, jt * kTok); }

// Bounded wait.  The hardware suspends a failed try for a while by itself, so the
// clock is read, and the abort flag of a role that gave up looked at, only every
// 32 tries: a timer read costs as much as several hand-overs.
__device__ __forceinline__ bool bar_wait(int* abort, uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  uint64_t t0 = 0;
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (*(volatile int*)abort != 0) return false;
    const uint64_t now = globaltimer_ns();
    if (t0 == 0) {
      t0 = now;
    } else if (now - t0 > g_wait_limit_ns) {
      atomicExch(abort, 1);
      atomicExch(&g_token_status, 1);
      return false;
    }
  }
}
// The same for a whole warp, with one answer for all its lanes.
__device__ __forceinline__ bool bar_wait_warp(int* abort, uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, bar_wait(abort, bar, parity));
}

__device__ __forceinline__ uint64_t pk2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void up2(uint64_t r, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float absmax3(float a, float b, float c) {
  float r;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The cap in log2 units: cap' tanh(k s) with cap' = cap log2(e), k = scale / cap.
// tanh(z) / z by least-squares polynomials in z^2: degree 2 for |z| <= 0.3 with
// equalised error of tanh (1.7e-7, below what the rounding of P leaves), degree 4
// for |z| <= 0.5 with equalised relative error (1.3e-8: where weights leave in
// float32, kTanh in oc_token.cuh); beyond, tanhf.
constexpr float kCapPoly2 = 0.3f;
struct CapFn {
  float k, cap2;             // k_in, cap * log2(e)
  float b0, b1, b2;          // degree 2 in s^2, times cap' k
  float a0, a1, a2, a3, a4;  // degree 4
  __device__ __forceinline__ CapFn(const TcArgs& x) {
    k = x.k_in;
    cap2 = x.t.cap * kLog2e;
    const float k2 = k * k, c = cap2 * k;
    b0 = c * 0.9999960064888f;
    b1 = c * k2 * -0.33297479152679443f;
    b2 = c * k2 * k2 * 0.12522591650485992f;
    a0 = c;
    a1 = c * k2 * kTanh[0];
    a2 = c * k2 * k2 * kTanh[1];
    a3 = c * k2 * k2 * k2 * kTanh[2];
    a4 = c * k2 * k2 * k2 * k2 * kTanh[3];
  }
  __device__ __forceinline__ float exact(float s) const { return cap2 * tanhf(k * s); }
  template <int DEG>
  __device__ __forceinline__ uint64_t poly2(uint64_t s, uint64_t off) const {  // cap' tanh(k s) + off
    const uint64_t u = mul2(s, s);
    uint64_t p;
    if (DEG == 2) {
      p = fma2(pk2(b2, b2), u, pk2(b1, b1));
      p = fma2(p, u, pk2(b0, b0));
    } else {
      p = fma2(pk2(a4, a4), u, pk2(a3, a3));
      p = fma2(p, u, pk2(a2, a2));
      p = fma2(p, u, pk2(a1, a1));
      p = fma2(p, u, pk2(a0, a0));
    }
    return fma2(p, s, off);
  }
};

// Is any of the warp's 32 x N scores beyond the polynomial?  (NaN may pass: it
// stays NaN in the polynomial.)
template <int N>
__device__ __forceinline__ bool cap_far(const float* s, float k_in) {
  float top[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) top[k] = absmax3(s[k], s[4 + k], 0.f);
#pragma unroll
  for (int i = 8; i < N; i += 8)
#pragma unroll
    for (int k = 0; k < 4; ++k) top[k] = absmax3(top[k], s[i + k], s[i + 4 + k]);
  return __any_sync(0xffffffffu, !(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * k_in <= kTanhMax));
}

// 2^x of a pair on the FMA pipe, x clamped to >= -126: x = n + f, n = floor(x) by
// adding 1.5 * 2^23 with rounding toward -inf (its low bits are then n), 2^f on [0,
// 1) a least-squares polynomial with equalised relative error (degree 4: 2.6e-6,
// degree 5: 7.5e-8), times 2^n built in the exponent field.  NaN stays NaN.
template <int DEG>
__device__ __forceinline__ uint64_t poly_ex2(uint64_t x) {
  float a, b;
  up2(x, a, b);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(-126.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(-126.f));
  x = pk2(a, b);
  uint64_t t, n, f;
  const uint64_t magic = pk2(12582912.f, 12582912.f);
  asm("add.rm.f32x2 %0, %1, %2;" : "=l"(t) : "l"(x), "l"(magic));
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(n) : "l"(t), "l"(magic));
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(f) : "l"(x), "l"(n));
  uint64_t p;
  if (DEG == 4) {
    p = fma2(pk2(0.013534166850149632f, 0.013534166850149632f), f, pk2(0.052011460065841675f, 0.052011460065841675f));
    p = fma2(p, f, pk2(0.2414427548646927f, 0.2414427548646927f));
    p = fma2(p, f, pk2(0.6930038332939148f, 0.6930038332939148f));
    p = fma2(p, f, pk2(1.0000026226043701f, 1.0000026226043701f));
  } else {
    p = fma2(pk2(0.0018775765784084797f, 0.0018775765784084797f), f, pk2(0.008989340625703335f, 0.008989340625703335f));
    p = fma2(p, f, pk2(0.05582631751894951f, 0.05582631751894951f));
    p = fma2(p, f, pk2(0.24015361070632935f, 0.24015361070632935f));
    p = fma2(p, f, pk2(0.6931530833244324f, 0.6931530833244324f));
    p = fma2(p, f, pk2(0.9999999403953552f, 0.9999999403953552f));
  }
  float t0, t1;
  up2(t, t0, t1);
  return mul2(p, pk2(__uint_as_float(__float_as_uint(t0) * (1u << 23) + 0x3f800000u),
                     __uint_as_float(__float_as_uint(t1) * (1u << 23) + 0x3f800000u)));
}

// 2^(score - m) of 32 scores (columns 32 c ..) as bfloat16 pairs, and their sums;
// At head_dim 64 an eighth of the exponentials run on the FMA pipe (the products
// are half as long there; a 2048-token chunk on 32K: 884 -> 795 us; at 128, and
// with a cap's polynomial on that pipe already, it costs 0.3 to 8 %).
// DEG > 0: capped by the polynomial of that degree, with the largest |product| in
// top.
template <int D, int DEG, bool BIAS>
__device__ __forceinline__ void chunk_exp(const float* s, int c, uint32_t* pk, uint64_t (&r2)[4], float& top,
                                          float c_scale, uint64_t nm2, uint64_t sl2, float b0, const CapFn& cap) {
  uint64_t off4[4];
  if (BIAS) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      off4[i] = fma2(pk2((float)(32 * c + 2 * i), (float)(32 * c + 2 * i + 1)), sl2, pk2(b0, b0));
  }
  const uint64_t step = BIAS ? mul2(pk2(8.f, 8.f), sl2) : 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint64_t v = pk2(s[2 * i], s[2 * i + 1]);
    uint64_t off = nm2;
    if (BIAS) {
      off = off4[i & 3];
      off4[i & 3] = add2(off, step);
    }
    if (DEG) top = absmax3(top, s[2 * i], s[2 * i + 1]);
    const uint64_t e = DEG ? cap.poly2<DEG ? DEG : 2>(v, off) : fma2(v, pk2(c_scale, c_scale), off);
    float e0, e1;
    if (D == 64 && !DEG && i % 8 == 0) {
      up2(poly_ex2<4>(e), e0, e1);
    } else {
      up2(e, e0, e1);
      e0 = ex2(e0);
      e1 = ex2(e1);
    }
    r2[i & 3] = add2(r2[i & 3], pk2(e0, e1));
    pk[16 * c + i] = pack_bf16x2(e0, e1);
  }
}

// Does tile j of the unit hold tokens that no query may see?
__device__ __forceinline__ bool tc_dirty(const TcArgs& x, const TcUnit& w, int j) {
  const TokArgs& a = x.t;
  const int jt = tc_tile(w, j);
  if (j >= w.ncache) {
    const uint4 seen = x.tree_bits[((size_t)w.b * (a.Sq + 1) + a.Sq) * 2 + jt];
    return (seen.x & seen.y & seen.z & seen.w) != ~0u;
  }
  return jt * kTok + kTok > w.len || (a.table && tc_key_row(a, w.b, jt) < 0) ||
         (a.docs && x.key_docs[(size_t)w.b * x.nkt + jt].x < 0);
}

// The reference point m of a row's softmax is exact whatever it is, as long as
// 2^(score - m), its sums and its products with the values stay in range, and
// bfloat16 has the range of float32.  So a row takes the maximum of its first
// visible tile, and the tiles after it are exponentiated without looking for one; a
// tile whose sum comes to kRefMax or more is done over, with the rescaling.
//
// CAP 0: no cap.  CAP 1 (cap <= kCapFixed, no bias): m is 0, with no maximum to
// find, while |score| <= tanh(kTanhMax) cap, at most 41.4 in log2 units: 2^score is
// bounded by the polynomials' range, which is looked at anyway.  A tile beyond it, or
// masked, finds its rows' maxima, unless the cap is that small itself, and moves m
// where that is more than kCapSlack away (down as long as the row has summed nothing).
// (Looking at the sums of the fast tiles instead: a capped 2048-token chunk on 32K 1,104
// -> 1,174 us.)  CAP 2: larger caps, or with a bias.
//
// In all of them the weights of 128 keys sum to less than 2^49, those of 2^31 to
// less than 2^73: values up to 2^50, and their sums, stay far inside float32.
constexpr float kCapFixed = 62.f;
constexpr float kCapSlack = 42.f;
constexpr float kRefMax = 281474976710656.f;  // 2^48

template <int D, int CAP, bool BIAS>
__device__ void tc_softmax(TcSmem<D>& sm, const TcArgs& x, int t, uint32_t tmem) {
  const TokArgs& a = x.t;
  const int rl = threadIdx.x & 127, lane = threadIdx.x & 31;
  const uint32_t t_s = tmem + ((uint32_t)(threadIdx.x & 96) << 16) + t * 256;
  const uint32_t t_o = t_s + 128;
  const float c_scale = a.scale * kLog2e;
  const CapFn cap(x);
  uint32_t s_ph = 0, o_ph = 0;
  TcWalk walk(x, sm.pre);
  TcUnit w;
  while (walk.next(x, sm.pre, w)) {
    if (t >= w.ntile && !w.dual) continue;
    const int rt = w.dual ? 0 : t;  // row tile
    const int p0 = rt ? w.p0[1] : w.p0[0], min_hi = rt ? w.min_hi[1] : w.min_hi[0];
    const int pos_i = p0 + rl / x.Gp;  // query position of this row
    const int r = pos_i * a.G + (rt ? w.hs[1] : w.hs[0]) * x.Gp + rl % x.Gp;
    const int j_first = w.dual ? t : 0, j_step = w.dual ? 2 : 1;
    const bool any = j_first < w.n;  // is there a tile for this half?
    const bool real = pos_i < a.Sq;
    const TokRow row = tok_row(a, w.b, w.h, real ? r : a.R, w.len);
    int4 qd = make_int4(0, 0, 0, 0);
    if (a.docs) qd = x.query_docs[(size_t)w.b * x.npt + p0 / x.P];
    float m_used = CAP == 1 || !real ? 0.f : -INFINITY, l = 0.f;
    int level = a.lse ? 1 : 0;  // which of the cap's polynomials is in use
    // what a tile's masking depends on, loaded a tile ahead
    int2 kd = make_int2(0, 0);
    bool no_page = false;
    const auto look = [&](int j) {
      if (j >= w.ncache) return;
      if (a.docs) kd = x.key_docs[(size_t)w.b * x.nkt + tc_tile(w, j)];
      if (a.table) no_page = tc_key_row(a, w.b, tc_tile(w, j)) < 0;
    };
    look(j_first);
    for (int j = j_first; j < w.n; j += j_step) {
      // is every key of the tile visible to every row of it?
      const bool draft = j >= w.ncache;
      const int jt = tc_tile(w, j), j0 = jt * kTok;
      const bool hole = no_page && !draft;
      bool part = draft || j0 + kTok > min_hi || hole;
      if (a.docs && !draft) part = part || kd.x < 0 || kd.x != kd.y || qd.x != kd.x || qd.y != kd.x;
      look(j + j_step);
      if (!bar_wait_warp(&sm.abort, &sm.s_full[t], s_ph)) return;
      s_ph ^= 1;
      tc_fence_after();
      // Fast: every key visible, every row with a reference point (with CAP 1, the first).
      bool done = false;
      const float d0 = (float)(row.pos - j0);
      const bool behind = !BIAS || (a.causal && !a.prefix);
      if (!part && behind && level < 2 && (CAP == 1 || !__any_sync(0xffffffffu, m_used == -INFINITY))) {
        uint32_t pk[64];
        const float ref = CAP == 1 ? 0.f : m_used;
        const uint64_t nm2 = pk2(-ref, -ref);
        const uint64_t sl2 = pk2(row.slope2, row.slope2);
        // |d| = d behind the query: bias and reference point are linear along the tile
        const float b0 = fmaf(-row.slope2, d0, -ref);
        uint64_t r2[4] = {0, 0, 0, 0};
        float s[128], top = 0.f;
        tmem_ld128_wait(t_s, s);
        if (!CAP || level == 0) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            chunk_exp<D, CAP ? 2 : 0, BIAS>(s + 32 * c, c, pk, r2, top, c_scale, nm2, sl2, b0, cap);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) chunk_exp<D, 4, BIAS>(s + 32 * c, c, pk, r2, top, c_scale, nm2, sl2, b0, cap);
        }
        float q[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) up2(r2[i], q[2 * i], q[2 * i + 1]);
        const float sum = ((q[0] + q[1]) + (q[2] + q[3])) + ((q[4] + q[5]) + (q[6] + q[7]));
        // a score beyond the polynomial, or a sum that has grown too large?
        const bool far = CAP && __any_sync(0xffffffffu, !(top * x.k_in <= (level ? kTanhMax : kCapPoly2)));
        if (far) ++level;  // for the rest of the unit; 2: not this way
        const bool over = far || (CAP != 1 && real && !(sum < kRefMax));
        if (!__any_sync(0xffffffffu, over)) {
          tmem_st32u(t_s, pk);
          tmem_st32u(t_s + 32, pk + 32);
          l += sum;
          done = true;
        }
      }
      if (!done) {
        // which of the 128 keys the row sees, a bit each
        uint32_t vis[4] = {~0u, ~0u, ~0u, ~0u};
        if (part && draft) {
          const uint4 bits = real ? x.tree_bits[((size_t)w.b * (a.Sq + 1) + pos_i) * 2 + jt] : make_uint4(0, 0, 0, 0);
          vis[0] = bits.x;
          vis[1] = bits.y;
          vis[2] = bits.z;
          vis[3] = bits.w;
        } else if (part) {
          const int lim = hole ? 0 : row.hi - j0;
#pragma unroll
          for (int y = 0; y < 4; ++y) vis[y] = lim >= 32 * y + 32 ? ~0u : lim <= 32 * y ? 0u : (1u << (lim - 32 * y)) - 1u;
          if (a.docs) {
            // one round per document among the warp's rows
            int d[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const int jj = j0 + 32 * y + lane;
              d[y] = jj < a.S ? a.docs[(size_t)w.b * a.S + jj] : -1;
            }
            uint32_t todo = ~0u;
            while (todo) {
              const int doc = __shfl_sync(0xffffffffu, row.doc, __ffs(todo) - 1);
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                const uint32_t same = __ballot_sync(0xffffffffu, d[y] == doc);
                if (row.doc == doc) vis[y] &= same;
              }
              todo &= ~__ballot_sync(0xffffffffu, row.doc == doc);
            }
          }
        }
        // 32 scores in log2 units, biased and masked.  They are read from tensor
        // memory once for the maximum and once for the exponentials: the code stays
        // a quarter as long (a CTA's first tile comes this way, with cold
        // instruction caches)
        const auto mask = [&](int c, float (&s)[32]) {
          const uint32_t word = c == 0 ? vis[0] : c == 1 ? vis[1] : c == 2 ? vis[2] : vis[3];
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(word >> i & 1)) s[i] = -INFINITY;
        };
        const auto scores = [&](int c, float (&s)[32]) {
          tmem_ld32_wait(t_s + 32 * c, s);
          if (CAP) {
            if (cap_far<32>(s, x.k_in)) {
#pragma unroll
              for (int i = 0; i < 32; ++i) s[i] = cap.exact(s[i]);
            } else {
#pragma unroll
              for (int i = 0; i < 32; i += 2) up2(cap.poly2<4>(pk2(s[i], s[i + 1]), 0), s[i], s[i + 1]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) s[i] *= c_scale;
          }
          if (BIAS) {
            const float dc = d0 - (float)(32 * c);
#pragma unroll
            for (int i = 0; i < 32; ++i) s[i] = fmaf(-row.slope2, fabsf(dc - (float)i), s[i]);
          }
          mask(c, s);
        };
        if (CAP != 1 || cap.cap2 > kCapSlack) {
          float mx = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float s[32];
            if (CAP == 1) {  // the cap keeps the order: the largest product has the largest score
              tmem_ld32_wait(t_s + 32 * c, s);
              mask(c, s);
            } else {
              scores(c, s);
            }
            float m4[4] = {mx, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 32; i += 8)
#pragma unroll
              for (int y = 0; y < 4; ++y) m4[y] = max3(m4[y], s[i + y], s[i + 4 + y]);
            mx = fmaxf(max3(m4[0], m4[1], m4[2]), m4[3]);
          }
          bool need;
          if (CAP == 1) {
            const bool sees = mx > -INFINITY;
            mx = cap.exact(mx);
            need = sees && (mx > m_used + kCapSlack || (l == 0.f && mx < m_used - kCapSlack));
          } else {
            need = mx > m_used + 8.f;
          }
          if (__any_sync(0xffffffffu, need)) {
            const float alpha = need ? ex2(m_used - mx) : 1.f;  // 0 on a row's first visible tile without a cap
            if (j > j_first) {
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                float o[32];
                tmem_ld32_wait(t_o + 32 * c, o);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] *= alpha;
                tmem_st32(t_o + 32 * c, o);
              }
            }
            l *= alpha;
            if (need) m_used = mx;
            if (CAP == 1) level = 2;  // the fast path takes 0
          }
        }
        const float base = m_used == -INFINITY ? 0.f : m_used;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {  // P of 32 keys takes 16 columns, behind the scores still to be read
          float s[32];
          uint32_t pk[16];
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
          scores(c, s);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float e0 = ex2(s[2 * i] - base), e1 = ex2(s[2 * i + 1] - base);
            sum[i & 3] += e0 + e1;
            pk[i] = pack_bf16x2(e0, e1);
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          tmem_st16u(t_s + 16 * c, pk);
        }
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.p_full[t]);
    }
    if (any) {
      if (!bar_wait_warp(&sm.abort, &sm.o_full[t], o_ph)) return;
      o_ph ^= 1;
      tc_fence_after();
    }
    if (l == 0.f) m_used = -INFINITY;
    const int64_t part = (int64_t)w.part * (128 * TcCfg<D>::kPerUnit) + t * 128 + rl;
    const int64_t at = tok_q_offset(a, w.b, w.h, real ? r : 0, D);
    if (real) {
      if (w.part >= 0) {
        a.pm[part] = m_used;
        a.pl[part] = l;
      } else if (a.lse) {
        a.lse[(int64_t)w.bh * a.R + r] = l == 0.f ? INFINITY : m_used + log2f(l);
      }
    }
    if (w.part >= 0) {
      // float32 rows leave in the accumulator layout: four lanes write 32 bytes of
      // a row (a thread writing its own row 16 bytes at a time takes 32 sectors an
      // instruction)
      const int64_t base = part - rl + (threadIdx.x & 96);
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        const int g = half * 16 + (lane >> 2);
        const bool put0 = __shfl_sync(0xffffffffu, real && m_used != -INFINITY, g);
        const bool put1 = __shfl_sync(0xffffffffu, real && m_used != -INFINITY, g + 8);
        if (!any) continue;
#pragma unroll 1
        for (int c = 0; c < D / 64; ++c) {
          float o[32];
          tmem_frag64_wait(t_o + ((uint32_t)(half * 16) << 16) + 64 * c, o);
          float* dst = a.po + (base + g) * D + 64 * c + 2 * (lane & 3);
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            if (put0) *reinterpret_cast<float2*>(dst + 8 * n) = make_float2(o[4 * n], o[4 * n + 1]);
            if (put1) *reinterpret_cast<float2*>(dst + 8 * D + 8 * n) = make_float2(o[4 * n + 2], o[4 * n + 3]);
          }
        }
      }
    } else {
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        float o[32];
        if (any) {
          tmem_ld32_wait(t_o + 32 * c, o);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.f;
        }
        if (!real) continue;
        if (a.out_dtype == OC_BF16) {
#pragma unroll
          for (int i = 0; i < 32; i += 8)
            *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + at + 32 * c + i) =
                make_uint4(pack_bf16x2(o[i] * inv, o[i + 1] * inv), pack_bf16x2(o[i + 2] * inv, o[i + 3] * inv),
                           pack_bf16x2(o[i + 4] * inv, o[i + 5] * inv), pack_bf16x2(o[i + 6] * inv, o[i + 7] * inv));
        } else {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at + 32 * c + i) =
                make_float4(o[i] * inv, o[i + 1] * inv, o[i + 2] * inv, o[i + 3] * inv);
        }
      }
    }
    if (any) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.o_free[t]);  // the next unit may overwrite O
    }
  }
}

// The K / V ring.  With one row tile per unit (dual) the second query buffer,
// which lies right before it, is a slot more: two streams of key tiles are in
// flight.
template <int D>
__device__ __forceinline__ unsigned char* tc_ring(TcSmem<D>& sm, const TcArgs& x) {
  return TcCfg<D>::kPerUnit == 2 && x.tiles == 1 ? sm.q[TcCfg<D>::kPerUnit - 1] : sm.kv[0];
}
template <int D>
__device__ __forceinline__ uint32_t tc_slots(const TcArgs& x) {
  return TcCfg<D>::kSlots + (TcCfg<D>::kPerUnit == 2 && x.tiles == 1 ? 1 : 0);
}

template <int D>
__device__ void tc_producer(TcSmem<D>& sm, const TcArgs& x, const CUtensorMap* mq, const CUtensorMap* mk,
                            const CUtensorMap* mv, const CUtensorMap* mdk, const CUtensorMap* mdv) {
  using C = TcCfg<D>;
  const TokArgs& a = x.t;
  uint32_t q_ph = 0, L = 0;
  unsigned char* ring = tc_ring<D>(sm, x);
  const uint32_t slots = tc_slots<D>(x);
  bool go = true;
  TcWalk walk(x, sm.pre);
  TcUnit w;
  while (go && walk.next(x, sm.pre, w)) {
    if (w.n == 0) continue;
    if (!bar_wait(&sm.abort, &sm.q_empty, q_ph ^ 1)) break;
    q_ph ^= 1;
    mbar_expect_tx(&sm.q_full, (uint32_t)(w.ntile * C::kTileBytes));
#pragma unroll
    for (int t = 0; t < C::kPerUnit; ++t)
      if (t < w.ntile)
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_3d(sm.q[t] + c * C::kBox, mq, &sm.q_full, 64 * c, w.h * a.G + w.hs[t] * x.Gp, w.b * a.Sq + w.p0[t]);
    for (int j = 0; go && j < w.n; ++j) {
      const bool draft = j >= w.ncache;
      int key = draft ? w.b * a.Sq + tc_tile(w, j) * kTok : tc_key_row(a, w.b, tc_tile(w, j));
      if (key < 0) key = 0;  // a page outside the pool: loaded from page 0, masked and zeroed
      // rolled: the roles share the instruction caches (capped 2048-token chunk on 32K 1,235 ->
      // 1,145 us, 8K prompt with a cap of 30 752 -> 711, 61 drafted tokens 182 -> 174;
      // uncapped 1,022 -> 1,032)
#pragma unroll 1
      for (int kv = 0; kv < 2; ++kv, ++L) {
        const uint32_t slot = L % slots;
        if (!bar_wait(&sm.abort, &sm.kv_empty[slot], ((L / slots) & 1) ^ 1)) {
          go = false;
          break;
        }
        mbar_expect_tx(&sm.kv_full[slot], C::kTileBytes);
        const CUtensorMap* m = kv ? (draft ? mdv : mv) : (draft ? mdk : mk);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_3d(ring + slot * C::kTileBytes + c * C::kBox, m, &sm.kv_full[slot], 64 * c, w.h, key);
      }
    }
  }
  // let the copies in flight land (bounded) before the CTA ends: this role, or another that
  // has not read them, may have given up
#pragma unroll 1
  for (uint32_t s = 0; s < slots && s < L; ++s) mbar_wait(&sm.kv_full[s], ((L - s - 1) / slots) & 1);
  mbar_wait(&sm.q_full, q_ph ^ 1);
}

// Where padding, pages or drafted tokens make it a matter of memory reads whether
// a tile is dirty, the cleaner passes every tile, and the issuing warp need not
// know.
__device__ __forceinline__ bool tc_look_always(const TokArgs& a) { return a.docs || a.table || a.dk; }

// Zeros over the values of tokens that nobody may see, before the tensor cores
// read the tile.  The warp looks at every load in order and takes part in the
// release of its slot, so that it neither lags nor runs ahead of the ring.
template <int D>
__device__ void tc_cleaner(TcSmem<D>& sm, const TcArgs& x) {
  using C = TcCfg<D>;
  const TokArgs& a = x.t;
  const int lane = threadIdx.x & 31;
  unsigned char* ring = tc_ring<D>(sm, x);
  const uint32_t slots = tc_slots<D>(x);
  uint32_t L = 0;
  TcWalk walk(x, sm.pre);
  TcUnit w;
  while (walk.next(x, sm.pre, w)) {
    for (int j = 0; j < w.n; ++j, L += 2) {
      const uint32_t kslot = L % slots, slot = (L + 1) % slots;
      if (!bar_wait_warp(&sm.abort, &sm.kv_full[kslot], (L / slots) & 1)) return;
      if (lane == 0) mbar_arrive(&sm.kv_empty[kslot]);
      if (!bar_wait_warp(&sm.abort, &sm.kv_full[slot], ((L + 1) / slots) & 1)) return;
      const bool dirty = tc_dirty(x, w, j);
      if (dirty) {
        const bool draft = j >= w.ncache;
        const int jt = tc_tile(w, j), j0 = jt * kTok;
        const uint32_t* seen = reinterpret_cast<const uint32_t*>(x.tree_bits) + ((size_t)w.b * (a.Sq + 1) + a.Sq) * 8;
        const bool no_page = !draft && a.table && tc_key_row(a, w.b, jt) < 0;
        for (int it = 0; it < kTok / 4; ++it) {
          const int rr = it * 4 + (lane >> 3), jj = j0 + rr;
          const bool keep = draft ? (seen[jj >> 5] >> (jj & 31) & 1) != 0
                                  : jj < w.len && !no_page && (!a.docs || a.docs[(size_t)w.b * a.S + jj] >= 0);
          if (!keep)
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
              *reinterpret_cast<uint4*>(ring + slot * C::kTileBytes + c * C::kBox + rr * 128 + (lane & 7) * 16) =
                  make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async();  // the tensor cores read through the async proxy
        __syncwarp();
      }
      if (lane == 0) {
        if (dirty || tc_look_always(a)) mbar_arrive(&sm.v_clean[slot]);
        mbar_arrive(&sm.kv_empty[slot]);
      }
    }
  }
}

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

// A place in the K / V ring.
struct RingPos {
  uint32_t slot, ph, slots;
  __device__ __forceinline__ RingPos ahead(uint32_t n) const {  // n <= slots
    RingPos r = *this;
    r.slot += n;
    if (r.slot >= slots) {
      r.slot -= slots;
      r.ph ^= 1;
    }
    return r;
  }
};

// The issuing warp.  All its lanes run the loop, so that the compiler keeps the
// operands of the products in uniform registers; one elected lane issues.  Every
// instruction here delays the tensor cores (the warp shares its scheduler with
// four that keep it busy), so the loop does what it can before the tile's P is
// awaited.
template <int D>
__device__ void tc_mma(TcSmem<D>& sm, const TcArgs& x, uint32_t tmem) {
  using C = TcCfg<D>;
  constexpr uint32_t kIdQK = tc_idesc_bf16(kRows, kTok, 0), kIdPV = tc_idesc_bf16(kRows, D, 1);
  const uint64_t qd0 = sdesc(__shfl_sync(0xffffffffu, smem_u32(sm.q[0]), 0), 16, 1024);
  const uint32_t kv = __shfl_sync(0xffffffffu, smem_u32(tc_ring<D>(sm, x)), 0);
  const uint64_t kd0 = sdesc(kv, 16, 1024), vd0 = sdesc(kv, C::kBox, 1024);
  tmem = __shfl_sync(0xffffffffu, tmem, 0);
  uint32_t q_ph = 0, p_ph[2] = {0, 0}, o_ph[2] = {1, 1}, clean_ph = 0;  // clean_ph: a bit per slot
  RingPos kp{0, 0, tc_slots<D>(x)};
  const bool always = tc_look_always(x.t);
  const auto wait_full = [&](const RingPos& r) { return bar_wait_warp(&sm.abort, &sm.kv_full[r.slot], r.ph); };
  const auto wait_clean = [&](const RingPos& r) {
    if (!bar_wait_warp(&sm.abort, &sm.v_clean[r.slot], (clean_ph >> r.slot) & 1)) return false;
    clean_ph ^= 1u << r.slot;
    return true;
  };
  // by the elected lane: S_t = Q K^T of the tile at kd; O_t (+)= P_t V
  const auto scores = [&](int t, uint64_t qd, const RingPos& r) {
    const uint64_t kd = kd0 + r.slot * (C::kTileBytes >> 4);
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      const uint32_t off = ((kk >> 2) * C::kBox + (kk & 3) * 32) >> 4;
      umma_bf16(tmem + t * 256, qd + off, kd + off, kIdQK, kk > 0 ? 1 : 0);
    }
  };
  const auto values = [&](int t, const RingPos& r, bool first) {
    const uint64_t vd = vd0 + r.slot * (C::kTileBytes >> 4);
#pragma unroll
    for (int kk = 0; kk < kTok / 16; ++kk)
      umma_bf16_ts(tmem + t * 256 + 128, tmem + t * 256 + kk * 8, vd + kk * 128, kIdPV, !first || kk > 0 ? 1 : 0);
  };
  TcWalk walk(x, sm.pre);
  TcUnit w;
  while (walk.next(x, sm.pre, w)) {
    const int n = __shfl_sync(0xffffffffu, w.n, 0), ntile = __shfl_sync(0xffffffffu, w.ntile, 0);
    const bool dual = __shfl_sync(0xffffffffu, (int)w.dual, 0) != 0;
    if (n == 0) continue;
    // is the first tile cut by the end of the sequence?
    const bool cut = (w.jt0 + w.ncache) * kTok > w.len && w.ncache > 0;
    if (!bar_wait_warp(&sm.abort, &sm.q_full, q_ph)) return;
    q_ph ^= 1;
    if (C::kPerUnit == 2 && dual) {
      // half t takes the key tiles t, t + 2, ...: K of tile j is load 2 j of the
      // unit, V load 2 j + 1
      for (int j = 0; j < n + 2; ++j) {
        const int t = j & 1;
        const RingPos kn = kp.ahead(4);  // of tile j + 2 (there are at least six slots)
        if (j >= 2) {                    // PV of tile j - 2
          const RingPos vp = kp.ahead(1);
          if (!wait_full(vp)) return;
          if ((always || (cut && j == 2)) && !wait_clean(vp)) return;
          if (j < 4) {  // the softmax has read the previous unit's O_t
            if (!bar_wait_warp(&sm.abort, &sm.o_free[t], o_ph[t])) return;
            o_ph[t] ^= 1;
          }
          if (j < n && !wait_full(kn)) return;
          if (!bar_wait_warp(&sm.abort, &sm.p_full[t], p_ph[t])) return;
          p_ph[t] ^= 1;
          tc_fence_after();
          if (elect_one()) {
            values(t, vp, j < 4);
            umma_commit(&sm.kv_empty[vp.slot]);
            if (j < n) {
              scores(t, qd0, kn);
              umma_commit(&sm.s_full[t]);
              umma_commit(&sm.kv_empty[kn.slot]);
              if (j == n - 1) umma_commit(&sm.q_empty);
            } else {
              umma_commit(&sm.o_full[t]);
            }
          }
          kp = kp.ahead(2);
        } else if (j < n) {  // the first S of each half
          const RingPos r = kp.ahead(2 * j);
          if (!wait_full(r)) return;
          tc_fence_after();
          if (elect_one()) {
            scores(t, qd0, r);
            umma_commit(&sm.s_full[t]);
            umma_commit(&sm.kv_empty[r.slot]);
            if (j == n - 1) umma_commit(&sm.q_empty);
          }
        } else {
          continue;
        }
        __syncwarp();
      }
      continue;
    }
    if (!wait_full(kp)) return;
    tc_fence_after();
    // S of the first key tile
#pragma unroll
    for (int t = 0; t < C::kPerUnit; ++t) {
      if (t < ntile && elect_one()) {
        scores(t, qd0 + t * (C::kTileBytes >> 4), kp);
        umma_commit(&sm.s_full[t]);
        if (t == ntile - 1) {
          umma_commit(&sm.kv_empty[kp.slot]);
          if (n == 1) umma_commit(&sm.q_empty);
        }
      }
      __syncwarp();
    }
    for (int j = 1; j <= n; ++j) {
      const RingPos vp = kp.ahead(1);  // V of tile j - 1; K of tile j after it
      kp = kp.ahead(2);
      if (!wait_full(vp)) return;
      if ((always || (cut && j == 1)) && !wait_clean(vp)) return;
      if (j < n && !wait_full(kp)) return;
#pragma unroll
      for (int t = 0; t < C::kPerUnit; ++t) {
        if (t >= ntile) break;
        if (j == 1) {  // the softmax has read the previous unit's O_t
          if (!bar_wait_warp(&sm.abort, &sm.o_free[t], o_ph[t])) return;
          o_ph[t] ^= 1;
        }
        if (!bar_wait_warp(&sm.abort, &sm.p_full[t], p_ph[t])) return;
        p_ph[t] ^= 1;
        tc_fence_after();
        if (elect_one()) {
          values(t, vp, j == 1);
          if (j < n) {
            scores(t, qd0 + t * (C::kTileBytes >> 4), kp);
            umma_commit(&sm.s_full[t]);  // covers PV of tile j - 1 too: O_t may be rescaled
          } else {
            umma_commit(&sm.o_full[t]);
          }
          if (t == ntile - 1) {
            umma_commit(&sm.kv_empty[vp.slot]);
            if (j < n) umma_commit(&sm.kv_empty[kp.slot]);
            if (j == n - 1) umma_commit(&sm.q_empty);
          }
        }
        __syncwarp();
      }
    }
  }
}

template <int D, int CAP, bool BIAS>
__global__ void __launch_bounds__(kThreads, 1)
    tok_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                  const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mdk,
                  const __grid_constant__ CUtensorMap mdv, const __grid_constant__ TcArgs x) {
  extern __shared__ unsigned char raw[];
  TcSmem<D>& sm = *reinterpret_cast<TcSmem<D>*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i <= TcCfg<D>::kSlots; ++i) {
      mbar_init(&sm.kv_full[i], 1);
      mbar_init(&sm.kv_empty[i], 2);  // the products and the cleaner
      mbar_init(&sm.v_clean[i], 1);
    }
    mbar_init(&sm.q_full, 1);
    mbar_init(&sm.q_empty, 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sm.s_full[t], 1);
      mbar_init(&sm.p_full[t], 4);
      mbar_init(&sm.o_full[t], 1);
      mbar_init(&sm.o_free[t], 4);
    }
    mbar_init(&sm.drain, 1);
    sm.abort = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();     // everything below, the lengths too, may come from the kernel before this one
  if (tok_followed(x.t)) pdl_trigger();  // the merge may find its parts meanwhile
  if (x.t.even && warp == 0) tok_prefix(x.t, sm.pre);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;

  // 384 threads x 168 registers = 256 x 208 + 128 x 88
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    tc_softmax<D, CAP, BIAS>(sm, x, warp >> 2, tmem);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == kProducerWarp) {
      if ((threadIdx.x & 31) == 0) tc_producer<D>(sm, x, &mq, &mk, &mv, &mdk, &mdv);
      __syncwarp();
    } else if (warp == kCleanWarp) {
      tc_cleaner<D>(sm, x);
    } else if (warp == kMmaWarp) {
      tc_mma<D>(sm, x, tmem);
      __syncwarp();
      if (elect_one()) {
        umma_commit(&sm.drain);  // every MMA in flight, before the memory is freed
        if (!mbar_wait(&sm.drain, 0)) atomicExch(&g_token_status, 1);
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// ---------------------------------------------------------------------------
// Column sums of the softmax, for the accumulating form with more rows than
// the scores are worth storing for: with the denominators known, the scores
// are multiplied again with the keys as the rows of the tile, S^T = K Q^T, so
// that a thread (a tensor-memory lane) owns one key and adds its weights over
// all query rows in its own registers, in the order of the rows: no exchange
// between threads, no atomics.  One MMA and one exponential per row and key:
// bound by the exponentials, five in sixteen of which run on the FMA pipe (2 x
// 1024 rows on 8K keys: 235 -> 221 us; more, or any beside a cap's polynomial,
// costs).  A unit is two tiles of 128 keys of one (b, h)
// that share every query tile; two score buffers per key tile in tensor memory
// let the products run ahead of the exponentials.
// ---------------------------------------------------------------------------
template <int D>
struct TwSmem {
  unsigned char k[TcCfg<D>::kKeyTiles][TcCfg<D>::kTileBytes];
  unsigned char q[TcCfg<D>::kQuerySlots][TcCfg<D>::kTileBytes];
  float lse[TcCfg<D>::kQuerySlots][kRows];
  uint64_t k_full, k_empty;
  uint64_t q_full[TcCfg<D>::kQuerySlots], q_empty[TcCfg<D>::kQuerySlots];
  uint64_t s_full[2][2], s_empty[2][2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
};

struct TwUnit {
  int b, h, bh, len, j0, ntile, r0, n;  // first key, key tiles with keys, first row tile, row tiles
};

template <int D>
__device__ __forceinline__ TwUnit tw_unit(const TcArgs& x, int u) {
  const TokArgs& a = x.t;
  TwUnit w;
  const int BH = a.B * a.Hkv;
  w.bh = u % BH;
  w.b = w.bh / a.Hkv;
  w.h = w.bh % a.Hkv;
  w.len = tok_len(a, w.b);
  w.j0 = u / BH * TcCfg<D>::kKeyTiles * kTok;  // the first keys, which most rows see, come first
  w.ntile = TcCfg<D>::kKeyTiles == 2 && w.j0 + kTok < w.len ? 2 : 1;
  const int before = w.j0 - (w.len - a.Sq);  // query positions that lie before the unit's first key
  w.r0 = (before > 0 ? before / x.P : 0) * x.nhs;
  w.n = w.j0 < w.len ? max(0, x.tiles - w.r0) : 0;
  return w;
}

template <int D>
__device__ void tw_producer(TwSmem<D>& sm, const TcArgs& x, const CUtensorMap* mq, const CUtensorMap* mk) {
  using C = TcCfg<D>;
  const TokArgs& a = x.t;
  const int lane = threadIdx.x & 31;
  uint32_t k_ph = 0, L = 0;
  bool go = true;
  for (int k = 0; go && k * (int)gridDim.x < x.units; ++k) {
    const int u = tc_deal(k);
    if (u >= x.units) continue;
    const TwUnit w = tw_unit<D>(x, u);
    if (w.n == 0) continue;
    if (!bar_wait_warp(&sm.abort, &sm.k_empty, k_ph ^ 1)) break;
    k_ph ^= 1;
    if (lane == 0) {
      mbar_expect_tx(&sm.k_full, (uint32_t)(w.ntile * C::kTileBytes));
      for (int t = 0; t < w.ntile; ++t)
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_3d(sm.k[t] + c * C::kBox, mk, &sm.k_full, 64 * c, w.h, w.b * a.S + w.j0 + t * kTok);
    }
    for (int i = 0; i < w.n; ++i, ++L) {
      const int r = w.r0 + i, p0 = r / x.nhs * x.P, hs = r % x.nhs;
      float lse[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int col = 32 * k + lane, pos = p0 + col / x.Gp;
        lse[k] = pos < a.Sq ? a.lse[(int64_t)w.bh * a.R + (int64_t)pos * a.G + hs * x.Gp + col % x.Gp] : INFINITY;
      }
      const uint32_t slot = L % TcCfg<D>::kQuerySlots;
      if (!bar_wait_warp(&sm.abort, &sm.q_empty[slot], ((L / TcCfg<D>::kQuerySlots) & 1) ^ 1)) {
        go = false;
        break;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) sm.lse[slot][32 * k + lane] = lse[k];
      if (lane == 0) {
        mbar_expect_tx(&sm.q_full[slot], C::kTileBytes);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_3d(sm.q[slot] + c * C::kBox, mq, &sm.q_full[slot], 64 * c, w.h * a.G + hs * x.Gp, w.b * a.Sq + p0);
      } else {
        mbar_arrive(&sm.q_full[slot]);
      }
    }
  }
  // the copies in flight land (bounded) before the CTA ends, as above
#pragma unroll 1
  for (uint32_t s = 0; s < TcCfg<D>::kQuerySlots && s < L; ++s)
    mbar_wait(&sm.q_full[s], ((L - s - 1) / TcCfg<D>::kQuerySlots) & 1);
  mbar_wait(&sm.k_full, k_ph ^ 1);
}

template <int D>
__device__ void tw_mma(TwSmem<D>& sm, const TcArgs& x, uint32_t tmem) {
  using C = TcCfg<D>;
  constexpr uint32_t kId = tc_idesc_bf16(kTok, kRows, 0);
  const uint64_t kd0 = sdesc(__shfl_sync(0xffffffffu, smem_u32(sm.k[0]), 0), 16, 1024);
  const uint64_t qd0 = sdesc(__shfl_sync(0xffffffffu, smem_u32(sm.q[0]), 0), 16, 1024);
  tmem = __shfl_sync(0xffffffffu, tmem, 0);
  uint32_t k_ph = 0, slot = 0, ph = 0, use[2] = {0, 0};
  for (int k = 0; k * (int)gridDim.x < x.units; ++k) {
    const int u = tc_deal(k);
    if (u >= x.units) continue;
    const TwUnit w = tw_unit<D>(x, u);
    const int n = __shfl_sync(0xffffffffu, w.n, 0), ntile = __shfl_sync(0xffffffffu, w.ntile, 0);
    if (n == 0) continue;
    if (!bar_wait_warp(&sm.abort, &sm.k_full, k_ph)) return;
    k_ph ^= 1;
    for (int i = 0; i < n; ++i) {
      const uint64_t qd = qd0 + slot * (C::kTileBytes >> 4);
      if (!bar_wait_warp(&sm.abort, &sm.q_full[slot], ph)) return;
#pragma unroll
      for (int t = 0; t < C::kKeyTiles; ++t) {
        if (t >= ntile) break;
        const uint32_t buf = use[t] & 1;
        if (!bar_wait_warp(&sm.abort, &sm.s_empty[t][buf], ((use[t] >> 1) & 1) ^ 1)) return;
        ++use[t];
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = ((kk >> 2) * C::kBox + (kk & 3) * 32) >> 4;
            umma_bf16(tmem + t * 256 + buf * 128, kd0 + t * (C::kTileBytes >> 4) + off, qd + off, kId, kk > 0 ? 1 : 0);
          }
          umma_commit(&sm.s_full[t][buf]);
          if (t == ntile - 1) {
            umma_commit(&sm.q_empty[slot]);
            if (i == n - 1) umma_commit(&sm.k_empty);
          }
        }
        __syncwarp();
      }
      if (++slot == TcCfg<D>::kQuerySlots) {
        slot = 0;
        ph ^= 1;
      }
    }
  }
}

template <int D, bool CAP>
__device__ void tw_sum(TwSmem<D>& sm, const TcArgs& x, int t, uint32_t tmem, const float* w_in, float* w_out) {
  const TokArgs& a = x.t;
  const int lane = threadIdx.x & 31, kl = threadIdx.x & 127;
  const uint32_t t_s = tmem + ((uint32_t)(threadIdx.x & 96) << 16) + t * 256;
  const float c_scale = a.scale * kLog2e;
  const CapFn cap(x);
  uint32_t L = 0, use = 0;
  for (int k = 0; k * (int)gridDim.x < x.units; ++k) {
    const int u = tc_deal(k);
    if (u >= x.units) continue;
    const TwUnit w = tw_unit<D>(x, u);
    const int j = w.j0 + t * kTok + kl;
    uint64_t acc[4] = {0, 0, 0, 0};
    float edge = 0.f;
    for (int i = 0; i < w.n; ++i, ++L) {
      const uint32_t slot = L % TcCfg<D>::kQuerySlots;
      if (!bar_wait_warp(&sm.abort, &sm.q_full[slot], (L / TcCfg<D>::kQuerySlots) & 1)) return;  // the denominators
      if (t < w.ntile) {
        const uint32_t buf = use & 1;
        if (!bar_wait_warp(&sm.abort, &sm.s_full[t][buf], (use >> 1) & 1)) return;
        ++use;
        tc_fence_after();
        float s[128];
        tmem_ld128_wait(t_s + buf * 128, s);
        tc_fence_before();
        mbar_arrive(&sm.s_empty[t][buf]);
        const int r = w.r0 + i, p0 = r / x.nhs * x.P, pos0 = w.len - a.Sq + p0;
        const float4* lse = reinterpret_cast<const float4*>(sm.lse[slot]);
        // rows [lo, hi) of the tile see this thread's key
        const bool part = w.j0 + t * kTok + kTok - 1 > pos0 || p0 + x.P > a.Sq;
        const bool far = CAP && cap_far<128>(s, x.k_in);
        if (!part && !far) {
          const uint64_t sc2 = pk2(c_scale, c_scale);
#pragma unroll
          for (int k = 0; k < 128; k += 4) {
            const float4 z = lse[k / 4];
            const uint64_t nz[2] = {pk2(-z.x, -z.y), pk2(-z.z, -z.w)};
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const uint64_t v = pk2(s[k + 2 * y], s[k + 2 * y + 1]);
              uint64_t e = CAP ? cap.poly2<4>(v, nz[y]) : fma2(v, sc2, nz[y]);
              if (!CAP && (k / 2 + y) % 16 < 5) {
                e = poly_ex2<5>(e);
              } else {
                float e0, e1;
                up2(e, e0, e1);
                e = pk2(ex2(e0), ex2(e1));
              }
              acc[(k / 2 + y) & 3] = add2(acc[(k / 2 + y) & 3], e);
            }
          }
        } else {
          const int lo = max(0, (j - pos0) * x.Gp), hi = min(kRows, (a.Sq - p0) * x.Gp);
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < 128; ++k) {
            const float v = CAP ? cap.exact(s[k]) : s[k] * c_scale;
            const float z = sm.lse[slot][k];
            const float e = ex2(v - z);
            if (k >= lo && k < hi && z != INFINITY) sum[k & 3] += e;
          }
          edge += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_empty[slot]);
    }
    if (t < TcCfg<D>::kKeyTiles && j < a.S) {
      const int64_t at = (int64_t)w.bh * a.S + j;
      float q[8];
#pragma unroll
      for (int y = 0; y < 4; ++y) up2(acc[y], q[2 * y], q[2 * y + 1]);
      float sum = ((q[0] + q[1]) + (q[2] + q[3])) + ((q[4] + q[5]) + (q[6] + q[7])) + edge;
      if (j >= w.len) sum = 0.f;
      w_out[at] = (w_in ? w_in[at] : 0.f) + sum;
    }
  }
}

template <int D, bool CAP>
__global__ void __launch_bounds__(kThreads, 1)
    tok_tc_weights_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                          const __grid_constant__ TcArgs x, const float* w_in, float* w_out) {
  extern __shared__ unsigned char raw[];
  TwSmem<D>& sm = *reinterpret_cast<TwSmem<D>*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    mbar_init(&sm.k_full, 1);
    mbar_init(&sm.k_empty, 1);
    for (int i = 0; i < TcCfg<D>::kQuerySlots; ++i) {
      mbar_init(&sm.q_full[i], 32);  // 31 lanes, and the one that announces the copy
      mbar_init(&sm.q_empty[i], 9);  // eight summing warps and the tensor cores
    }
    for (int t = 0; t < 2; ++t)
      for (int i = 0; i < 2; ++i) {
        mbar_init(&sm.s_full[t][i], 1);
        mbar_init(&sm.s_empty[t][i], 128);
      }
    mbar_init(&sm.drain, 1);
    sm.abort = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    tw_sum<D, CAP>(sm, x, warp >> 2, tmem, w_in, w_out);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == kProducerWarp) {
      tw_producer<D>(sm, x, &mq, &mk);
      __syncwarp();
    } else if (warp == kMmaWarp) {
      tw_mma<D>(sm, x, tmem);
      __syncwarp();
      if (elect_one()) {
        umma_commit(&sm.drain);
        if (!mbar_wait(&sm.drain, 0)) atomicExch(&g_token_status, 1);
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// Ancestor bits of a tree's nodes (row i: 256 bits) and, in row T, the drafted
// tokens that any node sees.  One CTA per batch row, a warp per node.
__global__ void __launch_bounds__(1024) tok_tree_bits_kernel(const uint8_t* tree, int64_t bstride, int T, uint32_t* bits) {
  __shared__ uint32_t seen[8];
  if (threadIdx.x < 8) seen[threadIdx.x] = 0;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  const uint8_t* tm = tree + blockIdx.x * bstride;
  uint32_t* out = bits + (size_t)blockIdx.x * (T + 1) * 8;
  for (int i = threadIdx.x >> 5; i < T; i += 32) {
    uint32_t mine = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const int s = w * 32 + lane;
      const uint32_t word = __ballot_sync(0xffffffffu, s < T && tm[(int64_t)i * T + s] != 0);
      if (lane == w) mine = word;
    }
    if (lane < 8) {
      out[i * 8 + lane] = mine;
      if (mine) atomicOr(&seen[lane], mine);
    }
  }
  __syncthreads();
  if (threadIdx.x < 8) out[T * 8 + threadIdx.x] = seen[threadIdx.x];
}

// Least and largest document of every 128-key tile (keys behind the sequence
// count as padding); one warp per tile.
__global__ void __launch_bounds__(128) tok_key_docs_kernel(const TokArgs a, int nkt, int2* key_docs) {
  const int tile = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (tile >= a.B * nkt) return;
  const int b = tile / nkt, j0 = tile % nkt * kTok, len = tok_len(a, b);
  int lo = INT32_MAX, hi = -1;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int j = j0 + 32 * k + lane;
    const int d = j < len ? a.docs[(size_t)b * a.S + j] : -1;
    lo = min(lo, d < 0 ? -1 : d);
    hi = max(hi, d);
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (lane == 0) key_docs[tile] = make_int2(lo, hi);
}

// Least (-1 with padding among them) and largest document of the P query
// positions of a position tile, and the span of key tiles that hold any
// document between; one warp per tile.
__global__ void __launch_bounds__(128) tok_query_docs_kernel(const TokArgs a, int P, int npt, int nkt,
                                                             const int2* key_docs, int4* query_docs) {
  pdl_wait();
  const int tile = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (tile >= a.B * npt) return;
  const int b = tile / npt, p0 = tile % npt * P, len = tok_len(a, b);
  int lo = INT32_MAX, least = INT32_MAX, hi = -1;
  for (int i = p0 + lane; i < min(p0 + P, a.Sq); i += 32) {
    const int pos = len - a.Sq + i;
    const int d = pos >= 0 ? a.docs[(size_t)b * a.S + pos] : -1;
    lo = min(lo, d < 0 ? -1 : d);
    if (d >= 0) least = min(least, d);
    hi = max(hi, d);
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  least = __reduce_min_sync(0xffffffffu, least);
  hi = __reduce_max_sync(0xffffffffu, hi);
  int first = INT32_MAX, last = 0;
  for (int k = lane; k < nkt; k += 32) {
    const int2 kd = key_docs[(size_t)b * nkt + k];
    if (kd.x <= hi && kd.y >= least) {
      first = min(first, k);
      last = max(last, k + 1);
    }
  }
  first = __reduce_min_sync(0xffffffffu, first);
  last = __reduce_max_sync(0xffffffffu, last);
  if (lane == 0) query_docs[tile] = make_int4(lo, hi, first, last);
}

int tc_map(CUtensorMap* m, const void* base, int D, int heads, int64_t rows, int box_heads, int box_rows,
           const char* fn) {
  const uint64_t dims[3] = {(uint64_t)D, (uint64_t)heads, (uint64_t)rows};
  const uint64_t strides[2] = {(uint64_t)D * 2, (uint64_t)heads * D * 2};
  const uint32_t box[3] = {64, (uint32_t)box_heads, (uint32_t)box_rows};
  const int r = encode_map_3d(m, base, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dims, strides, box, true);
  if (r) return set_error(OC_ERR_CUDA, "%s: tensor map failed (CUresult %d)", fn, r);
  return OC_OK;
}

template <int D, int CAP, bool BIAS>
int launch_tc(const CUtensorMap (&m)[5], const TcArgs& x, cudaStream_t st) {
  const size_t smem = sizeof(TcSmem<D>) + 1024;
  auto kern = tok_tc_kernel<D, CAP, BIAS>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(done, kern, smem);
  if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "tok_tc_kernel: %s", cudaGetErrorString(e));
  const int sms = device_sm_count();
  const dim3 grid((unsigned)(x.t.even ? x.t.ncta : x.units < sms ? x.units : sms));
  if (x.tree_bits || x.query_docs) {
    e = launch_pdl(kern, grid, dim3(kThreads), smem, st, m[0], m[1], m[2], m[3], m[4], x);
  } else {
    kern<<<grid, kThreads, smem, st>>>(m[0], m[1], m[2], m[3], m[4], x);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "tok_tc_kernel: %s", cudaGetErrorString(e));
  return OC_OK;
}

template <int D>
int launch_tc_form(const CUtensorMap (&m)[5], const TcArgs& x, cudaStream_t st) {
  const bool bias = x.t.slopes != nullptr;
  if (x.t.cap > 0.f && bias) return launch_tc<D, 2, true>(m, x, st);
  if (x.t.cap > 0.f) return x.t.cap > kCapFixed ? launch_tc<D, 2, false>(m, x, st) : launch_tc<D, 1, false>(m, x, st);
  return bias ? launch_tc<D, 0, true>(m, x, st) : launch_tc<D, 0, false>(m, x, st);
}

}  // namespace

// Row tiles: Gp heads x P positions.
TokTcShape tok_tc_shape(int q_len, int G, int head_dim) {
  TokTcShape s;
  s.Gp = 1;
  while (s.Gp < kRows && G % (2 * s.Gp) == 0) s.Gp *= 2;
  s.nhs = G / s.Gp;
  s.P = kRows / s.Gp;
  s.npt = (q_len + s.P - 1) / s.P;
  s.per_unit = head_dim == 256 ? TcCfg<256>::kPerUnit : TcCfg<128>::kPerUnit;
  s.units = (s.npt * s.nhs + s.per_unit - 1) / s.per_unit;
  return s;
}

size_t tok_tc_prep_bytes(int batch, int q_len, int G, int head_dim, int seq_len) {
  const TokTcShape s = tok_tc_shape(q_len, G, head_dim);
  const size_t tree = q_len <= kMaxNodes ? (size_t)batch * (q_len + 1) * 32 : 0;
  const size_t docs = (size_t)batch * s.npt * sizeof(int4) + (size_t)batch * ((seq_len + kTok - 1) / kTok) * sizeof(int2);
  return tree > docs ? tree : docs;
}

int tok_tc(const char* fn, const TokArgs& a, int head_dim, void* prep, cudaStream_t st) {
  const TokTcShape s = tok_tc_shape(a.Sq, a.G, head_dim);
  TcArgs x = {};
  x.t = a;
  x.Gp = s.Gp;
  x.nhs = s.nhs;
  x.P = s.P;
  x.tiles = s.npt * s.nhs;
  x.per_unit = s.per_unit;
  x.upb = s.units;
  x.units = a.B * a.Hkv * s.units;
  x.nkt = (a.S + kTok - 1) / kTok;
  x.npt = s.npt;
  x.k_in = a.cap > 0.f ? a.scale / a.cap : 0.f;
  CUtensorMap m[5];
  int rc = tc_map(&m[0], a.q, head_dim, a.Hq, (int64_t)a.B * a.Sq, s.Gp, s.P, fn);
  if (rc) return rc;
  m[1] = m[2] = m[3] = m[4] = m[0];
  if (a.S > 0) {
    const int64_t rows = a.table ? (int64_t)a.num_pages * a.page : (int64_t)a.B * a.S;
    rc = tc_map(&m[1], a.k, head_dim, a.Hkv, rows, 1, kTok, fn);
    if (!rc) rc = tc_map(&m[2], a.v, head_dim, a.Hkv, rows, 1, kTok, fn);
    if (rc) return rc;
  }
  if (a.dk) {
    rc = tc_map(&m[3], a.dk, head_dim, a.Hkv, (int64_t)a.B * a.Sq, 1, kTok, fn);
    if (!rc) rc = tc_map(&m[4], a.dv, head_dim, a.Hkv, (int64_t)a.B * a.Sq, 1, kTok, fn);
    if (rc) return rc;
    x.tree_bits = static_cast<const uint4*>(prep);
    tok_tree_bits_kernel<<<a.B, 1024, 0, st>>>(a.tree, a.tree_bstride, a.Sq, static_cast<uint32_t*>(prep));
    rc = check_launch("tok_tree_bits_kernel");
    if (rc) return rc;
  } else if (a.docs && a.S > 0) {
    int4* qd = static_cast<int4*>(prep);
    int2* kd = reinterpret_cast<int2*>(qd + (size_t)a.B * s.npt);
    x.query_docs = qd;
    x.key_docs = kd;
    tok_key_docs_kernel<<<(unsigned)(((int64_t)a.B * x.nkt + 3) / 4), 128, 0, st>>>(a, x.nkt, kd);
    rc = check_launch("tok_key_docs_kernel");
    if (rc) return rc;
    cudaError_t e = launch_pdl(tok_query_docs_kernel, dim3((unsigned)(((int64_t)a.B * s.npt + 3) / 4)), dim3(128), 0, st,
                               a, s.P, s.npt, x.nkt, static_cast<const int2*>(kd), qd);
    if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "tok_query_docs_kernel: %s", cudaGetErrorString(e));
  } else if (a.docs) {
    x.t.docs = nullptr;  // an empty cache: no row sees anything
  }
  if (head_dim == 64) return launch_tc_form<64>(m, x, st);
  return head_dim == 128 ? launch_tc_form<128>(m, x, st) : launch_tc_form<256>(m, x, st);
}

namespace {
template <int D, bool CAP>
int launch_tw(const CUtensorMap& mq, const CUtensorMap& mk, const TcArgs& x, const float* w_in, float* w_out,
              cudaStream_t st) {
  const size_t smem = sizeof(TwSmem<D>) + 1024;
  auto kern = tok_tc_weights_kernel<D, CAP>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(done, kern, smem);
  if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "tok_tc_weights_kernel: %s", cudaGetErrorString(e));
  const int sms = device_sm_count();
  kern<<<(unsigned)(x.units < sms ? x.units : sms), kThreads, smem, st>>>(mq, mk, x, w_in, w_out);
  return check_launch("tok_tc_weights_kernel");
}
}  // namespace

int tok_tc_weights(const char* fn, const TokArgs& a, int head_dim, const float* w_in, float* w_out, cudaStream_t st) {
  const TokTcShape s = tok_tc_shape(a.Sq, a.G, head_dim);
  TcArgs x = {};
  x.t = a;
  x.Gp = s.Gp;
  x.nhs = s.nhs;
  x.P = s.P;
  x.tiles = s.npt * s.nhs;
  const int keys = kTok * (head_dim == 256 ? TcCfg<256>::kKeyTiles : TcCfg<128>::kKeyTiles);
  const int64_t units = (int64_t)((a.S + keys - 1) / keys) * a.B * a.Hkv;
  OC_REQUIRE(units < INT32_MAX, OC_ERR_SHAPE, "%s: too many work units", fn);
  x.units = (int)units;
  x.k_in = a.cap > 0.f ? a.scale / a.cap : 0.f;
  CUtensorMap mq, mk;
  int rc = tc_map(&mq, a.q, head_dim, a.Hq, (int64_t)a.B * a.Sq, s.Gp, s.P, fn);
  if (!rc) rc = tc_map(&mk, a.k, head_dim, a.Hkv, (int64_t)a.B * a.S, 1, kTok, fn);
  if (rc) return rc;
  const bool cap = a.cap > 0.f;
  if (head_dim == 64)
    return cap ? launch_tw<64, true>(mq, mk, x, w_in, w_out, st) : launch_tw<64, false>(mq, mk, x, w_in, w_out, st);
  if (head_dim == 128)
    return cap ? launch_tw<128, true>(mq, mk, x, w_in, w_out, st) : launch_tw<128, false>(mq, mk, x, w_in, w_out, st);
  return cap ? launch_tw<256, true>(mq, mk, x, w_in, w_out, st) : launch_tw<256, false>(mq, mk, x, w_in, w_out, st);
}

int wait_limit_token(unsigned long long ns) { return set_wait_limit_here(ns); }
int token_status(int* status, int reset) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_token_status, sizeof(int));
  if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "oc_device_status: %s", cudaGetErrorString(e));
  if (reset) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_token_status, &zero, sizeof(int));
    if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "oc_device_status: %s", cudaGetErrorString(e));
  }
  return OC_OK;
}

}  // namespace oc
