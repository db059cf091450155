// Token-level attention over a KV cache: what the tree, chunk and
// accumulating forms share.
//
// For batch row b and KV head h the query rows of the G = Hq / Hkv heads that
// read it are numbered r = i * G + g (query position i, head h * G + g).  Row
// r may see key j of the cache iff
//     j < hi_r   and   (no documents, or documents[b, j] == doc_r),
// where hi_r folds the sequence length, the causal limit and the prefix (a
// row that has no position, or lies in padding, has hi_r = 0), and drafted
// key s iff tree[b, i, s].  Its score is, in log2 units,
//     s2 = log2(e) * (cap * tanh(scale * q.k / cap) - slope * |pos_r - j|)
// (without the tanh when cap is 0; the float32 kernel leaves log2(e) to the
// exponential), and the output softmax(s) . v; a row that sees nothing is zero.
#pragma once

#include "oc_common.cuh"

namespace oc {

constexpr float kLog2e = 1.4426950408889634f;
// tanh(z) = z (1 + u (c0 + u (c1 + u (c2 + u c3)))), u = z^2, |z| <= kTanhMax: a
// least-squares fit with equalised relative error (1.3e-8).
__device__ constexpr float kTanh[4] = {-0.3333306908607483f, 0.13324779272079468f, -0.05298607423901558f,
                                       0.017135007306933403f};
constexpr float kTanhMax = 0.5f;
__device__ __forceinline__ float tok_tanh(float z) {
  const float u = z * z;
  float p = fmaf(kTanh[3], u, kTanh[2]);
  p = fmaf(p, u, kTanh[1]);
  p = fmaf(p, u, kTanh[0]);
  return fmaf(z * u, p, z);
}
constexpr int kMaxNodes = 256;  // drafted tokens of one tree

struct TokArgs {
  const void *q, *k, *v;
  const void *dk, *dv;        // drafted keys / values (B, Sq, Hkv, D); NULL: chunk form
  const uint8_t* tree;        // (1 or B, Sq, Sq)
  int64_t tree_bstride;       // 0 or Sq * Sq
  const int32_t* lengths;     // (B) or NULL (= S)
  const int32_t* table;       // (B, table_stride) pool pages, or NULL: k, v are (B, S, Hkv, D)
  int table_stride, page, num_pages;
  const int32_t *prefix, *docs;  // (B), (B, S); nullable
  const float* slopes;           // (Hq) nullable
  int causal;
  int B, Sq, Hq, Hkv, G, R, S;   // R = Sq * G rows per KV head; S keys of capacity per batch row
  float scale, cap;
  void* out;
  int out_dtype;
  // A unit is a row tile of one (b, h): units of batch row b are numbered h *
  // nrt + rt.  Either every unit is one CTA's (even = 0), or the key tiles of
  // all units, laid end to end, are cut into equal runs, ncta in all (even = 1).
  int nrt, even, ncta, tile;  // row tiles per (b, h); keys of a tile
  int hg;                     // heads that are cut alike; divides Hkv and ncta
  int unit_rows;              // rows of a unit's partial
  float *pm, *pl, *po;        // partials: [part][unit_rows][(D)], parts 2 * cta and 2 * cta + 1
  // (B * Hkv, R, logit_stride) scores in the units of pm, -inf where masked, written for the
  // key tiles that a row's unit visits (with a causal mask: all that the row sees); nullable
  float* logits;
  int64_t logit_stride;
  float* lse;                    // (B * Hkv, R) log of the softmax denominator, +inf for empty rows; nullable
  float unit;                    // 2^(unit * x) = e^x in the units of pm and lse: log2(e) for natural ones, else 1
};

__device__ __forceinline__ int tok_len(const TokArgs& a, int b) {
  if (!a.lengths) return a.S;
  const int n = a.lengths[b];
  return n < 0 ? 0 : (n > a.S ? a.S : n);
}

// Does another kernel of the same call follow the attention kernel?  Only then may it
// let the next one start early: a kernel of another call may read its queries before
// it waits, and they may be this call's output.
__device__ __forceinline__ bool tok_followed(const TokArgs& a) { return a.even || (a.lse && a.S > 0); }

// What one query row may see and how its scores are biased.
struct TokRow {
  int hi;       // keys [0, hi)
  int pos;      // position of the query in its sequence
  int doc;      // document of the query (only with documents)
  float slope2; // slope * log2(e), 0 without a bias
};

__device__ __forceinline__ TokRow tok_row(const TokArgs& a, int b, int h, int r, int len) {
  TokRow w;
  w.hi = 0;
  w.pos = 0;
  w.doc = 0;
  w.slope2 = 0.f;
  if (r >= a.R) return w;
  const int i = r / a.G;
  if (a.dk) {
    w.hi = len;
    w.pos = len;
    return w;
  }
  w.pos = len - a.Sq + i;
  if (a.slopes) w.slope2 = a.slopes[h * a.G + r % a.G] * kLog2e;
  if (w.pos < 0) return w;
  int hi = len;
  if (a.causal) {
    hi = w.pos + 1;
    if (a.prefix && a.prefix[b] > hi) hi = a.prefix[b];
    if (hi > len) hi = len;
  }
  if (a.docs) {
    w.doc = a.docs[(size_t)b * a.S + w.pos];
    if (w.doc < 0) hi = 0;
  }
  w.hi = hi;
  return w;
}

// ---- the even cut ---------------------------------------------------------
// The lengths are on the device, so the cut is made there: every CTA adds up
// the rows' tiles (at most kMaxEvenBatch of them) and finds its run.  A run
// begins and ends inside a unit at most; those two pieces are partials, which
// tok_merge_kernel joins.  hg neighbouring heads, whose keys lie side by side in
// memory, are cut alike and go to hg neighbouring CTAs, which read the same
// tokens at about the same time: DRAM pages are then opened for hg heads' bytes
// instead of one's.
constexpr int kMaxEvenBatch = 256;

__device__ __forceinline__ int tok_tiles(const TokArgs& a, int b) {
  const int n = (tok_len(a, b) + a.tile - 1) / a.tile + (a.dk ? (a.Sq + a.tile - 1) / a.tile : 0);
  return n > 0 ? n : 1;  // a unit without keys still has rows to write
}

// pre[b] = tiles of a unit of the rows before b (one warp).
__device__ __forceinline__ void tok_prefix(const TokArgs& a, int* pre) {
  const int lane = threadIdx.x & 31;
  int run = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    int n = b0 + lane < a.B ? tok_tiles(a, b0 + lane) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) n += y;
    }
    if (b0 + lane < a.B) pre[b0 + lane + 1] = run + n;
    run += __shfl_sync(0xffffffffu, n, 31);
  }
  if (lane == 0) pre[0] = 0;
}

struct TokSeg {
  int b, unit, t0, t1;  // tiles [t0, t1) of the unit
  int part;             // -1: the whole unit
};

// The cut of `total` tiles into n runs: the first `rem` have one tile more.  (All
// in 32 bits: a 64-bit division costs a CTA's set-up a microsecond.)
struct TokCut {
  int n, q, rem;
  __device__ __forceinline__ TokCut(const TokArgs& a, int total) {
    n = a.ncta / a.hg;
    if (n > total) n = total > 0 ? total : 1;  // none is empty
    q = (int)((unsigned)total / (unsigned)n);
    rem = total - q * n;
  }
  __device__ __forceinline__ int first(int i) const { return i * q + min(i, rem); }  // first tile of run i
  __device__ __forceinline__ int run(int t) const {                                  // run of tile t
    const int big = rem * (q + 1);
    return t < big ? (int)((unsigned)t / (unsigned)(q + 1)) : rem + (int)((unsigned)(t - big) / (unsigned)q);
  }
};

struct TokWalk {
  int x, lo, hi, b;
  __device__ __forceinline__ TokWalk(const TokArgs& a, const int* pre, int cta) {
    const int total = a.even ? a.Hkv / a.hg * a.nrt * pre[a.B] : 0;
    const TokCut cut(a, total);
    const int i = cta / a.hg;
    lo = i < cut.n ? cut.first(i) : 0;
    hi = i < cut.n && total ? cut.first(i + 1) : 0;
    x = lo;
    b = 0;
  }
  __device__ __forceinline__ bool next(const TokArgs& a, const int* pre, int cta, TokSeg& s) {
    if (x >= hi) return false;
    const int upb = a.Hkv / a.hg * a.nrt;
    while (x >= upb * pre[b + 1]) ++b;
    const int rel = x - upb * pre[b], nt = pre[b + 1] - pre[b];
    const int u = (int)((unsigned)rel / (unsigned)nt);  // head group * nrt + row tile
    const int hgroup = a.nrt == 1 ? u : u / a.nrt;
    s.b = b;
    s.unit = (hgroup * a.hg + cta % a.hg) * a.nrt + u - hgroup * a.nrt;
    s.t0 = rel - u * nt;
    s.t1 = min(nt, s.t0 + hi - x);
    s.part = s.t0 == 0 && s.t1 == nt ? -1 : 2 * cta + (x == lo ? 0 : 1);
    x += s.t1 - s.t0;
    return true;
  }
};

// Row (of the (rows, Hkv, D) view of k / v) of token j of batch row b; -1 for
// a token whose page lies outside the pool.
__device__ __forceinline__ int64_t tok_kv_row(const TokArgs& a, int b, int j) {
  if (!a.table) return (int64_t)b * a.S + j;
  const int n = j / a.page, p = a.table[(size_t)b * a.table_stride + n];
  return p < 0 || p >= a.num_pages ? -1 : (int64_t)p * a.page + (j - n * a.page);
}

// Element offset of the first channel of output / query row r of (b, h).
__device__ __forceinline__ int64_t tok_q_offset(const TokArgs& a, int b, int h, int r, int D) {
  return (((int64_t)b * a.Sq + r / a.G) * a.Hq + (int64_t)h * a.G + r % a.G) * D;
}

// The score from the dot product, in natural units (the float32 kernel keeps
// them: log2(e) times a score would round once more, and the exponential would
// magnify that; here it multiplies the difference to the maximum).
__device__ __forceinline__ float tok_score(const TokArgs& a, float dot, float slope2, int pos, int j) {
  float x = dot * a.scale;
  if (a.cap > 0.f) x = a.cap * tanhf(x / a.cap);
  return slope2 != 0.f ? fmaf(-slope2 * (1.f / kLog2e), fabsf((float)(pos - j)), x) : x;
}

// The bfloat16 kernel for few rows (oc_token_mma.cu); row_tile 16, 32 or 64.
int tok_mma(const TokArgs& a, int head_dim, int row_tile, cudaStream_t st);
int tok_mma_tile(int head_dim);  // keys of its tiles

// The float32 kernel for few rows (oc_token_few.cu): units of 16 rows.
int tok_few(const TokArgs& a, int head_dim, cudaStream_t st);
int tok_few_tile(int head_dim);

// The bfloat16 kernel on the tcgen05 tensor cores (oc_token_tc.cu) for
// a positive scale; a unit is one or two row tiles.
// prep: tok_tc_prep_bytes of scratch.
struct TokTcShape {
  int Gp, nhs, P, npt;  // heads and positions of a row tile; head groups, position tiles
  int per_unit, units;  // row tiles of a unit (one at head_dim 256, else two); units per (b, h)
};
TokTcShape tok_tc_shape(int q_len, int G, int head_dim);
size_t tok_tc_prep_bytes(int batch, int q_len, int G, int head_dim, int seq_len);
int tok_tc(const char* fn, const TokArgs& a, int head_dim, void* prep, cudaStream_t st);

// Column sums of the softmax on the tcgen05 tensor cores, from a.lse
// (bfloat16, contiguous keys, positive scale).
int tok_tc_weights(const char* fn, const TokArgs& a, int head_dim, const float* w_in, float* w_out, cudaStream_t st);

// Merge of the partials of the even cut (oc_token_attention.cu).
int tok_merge(const TokArgs& a, int head_dim, bool tc, cudaStream_t st);

}  // namespace oc
