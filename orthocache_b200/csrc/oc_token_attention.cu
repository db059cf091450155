// Token-level attention: entry points, the float32-arithmetic kernel that
// serves every type and size, the merge of partials split over the keys, and
// the column sums of the attention weights.
//
// oc_tree_attention: T drafted tokens, arranged in a tree, attend to a
// cache and to their own ancestors.  oc_chunk_attention: a query chunk at the
// end of each sequence, with a causal, prefix or document mask, capped scores
// and a distance bias.  oc_accumulate_attention: causal chunk attention that
// also adds the attention weight of every key, summed over the query rows of
// its KV head, to a running sum.  No counterpart in the reference, whose
// attention takes whole 512-token blocks without a mask
// (src/orthocache/indirect_attention.py:29-170).
#include <math.h>

#include "oc_token.cuh"

namespace oc {
namespace {

constexpr int kSimtThreads = 256;
constexpr int kSimtTok = 64;  // keys per tile

template <int D, int RPT>
struct SimtSmem {
  float q[16 * RPT][D];
  float k[kSimtTok][D + 4];  // +4: the 16 keys a half-warp reads at once fall into different banks
  float v[kSimtTok][D];
  float p[16 * RPT][kSimtTok];
  TokRow row[16 * RPT];
  int doc[kSimtTok];
  int seen[kSimtTok];
  int hi, lo;
};

// Load keys [j0, j0 + 64) of the cache (or of the drafted tokens) as float32.
// Keys that no row may see (behind the sequence, padding, pages outside the
// pool) become zero, so that whatever the memory holds there cannot reach a
// result.
template <typename T, int D>
__device__ __forceinline__ void simt_load_vec(const T* src, float* dst) {
  constexpr int kVec = Elem<T>::kVec;
  const uint4 w = *reinterpret_cast<const uint4*>(src);
  float f[kVec];
  unpack16<T>(w, f);
#pragma unroll
  for (int c = 0; c < kVec; ++c) dst[c] = f[c];
}

// Row tiles of 16 * RPT query rows against tiles of 64 keys, one pass with
// the running maximum and sum of the softmax; 256 threads as 16 x 16: thread
// (ty, tx) owns rows ty + 16 i, the scores of keys tx + 16 n, and the output
// channels 4 tx + 64 c of its rows, so that the softmax statistics stay in
// registers (reduced over the 16 lanes of a half-warp).  Bound by the
// shared-memory reads of the score product, about 1.2 per four FMA.
template <typename T, int D, int RPT>
__global__ void __launch_bounds__(kSimtThreads) tok_simt_kernel(const TokArgs a) {
  extern __shared__ __align__(16) unsigned char raw[];
  SimtSmem<D, RPT>& sm = *reinterpret_cast<SimtSmem<D, RPT>*>(raw);
  constexpr int RT = 16 * RPT, kVec = Elem<T>::kVec, NC = D / 64;
  const int bh = blockIdx.x % (a.B * a.Hkv);
  const int rt = a.nrt - 1 - blockIdx.x / (a.B * a.Hkv);  // the rows with most keys first
  const int b = bh / a.Hkv, h = bh % a.Hkv, c = blockIdx.y;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int len = tok_len(a, b);
  const T* kbase = static_cast<const T*>(a.k);
  const T* vbase = static_cast<const T*>(a.v);

  if (tid == 0) {
    sm.hi = 0;
    sm.lo = INT32_MAX;
  }
  __syncthreads();
  for (int r = tid; r < RT; r += kSimtThreads) {
    sm.row[r] = tok_row(a, b, h, rt * RT + r, len);
    if (sm.row[r].hi > 0) atomicMax(&sm.hi, sm.row[r].hi);
  }
  for (int e = tid; e < RT * (D / kVec); e += kSimtThreads) {
    const int r = e / (D / kVec), x = e % (D / kVec) * kVec;
    if (rt * RT + r < a.R)
      simt_load_vec<T, D>(static_cast<const T*>(a.q) + tok_q_offset(a, b, h, rt * RT + r, D) + x, &sm.q[r][x]);
    else
#pragma unroll
      for (int y = 0; y < kVec; ++y) sm.q[r][x + y] = 0.f;
  }
  __syncthreads();
  const int t0 = c * a.chunk;
  int t1 = min(sm.hi, t0 + a.chunk);
  if (t1 < t0) t1 = t0;
  const int ncache = (t1 - t0 + kSimtTok - 1) / kSimtTok;
  const int ndraft = a.dk && c == a.nchunk - 1 ? (a.Sq + kSimtTok - 1) / kSimtTok : 0;

  TokRow row[RPT];
  float m[RPT], l[RPT], o[RPT][NC * 4];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    row[i] = sm.row[ty + 16 * i];
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int x = 0; x < NC * 4; ++x) o[i][x] = 0.f;
  }

  for (int tile = 0; tile < ncache + ndraft; ++tile) {
    const bool draft = tile >= ncache;
    const int j0 = draft ? (tile - ncache) * kSimtTok : t0 + tile * kSimtTok;
    __syncthreads();  // the previous tile's keys and values are read
    if (tid < kSimtTok) {
      const int j = j0 + tid;
      int seen = 0, doc = -1;
      if (draft) {
        if (j < a.Sq)
          for (int i = 0; i < a.Sq && !seen; ++i) seen = a.tree[b * a.tree_bstride + (int64_t)i * a.Sq + j] != 0;
      } else if (j < len) {
        doc = a.docs ? a.docs[(size_t)b * a.S + j] : 0;
        seen = doc >= 0 && tok_kv_row(a, b, j) >= 0;
      }
      sm.doc[tid] = doc;
      sm.seen[tid] = seen;
    }
    __syncthreads();
    for (int e = tid; e < kSimtTok * (D / kVec); e += kSimtThreads) {
      const int t = e / (D / kVec), x = e % (D / kVec) * kVec, j = j0 + t;
      if (sm.seen[t]) {
        const int64_t at = draft ? (((int64_t)b * a.Sq + j) * a.Hkv + h) * D + x
                                 : (tok_kv_row(a, b, j) * a.Hkv + h) * D + x;
        simt_load_vec<T, D>((draft ? static_cast<const T*>(a.dk) : kbase) + at, &sm.k[t][x]);
        simt_load_vec<T, D>((draft ? static_cast<const T*>(a.dv) : vbase) + at, &sm.v[t][x]);
      } else {
#pragma unroll
        for (int y = 0; y < kVec; ++y) sm.k[t][x + y] = sm.v[t][x + y] = 0.f;
      }
    }
    __syncthreads();

    float s[RPT][4];
#pragma unroll
    for (int i = 0; i < RPT; ++i)
#pragma unroll
      for (int n = 0; n < 4; ++n) s[i][n] = 0.f;
#pragma unroll 4
    for (int x = 0; x < D; x += 4) {
      float4 kk[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) kk[n] = *reinterpret_cast<const float4*>(&sm.k[tx + 16 * n][x]);
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const float4 qq = *reinterpret_cast<const float4*>(&sm.q[ty + 16 * i][x]);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          s[i][n] = fmaf(qq.x, kk[n].x, s[i][n]);
          s[i][n] = fmaf(qq.y, kk[n].y, s[i][n]);
          s[i][n] = fmaf(qq.z, kk[n].z, s[i][n]);
          s[i][n] = fmaf(qq.w, kk[n].w, s[i][n]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int r = rt * RT + ty + 16 * i;
      float mx = -INFINITY;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int t = tx + 16 * n, j = j0 + t;
        bool vis = sm.seen[t] != 0;
        if (draft)
          vis = vis && r < a.R && a.tree[b * a.tree_bstride + (int64_t)(r / a.G) * a.Sq + j] != 0;
        else
          vis = vis && j < row[i].hi && j < t1 && (!a.docs || sm.doc[t] == row[i].doc);
        s[i][n] = vis ? tok_score(a, s[i][n], row[i].slope2, row[i].pos, j) : -INFINITY;
        mx = fmaxf(mx, s[i][n]);
      }
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
      const float m_new = fmaxf(m[i], mx);
      const float base = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = exp2f(m[i] - base);
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float p = exp2f(s[i][n] - base);
        sm.p[ty + 16 * i][tx + 16 * n] = p;
        sum += p;
      }
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      l[i] = l[i] * alpha + sum;
      m[i] = m_new;
#pragma unroll
      for (int x = 0; x < NC * 4; ++x) o[i][x] *= alpha;
    }
    __syncwarp();  // a half-warp reads back only the rows it wrote
#pragma unroll 2
    for (int t = 0; t < kSimtTok; t += 4) {
      float4 p[RPT];
#pragma unroll
      for (int i = 0; i < RPT; ++i) p[i] = *reinterpret_cast<const float4*>(&sm.p[ty + 16 * i][t]);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
#pragma unroll
        for (int cc = 0; cc < NC; ++cc) {
          const float4 vv = *reinterpret_cast<const float4*>(&sm.v[t + u][4 * tx + 64 * cc]);
#pragma unroll
          for (int i = 0; i < RPT; ++i) {
            const float pp = u == 0 ? p[i].x : u == 1 ? p[i].y : u == 2 ? p[i].z : p[i].w;
            o[i][4 * cc + 0] = fmaf(pp, vv.x, o[i][4 * cc + 0]);
            o[i][4 * cc + 1] = fmaf(pp, vv.y, o[i][4 * cc + 1]);
            o[i][4 * cc + 2] = fmaf(pp, vv.z, o[i][4 * cc + 2]);
            o[i][4 * cc + 3] = fmaf(pp, vv.w, o[i][4 * cc + 3]);
          }
        }
      }
    }
  }

  // results: the output itself when the keys are not split, else a partial
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int rl = ty + 16 * i, r = rt * RT + rl;
    if (r >= a.R) continue;
    if (a.nchunk > 1) {
      const int64_t part = ((int64_t)(bh * a.nrt + rt) * a.nchunk + c) * RT + rl;
      if (tx == 0) {
        a.pm[part] = m[i];
        a.pl[part] = l[i];
      }
      if (m[i] == -INFINITY) continue;
#pragma unroll
      for (int cc = 0; cc < NC; ++cc)
        *reinterpret_cast<float4*>(&a.po[part * D + 4 * tx + 64 * cc]) =
            make_float4(o[i][4 * cc], o[i][4 * cc + 1], o[i][4 * cc + 2], o[i][4 * cc + 3]);
      continue;
    }
    const float inv = l[i] > 0.f ? 1.f / l[i] : (l[i] == 0.f ? 0.f : l[i]);  // NaN stays NaN
    if (a.lse && tx == 0) a.lse[(int64_t)bh * a.R + r] = l[i] == 0.f ? INFINITY : m[i] + log2f(l[i]);
    const int64_t at = tok_q_offset(a, b, h, r, D);
#pragma unroll
    for (int cc = 0; cc < NC; ++cc)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float val = o[i][4 * cc + y] * inv;
        if (a.out_dtype == OC_BF16)
          static_cast<__nv_bfloat16*>(a.out)[at + 4 * tx + 64 * cc + y] = __float2bfloat16_rn(val);
        else
          static_cast<float*>(a.out)[at + 4 * tx + 64 * cc + y] = val;
      }
  }
}

// One warp per query row: out = sum_c 2^(m_c - M) o_c / sum_c 2^(m_c - M) l_c.
template <int D>
__global__ void __launch_bounds__(128) tok_merge_kernel(const TokArgs a, int row_tile) {
  pdl_wait();
  const int64_t gr = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (gr >= (int64_t)a.B * a.Hkv * a.R) return;
  const int bh = (int)(gr / a.R), r = (int)(gr % a.R);
  const int rt = r / row_tile, rl = r % row_tile;
  const int64_t base = (int64_t)(bh * a.nrt + rt) * a.nchunk;
  float M = -INFINITY;
  for (int c = lane; c < a.nchunk; c += 32) M = fmaxf(M, a.pm[(base + c) * row_tile + rl]);
  M = warp_max(M);
  float o[D / 32], L = 0.f;
#pragma unroll
  for (int x = 0; x < D / 32; ++x) o[x] = 0.f;
  const float ref = M == -INFINITY ? 0.f : M;
  for (int c = 0; c < a.nchunk; ++c) {
    const int64_t part = (base + c) * row_tile + rl;
    const float mc = a.pm[part];
    if (mc == -INFINITY) {
      L += a.pl[part];  // 0, or NaN when every visible score was NaN
      continue;
    }
    const float w = exp2f(mc - ref);
    L += w * a.pl[part];
#pragma unroll
    for (int x = 0; x < D / 128 + (D < 128); ++x) {
      constexpr int kV = D < 128 ? 2 : 4;
#pragma unroll
      for (int y = 0; y < kV; ++y) o[x * kV + y] += w * a.po[part * D + x * 32 * kV + lane * kV + y];
    }
  }
  if (a.lse && lane == 0) a.lse[gr] = L == 0.f ? INFINITY : M + log2f(L);
  const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
  const int64_t at = tok_q_offset(a, bh / a.Hkv, bh % a.Hkv, r, D);
#pragma unroll
  for (int x = 0; x < D / 128 + (D < 128); ++x) {
    constexpr int kV = D < 128 ? 2 : 4;
#pragma unroll
    for (int y = 0; y < kV; ++y) {
      const int64_t e = at + x * 32 * kV + lane * kV + y;
      const float val = o[x * kV + y] * inv;
      if (a.out_dtype == OC_BF16)
        static_cast<__nv_bfloat16*>(a.out)[e] = __float2bfloat16_rn(val);
      else
        static_cast<float*>(a.out)[e] = val;
    }
  }
}

// Column sums of the softmax: for 64 keys of (b, h), the weights 2^(s - lse_r)
// of every query row, added in row order (no atomics: the same inputs give the
// same sums).  The scores are recomputed from q and k, since the softmax
// denominators are known only after all keys have been seen.
template <typename T, int D>
struct WeightSmem {
  float k[kSimtTok][D + 4];
  float q[32][D];
  TokRow row[32];
  float lse[32];
  float sum[16][kSimtTok];
};

template <typename T, int D>
__global__ void __launch_bounds__(kSimtThreads) tok_weights_kernel(const TokArgs a, const float* w_in, float* w_out) {
  extern __shared__ __align__(16) unsigned char raw[];
  WeightSmem<T, D>& sm = *reinterpret_cast<WeightSmem<T, D>*>(raw);
  constexpr int kVec = Elem<T>::kVec;
  const int bh = blockIdx.x % (a.B * a.Hkv), j0 = blockIdx.x / (a.B * a.Hkv) * kSimtTok;
  const int b = bh / a.Hkv, h = bh % a.Hkv;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int len = tok_len(a, b);
  for (int e = tid; e < kSimtTok * (D / kVec); e += kSimtThreads) {
    const int t = e / (D / kVec), x = e % (D / kVec) * kVec;
    if (j0 + t < len)
      simt_load_vec<T, D>(static_cast<const T*>(a.k) + (((int64_t)b * a.S + j0 + t) * a.Hkv + h) * D + x, &sm.k[t][x]);
    else
#pragma unroll
      for (int y = 0; y < kVec; ++y) sm.k[t][x + y] = 0.f;
  }
  pdl_wait();  // the softmax denominators come from the kernel before this one
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  // rows before the first position that sees key j0 have no weight here
  int first = 0;
  if (a.causal) first = max(0, j0 - (len - a.Sq)) * a.G;
  if (j0 >= len) first = a.R;
  for (int r0 = first; r0 < a.R; r0 += 32) {
    __syncthreads();
    if (tid < 32) {
      sm.row[tid] = tok_row(a, b, h, r0 + tid, len);
      sm.lse[tid] = r0 + tid < a.R ? a.lse[(int64_t)bh * a.R + r0 + tid] : INFINITY;
    }
    for (int e = tid; e < 32 * (D / kVec); e += kSimtThreads) {
      const int r = e / (D / kVec), x = e % (D / kVec) * kVec;
      if (r0 + r < a.R)
        simt_load_vec<T, D>(static_cast<const T*>(a.q) + tok_q_offset(a, b, h, r0 + r, D) + x, &sm.q[r][x]);
      else
#pragma unroll
        for (int y = 0; y < kVec; ++y) sm.q[r][x + y] = 0.f;
    }
    __syncthreads();
    float s[2][4] = {};
#pragma unroll 4
    for (int x = 0; x < D; x += 4) {
      float4 kk[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) kk[n] = *reinterpret_cast<const float4*>(&sm.k[tx + 16 * n][x]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 qq = *reinterpret_cast<const float4*>(&sm.q[ty + 16 * i][x]);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          s[i][n] = fmaf(qq.x, kk[n].x, s[i][n]);
          s[i][n] = fmaf(qq.y, kk[n].y, s[i][n]);
          s[i][n] = fmaf(qq.z, kk[n].z, s[i][n]);
          s[i][n] = fmaf(qq.w, kk[n].w, s[i][n]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const TokRow row = sm.row[ty + 16 * i];
      const float lse = sm.lse[ty + 16 * i];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int j = j0 + tx + 16 * n;
        if (j < row.hi && lse != INFINITY) acc[n] += exp2f(tok_score(a, s[i][n], row.slope2, row.pos, j) - lse);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < 4; ++n) sm.sum[ty][tx + 16 * n] = acc[n];
  __syncthreads();
  if (tid < kSimtTok && j0 + tid < a.S) {
    const int64_t at = (int64_t)bh * a.S + j0 + tid;
    float w = 0.f;
#pragma unroll
    for (int y = 0; y < 16; ++y) w += sm.sum[y][tid];
    w_out[at] = (w_in ? w_in[at] : 0.f) + w;
  }
}

// Column sums from stored scores (few rows): a thread per key, rows in order.
__global__ void __launch_bounds__(256) tok_sum_kernel(const TokArgs a, const float* w_in, float* w_out) {
  const int bh = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x;
  if (j >= a.S) return;
  const int64_t at = (int64_t)bh * a.S + j;
  const int len = tok_len(a, bh / a.Hkv);
  pdl_wait();
  const float before = w_in ? w_in[at] : 0.f;
  float sum = 0.f;
  if (j < len) {
    const float* s = a.logits + (int64_t)bh * a.R * a.logit_stride + j;
#pragma unroll 8
    for (int r = 0; r < a.R; ++r) sum += exp2f(s[r * a.logit_stride] - a.lse[(int64_t)bh * a.R + r]);
  }
  w_out[at] = before + sum;
}

}  // namespace

int tok_merge(const TokArgs& a, int head_dim, int row_tile, cudaStream_t st) {
  const int64_t rows = (int64_t)a.B * a.Hkv * a.R;
  const dim3 grid((unsigned)((rows + 3) / 4));
  cudaError_t e;
  if (head_dim == 64)
    e = launch_pdl(tok_merge_kernel<64>, grid, dim3(128), 0, st, a, row_tile);
  else if (head_dim == 128)
    e = launch_pdl(tok_merge_kernel<128>, grid, dim3(128), 0, st, a, row_tile);
  else
    e = launch_pdl(tok_merge_kernel<256>, grid, dim3(128), 0, st, a, row_tile);
  if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "tok_merge_kernel: %s", cudaGetErrorString(e));
  return OC_OK;
}

namespace {

// How a call is cut.
struct TokPlan {
  bool tc;            // the tcgen05 kernel
  int row_tile, nrt;  // rows per tile, row tiles per (b, h)
  int chunk, nchunk;  // keys per chunk, chunks
  size_t lse_off, m_off, l_off, o_off, prep_off, logit_off, logit_stride, bytes;  // logit_stride 0: none
};

inline size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// Kernel: float32 takes the float32-arithmetic kernel (row tiles of 16 or 64);
// bfloat16 the m16n8k16 kernel (16, 32 or 64 rows, what the rows fill) or, for
// more than kTcRows rows per KV head at head_dim 64 and 128, the tcgen05 one.
//
// Split of the keys: the CTAs of all (row tile, batch row, KV head, chunk) run
// in waves of one (tcgen05) or two per SM; of the possible numbers of chunks
// the one with the least waves x (keys of a chunk + what a CTA's set-up costs, in
// keys) plus the traffic of the partials is taken.  Row tiles of a causal chunk
// as long as a good part of its sequence differ in work and fill the SMs evenly
// by themselves; documents shorten the spans to a length the host does not
// know: then keys are split only while there are fewer row tiles than SMs.
constexpr int kTcRows = 64;

// The accumulating form needs every score again once the denominators are
// known.  Up to kLogitRows rows per KV head the bfloat16 kernel stores them
// (4 bytes a row and key, against 2 D bytes of a key to multiply again: at 16
// rows and 128 channels 64 against 256); beyond, they are recomputed.
constexpr int kLogitRows = 16;

TokPlan tok_plan(int dtype, int batch, int q_len, int q_heads, int kv_heads, int head_dim, int seq_len, float scale,
                 bool uneven, bool lse) {
  TokPlan p;
  const int G = q_heads / kv_heads;
  const int64_t R = (int64_t)q_len * G;
  p.tc = dtype == OC_BF16 && head_dim <= 128 && R > kTcRows && scale > 0.f;
  int64_t units, slots = device_sm_count();
  int step, setup;
  if (p.tc) {
    units = (int64_t)batch * kv_heads * tok_tc_shape(q_len, G).npairs;
    p.row_tile = (int)R;
    p.nrt = 1;
    step = 128;
    setup = 512;
  } else {
    p.row_tile = R <= 16 ? 16 : R <= 32 ? (dtype == OC_BF16 ? 32 : 16) : 64;
    p.nrt = (int)((R + p.row_tile - 1) / p.row_tile);
    units = (int64_t)batch * kv_heads * p.nrt;
    slots *= 2;
    step = 64;
    setup = dtype == OC_BF16 ? 160 : 32;
  }
  int64_t most = seq_len / (2 * step);
  if (most > 2 * slots / units + 4) most = 2 * slots / units + 4;
  if (uneven && units >= slots) most = 1;
  // partials: rows x head_dim floats written and read at about 6 TB/s, in keys of
  // one CTA (the tcgen05 kernel takes 67 keys a microsecond, the others less)
  const double part_keys = p.tc ? 256.0 * head_dim * 8 / 6e6 * 67 : 0.0;
  double best = 0;
  p.nchunk = 1;
  p.chunk = seq_len < step ? step : (seq_len + step - 1) / step * step;
  for (int64_t n = 1; n <= most; ++n) {
    const int64_t keys = ((seq_len + n - 1) / n + step - 1) / step * step;
    const double cost =
        (double)((units * n + slots - 1) / slots) * (keys + (n > 1 ? setup : 0)) + (n > 1 ? units * n * part_keys : 0);
    if (n == 1 || cost < best) {
      best = cost;
      p.chunk = (int)keys;
      p.nchunk = (int)((seq_len + keys - 1) / keys);
    }
  }
  if (p.nchunk < 1) p.nchunk = 1;
  const size_t parts = p.nchunk > 1 ? (size_t)batch * kv_heads * p.nrt * p.nchunk * p.row_tile : 0;
  size_t off = 0;
  p.lse_off = off;
  if (lse) off += up256((size_t)batch * kv_heads * R * sizeof(float));
  p.m_off = off;
  off += up256(parts * sizeof(float));
  p.l_off = off;
  off += up256(parts * sizeof(float));
  p.o_off = off;
  off += up256(parts * head_dim * sizeof(float));
  p.prep_off = off;
  if (p.tc) off += up256(tok_tc_prep_bytes(batch, q_len, G, seq_len));
  p.logit_off = off;
  p.logit_stride = 0;
  if (lse && dtype == OC_BF16 && R <= kLogitRows) {
    p.logit_stride = (seq_len + 63) / 64 * 64;  // whole tiles
    off += up256((size_t)batch * kv_heads * R * p.logit_stride * sizeof(float));
  }
  p.bytes = off;
  return p;
}

template <typename T, int D, int RPT>
int launch_simt(const TokArgs& a, cudaStream_t st) {
  const size_t smem = sizeof(SimtSmem<D, RPT>);
  static std::atomic<uint64_t> done{0};
  if (first_on_device(done)) {
    cudaError_t e = cudaFuncSetAttribute(tok_simt_kernel<T, D, RPT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem);
    if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "tok_simt_kernel: %s", cudaGetErrorString(e));
  }
  tok_simt_kernel<T, D, RPT><<<dim3((unsigned)(a.B * a.Hkv * a.nrt), (unsigned)a.nchunk), kSimtThreads, smem, st>>>(a);
  return check_launch("tok_simt_kernel");
}

template <typename T>
int dispatch_simt(const TokArgs& a, int D, int row_tile, cudaStream_t st) {
  if (D == 64) return row_tile == 16 ? launch_simt<T, 64, 1>(a, st) : launch_simt<T, 64, 4>(a, st);
  if (D == 128) return row_tile == 16 ? launch_simt<T, 128, 1>(a, st) : launch_simt<T, 128, 4>(a, st);
  return row_tile == 16 ? launch_simt<T, 256, 1>(a, st) : launch_simt<T, 256, 4>(a, st);
}

template <typename T, int D>
int launch_weights(const TokArgs& a, const float* w_in, float* w_out, cudaStream_t st) {
  const size_t smem = sizeof(WeightSmem<T, D>);
  static std::atomic<uint64_t> done{0};
  if (first_on_device(done)) {
    cudaError_t e = cudaFuncSetAttribute(tok_weights_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem);
    if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "tok_weights_kernel: %s", cudaGetErrorString(e));
  }
  const int64_t blocks = (int64_t)((a.S + kSimtTok - 1) / kSimtTok) * a.B * a.Hkv;
  cudaError_t e = launch_pdl(tok_weights_kernel<T, D>, dim3((unsigned)blocks), dim3(kSimtThreads), smem, st, a, w_in,
                             w_out);
  if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "tok_weights_kernel: %s", cudaGetErrorString(e));
  return OC_OK;
}

template <typename T>
int dispatch_weights(const TokArgs& a, int D, const float* w_in, float* w_out, cudaStream_t st) {
  if (D == 64) return launch_weights<T, 64>(a, w_in, w_out, st);
  if (D == 128) return launch_weights<T, 128>(a, w_in, w_out, st);
  return launch_weights<T, 256>(a, w_in, w_out, st);
}

// Checks shared by the three entry points; fills the sizes of `a`.
int tok_common(const char* fn, TokArgs& a, const void* q, const void* k, const void* v, int dtype, int batch,
               int q_len, int q_heads, int kv_heads, int head_dim, int seq_len, float cap, float scale, void* out,
               int out_dtype) {
  OC_REQUIRE(q && out && (seq_len == 0 || (k && v)), OC_ERR_NULL, "%s: NULL pointer", fn);
  OC_REQUIRE(dtype == OC_F32 || dtype == OC_BF16, OC_ERR_DTYPE, "%s: bad dtype %d", fn, dtype);
  OC_REQUIRE(out_dtype == OC_F32 || out_dtype == OC_BF16, OC_ERR_DTYPE, "%s: bad out dtype %d", fn, out_dtype);
  OC_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, OC_ERR_SHAPE,
             "%s: head_dim %d is not 64, 128 or 256", fn, head_dim);
  OC_REQUIRE(batch >= 1 && q_len >= 1, OC_ERR_SHAPE, "%s: batch %d, q_len %d", fn, batch, q_len);
  OC_REQUIRE(kv_heads >= 1 && q_heads >= kv_heads && q_heads % kv_heads == 0, OC_ERR_SHAPE,
             "%s: q_heads %d is not a multiple of kv_heads %d", fn, q_heads, kv_heads);
  OC_REQUIRE(seq_len >= 0, OC_ERR_SHAPE, "%s: seq_len %d", fn, seq_len);
  OC_REQUIRE((int64_t)batch * seq_len < INT32_MAX && (int64_t)batch * q_len * q_heads < INT32_MAX &&
                 (int64_t)seq_len + q_len < INT32_MAX,
             OC_ERR_SHAPE, "%s: too many rows", fn);
  OC_REQUIRE(isfinite(cap) && cap >= 0.f, OC_ERR_SHAPE, "%s: cap must be finite and >= 0 (0: none)", fn);
  OC_REQUIRE(isfinite(scale), OC_ERR_SHAPE, "%s: scale must be finite", fn);
  OC_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out), OC_ERR_ALIGN,
             "%s: q/k/v/out must be 16-byte aligned", fn);
  a = TokArgs{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.out_dtype = out_dtype;
  a.B = batch;
  a.Sq = q_len;
  a.Hq = q_heads;
  a.Hkv = kv_heads;
  a.G = q_heads / kv_heads;
  a.R = q_len * a.G;
  a.S = seq_len;
  a.cap = cap;
  a.scale = scale;
  return OC_OK;
}

int tok_run(const char* fn, TokArgs& a, int dtype, int head_dim, bool lse, void* workspace, size_t workspace_bytes,
            cudaStream_t st, const float* w_in = nullptr, float* w_out = nullptr) {
  const bool uneven = a.docs || (a.causal && a.Sq > a.S / 4);
  const TokPlan p = tok_plan(dtype, a.B, a.Sq, a.Hq, a.Hkv, head_dim, a.S, a.scale, uneven, lse);
  OC_REQUIRE((int64_t)a.B * a.Hkv * p.nchunk * (p.tc ? tok_tc_shape(a.Sq, a.G).npairs : p.nrt) < INT32_MAX &&
                 p.nchunk <= 65535,
             OC_ERR_SHAPE, "%s: too many work units", fn);
  OC_REQUIRE(workspace_bytes >= p.bytes, OC_ERR_CAPACITY, "%s: workspace %zu < %zu bytes", fn, workspace_bytes,
             p.bytes);
  OC_REQUIRE(p.bytes == 0 || (workspace && aligned16(workspace)), p.bytes && !workspace ? OC_ERR_NULL : OC_ERR_ALIGN,
             "%s: workspace must be a 16-byte aligned device pointer", fn);
  char* w = static_cast<char*>(workspace);
  a.nrt = p.nrt;
  a.chunk = p.chunk;
  a.nchunk = p.nchunk;
  a.pm = reinterpret_cast<float*>(w + p.m_off);
  a.pl = reinterpret_cast<float*>(w + p.l_off);
  a.po = reinterpret_cast<float*>(w + p.o_off);
  a.lse = lse ? reinterpret_cast<float*>(w + p.lse_off) : nullptr;
  a.logits = p.logit_stride ? reinterpret_cast<float*>(w + p.logit_off) : nullptr;
  a.logit_stride = (int64_t)p.logit_stride;
  int rc = p.tc ? tok_tc(fn, a, head_dim, w + p.prep_off, st)
           : dtype == OC_BF16 ? tok_mma(a, head_dim, p.row_tile, st)
                              : dispatch_simt<float>(a, head_dim, p.row_tile, st);
  if (rc) return rc;
  if (p.nchunk > 1) rc = tok_merge(a, head_dim, p.row_tile, st);
  if (rc || !w_out || a.S == 0) return rc;
  // the column sums
  if (a.logits) {
    const dim3 grid((unsigned)((a.S + 255) / 256), (unsigned)(a.B * a.Hkv));
    OC_REQUIRE(grid.y <= 65535, OC_ERR_SHAPE, "%s: too many heads", fn);
    cudaError_t e = launch_pdl(tok_sum_kernel, grid, dim3(256), 0, st, a, w_in, w_out);
    if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "tok_sum_kernel: %s", cudaGetErrorString(e));
    return OC_OK;
  }
  if (dtype == OC_BF16 && head_dim <= 128 && a.scale > 0.f) return tok_tc_weights(fn, a, head_dim, w_in, w_out, st);
  return dtype == OC_BF16 ? dispatch_weights<__nv_bfloat16>(a, head_dim, w_in, w_out, st)
                          : dispatch_weights<float>(a, head_dim, w_in, w_out, st);
}

}  // namespace
}  // namespace oc

using namespace oc;

extern "C" size_t oc_token_attention_workspace_bytes(int dtype, int batch, int q_len, int q_heads, int kv_heads,
                                                     int head_dim, int seq_len, int accumulate) {
  if (batch < 1 || q_len < 1 || kv_heads < 1 || q_heads < kv_heads || q_heads % kv_heads || seq_len < 0 ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return 0;
  // the most that any call of these sizes needs
  size_t most = 0;
  for (int i = 0; i < 4; ++i) {
    const size_t n = tok_plan(dtype, batch, q_len, q_heads, kv_heads, head_dim, seq_len, i & 1 ? 1.f : 0.f, (i & 2) != 0,
                              accumulate != 0).bytes;
    if (n > most) most = n;
  }
  return most;
}

extern "C" int oc_tree_attention(const void* q, const void* k, const void* v, int dtype, const int32_t* block_table,
                                 int table_stride, int num_pages, int block_size, const int32_t* lengths,
                                 const void* draft_k, const void* draft_v, const uint8_t* tree_mask,
                                 int mask_batched, int batch, int nodes, int q_heads, int kv_heads, int head_dim,
                                 int seq_len, float cap, float scale, void* out, int out_dtype, void* workspace,
                                 size_t workspace_bytes, oc_stream_t stream) {
  TokArgs a;
  int rc = tok_common("oc_tree_attention", a, q, k, v, dtype, batch, nodes, q_heads, kv_heads, head_dim, seq_len, cap,
                      scale, out, out_dtype);
  if (rc) return rc;
  OC_REQUIRE(draft_k && draft_v && tree_mask, OC_ERR_NULL, "oc_tree_attention: NULL pointer");
  OC_REQUIRE(aligned16(draft_k) && aligned16(draft_v), OC_ERR_ALIGN,
             "oc_tree_attention: draft keys / values must be 16-byte aligned");
  OC_REQUIRE(nodes <= kMaxNodes, OC_ERR_CAPACITY, "oc_tree_attention: %d nodes, at most %d", nodes, kMaxNodes);
  if (block_table) {
    OC_REQUIRE(block_size >= 128 && block_size % 128 == 0, OC_ERR_SHAPE,
               "oc_tree_attention: block_size %d is not a multiple of 128", block_size);
    OC_REQUIRE(num_pages >= 1 && table_stride >= 0 && (int64_t)table_stride * block_size == seq_len, OC_ERR_SHAPE,
               "oc_tree_attention: table of %d pages of %d tokens, seq_len %d, num_pages %d", table_stride, block_size,
               seq_len, num_pages);
    OC_REQUIRE((int64_t)num_pages * block_size < INT32_MAX, OC_ERR_SHAPE, "oc_tree_attention: pool too large");
  }
  a.table = block_table;
  a.table_stride = table_stride;
  a.num_pages = num_pages;
  a.page = block_size;
  a.lengths = lengths;
  a.dk = draft_k;
  a.dv = draft_v;
  a.tree = tree_mask;
  a.tree_bstride = mask_batched ? (int64_t)nodes * nodes : 0;
  return tok_run("oc_tree_attention", a, dtype, head_dim, false, workspace, workspace_bytes,
                 reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int oc_chunk_attention(const void* q, const void* k, const void* v, int dtype, const int32_t* lengths,
                                  int causal, const int32_t* prefix, const int32_t* documents, const float* slopes,
                                  int batch, int q_len, int q_heads, int kv_heads, int head_dim, int seq_len,
                                  float cap, float scale, void* out, int out_dtype, void* workspace,
                                  size_t workspace_bytes, oc_stream_t stream) {
  TokArgs a;
  int rc = tok_common("oc_chunk_attention", a, q, k, v, dtype, batch, q_len, q_heads, kv_heads, head_dim, seq_len, cap,
                      scale, out, out_dtype);
  if (rc) return rc;
  a.lengths = lengths;
  a.causal = causal != 0;
  a.prefix = prefix;
  a.docs = documents;
  a.slopes = slopes;
  return tok_run("oc_chunk_attention", a, dtype, head_dim, false, workspace, workspace_bytes,
                 reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int oc_accumulate_attention(const void* q, const void* k, const void* v, int dtype, const int32_t* lengths,
                                       const float* weights_in, float* weights_out, int batch, int q_len, int q_heads,
                                       int kv_heads, int head_dim, int seq_len, float cap, float scale, void* out,
                                       int out_dtype, void* workspace, size_t workspace_bytes, oc_stream_t stream) {
  TokArgs a;
  int rc = tok_common("oc_accumulate_attention", a, q, k, v, dtype, batch, q_len, q_heads, kv_heads, head_dim, seq_len,
                      cap, scale, out, out_dtype);
  if (rc) return rc;
  OC_REQUIRE(weights_out || seq_len == 0, OC_ERR_NULL, "oc_accumulate_attention: NULL pointer");
  a.lengths = lengths;
  a.causal = 1;
  return tok_run("oc_accumulate_attention", a, dtype, head_dim, true, workspace, workspace_bytes,
                 reinterpret_cast<cudaStream_t>(stream), weights_in, weights_out);
}
