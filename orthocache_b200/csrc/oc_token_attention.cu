// Token-level attention: entry points, the float32 kernel for more than a few
// rows, the merge of partials split over the keys, and the column sums of the
// attention weights.
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

#include "oc_mma.cuh"
#include "oc_tma.cuh"
#include "oc_token.cuh"

namespace oc {
namespace {

constexpr int kSimtThreads = 256;
constexpr int kSimtTok = 64;  // keys per tile

// Rows are padded, so that the 16 keys a half-warp reads at once, and the rows of
// its two halves, fall into different banks.
template <int D, int kRpt>
struct SimtSmem {
  static constexpr int kStages = D == 64 ? 2 : 1;
  float q[16 * kRpt][D + 4];
  float k[kStages][kSimtTok][D + 4];
  float v[kStages][kSimtTok][D];
  float p[16 * kRpt][kSimtTok + 16];
  TokRow row[16 * kRpt];
  int doc[3][kSimtTok];
  int64_t src[3][kSimtTok];  // row of the key in its tensor, -1 for one that nobody sees
  int unseen[3];  // has the tile such keys?
  int hi, min_hi;
  int span[4];  // least and largest document of the rows, first key and last + 1 of those between
  int pre[kMaxEvenBatch + 1];
};

// Four floats to shared memory, or zeros.
__device__ __forceinline__ void simt_cp16(float* dst, const float* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(real ? 16 : 0)
               : "memory");
}

template <typename T>
__device__ __forceinline__ void simt_load_vec(const T* src, float* dst) {
  constexpr int kVec = Elem<T>::kVec;
  const uint4 w = *reinterpret_cast<const uint4*>(src);
  float f[kVec];
  unpack16<T>(w, f);
#pragma unroll
  for (int c = 0; c < kVec; ++c) dst[c] = f[c];
}

// Row tiles of 16 kRpt (64 or 128) query rows against tiles of 64 keys, one pass
// with the running maximum and sum of the softmax; 256 threads as 16 x 16: thread
// (ty, tx) owns rows ty + 16 i, the scores of keys tx + 16 n, and the output
// channels 4 tx + 64 c of its rows, so that the softmax statistics stay in
// registers (reduced over the 16 lanes of a half-warp).  Keys and values come by
// cp.async: at 64 channels the next tile while one is multiplied, beyond, where
// there is room for one, the next keys during the softmax and output of a tile and
// the next values during the scores.  Keys that no row may see (behind the
// sequence, padding, pages outside the pool) are filled with zeros, so that
// whatever the memory holds there cannot reach a result.  Bound by the FMA pipe and
// the latency of the shared-memory reads: 512 rows x 4K, 16 heads, D 128 take 435 us
// = 37 TFLOP/s (row tiles of 64: 562; loading each tile in turn and masking all of
// them: 784).
template <int D, int kRpt>
__global__ void __launch_bounds__(kSimtThreads, D == 64 ? 2 : 1) tok_simt_kernel(const TokArgs a) {
  extern __shared__ __align__(16) unsigned char raw[];
  using Smem = SimtSmem<D, kRpt>;
  Smem& sm = *reinterpret_cast<Smem*>(raw);
  constexpr int RT = 16 * kRpt, NC = D / 64, ST = Smem::kStages, kRow = D / 4;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const float* qbase = static_cast<const float*>(a.q);
  if (tok_followed(a)) pdl_trigger();  // the merge may find its parts meanwhile
  if (a.even) {
    if (tid < 32) tok_prefix(a, sm.pre);
    __syncthreads();
  }
  TokWalk walk(a, sm.pre, blockIdx.x);
  TokSeg seg;
  for (bool more = true; more;) {
    if (a.even) {
      if (!walk.next(a, sm.pre, blockIdx.x, seg)) break;
    } else {
      // a CTA per unit, the rows with most keys first
      const int bh = blockIdx.x % (a.B * a.Hkv);
      seg = TokSeg{bh / a.Hkv, bh % a.Hkv * a.nrt + a.nrt - 1 - (int)(blockIdx.x / (a.B * a.Hkv)), 0, INT32_MAX, -1};
      more = false;
    }
    const int b = seg.b, h = seg.unit / a.nrt, rt = seg.unit % a.nrt, bh = b * a.Hkv + h;
    const int len = tok_len(a, b);
    __syncthreads();  // the previous piece is done with shared memory
    if (tid == 0) {
      sm.hi = 0;
      sm.min_hi = INT32_MAX;
      sm.span[0] = sm.span[2] = INT32_MAX;
      sm.span[1] = sm.span[3] = -1;
    }
    for (int e = tid; e < RT * kRow; e += kSimtThreads) {
      const int r = e / kRow, x = e % kRow * 4;
      const bool real = rt * RT + r < a.R;
      simt_cp16(&sm.q[r][x], qbase + (real ? tok_q_offset(a, b, h, rt * RT + r, D) + x : 0), real);
    }
    __syncthreads();
    for (int r = tid; r < RT; r += kSimtThreads) {
      sm.row[r] = tok_row(a, b, h, rt * RT + r, len);
      if (rt * RT + r < a.R) {
        atomicMax(&sm.hi, sm.row[r].hi);
        atomicMin(&sm.min_hi, sm.row[r].hi);
        if (a.docs && sm.row[r].hi > 0) {
          atomicMin(&sm.span[0], sm.row[r].doc);
          atomicMax(&sm.span[1], sm.row[r].doc);
        }
      }
    }
    __syncthreads();
    const int nct = (len + kSimtTok - 1) / kSimtTok;  // tiles of the cache; drafted tokens follow
    int t0 = min(seg.t0, nct) * kSimtTok, t1 = max(t0, min(sm.hi, min(seg.t1, nct) * kSimtTok));
    if (a.docs && t0 < t1) {  // the tiles that hold any of the rows' documents
      int first = INT32_MAX, last = -1;
      for (int j = t0 + tid; j < t1; j += kSimtThreads) {
        const int d = a.docs[(size_t)b * a.S + j];
        if (d >= sm.span[0] && d <= sm.span[1]) {
          first = min(first, j);
          last = max(last, j + 1);
        }
      }
      if (last >= 0) {
        atomicMin(&sm.span[2], first);
        atomicMax(&sm.span[3], last);
      }
      __syncthreads();
      t1 = min(t1, max(t0, sm.span[3]));
      if (sm.span[2] < t1) t0 = sm.span[2] / kSimtTok * kSimtTok;
    }
    const int ncache = (t1 - t0 + kSimtTok - 1) / kSimtTok;
    const int d0 = max(seg.t0 - nct, 0);
    const int ndraft = a.dk && seg.t1 > nct ? min(seg.t1 - nct, (a.Sq + kSimtTok - 1) / kSimtTok) - d0 : 0;
    const int ntile = ncache + ndraft, min_hi = sm.min_hi;
    if (tid < 3) sm.unseen[tid] = -1;

    const auto first_key = [&](int tile) {
      return tile >= ncache ? (d0 + tile - ncache) * kSimtTok : t0 + tile * kSimtTok;
    };
    // where the tile's keys lie, and their documents
    const auto mark = [&](int tile) {
      if (tile >= ntile || tid >= kSimtTok) return;  // whole warps
      const int j = first_key(tile) + tid;
      int64_t src = -1;
      int doc = -1;
      if (tile >= ncache) {
        for (int i = 0; j < a.Sq && i < a.Sq && src < 0; ++i)
          if (a.tree[b * a.tree_bstride + (int64_t)i * a.Sq + j]) src = (int64_t)b * a.Sq + j;
      } else if (j < len) {
        doc = a.docs ? a.docs[(size_t)b * a.S + j] : 0;
        if (doc >= 0) src = tok_kv_row(a, b, j);
      }
      sm.doc[tile % 3][tid] = doc;
      sm.src[tile % 3][tid] = src;
      if (__any_sync(0xffffffffu, src < 0) && (tid & 31) == 0) sm.unseen[tile % 3] = tile;
    };
    const auto issue = [&](int tile, bool keys, bool values) {
      if (tile >= ntile) return;
      const float* kp = static_cast<const float*>(tile >= ncache ? a.dk : a.k);
      const float* vp = static_cast<const float*>(tile >= ncache ? a.dv : a.v);
#pragma unroll 4
      for (int e = tid; e < kSimtTok * kRow; e += kSimtThreads) {
        const int t = e / kRow, x = e % kRow * 4;
        const int64_t src = sm.src[tile % 3][t], at = (src * a.Hkv + h) * D + x;
        if (keys) simt_cp16(&sm.k[tile % ST][t][x], src >= 0 ? kp + at : qbase, src >= 0);
        if (values) simt_cp16(&sm.v[tile % ST][t][x], src >= 0 ? vp + at : qbase, src >= 0);
      }
    };
    const auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };

    TokRow rows[kRpt == 4 ? 4 : 1];  // in registers while there are enough
    const auto row_of = [&](int i) { return kRpt == 4 ? rows[kRpt == 4 ? i : 0] : sm.row[ty + 16 * i]; };
    float m[kRpt], l[kRpt], o[kRpt][NC * 4];
#pragma unroll
    for (int i = 0; i < kRpt; ++i) {
      if (kRpt == 4) rows[kRpt == 4 ? i : 0] = sm.row[ty + 16 * i];
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int x = 0; x < NC * 4; ++x) o[i][x] = 0.f;
    }

    __syncthreads();
    for (int t = 0; t < 2; ++t) mark(t);
    __syncthreads();
    issue(0, true, ST == 2);
    commit();
    if (ST == 1) {
      issue(0, false, true);
      commit();
    }
    for (int tile = 0; tile < ntile; ++tile) {
      const bool draft = tile >= ncache;
      const int j0 = first_key(tile);
      const int *doc = sm.doc[tile % 3];
      const int64_t* src = sm.src[tile % 3];
      const int at = tile % ST;
      if (ST == 2) {
        __syncthreads();  // the tile before is read
        issue(tile + 1, true, true);
        commit();
        mark(tile + 2);
      }
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncthreads();  // the keys are there
      const bool unseen = sm.unseen[tile % 3] == tile;

      float s[kRpt][4];
#pragma unroll
      for (int i = 0; i < kRpt; ++i)
#pragma unroll
        for (int n = 0; n < 4; ++n) s[i][n] = 0.f;
#pragma unroll 4
      for (int x = 0; x < D; x += 4) {
        float4 kk[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) kk[n] = *reinterpret_cast<const float4*>(&sm.k[at][tx + 16 * n][x]);
#pragma unroll
        for (int i = 0; i < kRpt; ++i) {
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
      if (ST == 1) {
        __syncthreads();  // the keys are read
        issue(tile + 1, true, false);
        commit();
      }
      // scale, cap, bias (natural units: log2(e) times a score would round once more,
      // and the exponential magnify that; here it multiplies the difference to the
      // maximum)
      const float in = a.cap > 0.f ? a.scale / a.cap : a.scale;
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < kRpt; ++i)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          s[i][n] *= in;
          top = fmaxf(top, fabsf(s[i][n]));
        }
      if (a.cap > 0.f) {
        if (__all_sync(0xffffffffu, top <= kTanhMax)) {  // (NaN may pass: it stays NaN)
#pragma unroll
          for (int i = 0; i < kRpt; ++i)
#pragma unroll
            for (int n = 0; n < 4; ++n) s[i][n] = a.cap * tok_tanh(s[i][n]);
        } else {
#pragma unroll
          for (int i = 0; i < kRpt; ++i)
#pragma unroll
            for (int n = 0; n < 4; ++n) s[i][n] = a.cap * tanhf(s[i][n]);
        }
      }
      if (a.slopes) {
#pragma unroll
        for (int i = 0; i < kRpt; ++i) {
          const TokRow row = row_of(i);
#pragma unroll
          for (int n = 0; n < 4; ++n)
            s[i][n] = fmaf(-row.slope2 * (1.f / kLog2e), fabsf((float)(row.pos - (j0 + tx + 16 * n))), s[i][n]);
        }
      }
      if (draft || a.docs || unseen || j0 + kSimtTok > min_hi) {  // else every row sees every key
#pragma unroll
        for (int i = 0; i < kRpt; ++i) {
          const TokRow row = row_of(i);
          const int r = rt * RT + ty + 16 * i;
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int t = tx + 16 * n, j = j0 + t;
            bool vis = src[t] >= 0;
            if (draft)
              vis = vis && r < a.R && a.tree[b * a.tree_bstride + (int64_t)(r / a.G) * a.Sq + j] != 0;
            else
              vis = vis && j < row.hi && (!a.docs || doc[t] == row.doc);
            if (!vis) s[i][n] = -INFINITY;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kRpt; ++i) {
        float mx = fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3]));
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        const float m_new = fmaxf(m[i], mx);
        const float base = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = exp2f((m[i] - base) * kLog2e);
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float p = exp2f((s[i][n] - base) * kLog2e);
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
      if (ST == 1) {
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncthreads();  // the values are there
      } else {
        __syncwarp();  // a half-warp reads back only the weights it wrote
      }
#pragma unroll 2
      for (int t = 0; t < kSimtTok; t += 4) {
        float4 p[kRpt];
#pragma unroll
        for (int i = 0; i < kRpt; ++i) p[i] = *reinterpret_cast<const float4*>(&sm.p[ty + 16 * i][t]);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
          for (int cc = 0; cc < NC; ++cc) {
            const float4 vv = *reinterpret_cast<const float4*>(&sm.v[at][t + u][4 * tx + 64 * cc]);
#pragma unroll
            for (int i = 0; i < kRpt; ++i) {
              const float pp = u == 0 ? p[i].x : u == 1 ? p[i].y : u == 2 ? p[i].z : p[i].w;
              o[i][4 * cc + 0] = fmaf(pp, vv.x, o[i][4 * cc + 0]);
              o[i][4 * cc + 1] = fmaf(pp, vv.y, o[i][4 * cc + 1]);
              o[i][4 * cc + 2] = fmaf(pp, vv.z, o[i][4 * cc + 2]);
              o[i][4 * cc + 3] = fmaf(pp, vv.w, o[i][4 * cc + 3]);
            }
          }
        }
      }
      if (ST == 1) {
        __syncthreads();  // the values are read
        issue(tile + 1, false, true);
        commit();
        mark(tile + 2);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");  // the queries of a piece without tiles

    // results: the output itself when the keys are not split, else a partial
#pragma unroll
    for (int i = 0; i < kRpt; ++i) {
      const int rl = ty + 16 * i, r = rt * RT + rl;
      if (r >= a.R) continue;
      if (seg.part >= 0) {
        const int64_t part = (int64_t)seg.part * RT + rl;
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
      if (a.lse && tx == 0) a.lse[(int64_t)bh * a.R + r] = l[i] == 0.f ? INFINITY : m[i] + logf(l[i]);
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
}

// out = sum_p 2^(m_p - M) o_p / sum_p 2^(m_p - M) l_p over the parts p of a row's
// unit.  A block takes rows of one unit (a unit without parts was written by its
// CTA): the parts are found once for all of them.  WPR warps share a row: eight
// when there are few rows with many parts, whose loads then run side by side,
// one when there are many rows.
constexpr int kMergeThreads = 256;
constexpr int kMergeMaxParts = 2 * 256;  // CTAs of the even cut, at most two per SM

template <int D, int WPR>
__global__ void __launch_bounds__(kMergeThreads) tok_merge_kernel(const TokArgs a, const TokTcShape tc, int blocks_per_unit) {
  __shared__ int s_part[kMergeMaxParts];
  __shared__ int s_tiles[3];  // tiles of a unit: of the rows before b, of all rows, of row b
  __shared__ float s_m[8], s_l[8], s_o[WPR > 1 ? 8 : 1][D];
  const int unit = blockIdx.x / blocks_per_unit, block = blockIdx.x % blocks_per_unit;
  const int upb = a.Hkv * a.nrt, b = unit / upb, h = unit % upb / a.nrt, rt = unit % a.nrt;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < 32) {
    int before = 0, all = 0, mine = 0;
    for (int y = lane; y < a.B; y += 32) {
      const int n = tok_tiles(a, y);
      all += n;
      if (y < b) before += n;
      if (y == b) mine = n;
    }
    all = __reduce_add_sync(0xffffffffu, all);
    before = __reduce_add_sync(0xffffffffu, before);
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) {
      s_tiles[0] = before;
      s_tiles[1] = all;
      s_tiles[2] = mine;
    }
  }
  __syncthreads();
  const int upg = a.Hkv / a.hg * a.nrt;
  const int start = upg * s_tiles[0] + (h / a.hg * a.nrt + rt) * s_tiles[2];
  const TokCut cut(a, upg * s_tiles[1]);
  const int c0 = cut.run(start), parts = cut.run(start + s_tiles[2] - 1) - c0 + 1;
  if (parts <= 1) {
    pdl_wait();  // what follows on the stream waits for this kernel alone, and through it for the partials' one
    return;
  }
  // a unit of one row tile has two partials of 128 rows a piece (both halves of its
  // CTA worked on it)
  const int sub = tc.per_unit == 2 && tc.npt * tc.nhs == 1 ? 2 : 1, nparts = parts * sub;
  for (int e = tid; e < nparts; e += kMergeThreads) {
    const int c = c0 + e / sub;
    s_part[e] = (2 * (c * a.hg + h % a.hg) + (cut.first(c) >= start ? 0 : 1)) * sub + e % sub;
  }
  __syncthreads();
  pdl_wait();

  constexpr int kV = D < 128 ? 2 : 4, kN = D / 32 / kV, kRows = 8 / WPR;  // rows of a block at a time
  const int rows = a.unit_rows / sub;
  for (int r0 = block * kRows; r0 < rows; r0 += blocks_per_unit * kRows) {
    const int rl = r0 + (WPR > 1 ? 0 : warp);
    // query row of local row rl of the unit
    int r;
    bool real = rl < rows;
    if (tc.Gp) {
      const int t = tc.per_unit * rt + rl / 128, i = t / tc.nhs * tc.P + rl % 128 / tc.Gp;
      real = real && t < tc.npt * tc.nhs && i < a.Sq;
      r = i * a.G + t % tc.nhs * tc.Gp + rl % 128 % tc.Gp;
    } else {
      r = rt * rows + rl;
      real = real && r < a.R;
    }
    if (!real) continue;  // with WPR > 1 the same for the whole block
    float M = -INFINITY, o[D / 32], L = 0.f;
#pragma unroll
    for (int x = 0; x < D / 32; ++x) o[x] = 0.f;
    // four parts at a time, everything of them requested at once
    for (int c = WPR > 1 ? warp : 0; c < nparts; c += 4 * WPR) {
      float mc[4], lc[4], v[4][D / 32];
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        mc[z] = -INFINITY;
        lc[z] = 0.f;
        if (c + z * WPR < nparts) {
          const int64_t part = (int64_t)s_part[c + z * WPR] * rows + rl;
          mc[z] = a.pm[part];
          lc[z] = a.pl[part];
#pragma unroll
          for (int x = 0; x < kN; ++x) {
            const float* src = a.po + part * D + x * 32 * kV + lane * kV;
            if (kV == 4)
              *reinterpret_cast<float4*>(&v[z][x * kV]) = *reinterpret_cast<const float4*>(src);
            else
              *reinterpret_cast<float2*>(&v[z][x * kV]) = *reinterpret_cast<const float2*>(src);
          }
        }
      }
      const float m_new = fmaxf(M, fmaxf(fmaxf(mc[0], mc[1]), fmaxf(mc[2], mc[3])));
      const float ref = m_new == -INFINITY ? 0.f : m_new, old = exp2f((M - ref) * a.unit);
      L *= old;
#pragma unroll
      for (int x = 0; x < D / 32; ++x) o[x] *= old;
      M = m_new;
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        const bool any = mc[z] != -INFINITY;  // else nothing was written but l: 0, or NaN when all its scores were
        const float w = any ? exp2f((mc[z] - ref) * a.unit) : 1.f;
        L += w * lc[z];
#pragma unroll
        for (int x = 0; x < D / 32; ++x)
          if (any) o[x] = fmaf(w, v[z][x], o[x]);
      }
    }
    if (WPR > 1) {  // add up the eight warps
      __syncthreads();
#pragma unroll
      for (int x = 0; x < kN; ++x)
#pragma unroll
        for (int y = 0; y < kV; ++y) s_o[warp][x * 32 * kV + lane * kV + y] = o[x * kV + y];
      if (lane == 0) {
        s_m[warp] = M;
        s_l[warp] = L;
      }
      __syncthreads();
      if (tid < D / 4) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        L = 0.f;
        M = s_m[0];
#pragma unroll
        for (int w = 1; w < 8; ++w) M = fmaxf(M, s_m[w]);
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          const float f = s_m[w] == -INFINITY ? 1.f : exp2f((s_m[w] - M) * a.unit);
          L += f * s_l[w];
#pragma unroll
          for (int y = 0; y < 4; ++y) acc[y] += f * s_o[w][4 * tid + y];
        }
        if (a.lse && tid == 0) a.lse[(int64_t)(b * a.Hkv + h) * a.R + r] = L == 0.f ? INFINITY : M + (a.unit == 1.f ? log2f(L) : logf(L));
        const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
        const int64_t at = tok_q_offset(a, b, h, r, D) + 4 * tid;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          if (a.out_dtype == OC_BF16)
            static_cast<__nv_bfloat16*>(a.out)[at + y] = __float2bfloat16_rn(acc[y] * inv);
          else
            static_cast<float*>(a.out)[at + y] = acc[y] * inv;
        }
      }
      continue;
    }
    if (a.lse && lane == 0) a.lse[(int64_t)(b * a.Hkv + h) * a.R + r] = L == 0.f ? INFINITY : M + (a.unit == 1.f ? log2f(L) : logf(L));
    const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
    const int64_t at = tok_q_offset(a, b, h, r, D);
#pragma unroll
    for (int x = 0; x < kN; ++x) {
      const int64_t e = at + x * 32 * kV + lane * kV;
      if (a.out_dtype == OC_BF16) {
#pragma unroll
        for (int y = 0; y < kV; y += 2)
          *reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(a.out) + e + y) =
              pack_bf16x2(o[x * kV + y] * inv, o[x * kV + y + 1] * inv);
      } else {
#pragma unroll
        for (int y = 0; y < kV; ++y) static_cast<float*>(a.out)[e + y] = o[x * kV + y] * inv;
      }
    }
  }
}

template <int D>
int launch_merge(const TokArgs& a, const TokTcShape& tc, cudaStream_t st) {
  const int units = a.B * a.Hkv * a.nrt;
  // rows of a unit that exist at most, and whether all rows together are few
  const int rows = a.R < a.unit_rows ? a.R : a.unit_rows;
  const bool few = (int64_t)units * rows <= 1184;
  int bpu = rows;
  if (!few) {  // about eight blocks per SM, at least a row per warp
    bpu = (1184 + units - 1) / units;
    if (bpu > (a.unit_rows + 7) / 8) bpu = (a.unit_rows + 7) / 8;
  }
  cudaError_t e = few ? launch_pdl(tok_merge_kernel<D, 8>, dim3(units * bpu), dim3(kMergeThreads), 0, st, a, tc, bpu)
                      : launch_pdl(tok_merge_kernel<D, 1>, dim3(units * bpu), dim3(kMergeThreads), 0, st, a, tc, bpu);
  if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "tok_merge_kernel: %s", cudaGetErrorString(e));
  return OC_OK;
}

// Column sums of the softmax: for 64 keys of (b, h), the weights 2^(s - lse_r)
// of every query row, added in row order (no atomics: the same inputs give the
// same sums).  The scores are recomputed from q and k, since the softmax
// denominators are known only after all keys have been seen.
template <typename T, int D, int RW>
struct WeightSmem {
  float k[kSimtTok][D + 4];
  float q[RW][D + 4];
  TokRow row[RW];
  float lse[RW];
  float sum[16][kSimtTok];
};

// RW query rows at a time: 64 (1,080 -> 931 us with the attention of 512 rows x 4K, 16
// heads, D 128), but 32 where there are no more (152 us against 177 for 20 rows x 8K, 4
// heads, D 256).
template <typename T, int D, int RW>
__global__ void __launch_bounds__(kSimtThreads) tok_weights_kernel(const TokArgs a, const float* w_in, float* w_out) {
  extern __shared__ __align__(16) unsigned char raw[];
  WeightSmem<T, D, RW>& sm = *reinterpret_cast<WeightSmem<T, D, RW>*>(raw);
  constexpr int kVec = Elem<T>::kVec;
  const int bh = blockIdx.x % (a.B * a.Hkv), j0 = blockIdx.x / (a.B * a.Hkv) * kSimtTok;
  const int b = bh / a.Hkv, h = bh % a.Hkv;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int len = tok_len(a, b);
  for (int e = tid; e < kSimtTok * (D / kVec); e += kSimtThreads) {
    const int t = e / (D / kVec), x = e % (D / kVec) * kVec;
    if (j0 + t < len)
      simt_load_vec<T>(static_cast<const T*>(a.k) + (((int64_t)b * a.S + j0 + t) * a.Hkv + h) * D + x, &sm.k[t][x]);
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
  for (int r0 = first; r0 < a.R; r0 += RW) {
    __syncthreads();
    if (tid < RW) {
      sm.row[tid] = tok_row(a, b, h, r0 + tid, len);
      sm.lse[tid] = r0 + tid < a.R ? a.lse[(int64_t)bh * a.R + r0 + tid] * (a.unit / kLog2e) : INFINITY;  // natural
    }
    for (int e = tid; e < RW * (D / kVec); e += kSimtThreads) {
      const int r = e / (D / kVec), x = e % (D / kVec) * kVec;
      if (r0 + r < a.R)
        simt_load_vec<T>(static_cast<const T*>(a.q) + tok_q_offset(a, b, h, r0 + r, D) + x, &sm.q[r][x]);
      else
#pragma unroll
        for (int y = 0; y < kVec; ++y) sm.q[r][x + y] = 0.f;
    }
    __syncthreads();
    float s[RW / 16][4] = {};
#pragma unroll 4
    for (int x = 0; x < D; x += 4) {
      float4 kk[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) kk[n] = *reinterpret_cast<const float4*>(&sm.k[tx + 16 * n][x]);
#pragma unroll
      for (int i = 0; i < RW / 16; ++i) {
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
    for (int i = 0; i < RW / 16; ++i) {
      const TokRow row = sm.row[ty + 16 * i];
      const float lse = sm.lse[ty + 16 * i];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int j = j0 + tx + 16 * n;
        if (j < row.hi && lse != INFINITY) acc[n] += exp2f((tok_score(a, s[i][n], row.slope2, row.pos, j) - lse) * kLog2e);
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

// Column sums from stored scores (few rows): a thread per key, rows in order, from the
// first that sees the key on.  Rows before it may lie in a unit that ends before the
// key, whose scores nobody has stored.  Bound by the latency of its reads (32 rows x
// 32K, 8 heads 11.5 us, 4 rows x 64K 9): only blocks at the end of the sequence start at
// a row of each key's own (in all blocks: 17 and 11 us).
__global__ void __launch_bounds__(256) tok_sum_kernel(const TokArgs a, int blocks, const float* w_in,
                                                      float* w_out) {
  const int bh = blockIdx.x / blocks, j0 = blockIdx.x % blocks * 256, j = j0 + threadIdx.x;
  if (j >= a.S) return;
  const int64_t at = (int64_t)bh * a.S + j;
  const int len = tok_len(a, bh / a.Hkv);
  pdl_wait();
  const float before = w_in ? w_in[at] : 0.f;
  float sum = 0.f;
  if (j < len) {
    const float* s = a.logits + (int64_t)bh * a.R * a.logit_stride + j;
    const float* lse = a.lse + (int64_t)bh * a.R;
    const int all = len - a.Sq;  // keys up to this one are seen by every row
    if (j0 + 255 <= all) {
#pragma unroll 8
      for (int r = 0; r < a.R; ++r) sum += exp2f((s[r * a.logit_stride] - lse[r]) * a.unit);
    } else {  // eight rows requested at a time, of those that are stored
      const int first = max(0, j - all) * a.G;
      for (int r = 0; r < a.R; r += 8) {
        float x[8];
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          const int row = min(max(r + y, first), a.R - 1);
          x[y] = s[row * a.logit_stride] - lse[row];
        }
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          const float e = exp2f(x[y] * a.unit);
          if (r + y >= first && r + y < a.R) sum += e;
        }
      }
    }
  }
  w_out[at] = before + sum;
}

}  // namespace

int tok_merge(const TokArgs& a, int head_dim, bool tc, cudaStream_t st) {
  const TokTcShape shape = tc ? tok_tc_shape(a.Sq, a.G, head_dim) : TokTcShape{};
  return head_dim == 64 ? launch_merge<64>(a, shape, st)
                        : head_dim == 128 ? launch_merge<128>(a, shape, st) : launch_merge<256>(a, shape, st);
}

namespace {

// How a call is cut.
struct TokPlan {
  bool tc, even;                          // the tcgen05 kernel; the even cut of the keys
  int row_tile, nrt, unit_rows;           // rows per tile, units per (b, h), rows of a unit
  int tile, ncta, hg;                     // keys per tile, CTAs of the even cut, heads cut alike
  int64_t units;
  size_t lse_off, m_off, l_off, o_off, prep_off, logit_off, logit_stride, bytes;  // logit_stride 0: none
};

inline size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// Kernel: float32 takes the one for few rows (units of 16) up to 32 rows, beyond the
// one with row tiles of 64 or 128 (16K tokens, 4 KV heads: 32 rows take 44 and 52 us at 64
// channels, 69 and 89 at 128, 116 and 144 at 256; 36 rows 58 and 52, 95 and 87, 163
// and 146).  bfloat16 takes the m16n8k16 kernel (16, 32 or 64 rows, what the rows
// fill) or the tcgen05 one, from the rows on where it is the faster (a tree over 64K
// tokens, 8 KV heads: at 128 channels 32 rows take 69 and 77 us, 64 rows 108 and 77;
// at 64 channels 48 rows 54 and 56, 96 rows 75 and 58; 32K tokens, 16 heads of 256
// channels: 16 rows 114 and 134, 24 rows 187 and 134).
//
// Cut: with few units (row tile, batch row, KV head) for the GPU, all their key
// tiles are dealt out evenly over one (tcgen05) or two CTAs per SM, so that
// ragged lengths and odd numbers of units cost nothing but the partials: at most
// two per CTA.  From four waves of units on, each is a CTA's own; from one wave on
// too where the units differ in work anyway (a causal chunk as long as a good
// part of its sequence; documents), since the dealing goes by length, and where
// a unit has fewer than eight tiles.  A CTA takes at least kMinTiles tiles, below
// which its set-up outweighs them.
constexpr int kMinTiles = 2;

// The accumulating form needs every score again once the denominators are
// known.  Up to kLogitRows rows per KV head the kernels for few rows store them (4
// bytes a row and key, against 2 D or 4 D bytes of a key to multiply again);
// beyond, they are recomputed.  Stored and recomputed, bfloat16: 32 rows x 32K, 8
// heads, D 128 take 57 and 77 us, 24 rows x 16K, 2 x 4 heads, D 64 32 and 48;
// float32: 239 and 337, 83 and 103.  Not where a positive scale takes the tcgen05
// kernel anyway, and in 512 MiB at most, so that no call needs the memory of its keys
// once more: a batch with more of them goes by groups of its rows (16 x 32 rows x 32K,
// 16 heads, D 128, bfloat16: three groups 1,111 us, at once with 1 GiB 1,102; half as many
// recomputed 776, stored 541).
constexpr int kLogitRows = 32;
constexpr size_t kLogitBytes = (size_t)512 << 20;

// Rows that the kernels for few rows take.
inline bool tok_few_rows(int dtype, int64_t R, int head_dim) {
  return dtype == OC_F32 || R <= (head_dim == 64 ? 64 : head_dim == 128 ? 32 : 16);
}

inline size_t tok_logit_stride(int seq_len) { return ((size_t)seq_len + 63) / 64 * 64; }  // whole tiles

// Batch rows of one pass of the accumulating form: all of them, or as many as have
// their scores stored within kLogitBytes.
int tok_batch_group(int dtype, int batch, int q_len, int q_heads, int kv_heads, int head_dim, int seq_len) {
  const int64_t R = (int64_t)q_len * (q_heads / kv_heads);
  if (R > kLogitRows || !tok_few_rows(dtype, R, head_dim) || seq_len == 0) return batch;
  const size_t n = kLogitBytes / ((size_t)kv_heads * R * tok_logit_stride(seq_len) * sizeof(float));
  if (n < 1 || n >= (size_t)batch) return batch;
  const int groups = (batch + (int)n - 1) / (int)n;
  return (batch + groups - 1) / groups;
}

TokPlan tok_plan(int dtype, int batch, int q_len, int q_heads, int kv_heads, int head_dim, int seq_len, int draft_len,
                 float scale, bool uneven, bool docs, bool lse) {
  TokPlan p;
  const int G = q_heads / kv_heads;
  const int64_t R = (int64_t)q_len * G;
  const bool few = tok_few_rows(dtype, R, head_dim);
  p.tc = !few && scale > 0.f;
  int64_t slots = device_sm_count();
  if (p.tc) {
    p.row_tile = 128;
    const TokTcShape shape = tok_tc_shape(q_len, G, head_dim);
    p.nrt = shape.units;
    p.unit_rows = 128 * shape.per_unit;
    p.tile = 128;
  } else {
    p.row_tile = R <= 16 ? 16 : R <= 32 ? (dtype == OC_BF16 ? 32 : 16) : 64;
    // float32 with 128 channels: a tile of 128 rows takes about 3/2 the time of one of
    // 64 (72 rows x 16K, 2 heads: 83 and 95 us), but visits more keys of other documents
    // (200-token documents: 111 and 71 us)
    if (dtype == OC_F32 && head_dim == 128 && R > 64 && !docs && 3 * ((R + 127) / 128) < 2 * ((R + 63) / 64))
      p.row_tile = 128;
    p.nrt = (int)((R + p.row_tile - 1) / p.row_tile);
    p.unit_rows = p.row_tile;
    p.tile = dtype == OC_BF16 ? tok_mma_tile(head_dim) : p.row_tile == 16 ? tok_few_tile(head_dim) : kSimtTok;
    // CTAs that an SM's shared memory holds
    slots *= dtype == OC_BF16 || head_dim == 64 || (head_dim == 128 && p.row_tile == 16) ? 2 : 1;
  }
  p.units = (int64_t)batch * kv_heads * p.nrt;
  const int64_t tiles = p.units * ((seq_len + p.tile - 1) / p.tile + (draft_len + p.tile - 1) / p.tile);
  int64_t ncta = tiles / kMinTiles;
  if (ncta > slots) ncta = slots;
  if (ncta > kMergeMaxParts) ncta = kMergeMaxParts;
  p.even = batch <= kMaxEvenBatch && tiles < (1 << 30) && (p.units < slots ? ncta > p.units
                                      : !uneven && p.units < 4 * slots && tiles >= 8 * p.units);
  p.hg = 1;
  for (int g = 2; g <= 8; ++g)
    if (kv_heads % g == 0 && g <= ncta) p.hg = g;
  p.ncta = (int)(ncta < 1 ? 1 : ncta / p.hg * p.hg);
  const size_t parts = p.even ? (size_t)2 * p.ncta * p.unit_rows : 0;
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
  if (p.tc) off += up256(tok_tc_prep_bytes(batch, q_len, G, head_dim, seq_len));
  p.logit_off = off;
  p.logit_stride = 0;
  if (lse && few && R <= kLogitRows) {
    const size_t stride = tok_logit_stride(seq_len);
    const size_t logit_bytes = (size_t)batch * kv_heads * R * stride * sizeof(float);
    if (logit_bytes <= kLogitBytes) {
      p.logit_stride = stride;
      off += up256(logit_bytes);
    }
  }
  p.bytes = off;
  return p;
}

template <int D, int kRpt>
int launch_simt(const TokArgs& a, cudaStream_t st) {
  const size_t smem = sizeof(SimtSmem<D, kRpt>);
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(done, tok_simt_kernel<D, kRpt>, smem);
  if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "tok_simt_kernel: %s", cudaGetErrorString(e));
  tok_simt_kernel<D, kRpt><<<a.even ? a.ncta : a.B * a.Hkv * a.nrt, kSimtThreads, smem, st>>>(a);
  return check_launch("tok_simt_kernel");
}

int dispatch_simt(const TokArgs& a, int D, int row_tile, cudaStream_t st) {
  if (D == 64) return launch_simt<64, 4>(a, st);
  if (D == 128) return row_tile == 64 ? launch_simt<128, 4>(a, st) : launch_simt<128, 8>(a, st);
  return launch_simt<256, 4>(a, st);
}

template <typename T, int D, int RW>
int launch_weights(const TokArgs& a, const float* w_in, float* w_out, cudaStream_t st) {
  const size_t smem = sizeof(WeightSmem<T, D, RW>);
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(done, tok_weights_kernel<T, D, RW>, smem);
  if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "tok_weights_kernel: %s", cudaGetErrorString(e));
  const int64_t blocks = (int64_t)((a.S + kSimtTok - 1) / kSimtTok) * a.B * a.Hkv;
  e = launch_pdl(tok_weights_kernel<T, D, RW>, dim3((unsigned)blocks), dim3(kSimtThreads), smem, st, a, w_in, w_out);
  if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "tok_weights_kernel: %s", cudaGetErrorString(e));
  return OC_OK;
}

template <typename T>
int dispatch_weights(const TokArgs& a, int D, const float* w_in, float* w_out, cudaStream_t st) {
  const bool few = a.R <= 32;
  if (D == 64) return few ? launch_weights<T, 64, 32>(a, w_in, w_out, st) : launch_weights<T, 64, 64>(a, w_in, w_out, st);
  if (D == 128)
    return few ? launch_weights<T, 128, 32>(a, w_in, w_out, st) : launch_weights<T, 128, 64>(a, w_in, w_out, st);
  return few ? launch_weights<T, 256, 32>(a, w_in, w_out, st) : launch_weights<T, 256, 64>(a, w_in, w_out, st);
}

constexpr float kMaxScaleOfCap = 4096.f;

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
  // the cap's polynomials have coefficients up to scale (scale / cap)^8
  OC_REQUIRE(cap == 0.f || fabsf(scale) <= kMaxScaleOfCap * cap, OC_ERR_SHAPE,
             "%s: cap %g is below a %gth of the scale %g", fn, cap, kMaxScaleOfCap, scale);
  OC_REQUIRE(cap == 0.f || fabsf(scale) <= kMaxScaleOfCap * kMaxScaleOfCap, OC_ERR_SHAPE, "%s: scale %g with a cap", fn,
             scale);
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
  const TokPlan p = tok_plan(dtype, a.B, a.Sq, a.Hq, a.Hkv, head_dim, a.S, a.dk ? a.Sq : 0, a.scale, uneven,
                            a.docs != nullptr, lse);
  OC_REQUIRE(p.units < INT32_MAX, OC_ERR_SHAPE, "%s: too many work units", fn);
  OC_REQUIRE(workspace_bytes >= p.bytes, OC_ERR_CAPACITY, "%s: workspace %zu < %zu bytes", fn, workspace_bytes,
             p.bytes);
  OC_REQUIRE(p.bytes == 0 || (workspace && aligned16(workspace)), p.bytes && !workspace ? OC_ERR_NULL : OC_ERR_ALIGN,
             "%s: workspace must be a 16-byte aligned device pointer", fn);
  char* w = static_cast<char*>(workspace);
  a.nrt = p.nrt;
  a.even = p.even;
  a.ncta = p.ncta;
  a.hg = p.hg;
  a.tile = p.tile;
  a.unit_rows = p.unit_rows;
  a.pm = reinterpret_cast<float*>(w + p.m_off);
  a.pl = reinterpret_cast<float*>(w + p.l_off);
  a.po = reinterpret_cast<float*>(w + p.o_off);
  a.lse = lse ? reinterpret_cast<float*>(w + p.lse_off) : nullptr;
  a.logits = p.logit_stride ? reinterpret_cast<float*>(w + p.logit_off) : nullptr;
  a.logit_stride = (int64_t)p.logit_stride;
  a.unit = dtype == OC_BF16 ? 1.f : kLog2e;
  int rc = p.tc ? tok_tc(fn, a, head_dim, w + p.prep_off, st)
           : dtype == OC_BF16 ? tok_mma(a, head_dim, p.row_tile, st)
           : p.row_tile == 16 ? tok_few(a, head_dim, st)
                              : dispatch_simt(a, head_dim, p.row_tile, st);
  if (rc) return rc;
  if (p.even) rc = tok_merge(a, head_dim, p.tc, st);
  if (rc || !w_out || a.S == 0) return rc;
  // the column sums
  if (a.logits) {
    const int blocks = (a.S + 255) / 256;  // per (b, h); fewer than 2^31 / 256 for all b
    cudaError_t e = launch_pdl(tok_sum_kernel, dim3((unsigned)blocks * a.B * a.Hkv), dim3(256), 0, st, a, blocks, w_in,
                               w_out);
    if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "tok_sum_kernel: %s", cudaGetErrorString(e));
    return OC_OK;
  }
  if (dtype == OC_BF16 && a.scale > 0.f) return tok_tc_weights(fn, a, head_dim, w_in, w_out, st);
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
  const int group = accumulate ? tok_batch_group(dtype, batch, q_len, q_heads, kv_heads, head_dim, seq_len) : batch;
  size_t most = 0;
  for (int i = 0; i < 32; ++i) {
    const int rows = i & 16 ? batch % group : group;  // the last group may be smaller
    if (rows == 0) continue;
    const size_t n = tok_plan(dtype, rows, q_len, q_heads, kv_heads, head_dim, seq_len, i & 4 ? q_len : 0,
                              i & 1 ? 1.f : 0.f, (i & 2) != 0, (i & 8) != 0, accumulate != 0).bytes;
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
  const uintptr_t wi = reinterpret_cast<uintptr_t>(weights_in), wo = reinterpret_cast<uintptr_t>(weights_out);
  const uintptr_t wn = (uintptr_t)batch * kv_heads * seq_len * sizeof(float);
  OC_REQUIRE(!weights_in || wi == wo || wi + wn <= wo || wo + wn <= wi, OC_ERR_SHAPE,
             "oc_accumulate_attention: weights_in overlaps weights_out in part");
  a.causal = 1;
  const int group = tok_batch_group(dtype, batch, q_len, q_heads, kv_heads, head_dim, seq_len);
  const size_t es = dtype == OC_BF16 ? 2 : 4, out_es = out_dtype == OC_BF16 ? 2 : 4;
  const size_t q_row = (size_t)q_len * q_heads * head_dim, k_row = (size_t)seq_len * kv_heads * head_dim;
  for (int b = 0; b < batch; b += group) {  // one after the other on the stream, in the same workspace
    TokArgs g = a;
    g.B = batch - b < group ? batch - b : group;
    g.q = static_cast<const char*>(q) + b * q_row * es;
    g.k = static_cast<const char*>(k) + b * k_row * es;
    g.v = static_cast<const char*>(v) + b * k_row * es;
    g.out = static_cast<char*>(out) + b * q_row * out_es;
    g.lengths = lengths ? lengths + b : nullptr;
    const size_t at = (size_t)b * kv_heads * seq_len;
    rc = tok_run("oc_accumulate_attention", g, dtype, head_dim, true, workspace, workspace_bytes,
                 reinterpret_cast<cudaStream_t>(stream), weights_in ? weights_in + at : nullptr, weights_out + at);
    if (rc) return rc;
  }
  return OC_OK;
}
