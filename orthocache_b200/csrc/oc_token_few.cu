// Token-level attention for few query rows per KV head (float32): decoded and
// drafted tokens, up to 16 rows a tile.
//
// Mathematics and masks: oc_token.cuh.  Bound by reading keys and values once
// where the rows are few; a 16-row tile takes 32 D multiply-adds per key on the
// FMA pipe, more than its bytes.  In between, shared memory is the narrow place:
// so every key and value element is read from it by one thread alone, which
// multiplies it with all RR rows (RR = 4, 8 or 16, what the rows fill), and only
// the queries and weights, the same for a whole warp, are read again.
//
// A tile of TOK tokens takes three steps, the next tile on its way meanwhile:
//   * scores: thread (token, channel group), RR partial dot products;
//   * softmax: a warp per row adds the groups' parts up, in order, keeps the
//     running maximum and sum of the row in registers and leaves the weights;
//   * output: thread (4 channels, token group), RR x 4 sums in registers, joined
//     over the token groups once, at the end.
// Measured (D = 128): 1 token x 64K, 8 heads 111 us = 4.8 TB/s; 4 rows a head x 16K,
// 8 heads 41 us; 16 rows x 32K, 4 heads 68 us = 2 TB/s.  A register tile of 1 row x 4
// keys read keys and values from shared memory once per two rows: 315, 96 and 98 us.
// Three stages instead of two (119, 46 us at four rows), and three CTAs per SM (120,
// 44 us), are slower.
#include "oc_mma.cuh"
#include "oc_tma.cuh"
#include "oc_token.cuh"

namespace oc {
namespace {

constexpr int kFewThreads = 256;

template <int D>
struct FewShape {
  static constexpr int TOK = D == 64 ? 64 : 32, ST = 2;
  static constexpr int CG = kFewThreads / TOK, CW = D / CG;     // channel groups of the scores, channels of one
  static constexpr int KG = kFewThreads / (D / 4), KW = TOK / KG;  // token groups of the output, tokens of one
};

template <int D, int RR>
struct FewSmem {
  using C = FewShape<D>;
  union {
    struct {
      float k[C::ST][C::TOK][D + 4];  // padded: neighbouring tokens in different banks
      float v[C::ST][C::TOK][D];
    };
    float join[C::KG][RR][D];
  };
  float q[RR][D];
  float part[C::CG][RR][C::TOK];
  float p[RR][C::TOK];
  float alpha[RR], m[RR], l[RR];
  TokRow row[RR];
  int doc[C::ST + 1][C::TOK];
  int64_t src[C::ST + 1][C::TOK];  // row of the token in its tensor, -1 for one that nobody sees
  int hi, span[4];  // keys of the rows; their least and largest document, first key and last + 1 of those between
  int pre[kMaxEvenBatch + 1];
};

__device__ __forceinline__ void few_cp16(float* dst, const float* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(real ? 16 : 0)
               : "memory");
}

template <int D, int RR>
__global__ void __launch_bounds__(kFewThreads, D == 256 ? 1 : 2) tok_few_kernel(const TokArgs a) {
  extern __shared__ __align__(16) unsigned char raw[];
  using C = FewShape<D>;
  constexpr int TOK = C::TOK, ST = C::ST, kRow = D / 4, kMine = (RR + 7) / 8;  // rows of a warp in the softmax
  FewSmem<D, RR>& sm = *reinterpret_cast<FewSmem<D, RR>*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int tok = tid % TOK, cg = tid / TOK;        // scores
  const int xo = tid % kRow * 4, kg = tid / kRow;   // output
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
      const int u = blockIdx.x % (a.B * a.Hkv);
      seg = TokSeg{u / a.Hkv, u % a.Hkv * a.nrt + a.nrt - 1 - (int)(blockIdx.x / (a.B * a.Hkv)), 0, INT32_MAX, -1};
      more = false;
    }
    const int b = seg.b, h = seg.unit / a.nrt, rt = seg.unit % a.nrt, bh = b * a.Hkv + h;
    const int len = tok_len(a, b), r_first = rt * 16;  // a unit is 16 rows; RR < 16 when there are no more in all
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // the previous piece is done with shared memory
    if (tid == 0) {
      sm.hi = 0;
      sm.span[0] = sm.span[2] = INT32_MAX;
      sm.span[1] = sm.span[3] = -1;
    }
    for (int e = tid; e < RR * kRow; e += kFewThreads) {
      const int r = e / kRow, x = e % kRow * 4;
      const bool real = r_first + r < a.R;
      few_cp16(&sm.q[r][x], qbase + (real ? tok_q_offset(a, b, h, r_first + r, D) + x : 0), real);
    }
    __syncthreads();
    if (tid < RR) {
      const TokRow w = tok_row(a, b, h, r_first + tid, len);
      sm.row[tid] = w;
      if (w.hi > 0) {
        atomicMax(&sm.hi, w.hi);
        if (a.docs) {
          atomicMin(&sm.span[0], w.doc);
          atomicMax(&sm.span[1], w.doc);
        }
      }
    }
    __syncthreads();
    const int nct = (len + TOK - 1) / TOK;  // tiles of the cache; drafted tokens follow
    int t0 = min(seg.t0, nct) * TOK, t1 = max(t0, min(sm.hi, min(seg.t1, nct) * TOK));
    if (a.docs && t0 < t1) {  // the tiles that hold any of the rows' documents
      int first = INT32_MAX, last = -1;
      for (int j = t0 + tid; j < t1; j += kFewThreads) {
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
      if (sm.span[2] < t1) t0 = sm.span[2] / TOK * TOK;
    }
    const int ncache = (t1 - t0 + TOK - 1) / TOK;
    const int d0 = max(seg.t0 - nct, 0);
    const int ntile = ncache + (a.dk && seg.t1 > nct ? min(seg.t1 - nct, (a.Sq + TOK - 1) / TOK) - d0 : 0);

    const auto first_key = [&](int tile) { return tile >= ncache ? (d0 + tile - ncache) * TOK : t0 + tile * TOK; };
    // where the tile's tokens lie, and their documents
    const auto mark = [&](int tile) {
      if (tile >= ntile || tid >= TOK) return;
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
      sm.doc[tile % (ST + 1)][tid] = doc;
      sm.src[tile % (ST + 1)][tid] = src;
    };
    const auto issue = [&](int tile) {
      if (tile < ntile) {
        const float* kp = static_cast<const float*>(tile >= ncache ? a.dk : a.k);
        const float* vp = static_cast<const float*>(tile >= ncache ? a.dv : a.v);
#pragma unroll
        for (int i = 0; i < TOK * kRow / kFewThreads; ++i) {
          const int e = tid + i * kFewThreads, t = e / kRow, x = e % kRow * 4;
          const int64_t src = sm.src[tile % (ST + 1)][t], at = (src * a.Hkv + h) * D + x;
          few_cp16(&sm.k[tile % ST][t][x], src >= 0 ? kp + at : qbase, src >= 0);
          few_cp16(&sm.v[tile % ST][t][x], src >= 0 ? vp + at : qbase, src >= 0);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };

    float m[kMine], l[kMine], o[RR][4];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;  // this lane's tokens; joined at the end
    }
#pragma unroll
    for (int r = 0; r < RR; ++r)
#pragma unroll
      for (int y = 0; y < 4; ++y) o[r][y] = 0.f;
    const float in = a.cap > 0.f ? a.scale / a.cap : a.scale;

    for (int t = 0; t < ST; ++t) mark(t);
    __syncthreads();
    issue(0);
    for (int tile = 0; tile < ntile; ++tile) {
      const int at = tile % ST;
      __syncthreads();  // the tile before is read, the next one marked
      issue(tile + 1);
      mark(tile + 2);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncthreads();

      float s[RR];
#pragma unroll
      for (int r = 0; r < RR; ++r) s[r] = 0.f;
#pragma unroll
      for (int x = 0; x < C::CW; x += 4) {
        const float4 kk = *reinterpret_cast<const float4*>(&sm.k[at][tok][cg * C::CW + x]);
#pragma unroll
        for (int r = 0; r < RR; ++r) {
          const float4 qq = *reinterpret_cast<const float4*>(&sm.q[r][cg * C::CW + x]);
          s[r] = fmaf(qq.x, kk.x, s[r]);
          s[r] = fmaf(qq.y, kk.y, s[r]);
          s[r] = fmaf(qq.z, kk.z, s[r]);
          s[r] = fmaf(qq.w, kk.w, s[r]);
        }
      }
#pragma unroll
      for (int r = 0; r < RR; ++r) sm.part[cg][r][tok] = s[r];
      __syncthreads();

      const bool draft = tile >= ncache;
      const int j0 = first_key(tile);
      const int* doc = sm.doc[tile % (ST + 1)];
      const int64_t* src = sm.src[tile % (ST + 1)];
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int rl = warp + 8 * i, r = r_first + rl;
        if (rl >= RR) break;
        const TokRow row = sm.row[rl];
        float x[TOK / 32], mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < TOK / 32; ++n) {
          const int t = lane + 32 * n, j = j0 + t;
          float z = 0.f;
#pragma unroll
          for (int g = 0; g < C::CG; ++g) z += sm.part[g][rl][t];
          z *= in;
          if (a.cap > 0.f) z = a.cap * (fabsf(z) <= kTanhMax ? tok_tanh(z) : tanhf(z));
          if (a.slopes) z = fmaf(-row.slope2 * (1.f / kLog2e), fabsf((float)(row.pos - j)), z);
          bool vis = src[t] >= 0;
          if (draft)
            vis = vis && r < a.R && a.tree[b * a.tree_bstride + (int64_t)(r / a.G) * a.Sq + j] != 0;
          else
            vis = vis && j < row.hi && (!a.docs || doc[t] == row.doc);
          x[n] = vis ? z : -INFINITY;
          mx = fmaxf(mx, x[n]);
          if (a.logits && r < a.R) a.logits[((int64_t)bh * a.R + r) * a.logit_stride + j] = x[n];  // for the column sums
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        const float m_new = fmaxf(m[i], mx), base = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = exp2f((m[i] - base) * kLog2e);
        l[i] *= alpha;
        m[i] = m_new;
#pragma unroll
        for (int n = 0; n < TOK / 32; ++n) {
          const float p = exp2f((x[n] - base) * kLog2e);
          sm.p[rl][lane + 32 * n] = p;
          l[i] += p;
        }
        if (lane == 0) sm.alpha[rl] = alpha;
      }
      __syncthreads();

#pragma unroll
      for (int r = 0; r < RR; ++r) {
        const float alpha = sm.alpha[r];
#pragma unroll
        for (int y = 0; y < 4; ++y) o[r][y] *= alpha;
      }
#pragma unroll
      for (int t = 0; t < C::KW; t += 4) {
        float4 vv[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) vv[u] = *reinterpret_cast<const float4*>(&sm.v[at][kg * C::KW + t + u][xo]);
#pragma unroll
        for (int r = 0; r < RR; ++r) {
          const float4 p = *reinterpret_cast<const float4*>(&sm.p[r][kg * C::KW + t]);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float pp = u == 0 ? p.x : u == 1 ? p.y : u == 2 ? p.z : p.w;
            o[r][0] = fmaf(pp, vv[u].x, o[r][0]);
            o[r][1] = fmaf(pp, vv[u].y, o[r][1]);
            o[r][2] = fmaf(pp, vv[u].z, o[r][2]);
            o[r][3] = fmaf(pp, vv[u].w, o[r][3]);
          }
        }
      }
    }

    // join the token groups
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // the ring is free: the join reuses it
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int rl = warp + 8 * i;
      if (rl >= RR) break;
      const float sum = warp_sum(l[i]);
      if (lane == 0) {
        sm.m[rl] = m[i];
        sm.l[rl] = sum;
      }
    }
#pragma unroll
    for (int r = 0; r < RR; ++r)
      *reinterpret_cast<float4*>(&sm.join[kg][r][xo]) = make_float4(o[r][0], o[r][1], o[r][2], o[r][3]);
    __syncthreads();
    for (int e = tid; e < RR * kRow; e += kFewThreads) {
      const int rl = e / kRow, x = e % kRow * 4, r = r_first + rl;
      if (r >= a.R) continue;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int g = 0; g < C::KG; ++g) {
        const float4 ov = *reinterpret_cast<const float4*>(&sm.join[g][rl][x]);
        acc.x += ov.x;
        acc.y += ov.y;
        acc.z += ov.z;
        acc.w += ov.w;
      }
      const float M = sm.m[rl], L = sm.l[rl];
      if (seg.part >= 0) {
        const int64_t part = (int64_t)seg.part * 16 + rl;
        if (x == 0) {
          a.pm[part] = M;
          a.pl[part] = L;
        }
        if (M != -INFINITY) *reinterpret_cast<float4*>(&a.po[part * D + x]) = acc;
        continue;
      }
      if (a.lse && x == 0) a.lse[(int64_t)bh * a.R + r] = L == 0.f ? INFINITY : M + logf(L);
      const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);  // NaN stays NaN
      const int64_t out = tok_q_offset(a, b, h, r, D) + x;
      if (a.out_dtype == OC_BF16)
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + out) =
            make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
      else
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + out) =
            make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    }
  }
}

template <int D, int RR>
int launch_few(const TokArgs& a, cudaStream_t st) {
  constexpr size_t smem = sizeof(FewSmem<D, RR>);
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(done, tok_few_kernel<D, RR>, smem);
  if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "tok_few_kernel: %s", cudaGetErrorString(e));
  tok_few_kernel<D, RR><<<a.even ? a.ncta : a.B * a.Hkv * a.nrt, kFewThreads, smem, st>>>(a);
  return check_launch("tok_few_kernel");
}

template <int D>
int launch_few_rows(const TokArgs& a, cudaStream_t st) {
  if (a.R <= 4) return launch_few<D, 4>(a, st);
  if (a.R <= 8) return launch_few<D, 8>(a, st);
  return launch_few<D, 16>(a, st);
}

}  // namespace

int tok_few_tile(int head_dim) { return head_dim == 64 ? FewShape<64>::TOK : FewShape<128>::TOK; }

int tok_few(const TokArgs& a, int head_dim, cudaStream_t st) {
  if (head_dim == 64) return launch_few_rows<64>(a, st);
  if (head_dim == 128) return launch_few_rows<128>(a, st);
  return launch_few_rows<256>(a, st);
}

}  // namespace oc
