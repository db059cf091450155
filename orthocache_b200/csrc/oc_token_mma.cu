// Token-level attention for few query rows per KV head (bfloat16): decoded
// and drafted tokens, up to 64 rows a tile.
//
// Mathematics and masks: oc_token.cuh.  What bounds it is reading keys and
// values once: at 16 rows a token costs 8 D multiply-adds per byte of its keys
// and values, far below the balance of the tensor cores even at the rate of
// the warp-level m16n8k16 instructions; at 64 rows the two are about even, and
// more rows go to the tcgen05 kernel (oc_token_tc.cu).
//
// Layout.  A CTA works on a tile of 16 WR rows of one (batch row, KV head) and a
// run of its keys at a time; its warps are WR row groups x WT token groups x WD
// channel groups, so that every warp multiplies full 16-row fragments:
//   * keys and values stream through shared memory in tiles of TOK tokens,
//     STAGES deep, by 16-byte cp.async (it zero-fills the tokens nobody may
//     see, so garbage behind a sequence never reaches a product), in the
//     128-byte swizzle that makes the ldmatrix reads conflict-free;
//   * scores are Q.K^T fragments (rows x tokens), which after the softmax are
//     the A fragments of P.V as they stand: P stays in registers, rounded to
//     bfloat16 (half a step, 2^-8 relative, of each weight; the row sums are
//     taken before the rounding, in float32);
//   * each warp keeps its own running maximum and sum; the WT token groups are
//     joined once, at the end, in shared memory, and the runs by
//     tok_merge_kernel.
#include "oc_mma.cuh"
#include "oc_token.cuh"
#include "oc_tma.cuh"

namespace oc {
namespace {

template <int D> struct MmaTile;
template <> struct MmaTile<64> { static constexpr int kTok = 64, kWD = 1, kStages = 4; };
template <> struct MmaTile<128> { static constexpr int kTok = 64, kWD = 1, kStages = 3; };
template <> struct MmaTile<256> { static constexpr int kTok = 32, kWD = 2, kStages = 3; };

template <int D, int WR>
struct MmaShape {
  static constexpr int TOK = MmaTile<D>::kTok, WD = MmaTile<D>::kWD, ST = MmaTile<D>::kStages;
  static constexpr int WT = TOK / 16 / WR > 0 ? TOK / 16 / WR : 1;
  static constexpr int WARPS = WR * WT * WD, THREADS = 32 * WARPS;
  static constexpr int RT = 16 * WR;        // rows of the tile
  static constexpr int TPW = TOK / WT;      // tokens of a warp per tile
  static constexpr int NT = TPW / 8;        // n-tiles of the scores
  static constexpr int DW = D / WD;         // output channels of a warp
  static constexpr int kTileBytes = TOK * D * 2;
  static constexpr int kRing = ST * 2 * kTileBytes;
  static constexpr int kJoin = WT * RT * D * 4;
  static constexpr int kQOff = kRing > kJoin ? kRing : kJoin;
  static constexpr int kTreeOff = kQOff + RT * D * 2;  // ancestor bits of the tile's rows, then the seen bits
  static constexpr int kSmem = kTreeOff + (RT + 1) * (kMaxNodes / 32) * 4 + WT * RT * 2 * 4 + 64 + (kMaxEvenBatch + 1) * 4;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int D, int WR>
__global__ void __launch_bounds__(MmaShape<D, WR>::THREADS) tok_mma_kernel(const TokArgs a) {
  using C = MmaShape<D, WR>;
  constexpr int TOK = C::TOK, ST = C::ST, RT = C::RT, WT = C::WT, THREADS = C::THREADS, CPR = D / 8;
  extern __shared__ __align__(1024) unsigned char sm[];
  uint32_t* tree_bits = reinterpret_cast<uint32_t*>(sm + C::kTreeOff);  // [RT][8]
  uint32_t* seen_bits = tree_bits + RT * (kMaxNodes / 32);              // [8]
  float* st_m = reinterpret_cast<float*>(seen_bits + kMaxNodes / 32);   // [WT][RT]
  float* st_l = st_m + WT * RT;
  int* s_int = reinterpret_cast<int*>(st_l + WT * RT);  // hi max, hi min, doc min, doc max, first, last
  const uint32_t sbase = smem_u32(sm);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int wd = warp % C::WD, wt = warp / C::WD % WT, wr = warp / C::WD / WT;
  const int g = lane >> 2, c2 = (lane & 3) * 2;
  int* pre = s_int + 16;
  if (tok_followed(a)) pdl_trigger();  // the merge may find its parts meanwhile
  if (a.even) {
    if (tid < 32) tok_prefix(a, pre);
    __syncthreads();
  }
  TokWalk walk(a, pre, blockIdx.x);
  TokSeg seg;
  for (bool more = true; more;) {
    if (a.even) {
      if (!walk.next(a, pre, blockIdx.x, seg)) break;
    } else {
      // a CTA per unit, the rows with most keys first
      const int u = blockIdx.x % (a.B * a.Hkv);
      seg = TokSeg{u / a.Hkv, u % a.Hkv * a.nrt + a.nrt - 1 - (int)(blockIdx.x / (a.B * a.Hkv)), 0, INT32_MAX, -1};
      more = false;
    }
    const int b = seg.b, h = seg.unit / a.nrt, rt = seg.unit % a.nrt, bh = b * a.Hkv + h;
    const int len = tok_len(a, b);
    const int nct = (len + TOK - 1) / TOK;  // tiles of the cache; drafted tokens follow
    const bool has_draft = a.dk && seg.t1 > nct;
    __syncthreads();  // the previous piece is done with shared memory

    // queries of the tile (swizzled like the keys), first in the copy queue
    for (int e = tid; e < RT * CPR; e += THREADS) {
      const int r = e / CPR, c = e % CPR;
      const bool real = rt * RT + r < a.R;
      const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(a.q) +
                                 (real ? tok_q_offset(a, b, h, rt * RT + r, D) + c * 8 : 0);
      cp16(sbase + C::kQOff + swz<RT>(r, c), src, real);
    }
    if (tid == 0) {
      s_int[0] = 0;
      s_int[1] = INT32_MAX;
      s_int[2] = INT32_MAX;
      s_int[3] = -1;
      s_int[4] = INT32_MAX;
      s_int[5] = 0;
    }
    if (has_draft)
      for (int e = tid; e < (RT + 1) * (kMaxNodes / 32); e += THREADS) tree_bits[e] = 0;
    __syncthreads();
    TokRow row[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) row[i] = tok_row(a, b, h, rt * RT + wr * 16 + g + 8 * i, len);
    for (int r = tid; r < RT; r += THREADS) {
      if (rt * RT + r >= a.R) continue;
      const TokRow w = tok_row(a, b, h, rt * RT + r, len);
      atomicMax(&s_int[0], w.hi);
      atomicMin(&s_int[1], w.hi);
      if (w.hi > 0 && a.docs) {
        atomicMin(&s_int[2], w.doc);
        atomicMax(&s_int[3], w.doc);
      }
    }
    if (has_draft) {
      // ancestor bits of the tile's rows, and which drafted tokens any row of
      // the tree sees (a padded one may hold anything)
      const uint8_t* tm = a.tree + b * a.tree_bstride;
      for (int e = tid; e < a.Sq * a.Sq; e += THREADS) {
        if (!tm[e]) continue;
        const int i = e / a.Sq, s = e % a.Sq;
        atomicOr(&seen_bits[s >> 5], 1u << (s & 31));
        const int r0 = max(i * a.G - rt * RT, 0), r1 = min((i + 1) * a.G - rt * RT, RT);
        for (int r = r0; r < r1; ++r) atomicOr(&tree_bits[r * (kMaxNodes / 32) + (s >> 5)], 1u << (s & 31));
      }
    }
    __syncthreads();
    int t0 = min(seg.t0, nct) * TOK, t1 = min(s_int[0], min(seg.t1, nct) * TOK);
    const int min_hi = s_int[1];
    if (a.docs && t0 < t1) {  // the span of this chunk that holds any of the rows' documents
      const int d0 = s_int[2], d1 = s_int[3];
      int first = INT32_MAX, last = 0;
      for (int j = t0 + tid; j < t1; j += THREADS) {
        const int d = a.docs[(size_t)b * a.S + j];
        if (d >= d0 && d <= d1) {
          first = min(first, j);
          last = max(last, j + 1);
        }
      }
      if (last) {
        atomicMin(&s_int[4], first);
        atomicMax(&s_int[5], last);
      }
      __syncthreads();
      t1 = min(t1, s_int[5]);
      if (s_int[4] < t1) t0 = s_int[4] / TOK * TOK;
    }
    const int ncache = t1 > t0 ? (t1 - t0 + TOK - 1) / TOK : 0;
    const int d0 = max(seg.t0 - nct, 0);  // first drafted tile
    const int ntile = ncache + (has_draft ? min(seg.t1 - nct, (a.Sq + TOK - 1) / TOK) - d0 : 0);

    // this thread's 16-byte column and rows r0, r0 + kStep, ... of a tile
    constexpr int kStep = THREADS / CPR;
    const int c_mine = tid % CPR, r0 = tid / CPR;
    const int64_t row_bytes = (int64_t)a.Hkv * D * 2;
    auto issue = [&](int t) {
      if (t < ntile) {
        const uint32_t slot = sbase + (t % ST) * 2 * C::kTileBytes;
        const bool draft = t >= ncache;
        const int j0 = draft ? (d0 + t - ncache) * TOK : t0 + t * TOK;
        const int64_t row0 = draft ? (int64_t)b * a.Sq + j0 : tok_kv_row(a, b, j0);  // a tile lies inside one page
        const char* kp = static_cast<const char*>(draft ? a.dk : a.k);
        const char* vp = static_cast<const char*>(draft ? a.dv : a.v);
        if (tid == 0) s_int[6 + t % ST] = row0 < 0;  // a page outside the pool
        const int64_t off0 = (row0 + r0) * row_bytes + (h * D + c_mine * 8) * 2;
        if (!draft && !a.docs && row0 >= 0 && j0 + TOK <= len) {
          kp += off0;
          vp += off0;
#pragma unroll
          for (int i = 0; i < TOK / kStep; ++i) {
            const uint32_t dst = slot + swz<TOK>(r0 + i * kStep, c_mine);
            cp16(dst, kp, true);
            cp16(dst + C::kTileBytes, vp, true);
            kp += kStep * row_bytes;
            vp += kStep * row_bytes;
          }
        } else {
#pragma unroll 1
          for (int i = 0; i < TOK / kStep; ++i) {
            const int r = r0 + i * kStep, j = j0 + r;
            bool real;
            if (draft)
              real = j < a.Sq && (seen_bits[j >> 5] >> (j & 31) & 1);
            else
              real = j < len && row0 >= 0 && (!a.docs || a.docs[(size_t)b * a.S + j] >= 0);
            const int64_t at = off0 + i * kStep * row_bytes;
            const uint32_t dst = slot + swz<TOK>(r, c_mine);
            cp16(dst, real ? kp + at : static_cast<const char*>(a.q), real);
            cp16(dst + C::kTileBytes, real ? vp + at : static_cast<const char*>(a.q), real);
          }
        }
      }
      cp_commit();
    };
#pragma unroll
    for (int t = 0; t < ST - 1; ++t) issue(t);

    constexpr int KQ = D <= 128 ? D / 16 : 1;  // query fragments kept in registers (64 of them at D = 256 are reread)
    uint32_t qf[KQ][4];
    float o[C::DW / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < C::DW / 8; ++i)
#pragma unroll
      for (int y = 0; y < 4; ++y) o[i][y] = 0.f;
    const float c_scale = a.scale * kLog2e, c_cap = a.cap * kLog2e, c_in = a.cap > 0.f ? a.scale / a.cap : 0.f;
    // ldmatrix addresses: lanes 0-15 give rows (lane % 16) of the first 8
    // channels, lanes 16-31 of the next 8
    const int q_row = wr * 16 + (lane & 15), q_c = lane >> 4;

    for (int t = 0; t < ntile; ++t) {
      cp_wait<ST - 2>();
      __syncthreads();
      issue(t + ST - 1);
      const uint32_t kt = sbase + (t % ST) * 2 * C::kTileBytes, vt = kt + C::kTileBytes;
      if (t == 0 && D <= 128) {
#pragma unroll
        for (int kk = 0; kk < KQ; ++kk) ldsm_x4(qf[kk], sbase + C::kQOff + swz<RT>(q_row, 2 * kk + q_c));
      }
      const bool draft = t >= ncache, hole = s_int[6 + t % ST] != 0;
      const int j0 = (draft ? (d0 + t - ncache) * TOK : t0 + t * TOK) + wt * C::TPW;

      // scores of this warp's tokens: B fragments are 8 tokens x 16 channels of
      // the keys as they lie
      float s[C::NT][4];
#pragma unroll
      for (int n = 0; n < C::NT; ++n)
#pragma unroll
        for (int y = 0; y < 4; ++y) s[n][y] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t qa[4];
        if (D <= 128) {
#pragma unroll
          for (int y = 0; y < 4; ++y) qa[y] = qf[kk < KQ ? kk : 0][y];
        } else {
          ldsm_x4(qa, sbase + C::kQOff + swz<RT>(q_row, 2 * kk + q_c));
        }
#pragma unroll
        for (int n = 0; n < C::NT; n += 2) {
          uint32_t kb[4];
          ldsm_x4(kb, kt + swz<TOK>(wt * C::TPW + n * 8 + (lane & 7) + ((lane >> 4) << 3), 2 * kk + ((lane >> 3) & 1)));
          mma_bf16_16816(s[n], qa, kb[0], kb[1]);
          mma_bf16_16816(s[n + 1], qa, kb[2], kb[3]);
        }
      }

      // log2 units: scale, cap, bias, masks
      if (a.cap > 0.f) {
        float top = 0.f;
#pragma unroll
        for (int n = 0; n < C::NT; ++n)
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            s[n][y] *= c_in;  // scale / cap
            top = fmaxf(top, fabsf(s[n][y]));
          }
        if (__all_sync(0xffffffffu, top <= kTanhMax)) {  // (NaN may pass: it stays NaN)
#pragma unroll
          for (int n = 0; n < C::NT; ++n)
#pragma unroll
            for (int y = 0; y < 4; ++y) s[n][y] = c_cap * tok_tanh(s[n][y]);
        } else {
#pragma unroll
          for (int n = 0; n < C::NT; ++n)
#pragma unroll
            for (int y = 0; y < 4; ++y) s[n][y] = c_cap * tanhf(s[n][y]);
        }
      } else {
#pragma unroll
        for (int n = 0; n < C::NT; ++n)
#pragma unroll
          for (int y = 0; y < 4; ++y) s[n][y] *= c_scale;
      }
      if (a.slopes) {
#pragma unroll
        for (int n = 0; n < C::NT; ++n)
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const TokRow& w = row[y >> 1];
            s[n][y] = fmaf(-w.slope2, fabsf((float)(w.pos - (j0 + n * 8 + c2 + (y & 1)))), s[n][y]);
          }
      }
      if (draft) {
#pragma unroll
        for (int n = 0; n < C::NT; ++n)
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int j = j0 + n * 8 + c2 + (y & 1);
            const uint32_t bits = j < kMaxNodes ? tree_bits[(wr * 16 + g + (y >> 1) * 8) * (kMaxNodes / 32) + (j >> 5)] : 0;
            if (!(bits >> (j & 31) & 1)) s[n][y] = -INFINITY;
          }
      } else if (a.docs || hole || j0 + C::TPW > min_hi) {
#pragma unroll
        for (int n = 0; n < C::NT; ++n)
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int j = j0 + n * 8 + c2 + (y & 1);
            const TokRow& w = row[y >> 1];
            if (!(!hole && j < w.hi && (!a.docs || a.docs[(size_t)b * a.S + j] == w.doc))) s[n][y] = -INFINITY;
          }
      }

      if (WR <= 2 && a.logits && wd == 0) {  // kept for the column sums (few rows only)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = rt * RT + wr * 16 + g + 8 * i;
          if (r >= a.R) continue;
          float* dst = a.logits + ((int64_t)bh * a.R + r) * a.logit_stride + j0 + c2;
#pragma unroll
          for (int n = 0; n < C::NT; ++n) *reinterpret_cast<float2*>(dst + n * 8) = make_float2(s[n][2 * i], s[n][2 * i + 1]);
        }
      }

      // running softmax of the warp's 16 rows (a row's tokens lie in 4 lanes)
      uint32_t p[C::NT][2];
      float alpha[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < C::NT; ++n) mx = fmaxf(mx, fmaxf(s[n][2 * i], s[n][2 * i + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_new = fmaxf(m[i], mx);
        const float base = m_new == -INFINITY ? 0.f : m_new;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(alpha[i]) : "f"(m[i] - base));
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < C::NT; ++n) {
          float p0, p1;
          asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p0) : "f"(s[n][2 * i] - base));
          asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p1) : "f"(s[n][2 * i + 1] - base));
          sum += p0 + p1;
          p[n][i] = pack_bf16x2(p0, p1);
        }
        l[i] = l[i] * alpha[i] + sum;  // this lane's tokens; joined over the 4 lanes at the end
        m[i] = m_new;
      }
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int x = 0; x < C::DW / 8; ++x) {
          o[x][0] *= alpha[0];
          o[x][1] *= alpha[0];
          o[x][2] *= alpha[1];
          o[x][3] *= alpha[1];
        }
      }

      // O += P V: 16 tokens a step, B fragments by transposing loads
#pragma unroll
      for (int kk = 0; kk < C::NT / 2; ++kk) {
        const uint32_t pa[4] = {p[2 * kk][0], p[2 * kk][1], p[2 * kk + 1][0], p[2 * kk + 1][1]};
#pragma unroll
        for (int x = 0; x < C::DW / 8; x += 2) {
          uint32_t vb[4];
          ldsm_x4_t(vb, vt + swz<TOK>(wt * C::TPW + kk * 16 + (lane & 15), wd * (C::DW / 8) + x + (lane >> 4)));
          mma_bf16_16816(o[x], pa, vb[0], vb[1]);
          mma_bf16_16816(o[x + 1], pa, vb[2], vb[3]);
        }
      }
    }
    cp_wait<0>();
    __syncthreads();  // the ring is free: the join reuses it

    float* jo = reinterpret_cast<float*>(sm);  // [WT][RT][D]
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      const int r = wr * 16 + g + 8 * i;
      if (wd == 0 && (lane & 3) == 0) {
        st_m[wt * RT + r] = m[i];
        st_l[wt * RT + r] = l[i];
      }
#pragma unroll
      for (int x = 0; x < C::DW / 8; ++x)
        *reinterpret_cast<float2*>(&jo[(wt * RT + r) * D + wd * C::DW + x * 8 + c2]) =
            make_float2(o[x][2 * i], o[x][2 * i + 1]);
    }
    __syncthreads();
    for (int e = tid; e < RT * (D / 4); e += THREADS) {
      const int rl = e / (D / 4), x = e % (D / 4) * 4, r = rt * RT + rl;
      if (r >= a.R) continue;
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int w = 0; w < WT; ++w) M = fmaxf(M, st_m[w * RT + rl]);
      const float base = M == -INFINITY ? 0.f : M;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WT; ++w) {
        const float f = exp2f(st_m[w * RT + rl] - base);
        const float4 ov = *reinterpret_cast<const float4*>(&jo[(w * RT + rl) * D + x]);
        L += f * st_l[w * RT + rl];
        acc.x += f * ov.x;
        acc.y += f * ov.y;
        acc.z += f * ov.z;
        acc.w += f * ov.w;
      }
      if (seg.part >= 0) {
        const int64_t part = (int64_t)seg.part * RT + rl;
        if (x == 0) {
          a.pm[part] = M;
          a.pl[part] = L;
        }
        if (M != -INFINITY) *reinterpret_cast<float4*>(&a.po[part * D + x]) = acc;
        continue;
      }
      if (a.lse && x == 0) a.lse[(int64_t)bh * a.R + r] = L == 0.f ? INFINITY : M + log2f(L);
      const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
      const int64_t at = tok_q_offset(a, b, h, r, D) + x;
      if (a.out_dtype == OC_BF16)
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + at) =
            make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
      else
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) =
            make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    }
  }
}

template <int D, int WR>
int launch_mma(const TokArgs& a, cudaStream_t st) {
  using C = MmaShape<D, WR>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(done, tok_mma_kernel<D, WR>, C::kSmem);
  if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "tok_mma_kernel: %s", cudaGetErrorString(e));
  tok_mma_kernel<D, WR><<<a.even ? a.ncta : a.B * a.Hkv * a.nrt, C::THREADS, C::kSmem, st>>>(a);
  return check_launch("tok_mma_kernel");
}

template <int D>
int launch_mma_rows(const TokArgs& a, int row_tile, cudaStream_t st) {
  if (row_tile == 16) return launch_mma<D, 1>(a, st);
  if (row_tile == 32) return launch_mma<D, 2>(a, st);
  return launch_mma<D, 4>(a, st);
}

}  // namespace

int tok_mma_tile(int head_dim) { return head_dim == 256 ? MmaTile<256>::kTok : MmaTile<128>::kTok; }

int tok_mma(const TokArgs& a, int head_dim, int row_tile, cudaStream_t st) {
  if (head_dim == 64) return launch_mma_rows<64>(a, row_tile, st);
  if (head_dim == 128) return launch_mma_rows<128>(a, row_tile, st);
  return launch_mma_rows<256>(a, row_tile, st);
}

}  // namespace oc
