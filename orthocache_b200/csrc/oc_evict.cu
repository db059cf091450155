// Eviction of cache tokens by accumulated attention weight.
//
// Per batch row b and KV head h, of the n = lengths[b] tokens the `recent`
// last ones stay and, of the others, the keep - recent with the largest
// weights (equal weights: the lower position; NaN counts as the largest);
// all stay when n <= keep.  The kept tokens' keys, values and weights are
// written in order of position to a cache of `keep` tokens, with the source
// position of each.  The reference evicts whole 512-token blocks by their
// spectrum (src/orthocache/compaction.py:28-100); this is the token-level
// counterpart by attention weight.
//
// Selection is bound by latency, not bytes (a head's weights are 4 bytes a token,
// its kept keys and values 4 D): a head's weights are read once into the shared
// memory of a cluster of CTAs, and the threshold found by three histograms of 11,
// 11 and 10 bits of the order-preserving key, added up over the cluster through
// distributed shared memory, an eighth of the bins by each CTA (every CTA reading
// all histograms took 8,000 cycles a pass, this 2,500).  The gather is bound by
// memory: every kept row read and written once.
#include <cooperative_groups.h>

#include "oc_common.cuh"

namespace oc {
namespace {

namespace cg = cooperative_groups;

constexpr int kSelThreads = 1024;
constexpr int kBins = 2048;
constexpr int kSelCached = 48 * 1024;  // weights of one CTA that fit its shared memory

// Order-preserving 32-bit key of a weight: larger weight, larger key; -0 = +0;
// NaN above everything.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive scan of two values per thread over the block, with the totals.
__device__ __forceinline__ int2 block_scan2(int2 v, int2* warp_sums, int2& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int2 x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, x.x, o), b = __shfl_up_sync(0xffffffffu, x.y, o);
    if (lane >= o) {
      x.x += a;
      x.y += b;
    }
  }
  __syncthreads();  // the previous scan's sums are read
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int2 s = warp_sums[lane];  // 32 warps: every warp scans the sums
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, s.x, o), b = __shfl_up_sync(0xffffffffu, s.y, o);
    if (lane >= o) {
      s.x += a;
      s.y += b;
    }
  }
  total = make_int2(__shfl_sync(0xffffffffu, s.x, 31), __shfl_sync(0xffffffffu, s.y, 31));
  const int2 before = make_int2(__shfl_sync(0xffffffffu, s.x, warp ? warp - 1 : 0),
                                __shfl_sync(0xffffffffu, s.y, warp ? warp - 1 : 0));
  return make_int2(x.x - v.x + (warp ? before.x : 0), x.y - v.y + (warp ? before.y : 0));
}

struct SelSmem {
  int hist[kBins];
  int all[kBins];  // the cluster's
  int2 warp_sums[kSelThreads / 32];
  int2 sums;  // this CTA's kept by value, equal to the threshold
  uint32_t digit;
  int need;
};

// One cluster of CS CTAs per (b, h); CTA r holds the r-th segment of the tokens.
// CACHED: its weights lie in shared memory behind SelSmem.
template <int CS, bool CACHED>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const float* weights, const int32_t* lengths,
                                                                   int S, int H, int keep, int recent, int32_t* index,
                                                                   float* weights_out, int32_t* new_lengths) {
  extern __shared__ __align__(16) unsigned char raw[];
  SelSmem& sm = *reinterpret_cast<SelSmem*>(raw);
  float* cache = reinterpret_cast<float*>(raw + sizeof(SelSmem));
  const int bh = blockIdx.x / CS, rank = blockIdx.x % CS, b = bh / H, tid = threadIdx.x;
  int n = lengths ? lengths[b] : S;
  n = n < 0 ? 0 : (n > S ? S : n);
  const float* w = weights + (int64_t)bh * S;
  int32_t* idx = index + (int64_t)bh * keep;
  float* wo = weights_out + (int64_t)bh * keep;
  if (bh % H == 0 && rank == 0 && tid == 0) new_lengths[b] = min(n, keep);
  if (n <= keep) {  // the same for the whole cluster
    for (int i = rank * kSelThreads + tid; i < keep; i += CS * kSelThreads) {
      idx[i] = i < n ? i : -1;
      wo[i] = i < n ? w[i] : 0.f;
    }
    return;
  }
  const int cand = n - recent;  // tokens that compete
  const int want = keep - recent;
  const int seg = (n + CS - 1) / CS, s0 = min(n, rank * seg), cnt = min(n, s0 + seg) - s0;
  const int comp = max(0, min(cnt, cand - s0));  // of them, those that compete
  if (CACHED) {
#pragma unroll 8
    for (int i = tid; i < cnt; i += kSelThreads) cache[i] = w[s0 + i];
  }
  const float* mine = CACHED ? cache : w + s0;

  // threshold key: the want-th largest; need: how many equal to it are taken
  uint32_t prefix = 0;
  int need = want;
  if (want > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      for (int i = tid; i < kBins; i += kSelThreads) sm.hist[i] = 0;
      __syncthreads();
#pragma unroll 4
      for (int j0 = 0; j0 < comp; j0 += kSelThreads) {
        const bool valid = j0 + tid < comp;
        const uint32_t key = valid ? weight_key(mine[j0 + tid]) : 0;
        const bool in = valid && (pass == 0 || (key >> (shift + bits)) == (prefix >> (shift + bits)));
        const uint32_t digit = (key >> shift) & ((1u << bits) - 1u);
        // equal weights crowd one bin: one addition when a warp agrees
        const uint32_t first = __shfl_sync(0xffffffffu, digit, 0);
        if (__all_sync(0xffffffffu, in && digit == first)) {
          if ((tid & 31) == 0) atomicAdd(&sm.hist[digit], 32);
        } else if (in) {
          atomicAdd(&sm.hist[digit], 1);
        }
      }
      if (CS > 1) {
        // CTA r adds up the r-th part of the bins and hands the sums to all
        constexpr int kPart = kBins / CS;
        cg::this_cluster().sync();
        if (tid < kPart) {
          const int bin = rank * kPart + tid;
          int sum = 0;
#pragma unroll
          for (int r = 0; r < CS; ++r) sum += cg::this_cluster().map_shared_rank(sm.hist, r)[bin];
#pragma unroll
          for (int r = 0; r < CS; ++r) cg::this_cluster().map_shared_rank(sm.all, r)[bin] = sum;
        }
        cg::this_cluster().sync();
      } else {
        __syncthreads();
      }
      // from the top: thread t has bins kBins - 1 - 2 t and the one below
      const int* h = CS > 1 ? sm.all : sm.hist;
      const int hi = kBins - 1 - 2 * tid, c0 = h[hi], c1 = h[hi - 1];
      int2 total;
      const int before = block_scan2(make_int2(c0 + c1, 0), sm.warp_sums, total).x;
      if (before < need && need <= before + c0) {
        sm.digit = hi;
        sm.need = need - before;
      } else if (before + c0 < need && need <= before + c0 + c1) {
        sm.digit = hi - 1;
        sm.need = need - before - c0;
      }
      __syncthreads();
      prefix |= sm.digit << shift;
      need = sm.need;
    }
  }

  // in order of position: everything above the threshold and the recent tokens,
  // and the first `need` equal to it; a thread has a run of tokens
  const int per = (cnt + kSelThreads - 1) / kSelThreads, i0 = min(cnt, tid * per), i1 = min(cnt, i0 + per);
  int2 have = make_int2(0, 0);
  if (CACHED) __syncthreads();
  for (int i = i0; i < i1; ++i) {
    if (i >= comp) {
      ++have.x;
    } else if (want > 0) {
      const uint32_t key = weight_key(mine[i]);
      have.x += key > prefix;
      have.y += key == prefix;
    }
  }
  int2 total;
  int2 at = block_scan2(have, sm.warp_sums, total);
  if (CS > 1) {
    if (tid == 0) sm.sums = total;
    cg::this_cluster().sync();
    for (int r = 0; r < rank; ++r) {
      const int2 o = *cg::this_cluster().map_shared_rank(&sm.sums, r);
      at.x += o.x;
      at.y += o.y;
    }
  }
  for (int i = i0; i < i1; ++i) {
    const float wi = mine[i];
    bool above = true, equal = false;
    if (i < comp) {
      const uint32_t key = weight_key(wi);
      above = want > 0 && key > prefix;
      equal = want > 0 && key == prefix;
    }
    if (above || (equal && at.y < need)) {
      const int slot = at.x + min(at.y, need);
      idx[slot] = s0 + i;
      wo[slot] = wi;
    }
    at.x += above;
    at.y += equal;
  }
  if (CS > 1) cg::this_cluster().sync();  // no CTA leaves while others read its sums
}

template <int CS, bool CACHED>
cudaError_t launch_select(int heads, size_t smem, cudaStream_t st, const float* weights, const int32_t* lengths, int S,
                          int H, int keep, int recent, int32_t* index, float* weights_out, int32_t* new_lengths) {
  auto kern = evict_select_kernel<CS, CACHED>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(done, kern, sizeof(SelSmem) + (CACHED ? kSelCached * 4 : 0));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(heads * CS));
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CS;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CS > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, weights, lengths, S, H, keep, recent, index, weights_out, new_lengths);
}

// Rows of keys and values: one 16-byte vector per thread; output row (b, i, h)
// from source row (b, index[b, h, i], h), zero behind the last kept token.
__global__ void __launch_bounds__(256) evict_gather_kernel(const uint4* k, const uint4* v, const int32_t* index, int S,
                                                           int H, int keep, int vecs, int64_t total, uint4* ko,
                                                           uint4* vo) {
  pdl_wait();
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= total) return;
  const int x = (int)(e % vecs);
  const int64_t row = e / vecs;
  const int h = (int)(row % H);
  const int64_t bi = row / H;
  const int i = (int)(bi % keep);
  const int b = (int)(bi / keep);
  const int src = index[((int64_t)b * H + h) * keep + i];
  uint4 kk = make_uint4(0, 0, 0, 0), vv = kk;
  if (src >= 0) {
    const int64_t at = (((int64_t)b * S + src) * H + h) * vecs + x;
    kk = ldg_stream(k + at);
    vv = ldg_stream(v + at);
  }
  ko[e] = kk;
  vo[e] = vv;
}

}  // namespace
}  // namespace oc

using namespace oc;

extern "C" int oc_evict_tokens(const void* k, const void* v, int dtype, const float* weights, const int32_t* lengths,
                               int batch, int seq_len, int kv_heads, int head_dim, int keep, int recent, void* k_out,
                               void* v_out, float* weights_out, int32_t* index, int32_t* new_lengths,
                               oc_stream_t stream) {
  OC_REQUIRE(k && v && weights && k_out && v_out && weights_out && index && new_lengths, OC_ERR_NULL,
             "oc_evict_tokens: NULL pointer");
  OC_REQUIRE(dtype == OC_F32 || dtype == OC_BF16, OC_ERR_DTYPE, "oc_evict_tokens: bad dtype %d", dtype);
  OC_REQUIRE(batch >= 1 && kv_heads >= 1 && seq_len >= 1, OC_ERR_SHAPE, "oc_evict_tokens: batch %d, seq_len %d, kv_heads %d",
             batch, seq_len, kv_heads);
  const int es = dtype == OC_BF16 ? 2 : 4;
  OC_REQUIRE(head_dim >= 1 && (int64_t)head_dim * es % 16 == 0 && head_dim <= 65536, OC_ERR_SHAPE,
             "oc_evict_tokens: head_dim %d is not a multiple of 16 bytes", head_dim);
  OC_REQUIRE(keep >= 1 && keep <= seq_len, OC_ERR_SHAPE, "oc_evict_tokens: keep %d of %d tokens", keep, seq_len);
  OC_REQUIRE(recent >= 0 && recent <= keep, OC_ERR_SHAPE, "oc_evict_tokens: recent %d, keep %d", recent, keep);
  OC_REQUIRE(aligned16(k) && aligned16(v) && aligned16(k_out) && aligned16(v_out), OC_ERR_ALIGN,
             "oc_evict_tokens: keys / values must be 16-byte aligned");
  OC_REQUIRE(k_out != k && v_out != v && k_out != v_out && k_out != v && v_out != k && weights_out != weights, OC_ERR_SHAPE,
             "oc_evict_tokens: the kept tokens need buffers of their own");
  OC_REQUIRE((int64_t)batch * kv_heads < 65536 * 16, OC_ERR_SHAPE, "oc_evict_tokens: too many heads");
  const int vecs = head_dim * es / 16;
  const int64_t total = (int64_t)batch * keep * kv_heads * vecs;
  OC_REQUIRE((total + 255) / 256 < INT32_MAX, OC_ERR_SHAPE, "oc_evict_tokens: too many rows");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // a CTA per head up to 4096 tokens, a cluster of eight beyond (what a pass over
  // 8192 weights in one CTA takes is about what the cluster's barriers cost)
  const int heads = batch * kv_heads;
  cudaError_t e;
  if (seq_len <= 4096)
    e = launch_select<1, true>(heads, sizeof(SelSmem) + (size_t)seq_len * 4, st, weights, lengths, seq_len, kv_heads,
                               keep, recent, index, weights_out, new_lengths);
  else if ((seq_len + 7) / 8 <= kSelCached)
    e = launch_select<8, true>(heads, sizeof(SelSmem) + (size_t)((seq_len + 7) / 8) * 4, st, weights, lengths, seq_len,
                               kv_heads, keep, recent, index, weights_out, new_lengths);
  else
    e = launch_select<8, false>(heads, sizeof(SelSmem), st, weights, lengths, seq_len, kv_heads, keep, recent, index,
                                weights_out, new_lengths);
  if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "evict_select_kernel: %s", cudaGetErrorString(e));
  e = launch_pdl(evict_gather_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, st,
                 static_cast<const uint4*>(k), static_cast<const uint4*>(v), index, seq_len, kv_heads, keep, vecs,
                 total, static_cast<uint4*>(k_out), static_cast<uint4*>(v_out));
  if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "evict_gather_kernel: %s", cudaGetErrorString(e));
  return OC_OK;
}
