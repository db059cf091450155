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
#include "oc_common.cuh"

namespace oc {
namespace {

constexpr int kSelThreads = 1024;

// Order-preserving 32-bit key of a weight: larger weight, larger key; -0 = +0;
// NaN above everything.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive scan of one value per thread over the block; returns the total too.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // the previous scan's sums are read
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelThreads / 32; ++w) {
    const int s = warp_sums[w];
    if (w < warp) before += s;
    all += s;
  }
  total = all;
  return before + x - v;
}

// One CTA per (b, h): radix selection of the (keep - recent)-th largest key, 8
// bits a pass, then one pass in order of position that writes the kept
// positions.
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const float* weights, const int32_t* lengths,
                                                                   int S, int H, int keep, int recent, int32_t* index,
                                                                   float* weights_out, int32_t* new_lengths) {
  __shared__ int hist[256];
  __shared__ int warp_sums[kSelThreads / 32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int bh = blockIdx.x, b = bh / H, tid = threadIdx.x;
  int n = lengths ? lengths[b] : S;
  n = n < 0 ? 0 : (n > S ? S : n);
  const float* w = weights + (int64_t)bh * S;
  int32_t* idx = index + (int64_t)bh * keep;
  float* wo = weights_out + (int64_t)bh * keep;
  if (bh % H == 0 && tid == 0) new_lengths[b] = min(n, keep);
  if (n <= keep) {
    for (int i = tid; i < keep; i += kSelThreads) {
      idx[i] = i < n ? i : -1;
      wo[i] = i < n ? w[i] : 0.f;
    }
    return;
  }
  const int cand = n - recent;  // tokens that compete
  const int want = keep - recent;
  uint32_t prefix = 0;
  int need = want;  // of the tokens equal to the prefix so far, how many are still to be taken
  if (want > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < cand; i += kSelThreads) {
        const uint32_t key = weight_key(w[i]);
        if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int left = need, d = 255;
        while (d > 0 && hist[d] < left) left -= hist[d--];
        s_prefix = prefix | ((uint32_t)d << shift);
        s_need = left;
      }
      __syncthreads();
      prefix = s_prefix;
      need = s_need;
    }
  }
  // in order of position: everything above the threshold key, the first
  // `need` tokens equal to it, and the recent ones
  int base = 0, eq_base = 0;
  for (int i0 = 0; i0 < n; i0 += kSelThreads) {
    const int i = i0 + tid;
    int above = 0, equal = 0;
    float wi = 0.f;
    if (i < n) {
      wi = w[i];
      if (i >= cand) {
        above = 1;
      } else if (want > 0) {
        const uint32_t key = weight_key(wi);
        above = key > prefix;
        equal = key == prefix;
      }
    }
    int eq_total, total;
    const int eq_rank = eq_base + block_scan(equal, warp_sums, eq_total);
    eq_base += eq_total;
    const int take = above || (equal && eq_rank < need);
    const int slot = base + block_scan(take, warp_sums, total);
    base += total;
    if (take && slot < keep) {
      idx[slot] = i;
      wo[slot] = wi;
    }
  }
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
  OC_REQUIRE(k_out != k && v_out != v && k_out != v_out && k_out != v && v_out != k, OC_ERR_SHAPE,
             "oc_evict_tokens: the kept tokens need buffers of their own");
  OC_REQUIRE((int64_t)batch * kv_heads < 65536 * 16, OC_ERR_SHAPE, "oc_evict_tokens: too many heads");
  const int vecs = head_dim * es / 16;
  const int64_t total = (int64_t)batch * keep * kv_heads * vecs;
  OC_REQUIRE((total + 255) / 256 < INT32_MAX, OC_ERR_SHAPE, "oc_evict_tokens: too many rows");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  evict_select_kernel<<<batch * kv_heads, kSelThreads, 0, st>>>(weights, lengths, seq_len, kv_heads, keep, recent,
                                                                index, weights_out, new_lengths);
  int rc = check_launch("evict_select_kernel");
  if (rc) return rc;
  cudaError_t e = launch_pdl(evict_gather_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, st,
                             static_cast<const uint4*>(k), static_cast<const uint4*>(v), index, seq_len, kv_heads,
                             keep, vecs, total, static_cast<uint4*>(k_out), static_cast<uint4*>(v_out));
  if (e != cudaSuccess) return set_error(OC_ERR_CUDA, "evict_gather_kernel: %s", cudaGetErrorString(e));
  return OC_OK;
}
