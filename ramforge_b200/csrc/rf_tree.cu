// rf_tree.cu - attention of drafted tokens over a cached history and over the
// drafts' own tree (rf_tree_attention).
//
// out[t] = sum_p softmax_p(scale q[t] . k[p]) v[p] over the positions token t sees:
// the whole history p < L, and the drafts p = L + j whose bit j is set in its mask row.
// One pass over the keys carries the running maximum m, the sum l of exp(s - m) and
// the output sum, rescaled when m grows.
#include <cuda_bf16.h>

#include "rf_device.cuh"
#include "rf_verify.h"

namespace rf {
namespace {

struct TreeArgs {
  rf_kv_view c;
  const void* q;
  void* out;
  uint64_t q_stride, out_stride;
  uint32_t n_seqs, n_tokens, n_heads, words;  // words: mask words per token
  const int32_t *hist_len, *n_draft;
  const uint32_t* mask;
  float scale;
  unsigned* err;
};

// History length and draft count of sequence b; (0, 0) and the error bit where they do not fit the cache.
__device__ __forceinline__ void seq_lengths(const TreeArgs& a, uint32_t b, uint32_t* hist, uint32_t* drafts) {
  const int32_t L = a.hist_len[b], n = a.n_draft ? a.n_draft[b] : (int32_t)a.n_tokens;
  const bool ok = L >= 0 && n >= 0 && (uint32_t)n <= a.n_tokens && (uint64_t)L + (uint64_t)n <= a.c.capacity;
  if (!ok) atomicOr(a.err, kVerifyRange);
  *hist = ok ? (uint32_t)L : 0;
  *drafts = ok ? (uint32_t)n : 0;
}

__device__ __forceinline__ float act_get(const float* p) { return *p; }
__device__ __forceinline__ float act_get(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float act_get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void act_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void act_put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void act_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Element d of the cache row `slot` (value = code * scale rounded to f16).
template <bool Q8>
__device__ __forceinline__ float kv_value(const void* plane, const void* scale, uint64_t slot, uint32_t D, uint32_t d) {
  if constexpr (Q8) {
    const float s = __half2float(((const __half*)scale)[slot * (D / 32) + d / 32]);
    return __half2float(__float2half_rn((float)((const int8_t*)plane)[slot * D + d] * s));
  } else {
    return __half2float(((const __half*)plane)[slot * D + d]);
  }
}

// One CTA a (token, query head): warps take the keys in turn, lanes the head's dimensions.
template <class T, bool Q8, int D>
__global__ void __launch_bounds__(128) tree_simple_kernel(TreeArgs a) {
  constexpr int E = D / 32;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t h = blockIdx.x % a.n_heads, bt = blockIdx.x / a.n_heads, b = bt / a.n_tokens, t = bt % a.n_tokens;
  const uint32_t kh = h / (a.n_heads / a.c.n_kv_heads);
  uint32_t L, n;
  seq_lengths(a, b, &L, &n);
  const T* q = (const T*)a.q + bt * a.q_stride + h * D;
  T* out = (T*)a.out + bt * a.out_stride + h * D;
  float qv[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; e++) qv[e] = act_get(q + lane + 32 * e) * a.scale, o[e] = 0.f;
  const uint64_t base = ((uint64_t)b * a.c.n_kv_heads + kh) * a.c.capacity;
  const uint32_t end = t < n ? L + n : 0;
  for (uint32_t p = warp; p < end; p += 4) {
    if (p >= L) {
      const uint32_t j = p - L;
      const bool see = a.mask ? (a.mask[(uint64_t)bt * a.words + j / 32] >> (j % 32)) & 1u : j <= t;
      if (!see) continue;
    }
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; e++) s = fmaf(qv[e], kv_value<Q8>(a.c.k, a.c.k_scale, base + p, D, lane + 32 * e), s);
#pragma unroll
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.f : mn;
    const float c = expf(m - ref), w = expf(s - ref);
    l = l * c + w;
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = o[e] * c + w * kv_value<Q8>(a.c.v, a.c.v_scale, base + p, D, lane + 32 * e);
    m = mn;
  }
  __shared__ float sm[4], sl[4], so[4][D];
  if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
  for (int e = 0; e < E; e++) so[warp][lane + 32 * e] = o[e];
  __syncthreads();
  for (uint32_t d = threadIdx.x; d < D; d += 128) {
    const float M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), ref = M == -INFINITY ? 0.f : M;
    float num = 0.f, den = 0.f;
    for (int w = 0; w < 4; w++) {
      const float c = expf(sm[w] - ref);
      num += so[w][d] * c;
      den += sl[w] * c;
    }
    act_put(out + d, den == 0.f ? 0.f : num / den);
  }
}

template <class T, bool Q8>
cudaError_t launch_tree(const Launch& L, const TreeArgs& a) {
  const dim3 grid(a.n_seqs * a.n_tokens * a.n_heads);
  return launch_k(L, a.c.head_dim == 128 ? tree_simple_kernel<T, Q8, 128> : tree_simple_kernel<T, Q8, 64>, grid,
                  dim3(128), 0, a);
}

}  // namespace
}  // namespace rf

using namespace rf;

extern "C" {

int rf_tree_attention(const rf_kv_view* cache, const void* q, void* out, int act_type, uint32_t n_seqs,
                      uint32_t n_tokens, uint32_t n_heads, uint64_t q_stride, uint64_t out_stride,
                      const int32_t* hist_len, const int32_t* n_draft, const uint32_t* mask, float scale,
                      void* stream) {
  RF_TRY(check_kv_view(cache));
  const uint32_t es = act_bytes(act_type);
  if (!es) return set_error(RF_EINVAL, "activation type %d is not F32, F16 or BF16", act_type);
  if (!q || !out || !hist_len) return set_error(RF_EINVAL, "null argument");
  if (cache->head_dim != 64 && cache->head_dim != 128)
    return set_error(RF_EUNSUPPORTED, "tree attention covers head_dim 64 and 128, not %u", cache->head_dim);
  if (n_seqs > cache->n_seqs) return set_error(RF_EINVAL, "%u sequences, the cache holds %u", n_seqs, cache->n_seqs);
  if (!n_tokens || n_tokens > 1024) return set_error(RF_EINVAL, "n_tokens %u out of range 1..1024", n_tokens);
  if (!n_heads || n_heads % cache->n_kv_heads)
    return set_error(RF_EINVAL, "%u query heads are no multiple of %u KV heads", n_heads, cache->n_kv_heads);
  if (!(scale >= 0.f) || scale > 3.0e38f) return set_error(RF_EINVAL, "scale must be positive, or 0 for 1/sqrt(head_dim)");
  const uint64_t row = (uint64_t)n_heads * cache->head_dim;
  if (!q_stride) q_stride = row;
  if (!out_stride) out_stride = row;
  if (q_stride < row || out_stride < row) return set_error(RF_EINVAL, "a token stride is below its row's elements");
  if (!aligned_to(q, 16) || !aligned_to(out, 16) || q_stride * es % 16 || out_stride * es % 16)
    return set_error(RF_EINVAL, "query and output rows must be 16-byte aligned");
  if ((uint64_t)n_seqs * n_tokens * n_heads > 0x7fffffffull)
    return set_error(RF_EINVAL, "%u x %u tokens of %u heads are too many for one call", n_seqs, n_tokens, n_heads);
  if (!n_seqs) return RF_OK;
  TreeArgs a{};
  a.c = *cache;
  a.q = q, a.out = out;
  a.q_stride = q_stride, a.out_stride = out_stride;
  a.n_seqs = n_seqs, a.n_tokens = n_tokens, a.n_heads = n_heads, a.words = (n_tokens + 31) / 32;
  a.hist_len = hist_len, a.n_draft = n_draft, a.mask = mask;
  a.scale = scale > 0.f ? scale : 1.f / sqrtf((float)cache->head_dim);
  RF_TRY(verify_error_ptr(&a.err));
  const Launch L{(cudaStream_t)stream, false};
  const bool q8 = cache->type == RF_TYPE_Q8_0;
  switch (act_type) {
    case RF_ACT_F32: RF_CUDA((q8 ? launch_tree<float, true> : launch_tree<float, false>)(L, a)); break;
    case RF_ACT_F16: RF_CUDA((q8 ? launch_tree<__half, true> : launch_tree<__half, false>)(L, a)); break;
    default: RF_CUDA((q8 ? launch_tree<__nv_bfloat16, true> : launch_tree<__nv_bfloat16, false>)(L, a));
  }
  return RF_OK;
}

}  // extern "C"
