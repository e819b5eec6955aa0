// rf_tree.cuh - what the two kernels of rf_tree_attention share: the arguments, the
// split of the work over CTAs, visibility, and the softmax's constants.
#pragma once
#include <cuda_bf16.h>

#include "rf_device.cuh"
#include "rf_verify.h"

namespace rf {

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

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---------------------------------------------------------------------------
// The work split.  A unit is (sequence b, KV head h, row tile rt): up to ROWS of the
// n_b * G query rows (G query heads share a KV head; row r = token r / G, head r % G)
// against all its keys, in tiles of KT.  All tiles of all units, in that order, are
// cut into equal contiguous ranges, one a CTA (of as many CTAs as there are tiles, at
// most gridDim.x), whatever the histories: the lengths are read on the device.  A unit that lies in one CTA is finished there; the
// others leave partial results that tree_merge_kernel adds in order of the keys, so
// results do not depend on timing.  A CTA leaves at most two: slot 0 for the unit its
// range starts inside of, slot 1 for the one it ends inside of.
// ---------------------------------------------------------------------------
template <int KT, int ROWS>
struct Split {
  static __device__ __forceinline__ uint32_t tiles(uint32_t L, uint32_t n) { return n ? (L + n + KT - 1) / KT : 0; }
  static __device__ __forceinline__ uint32_t row_tiles(const TreeArgs& a, uint32_t n) {
    return (n * (a.n_heads / a.c.n_kv_heads) + ROWS - 1) / ROWS;
  }
  static __device__ __forceinline__ uint64_t work(const TreeArgs& a, uint32_t b) {
    if (b >= a.n_seqs) return 0;
    uint32_t L, n;
    seq_lengths(a, b, &L, &n);
    return (uint64_t)tiles(L, n) * row_tiles(a, n) * a.c.n_kv_heads;
  }
  // Whole warp: the tiles of all sequences, and (through *before) those of the sequences before b.
  static __device__ __forceinline__ uint64_t total(const TreeArgs& a, uint32_t b, uint64_t* before) {
    uint64_t t = 0, p = 0;
    for (uint32_t i = threadIdx.x & 31; i < a.n_seqs; i += 32) {
      const uint64_t w = work(a, i);
      t += w;
      if (i < b) p += w;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      t += __shfl_xor_sync(0xffffffffu, t, o);
      p += __shfl_xor_sync(0xffffffffu, p, o);
    }
    *before = p;
    return t;
  }
  // Whole warp: the sequence that holds tile w, and w's offset in it.
  static __device__ __forceinline__ uint32_t locate(const TreeArgs& a, uint64_t w, uint64_t* offset) {
    const uint32_t lane = threadIdx.x & 31;
    uint64_t acc = 0;
    for (uint32_t base = 0; base < a.n_seqs; base += 32) {
      uint64_t s = work(a, base + lane);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t up = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += up;
      }
      const unsigned past = __ballot_sync(0xffffffffu, acc + s > w);
      if (past) {
        const int first = __ffs(past) - 1;
        const uint64_t low = first ? __shfl_sync(0xffffffffu, s, first - 1) : 0;
        *offset = w - acc - low;
        return base + first;
      }
      acc += __shfl_sync(0xffffffffu, s, 31);
    }
    *offset = 0;
    return a.n_seqs;
  }
};

// A run of consecutive key tiles of one unit: what a CTA works on at a time.
struct Segment {
  uint32_t b, h, rt;          // sequence, KV head, row tile
  uint32_t k0, k1, tiles;     // the run [k0, k1) of the unit's tiles
  uint32_t hist, drafts, end; // lengths of the sequence; end = hist + drafts
  __device__ bool whole() const { return k0 == 0 && k1 == tiles; }
};

// The segments of this CTA, in order.
template <int KT, int ROWS>
struct Walk {
  using Sp = Split<KT, ROWS>;
  uint64_t w, w_end, rem;
  uint32_t b;
  // Whole warp.
  __device__ __forceinline__ Walk(const TreeArgs& a) {
    uint64_t ignore;
    const uint64_t all = Sp::total(a, 0, &ignore);
    const uint32_t ctas = (uint32_t)min((uint64_t)gridDim.x, all);  // no CTA without a tile
    w = w_end = 0;
    if (blockIdx.x >= ctas) return;
    w = all * blockIdx.x / ctas;
    w_end = all * (blockIdx.x + 1) / ctas;
    b = Sp::locate(a, w, &rem);
  }
  __device__ __forceinline__ bool next(const TreeArgs& a, Segment* s) {
    if (w >= w_end) return false;
    uint32_t L, n;
    seq_lengths(a, b, &L, &n);
    uint32_t tiles = Sp::tiles(L, n), rts = Sp::row_tiles(a, n);
    while (rem == (uint64_t)tiles * rts * a.c.n_kv_heads) {  // past this sequence (or it has no work)
      b++;
      rem = 0;
      seq_lengths(a, b, &L, &n);
      tiles = Sp::tiles(L, n), rts = Sp::row_tiles(a, n);
    }
    const uint32_t unit = (uint32_t)(rem / tiles);
    s->b = b, s->h = unit / rts, s->rt = unit % rts;
    s->k0 = (uint32_t)(rem % tiles);
    s->k1 = (uint32_t)min((uint64_t)tiles, s->k0 + (w_end - w));
    s->tiles = tiles;
    s->hist = L, s->drafts = n, s->end = L + n;
    w += s->k1 - s->k0;
    rem += s->k1 - s->k0;
    return true;
  }
};

// Floats of one partial result: ROWS x D output sums, then ROWS maxima and ROWS sums.
constexpr size_t part_floats(int rows, int D) { return (size_t)rows * (D + 2); }

// Visibility of position p for token t of sequence b (p < L + n).
__device__ __forceinline__ bool sees(const TreeArgs& a, uint32_t b, uint32_t t, uint32_t L, uint32_t p) {
  if (p < L) return true;
  const uint32_t j = p - L;
  return a.mask ? (a.mask[((uint64_t)b * a.n_tokens + t) * a.words + j / 32] >> (j % 32)) & 1u : j <= t;
}

// Softmax in base 2 with a running reference m that is only raised (and the sums
// rescaled) when some score passes it by 2^kRaise; weights are 2^(s - m + kWeightBias),
// below 2^15, so that f16 keeps 11 bits of every weight down to 2^-21 of the largest.
constexpr float kRaise = 8.f, kWeightBias = 7.f;

// ---------------------------------------------------------------------------
// One CTA a (token, query head): adds the partial results of a unit that several of
// the first kernel's CTAs shared (`grid` of them), and writes the zeros of tokens past a sequence's drafts.
// ---------------------------------------------------------------------------
template <class T, int D, int KT, int ROWS>
__global__ void __launch_bounds__(128) tree_merge_kernel(TreeArgs a, const float* __restrict__ part, uint32_t grid) {
  using Sp = Split<KT, ROWS>;
  constexpr int E = D / 32;
  __shared__ float s_o[4][D], s_l[4];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t hq = blockIdx.x % a.n_heads, bt = blockIdx.x / a.n_heads, b = bt / a.n_tokens, t = bt % a.n_tokens;
  const uint32_t G = a.n_heads / a.c.n_kv_heads, h = hq / G, r = t * G + hq % G;
  T* out = (T*)a.out + bt * a.out_stride + (uint64_t)hq * D;
  uint32_t L, n;
  seq_lengths(a, b, &L, &n);
  if (t >= n) {
    if (threadIdx.x < D) act_put(out + threadIdx.x, 0.f);
    return;
  }
  uint64_t before;
  const uint64_t all = Sp::total(a, b, &before);
  const uint32_t tiles = Sp::tiles(L, n);
  const uint64_t u0 = before + ((uint64_t)h * Sp::row_tiles(a, n) + r / ROWS) * tiles, u1 = u0 + tiles;
  const uint32_t ctas = (uint32_t)min((uint64_t)grid, all);  // CTA c holds [all c / ctas, all (c+1) / ctas)
  const uint32_t c0 = (uint32_t)(((u0 + 1) * ctas - 1) / all), c1 = (uint32_t)((u1 * ctas - 1) / all);
  if (c0 == c1) return;
  griddep_wait();
  const uint32_t rl = r % ROWS;
  auto slot = [&](uint32_t c) { return part + (2 * (size_t)c + (c == c0 ? 1 : 0)) * part_floats(ROWS, D); };
  float M = -INFINITY;
  for (uint32_t c = c0 + lane; c <= c1; c += 32) M = fmaxf(M, __ldcg(slot(c) + ROWS * D + rl));
#pragma unroll
  for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  float acc[E], den = 0.f;
#pragma unroll
  for (int e = 0; e < E; e++) acc[e] = 0.f;
#pragma unroll 4
  for (uint32_t c = c0 + warp; c <= c1; c += 4) {
    const float* s = slot(c);
    const float f = M == -INFINITY ? 1.f : ex2(__ldcg(s + ROWS * D + rl) - M);
    den += __ldcg(s + ROWS * D + ROWS + rl) * f;
#pragma unroll
    for (int e = 0; e < E; e++) acc[e] += __ldcg(s + (size_t)rl * D + lane + 32 * e) * f;
  }
#pragma unroll
  for (int e = 0; e < E; e++) s_o[warp][lane + 32 * e] = acc[e];
  if (lane == 0) s_l[warp] = den;
  __syncthreads();
  if (threadIdx.x < D) {
    const uint32_t d = threadIdx.x;
    const float l = s_l[0] + s_l[1] + s_l[2] + s_l[3];
    act_put(out + d, l == 0.f ? 0.f : (s_o[0][d] + s_o[1][d] + s_o[2][d] + s_o[3][d]) / l);
  }
}

// Scratch of one call: allocated in stream order from a pool of this library's own that keeps
// its memory, to be freed on the same stream, so calls on any stream, and captured ones, never
// share a buffer (rf_tree.cu).
int scratch_alloc(void** out, size_t bytes, cudaStream_t st);

// The kernel for many query rows a KV head (rf_tree_tc.cu).
int run_tree_tc(int act_type, const TreeArgs& a, cudaStream_t st);

}  // namespace rf
