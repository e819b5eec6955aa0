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
  const int32_t L = __ldg(a.hist_len + b), n = a.n_draft ? __ldg(a.n_draft + b) : (int32_t)a.n_tokens;
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

// Equal ranges of `all` tiles: the first `more` CTAs take `each` + 1, the others `each`.
struct Ranges {
  uint64_t all, each, more;
  uint32_t ctas;  // as many as there are tiles, at most the grid
  __device__ __forceinline__ Ranges(uint64_t all_, uint32_t grid) : all(all_), each(0), more(0) {
    ctas = all < grid ? (uint32_t)all : grid;
    if (!ctas) return;
    each = all >> 32 ? all / ctas : (uint32_t)all / ctas;
    more = all - each * ctas;
  }
  __device__ __forceinline__ uint64_t begin(uint32_t c) const { return each * c + min((uint64_t)c, more); }
  __device__ __forceinline__ uint32_t holder(uint64_t tile) const {  // the CTA of a tile
    const uint64_t wide = more * (each + 1);
    return tile < wide ? div(tile, each + 1) : (uint32_t)more + div(tile - wide, each);
  }
  static __device__ __forceinline__ uint32_t div(uint64_t x, uint64_t y) {
    return (x | y) >> 32 ? (uint32_t)(x / y) : (uint32_t)x / (uint32_t)y;
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
  uint64_t left, rem;  // tiles left, and the next one's offset in sequence b
  uint32_t b;
  // Whole warp.
  __device__ __forceinline__ Walk(const TreeArgs& a) {
    uint64_t ignore;
    const Ranges r(Sp::total(a, 0, &ignore), gridDim.x);
    left = 0;
    if (blockIdx.x >= r.ctas) return;
    const uint64_t w = r.begin(blockIdx.x);
    left = r.begin(blockIdx.x + 1) - w;
    b = Sp::locate(a, w, &rem);
  }
  __device__ __forceinline__ bool next(const TreeArgs& a, Segment* s) {
    if (!left) return false;
    uint32_t L, n;
    seq_lengths(a, b, &L, &n);
    uint32_t tiles = Sp::tiles(L, n), rts = Sp::row_tiles(a, n);
    while (rem == (uint64_t)tiles * rts * a.c.n_kv_heads) {  // past this sequence (or it has no work)
      b++;
      rem = 0;
      seq_lengths(a, b, &L, &n);
      tiles = Sp::tiles(L, n), rts = Sp::row_tiles(a, n);
    }
    const uint32_t unit = Ranges::div(rem, tiles);
    s->b = b, s->h = unit / rts, s->rt = unit - s->h * rts;
    s->k0 = (uint32_t)(rem - (uint64_t)unit * tiles);
    s->k1 = (uint32_t)min((uint64_t)tiles, s->k0 + left);
    s->tiles = tiles;
    s->hist = L, s->drafts = n, s->end = L + n;
    left -= s->k1 - s->k0;
    rem += s->k1 - s->k0;
    return true;
  }
};

// One partial result: output sums as [D / 4][ROWS] of 4 floats (rows side by side, so that
// threads that own a row write and read 16-byte pieces in a run), then ROWS maxima and ROWS sums.
constexpr size_t part_floats(int rows, int D) { return (size_t)rows * (D + 2); }
template <int ROWS>
__device__ __forceinline__ size_t part_at(uint32_t d, uint32_t r) { return ((size_t)(d / 4) * ROWS + r) * 4; }

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
// Joins the partial results of the units that several of the first kernel's CTAs shared
// (`grid` of them), in order of the keys, and writes the zeros of tokens past a sequence's drafts.
// A CTA takes 8 rows of a (sequence, KV head) and 32 dimensions, four threads to each piece
// of 4: each adds every fourth partial result.  What bounds it is latency, so many small CTAs.
// ---------------------------------------------------------------------------
template <class T, int D, int KT, int ROWS>
__global__ void __launch_bounds__(256) tree_merge_kernel(TreeArgs a, const float* __restrict__ part, uint32_t grid) {
  using Sp = Split<KT, ROWS>;
  __shared__ float4 s_o[4][64];
  __shared__ float s_l[4][8];
  const uint32_t tid = threadIdx.x, rx = tid & 7, dx = (tid >> 3) & 7, cx = tid >> 6;
  const uint32_t G = a.n_heads / a.c.n_kv_heads, groups = (a.n_tokens * G + 7) / 8;
  const uint32_t bh = blockIdx.x / groups, r0 = (blockIdx.x - bh * groups) * 8;
  const uint32_t b = bh / a.c.n_kv_heads, h = bh - b * a.c.n_kv_heads;
  const uint32_t r = r0 + rx, t = r / G, hq = h * G + (r - t * G), d = blockIdx.y * 32 + dx * 4;
  T* out = (T*)a.out + ((uint64_t)b * a.n_tokens + t) * a.out_stride + (uint64_t)hq * D + d;
  uint32_t L, n;
  seq_lengths(a, b, &L, &n);
  if (r < a.n_tokens * G && t >= n && cx == 0) act_put(out, 0.f), act_put(out + 1, 0.f), act_put(out + 2, 0.f), act_put(out + 3, 0.f);
  if (r0 >= n * G) return;
  uint64_t before;
  const Ranges ranges(Sp::total(a, b, &before), grid);
  const uint32_t tiles = Sp::tiles(L, n);
  const uint64_t u0 = before + ((uint64_t)h * Sp::row_tiles(a, n) + r0 / ROWS) * tiles;
  const uint32_t c0 = ranges.holder(u0), c1 = ranges.holder(u0 + tiles - 1);
  if (c0 == c1) return;  // finished by its CTA
  griddep_wait();
  const uint32_t rl = r % ROWS;
  auto slot = [&](uint32_t c) { return part + (2 * (size_t)c + (c == c0 ? 1 : 0)) * part_floats(ROWS, D); };
  float M = -INFINITY;
#pragma unroll 8
  for (uint32_t c = c0; c <= c1; c++) M = fmaxf(M, __ldcg(slot(c) + ROWS * D + rl));
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float den = 0.f;
#pragma unroll 8
  for (uint32_t c = c0 + cx; c <= c1; c += 4) {
    const float* s = slot(c);
    const float f = M == -INFINITY ? 1.f : ex2(__ldcg(s + ROWS * D + rl) - M);
    const float4 v = __ldcg(reinterpret_cast<const float4*>(s + part_at<ROWS>(d, rl)));
    den += __ldcg(s + ROWS * D + ROWS + rl) * f;
    acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
  }
  s_o[cx][tid & 63] = acc;
  if (dx == 0) s_l[cx][rx] = den;
  __syncthreads();
  if (cx == 0 && t < n) {
#pragma unroll
    for (int i = 1; i < 4; i++) {
      const float4 v = s_o[i][tid];
      acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
    }
    const float l = s_l[0][rx] + s_l[1][rx] + s_l[2][rx] + s_l[3][rx], inv = l == 0.f ? 0.f : 1.f / l;
    act_put(out, acc.x * inv), act_put(out + 1, acc.y * inv), act_put(out + 2, acc.z * inv), act_put(out + 3, acc.w * inv);
  }
}
template <class T, int D, int KT, int ROWS>
cudaError_t launch_merge(cudaStream_t st, const TreeArgs& a, const float* part, uint32_t grid) {
  const uint32_t groups = (a.n_tokens * (a.n_heads / a.c.n_kv_heads) + 7) / 8;
  return launch_k(Launch{st, true}, tree_merge_kernel<T, D, KT, ROWS>, dim3(a.n_seqs * a.c.n_kv_heads * groups, D / 32),
                  dim3(256), 0, a, part, grid);
}

// Scratch of one call: allocated in stream order from a pool of this library's own that keeps
// its memory, to be freed on the same stream, so calls on any stream, and captured ones, never
// share a buffer (rf_tree.cu).
int scratch_alloc(void** out, size_t bytes, cudaStream_t st);

// The kernel for many query rows a KV head (rf_tree_tc.cu).
int run_tree_tc(int act_type, const TreeArgs& a, cudaStream_t st);

}  // namespace rf
