// rf_tree.cuh - what the two kernels of rf_tree_attention share: the arguments, the
// split of the work over CTAs, visibility, and the softmax's constants.
#pragma once
#include <cuda_bf16.h>
#include <algorithm>

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
  uint32_t group, group_magic;  // query heads a KV head, and ceil(2^32 / group)
  float scale;
  unsigned* err;
};

// r / group for a query row r < 1024 * group, group <= kMaxGroup: the magic's excess times r stays below 2^32.
constexpr uint32_t kMaxGroup = 1024;
__device__ __forceinline__ uint32_t group_div(const TreeArgs& a, uint32_t r) {
  return a.group == 1 ? r : __umulhi(r, a.group_magic);
}

// History length and draft count of sequence b; (0, 0) and the error bit where they do not fit the cache.
// The read-only path, so that the compiler keeps them in registers: with plain loads, which the error word's
// atomics make it repeat, a 64-token tree over 32768 Q8_0 takes 59 us in place of 55.  They are read after the
// wait for the kernel before (tests/test_gpu_verify_chain.py has one that writes them until then).
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

// The powers of two that take a row of largest magnitude `top` to [1, 4) and back (1 for 0, infinity
// and NaN): products with them are exact.
__device__ __forceinline__ void pow2_scale(float top, float* down, float* up) {
  const int e = top > 0.f && top < INFINITY ? min(max(__float_as_int(top) >> 23, 1), 253) : 127;  // biased exponent
  *down = __int_as_float((254 - e) << 23);
  *up = __int_as_float(e << 23);
}

// ---------------------------------------------------------------------------
// The work split.  A unit is (sequence b, KV head h, row tile rt): up to ROWS of the
// n_b * G query rows (G query heads share a KV head; row r = token r / G, head r % G)
// against all its keys, in tiles of KT.  The lengths are read on the device, and every warp
// that needs the plan computes it.  Two ways to give the units to the CTAs:
//
//   by quota   each CTA gets at most `quota` tiles of one unit: the smallest quota for which the
//              grid has CTAs enough.  Nobody changes unit, which costs a CTA about 4 us.
//   in a row   all tiles of all units, in order, in equal ranges: the best balance, at the cost
//              of CTAs that end one unit and begin another.  For a quota that would be over
//              the even share by more than kSwitch tiles (or more units than CTAs).
//
// (16 tokens over 4095 Q8_0 positions, 32/8 heads: 20.0 us in a row, 15.4 by quota; 256 tokens over
// 32768, 64/8 heads: 129 tiles a CTA by quota, 112 in a row.)  A unit that lies in one CTA is
// finished there; the others leave partial results that tree_merge_kernel adds in order of
// the keys, so results do not depend on timing.  A CTA leaves at most two: slot 0 for the unit
// its tiles start inside of, slot 1 for the one they end inside of.
// ---------------------------------------------------------------------------
constexpr uint32_t kSwitch = 3;

// x / y, on the short path where both fit 32 bits.
__device__ __forceinline__ uint32_t div_u(uint64_t x, uint64_t y) {
  return (x | y) >> 32 ? (uint32_t)(x / y) : (uint32_t)x / (uint32_t)y;
}

// A run of consecutive key tiles of one unit: what a CTA works on at a time.
struct Segment {
  uint32_t b, h, rt;          // sequence, KV head, row tile
  uint32_t k0, k1, tiles;     // the run [k0, k1) of the unit's tiles
  uint32_t hist, drafts, end; // lengths of the sequence; end = hist + drafts
  __device__ bool whole() const { return k0 == 0 && k1 == tiles; }
};

template <int KT, int ROWS>
struct Plan {
  uint64_t all;         // tiles of all units
  uint32_t quota;       // most tiles of a CTA; 0: in a row
  uint32_t ctas;        // in a row: CTAs with work; the first `more` take `each` + 1 tiles, the others `each`
  uint64_t each, more;

  static __device__ __forceinline__ uint32_t tiles(uint32_t L, uint32_t n) { return n ? (L + n + KT - 1) / KT : 0; }
  static __device__ __forceinline__ uint32_t units(const TreeArgs& a, uint32_t n) {
    return (n * a.group + ROWS - 1) / ROWS * a.c.n_kv_heads;
  }
  // What sequence b takes: tiles (q = 0), or CTAs at a quota of q.
  static __device__ __forceinline__ uint64_t share(const TreeArgs& a, uint32_t b, uint32_t q) {
    if (b >= a.n_seqs) return 0;
    uint32_t L, n;
    seq_lengths(a, b, &L, &n);
    const uint32_t t = tiles(L, n);
    return (uint64_t)units(a, n) * (q ? (t + q - 1) / q : t);
  }
  // Whole warp: the shares of the sequences from `first` to before `limit`.
  static __device__ __forceinline__ uint64_t sum(const TreeArgs& a, uint32_t first, uint32_t limit, uint32_t q) {
    if (limit <= first + 1) return limit > first ? share(a, first, q) : 0;
    uint64_t t = 0;
    for (uint32_t i = first + (threadIdx.x & 31); i < limit; i += 32) t += share(a, i, q);
#pragma unroll
    for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    return t;
  }
  // Whole warp.
  __device__ __forceinline__ Plan(const TreeArgs& a, uint32_t grid) : each(0), more(0) {
    all = sum(a, 0, a.n_seqs, 0);
    ctas = all < grid ? (uint32_t)all : grid;
    quota = all <= grid;
    if (quota) return;
    each = div_u(all, ctas);
    more = all - each * ctas;
    const uint64_t least = each + (more ? 1 : 0);
    if (least >> 31) return;
    if (a.n_seqs == 1) {
      uint32_t L, n;
      seq_lengths(a, 0, &L, &n);
      const uint32_t u = units(a, n), per = u <= grid ? grid / u : 0, q = per ? (tiles(L, n) + per - 1) / per : 0;
      if (per && q <= least + kSwitch) quota = q;
      return;
    }
    // No quota does for more units than CTAs, which the largest quota tells (200 single tokens over 500 f16
    // positions, 32/8 heads: 97 us without that, 83 to 87 with it); with few (sequence, head) pairs it is not asked.
    constexpr uint32_t kMost = 1u << 31;
    uint32_t q = (uint64_t)a.n_seqs * a.c.n_kv_heads > grid ? kMost : (uint32_t)least;
#pragma unroll 1
    while (q == kMost || q <= least + kSwitch) {
      const bool fits = sum(a, 0, a.n_seqs, q) <= grid;
      if (fits && q != kMost) {
        quota = q;
        return;
      }
      if (!fits && q == kMost) return;
      q = q == kMost ? (uint32_t)least : q + 1;
    }
  }
  __device__ __forceinline__ uint64_t begin(uint32_t c) const { return each * c + min((uint64_t)c, more); }
  // In a row: the CTA that holds a tile.
  __device__ __forceinline__ uint32_t holder(uint64_t tile) const {
    const uint64_t wide = more * (each + 1);
    return tile < wide ? div_u(tile, each + 1) : (uint32_t)more + div_u(tile - wide, each);
  }
  // Whole warp: the sequence whose share holds w (w below the sum of all), and w's offset in it.
  static __device__ __forceinline__ uint32_t locate(const TreeArgs& a, uint64_t w, uint32_t q, uint64_t* offset) {
    const uint32_t lane = threadIdx.x & 31;
    *offset = w;
    if (a.n_seqs == 1) return w < share(a, 0, q) ? 0 : 1;
    uint64_t acc = 0;
    for (uint32_t base = 0; base < a.n_seqs; base += 32) {
      uint64_t s = share(a, base + lane, q);
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
    return a.n_seqs;
  }
};

// The segments of this CTA, in order.
template <int KT, int ROWS>
struct Walk {
  using P = Plan<KT, ROWS>;
  uint64_t left, rem;  // tiles left (by quota: 1 for the CTA's only segment), and the next one's offset in sequence b
  uint32_t b, quota;
  // Whole warp.
  __device__ __forceinline__ Walk(const TreeArgs& a) : left(0), rem(0), b(0) {
    const P p(a, gridDim.x);
    quota = p.quota;
    if (quota) {
      b = P::locate(a, blockIdx.x, quota, &rem);
      left = b < a.n_seqs;
    } else if (blockIdx.x < p.ctas) {
      const uint64_t w = p.begin(blockIdx.x);
      left = p.begin(blockIdx.x + 1) - w;
      b = P::locate(a, w, 0, &rem);
    }
  }
  __device__ __forceinline__ bool next(const TreeArgs& a, Segment* s) {
    if (!left) return false;
    uint32_t L, n;
    seq_lengths(a, b, &L, &n);
    uint32_t tiles = P::tiles(L, n), units = P::units(a, n);
    uint32_t unit;
    if (quota) {
      const uint32_t parts = (tiles + quota - 1) / quota, part = (uint32_t)rem % parts;
      unit = (uint32_t)rem / parts;
      s->k0 = (uint32_t)((uint64_t)tiles * part / parts), s->k1 = (uint32_t)((uint64_t)tiles * (part + 1) / parts);
      left = 0;
    } else {
      while (rem == (uint64_t)tiles * units) {  // past this sequence (or it has no work)
        b++;
        rem = 0;
        seq_lengths(a, b, &L, &n);
        tiles = P::tiles(L, n), units = P::units(a, n);
      }
      unit = div_u(rem, tiles);
      s->k0 = (uint32_t)(rem - (uint64_t)unit * tiles);
      s->k1 = (uint32_t)min((uint64_t)tiles, s->k0 + left);
      left -= s->k1 - s->k0;
      rem += s->k1 - s->k0;
    }
    const uint32_t rts = units / a.c.n_kv_heads;
    s->b = b, s->h = unit / rts, s->rt = unit - s->h * rts;
    s->tiles = tiles;
    s->hist = L, s->drafts = n, s->end = L + n;
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
// below 2^15, so that f16 keeps 11 bits of every weight down to 2^-21 of the largest.  With f16 and bf16
// activations a weight is that one f16, which is what their products take: a second term would double
// the products (f32 activations have it), and 2^-11 is what f16 outputs round by themselves.
constexpr float kRaise = 8.f, kWeightBias = 7.f;

// ---------------------------------------------------------------------------
// Joins the partial results of the units that several of the first kernel's CTAs shared
// (`grid` of them), in order of the keys, and writes the zeros of tokens past a sequence's drafts.
// A CTA takes 8 rows of a (sequence, KV head) and DPC dimensions; four threads share each
// piece of 4 dimensions, each adding every fourth partial result against a maximum of its own.
// Latency bounds it, so that what counts is the number of requests in flight on an SM:
//   few rows   a CTA for 32 dimensions, kAhead partial results with their maxima and sums
//              requested at once.  For a grid of up to two CTAs an SM with the registers for all of
//              them (one token over 131072 Q8_0 positions: 59.1 us with BLOCKS = 2, 60.1 with 4), above it
//              with as many CTAs an SM as fit (64 tokens over 8192, 32/8 heads: 28.2 with 4, 30.8 with 2).
//   many rows  a CTA for all dimensions, one partial result at a time, and a grid that fits the SMs,
//              since each CTA computes the plan: 24 sequences of 64 tokens over 500 positions, 32/8
//              heads, 80 us; with a CTA for each 8 rows and three partial results ahead 108.
// ---------------------------------------------------------------------------
template <class T, int D, int KT, int ROWS, int DPC, int BLOCKS>
__global__ void __launch_bounds__(256, BLOCKS)
    tree_merge_kernel(TreeArgs a, const float* __restrict__ part, uint32_t grid) {
  constexpr int X = DPC / 32, kAhead = X == 1 ? 6 : 1;
  __shared__ float4 s_o[4][64];
  __shared__ float2 s_ml[4][8];
  const uint32_t tid = threadIdx.x, rx = tid & 7, dx = (tid >> 3) & 7, cx = tid >> 6;
  const uint32_t groups = (a.n_tokens * a.group + 7) / 8;
  const uint32_t items = a.n_seqs * a.c.n_kv_heads * groups;
  griddep_launch();
  const Plan<KT, ROWS> plan(a, grid);
  uint64_t before = 0;  // what the sequences before `summed` take
  uint32_t summed = 0;
  for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
    const uint32_t bh = item / groups, r0 = (item - bh * groups) * 8;
    const uint32_t b = bh / a.c.n_kv_heads, h = bh - b * a.c.n_kv_heads;
    const uint32_t r = r0 + rx, t = group_div(a, r), hq = h * a.group + (r - t * a.group), d0 = blockIdx.y * DPC + dx * 4;
    T* out = (T*)a.out + ((uint64_t)b * a.n_tokens + t) * a.out_stride + (uint64_t)hq * D + d0;
    // the lengths were there before the first kernel began to read; every CTA waits for that kernel
    // before it ends, so that whoever waits for this one has waited for both
    uint32_t L, n;
    seq_lengths(a, b, &L, &n);
    if (t < a.n_tokens && t >= n && cx == 0) {
#pragma unroll
      for (int x = 0; x < X; x++)
#pragma unroll
        for (int i = 0; i < 4; i++) act_put(out + 32 * x + i, 0.f);
    }
    const uint32_t tiles = plan.tiles(L, n), parts = plan.quota ? (tiles + plan.quota - 1) / plan.quota : tiles;
    uint32_t c0 = 0, c1 = 0;  // the CTAs that shared the unit
    if (r0 < n * a.group) {
      if constexpr (DPC == D)
        before += plan.sum(a, summed, b, plan.quota), summed = b;
      else  // one piece of work a CTA
        before = plan.sum(a, 0, b, plan.quota);
      const uint64_t unit = (uint64_t)h * (plan.units(a, n) / a.c.n_kv_heads) + r0 / ROWS, u0 = before + unit * parts;
      c0 = plan.quota ? (uint32_t)u0 : plan.holder(u0);
      c1 = plan.quota ? (uint32_t)u0 + parts - 1 : plan.holder(u0 + tiles - 1);
    }
    griddep_wait();
    if (c0 == c1) continue;  // no rows, or finished by its CTA
    const uint32_t rl = r % ROWS;
    float M = -INFINITY, den = 0.f;
    float4 acc[X];
#pragma unroll
    for (int x = 0; x < X; x++) acc[x] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t c = c0 + cx; c <= c1; c += 4 * kAhead) {
      float m[kAhead], l[kAhead];
      float4 v[kAhead][X];
#pragma unroll
      for (int k = 0; k < kAhead; k++) {
        const uint32_t ck = c + 4 * k;
        m[k] = -INFINITY, l[k] = 0.f;
#pragma unroll
        for (int x = 0; x < X; x++) v[k][x] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (ck <= c1) {
          const float* s = part + (2 * (size_t)ck + (ck == c0 ? 1 : 0)) * part_floats(ROWS, D);
          m[k] = __ldcg(s + ROWS * D + rl), l[k] = __ldcg(s + ROWS * D + ROWS + rl);
#pragma unroll
          for (int x = 0; x < X; x++) v[k][x] = __ldcg(reinterpret_cast<const float4*>(s + part_at<ROWS>(d0 + 32 * x, rl)));
        }
      }
      float top = M;
#pragma unroll
      for (int k = 0; k < kAhead; k++) top = fmaxf(top, m[k]);
      const float old = top == -INFINITY ? 1.f : ex2(M - top);
      M = top;
      den *= old;
#pragma unroll
      for (int x = 0; x < X; x++) acc[x].x *= old, acc[x].y *= old, acc[x].z *= old, acc[x].w *= old;
#pragma unroll
      for (int k = 0; k < kAhead; k++) {
        const float f = top == -INFINITY ? 1.f : ex2(m[k] - top);
        den += l[k] * f;
#pragma unroll
        for (int x = 0; x < X; x++)
          acc[x].x += v[k][x].x * f, acc[x].y += v[k][x].y * f, acc[x].z += v[k][x].z * f, acc[x].w += v[k][x].w * f;
      }
    }
    if (dx == 0) s_ml[cx][rx] = make_float2(M, den);
    float f[4], inv = 0.f;
#pragma unroll
    for (int x = 0; x < X; x++) {
      if (x) __syncthreads();
      s_o[cx][tid & 63] = acc[x];
      __syncthreads();
      if (cx == 0 && t < n) {
        if (x == 0) {
          float top = -INFINITY, l = 0.f;
#pragma unroll
          for (int i = 0; i < 4; i++) top = fmaxf(top, s_ml[i][rx].x);
#pragma unroll
          for (int i = 0; i < 4; i++) {
            f[i] = top == -INFINITY ? 1.f : ex2(s_ml[i][rx].x - top);
            l += s_ml[i][rx].y * f[i];
          }
          inv = l == 0.f ? 0.f : 1.f / l;
        }
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float4 v = s_o[i][tid];
          o.x += v.x * f[i], o.y += v.y * f[i], o.z += v.z * f[i], o.w += v.w * f[i];
        }
        T* p = out + 32 * x;
        act_put(p, o.x * inv), act_put(p + 1, o.y * inv), act_put(p + 2, o.z * inv), act_put(p + 3, o.w * inv);
      }
    }
    __syncthreads();  // of s_ml and s_o, before the next rows
  }
}
// `carveout`: the first kernel's share of shared memory, kept so that the SMs need not change it between the two.
template <class T, int D, int KT, int ROWS>
cudaError_t launch_merge(cudaStream_t st, const TreeArgs& a, const float* part, uint32_t grid, int carveout) {
  const uint32_t blocks = a.n_seqs * a.c.n_kv_heads * ((a.n_tokens * a.group + 7) / 8), sms = (uint32_t)num_sms();
  const bool many = blocks > 2 * sms;
  auto* k = many                          ? tree_merge_kernel<T, D, KT, ROWS, D, 4>
            : blocks * (D / 32) > 2 * sms ? tree_merge_kernel<T, D, KT, ROWS, 32, 4>
                                          : tree_merge_kernel<T, D, KT, ROWS, 32, 2>;
  const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributePreferredSharedMemoryCarveout, carveout);
  if (e != cudaSuccess) return e;
  return launch_k(Launch{st, true}, k, dim3(many ? std::min(blocks, 4 * sms) : blocks, many ? 1 : D / 32), dim3(256), 0, a,
                  part, grid);
}

// Scratch of one call: allocated in stream order from a pool of this library's own that keeps
// its memory, to be freed on the same stream, so calls on any stream, and captured ones, never
// share a buffer (rf_tree.cu).
int scratch_alloc(void** out, size_t bytes, cudaStream_t st);

// The kernel for many query rows a KV head (rf_tree_tc.cu).
int run_tree_tc(int act_type, const TreeArgs& a, cudaStream_t st);

}  // namespace rf
