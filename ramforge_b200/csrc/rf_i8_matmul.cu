// rf_i8_matmul.cu - Y = X W^T in 8-bit integers with a scale for each token (row of X) and channel (row of W).
//
// The sums are whole 32-bit numbers and exact, so any split of the work gives the same bits:
//   y[t][n] = f32(f32(f32(sum) * x_scale[t]) * w_scale[n]) + bias[n], rounded to the output's type.
//
// The products run on tcgen05 (kind::i8) with channels as the rows of a tile and tokens as its columns: few tokens
// fill a tile of few columns, and a warp's 32 lanes of the accumulator are 32 consecutive outputs of one token.
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "rf_act.cuh"
#include "rf_device.cuh"
#include "rf_pair.cuh"
#include "rf_ring.cuh"
#include "rf_verify.h"

namespace rf {
namespace {

constexpr uint32_t kMaxIn = 65536;  // 65536 * 128 * 128 < 2^31

struct MatmulArgs {
  const int8_t *x, *w;
  const float *x_scale, *w_scale, *bias;
  void* y;
  uint64_t x_stride, w_stride, y_stride;
  uint32_t n_tokens, n_out, n_in;
};

// ---- waits, tensor memory, copies -------------------------------------------------------
// The value of lane 0, which the compiler then keeps in a uniform register, as descriptors want.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(~0u, x, 0); }
// True in one lane of the (whole) warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(p));
  return p != 0;
}
// 32 columns of the thread's lane (32 * (warp % 4) + lane).
__device__ __forceinline__ void tmem_ask_32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31"
      "}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
// What was asked for is there; the registers pass through so that no use moves above the wait.
__device__ __forceinline__ void tmem_have(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; i++) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_prefetch(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}
// K-major operand of 128-byte rows, 128-byte swizzle: groups of 8 rows 1024 bytes apart.
__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}
// kind::i8: signed codes, 32-bit sums, M x N.
__device__ __forceinline__ uint32_t idesc_i8(uint32_t m, uint32_t n) {
  return 2u << 4 | 1u << 7 | 1u << 10 | (n >> 3) << 17 | (m >> 4) << 24;
}
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{ .reg .pred p; setp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p; }" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
      : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// The address of `addr` in the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t map_cluster(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

// Four channels n .. n + 3 of token t.
template <class T>
__device__ __forceinline__ void put4(const MatmulArgs& a, uint32_t t, uint32_t n, const float (&v)[4], bool wide) {
  T* y = (T*)a.y + t * a.y_stride + n;
  if (wide && n + 4 <= a.n_out) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(y) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      T h[4];
#pragma unroll
      for (int i = 0; i < 4; i++) Act<T>::put(h + i, v[i]);
      *reinterpret_cast<uint2*>(y) = *reinterpret_cast<const uint2*>(h);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (n + i < a.n_out) Act<T>::put(y + i, v[i]);
  }
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Sums r of 32 tokens (rows of y from y on) of the channel nw + lane, a warp's 32 channels whole.  Of 16-bit outputs
// that lie in whole words (`wide`) the lanes 2i and 2i + 1 exchange one each, so that each stores two channels of one token.
template <class T, bool WIDE>
__device__ __forceinline__ void put_columns_as(T* y, uint64_t stride, uint32_t nw, uint32_t lane, const uint32_t (&r)[32],
                                               const float* sx, float sw, bool add, float bias) {
  const float2 w2 = make_float2(sw, sw);
  constexpr bool PAIR = sizeof(T) == 2 && WIDE;
  y += PAIR ? nw + (lane & 30) + (lane & 1) * stride : nw + lane;
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    const float4 x = *reinterpret_cast<const float4*>(sx + i);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int j = i + 2 * h;
      float2 v = make_float2((float)(int)r[j], (float)(int)r[j + 1]);
      v = pair_mul(pair_mul(v, h ? make_float2(x.z, x.w) : make_float2(x.x, x.y)), w2);
      if (add) v.x = __fadd_rn(v.x, bias), v.y = __fadd_rn(v.y, bias);
      if constexpr (PAIR) {
        const bool odd = lane & 1;
        const float other = __shfl_xor_sync(0xffffffffu, odd ? v.x : v.y, 1);
        *reinterpret_cast<uint32_t*>(y) = pack2<T>(odd ? other : v.x, odd ? v.y : other);
      } else {
        Act<T>::put(y, v.x);
        Act<T>::put(y + stride, v.y);
      }
      y += 2 * stride;
    }
  }
}
template <class T>
__device__ __forceinline__ void put_columns(T* y, uint64_t stride, uint32_t nw, uint32_t lane, const uint32_t (&r)[32],
                                            const float* sx, float sw, bool add, float bias, bool wide) {
  if (sizeof(T) == 2 && !wide)
    put_columns_as<T, false>(y, stride, nw, lane, r, sx, sw, add, bias);
  else
    put_columns_as<T, true>(y, stride, nw, lane, r, sx, sw, add, bias);
}
// The same for one channel (at y) and `count` tokens.
template <class T>
__device__ __forceinline__ void put_columns_any(T* y, uint64_t stride, uint32_t count, const uint32_t (&r)[32],
                                                const float* sx, float sw, bool add, float bias) {
#pragma unroll
  for (int i = 0; i < 32; i++) {
    if (i < count) {
      float v = __fmul_rn(__fmul_rn((float)(int)r[i], sx[i]), sw);
      if (add) v = __fadd_rn(v, bias);
      Act<T>::put(y, v);
    }
    y += stride;
  }
}

constexpr uint32_t TM = 128, TK = 128;  // channels of a tile, elements of a step

// ---------------------------------------------------------------------------
// One tile a cluster, its elements split over the cluster's CTAs: i8_split_kernel.
//
// A CTA has 128 channels x `cols` tokens and a run of the steps; warp 0 copies 128 bytes of each row a step through a
// ring of `stages`, warp 1 multiplies, and each CTA's sums go to the shared memory of the CTA that finishes their
// tokens.  (9 tokens through 128256 x 4096: 82 us, 0.98 of the copy rate; short calls are bound by their fixed parts, some 5 us of
// launch, first tile and meeting.)  Tensor memory is given back before the CTAs wait for one another, so that no two clusters can
// wait for each other's columns, and taken only after the kernel before has ended, whose CTAs may still need it.
// ---------------------------------------------------------------------------
constexpr uint32_t kMaxStages = 12;

struct SplitArgs {
  MatmulArgs a;
  uint32_t cols, stages, tmem_cols, steps, split;
  bool wide, wide4;  // y takes whole 4-byte words, four outputs at once
  unsigned* err;
};

template <class T>
__global__ void __launch_bounds__(256)
    i8_split_kernel(const SplitArgs s, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w) {
  extern __shared__ uint8_t dyn[];
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], done;
  __shared__ uint32_t s_tmem, s_stop;
  __shared__ __align__(16) float s_x[64];
  __shared__ float s_w[TM], s_b[TM];
  __shared__ uint32_t s_to[64];  // where a token's sums go
  const MatmulArgs& a = s.a;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t ring = (tc_smem_u32(dyn) + 1023) & ~1023u, stage = (TM + s.cols) * TK;
  const uint32_t rank = blockIdx.x % s.split, n0 = blockIdx.x / s.split * TM;
  const uint32_t k0 = s.steps * rank / s.split, k1 = s.steps * (rank + 1) / s.split;
  // each CTA of the cluster finishes a run of the tile's tokens: [CTA that sends][token][channel] behind the ring
  const uint32_t tokens = a.n_tokens, inbox = ring + s.stages * stage;
  const uint32_t first = tokens * rank / s.split, mine = tokens * (rank + 1) / s.split - first;
  const uint32_t room = (tokens + s.split - 1) / s.split * TM * 4;  // bytes of the inbox for each sender
  if (s.split > 1) cluster_arrive();
  if (tid == 0) {
    for (uint32_t i = 0; i < s.stages; i++) tc_mbar_init(tc_smem_u32(full + i), 1), tc_mbar_init(tc_smem_u32(empty + i), 1);
    tc_mbar_init(tc_smem_u32(&done), 1);
    tc_fence_barrier_init();
    s_stop = 0;
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
    for (uint32_t k = k0; k < min(k0 + s.stages, k1); k++) tma_prefetch(&map_w, k * TK, n0);  // into L2: safe before the wait
  }
  griddep_wait();
  if (warp == 2) tc_tmem_alloc(tc_smem_u32(&s_tmem), s.tmem_cols);
  if (tid < tokens) {
    s_x[tid] = a.x_scale[tid];
    if (s.split > 1) {
      const uint32_t to = ((tid + 1) * s.split - 1) / tokens;  // the CTA whose run holds the token
      s_to[tid] = map_cluster(inbox + rank * room + (tid - tokens * to / s.split) * TM * 4, to);
    }
  }
  if (tid < TM) {
    s_w[tid] = n0 + tid < a.n_out ? a.w_scale[n0 + tid] : 0.f;
    s_b[tid] = a.bias && n0 + tid < a.n_out ? a.bias[n0 + tid] : 0.f;
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  griddep_launch();
  const uint32_t tmem = s_tmem;
  volatile uint32_t* stop = &s_stop;

  // whole warps go round the ring, one lane issues: a loop of one lane keeps nothing in uniform registers, and its
  // products took 60 cycles each to issue
  if (warp == 0) {
    uint32_t slot = 0, phase = 0, k = k0;
    for (; k < k1; k++) {
      if (!wait_bar_warp(empty + slot, phase ^ 1, stop, s.err)) break;
      if (elect_one()) {
        const uint32_t bar = tc_smem_u32(full + slot), dst = ring + slot * stage;
        tc_mbar_expect_tx(bar, stage);
        tma_load(dst, &map_w, k * TK, n0, bar);
        tma_load(dst + TM * TK, &map_x, k * TK, 0, bar);
      }
      __syncwarp();
      if (++slot == s.stages) slot = 0, phase ^= 1;
    }
    if (k < k1)  // gave up: the copies in flight are waited for all the same
      for (uint32_t i = 0; i < min(k - k0, s.stages); i++) {
        if (slot-- == 0) slot = s.stages - 1, phase ^= 1;
        tc_mbar_wait(tc_smem_u32(full + slot), phase);
      }
  } else if (warp == 1) {
    const uint32_t idesc = idesc_i8(TM, s.cols);
    uint32_t slot = 0, phase = 0;
    for (uint32_t k = k0; k < k1; k++) {
      if (!wait_bar_warp(full + slot, phase, stop, s.err)) break;
      tc_fence_after_sync();
      const uint32_t at = uniform(ring + slot * stage);
      const uint64_t da = operand_desc(at), db = operand_desc(at + TM * TK);
      if (elect_one()) {
#pragma unroll
        for (int i = 0; i < 4; i++) mma_i8(tmem, da + 2 * i, db + 2 * i, idesc, k > k0 || i > 0);
        tc_commit(tc_smem_u32(empty + slot));
      }
      __syncwarp();
      if (++slot == s.stages) slot = 0, phase ^= 1;
    }
    if (elect_one()) tc_commit(tc_smem_u32(&done));
  }
  __syncwarp();
  const bool good = wait_bar_warp(&done, 0, stop, s.err);
  if (!good) tc_mbar_wait(tc_smem_u32(&done), 0);
  tc_fence_after_sync();

  __syncwarp();
  if (s.split > 1) cluster_wait();  // all CTAs of the cluster have begun: their shared memory may be written
  const uint32_t e = warp & 3;
  for (uint32_t c = 32 * (warp >> 2); c < tokens; c += 64) {
    uint32_t r[32];
    tmem_ask_32(tmem + (e << 21) + c, r), tmem_have(r);
    if (s.split > 1) {
#pragma unroll
      for (int i = 0; i < 32; i++)
        if (c + i < tokens)
          asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(s_to[c + i] + (32 * e + lane) * 4), "r"(r[i]) : "memory");
    } else if (good) {
      const uint32_t nw = n0 + 32 * e, n = nw + lane;
      const float sw = s_w[32 * e + lane], bias = s_b[32 * e + lane];
      T* y = (T*)a.y + (uint64_t)c * a.y_stride;
      if (nw + 32 <= a.n_out && c + 32 <= tokens)
        put_columns<T>(y, a.y_stride, nw, lane, r, s_x + c, sw, a.bias != nullptr, bias, s.wide);
      else if (n < a.n_out)
        put_columns_any<T>(y + n, a.y_stride, min(32u, tokens - c), r, s_x + c, sw, a.bias != nullptr, bias);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after_sync();
    tc_tmem_dealloc(tmem, s.tmem_cols);
  }
  __syncwarp();
  if (s.split == 1) return;
  cluster_arrive(), cluster_wait();
  // nothing of another CTA is touched from here on
  for (uint32_t i = tid; i < mine * (TM / 4); i += 256) {
    int4 sum = make_int4(0, 0, 0, 0);
    for (uint32_t r = 0; r < s.split; r++) {
      int4 v;
      asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(inbox + r * room + i * 16) : "memory");
      sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
    const uint32_t t = first + i / (TM / 4), c = i % (TM / 4) * 4;
    const int acc[4] = {sum.x, sum.y, sum.z, sum.w};
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      y[j] = __fmul_rn(__fmul_rn((float)acc[j], s_x[t]), s_w[c + j]);
      if (a.bias) y[j] = __fadd_rn(y[j], s_b[c + j]);
    }
    if (good) put4<T>(a, t, n0 + c, y, s.wide4);
  }
}

// ---------------------------------------------------------------------------
// Many tiles: i8_pair_kernel.
//
// A pair of CTAs (cta_group::2) has 256 channels x `cols` tokens: each holds 128 rows of W and half of the tokens'
// rows of X in its shared memory, and the sums of its channels in its tensor memory, so an SM reads 256 rows a step
// for 128 x 256 sums where a CTA alone reads 384 (4096 x 28672 x 4096: 303 us with pairs, 691 with CTAs of their own, one wave of
// tiles after the other).  At the tensor cores' full rate a step of 128 elements takes 512 cycles and 32 KB, 64 bytes a cycle and
// SM.  Long products are bound by the power cap's clock (3.2 PFLOP/s), short ones (n_in below about 1000) by the results.  Pairs stay and go from tile to tile; two accumulators, so that warps 4 to 11 write one out
// while the next fills.  Tokens' tiles come first in the order, so that a W tile is read by all of them at about one time.
//
//   warp 0  copies (both CTAs, completing on the first one's barriers)
//   warp 1  tcgen05.mma (the first CTA, for both)
//   warps 4 - 11  results
// ---------------------------------------------------------------------------
struct PairArgs {
  MatmulArgs a;
  uint32_t cols, n_tiles, tiles, stages, steps, sub;
  bool wide;  // y takes whole 4-byte words
  unsigned* err;
};
constexpr int kPairThreads = 384;

// A copy of one of the pair that completes on a barrier of either.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void mma_i8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{ .reg .pred p; setp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p; }" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
      : "memory");
}
// Arrive on `bar` of both CTAs when the products issued before are done.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"((uint16_t)3)
      : "memory");
}
template <class T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads)
    i8_pair_kernel(const PairArgs s, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w) {
  extern __shared__ uint8_t dyn[];
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_free[2];
  __shared__ uint32_t s_tmem, s_stop;
  __shared__ __align__(16) float s_x[8][256];
  const MatmulArgs& a = s.a;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = blockIdx.x & 1, pair = blockIdx.x >> 1;
  const uint32_t pairs = gridDim.x >> 1, half = s.cols / 2;
  const uint32_t ring = (tc_smem_u32(dyn) + 1023) & ~1023u, block = (TM + half) * TK, stage = s.sub * block;
  if (tid == 0) {
    for (uint32_t i = 0; i < s.stages; i++) tc_mbar_init(tc_smem_u32(full + i), 1), tc_mbar_init(tc_smem_u32(empty + i), 1);
    for (int i = 0; i < 2; i++) tc_mbar_init(tc_smem_u32(acc_full + i), 1), tc_mbar_init(tc_smem_u32(acc_free + i), 16);
    tc_fence_barrier_init();
    s_stop = 0;
  }
  griddep_wait();
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tc_smem_u32(&s_tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_arrive(), cluster_wait();
  tc_fence_after_sync();
  griddep_launch();
  const uint32_t tmem = s_tmem;
  volatile uint32_t* stop = &s_stop;

  if (warp == 0) {
    uint32_t slot = 0, phase = 0, uses = 0;
    bool ok = true;
    for (uint32_t tile = pair; tile < s.tiles && ok; tile += pairs) {
      const int n0 = tile / s.n_tiles * (2 * TM) + rank * TM, t0 = tile % s.n_tiles * s.cols + rank * half;
      for (uint32_t k = 0; k < s.steps; k++) {
        if (!(ok = wait_bar_warp(empty + slot, phase ^ 1, stop, s.err))) break;
        if (elect_one()) {
          const uint32_t bar = map_cluster(tc_smem_u32(full + slot), 0), dst = ring + slot * stage;
          if (rank == 0) tc_mbar_expect_tx(tc_smem_u32(full + slot), 2 * stage);
          for (uint32_t i = 0; i < s.sub; i++) {
            tma_load_pair(dst + i * block, &map_w, (k * s.sub + i) * TK, n0, bar);
            tma_load_pair(dst + i * block + TM * TK, &map_x, (k * s.sub + i) * TK, t0, bar);
          }
        }
        __syncwarp();
        uses++;
        if (++slot == s.stages) slot = 0, phase ^= 1;
      }
    }
    // the last products release their slots in both CTAs: neither ends before
    for (uint32_t i = 0; i < min(uses, s.stages) && ok; i++) {
      if (slot-- == 0) slot = s.stages - 1, phase ^= 1;
      ok = wait_bar_warp(empty + slot, phase, stop, s.err);
    }
    if (!ok) {  // gave up: copies in flight end within this time
      const long long t = clock64();
      while (clock64() - t < 4000000LL) {
      }
    }
  } else if (warp == 1 && rank == 0) {
    const uint32_t idesc = idesc_i8(2 * TM, s.cols);
    uint32_t slot = 0, phase = 0, buf = 0, turn = 0;
    bool ok = true;
    for (uint32_t tile = pair; tile < s.tiles && ok; tile += pairs) {
      ok = wait_bar_warp(acc_free + buf, turn ^ 1, stop, s.err);
      tc_fence_after_sync();
      for (uint32_t k = 0; k < s.steps && ok; k++) {
        if (!(ok = wait_bar_warp(full + slot, phase, stop, s.err))) break;
        tc_fence_after_sync();
        const uint32_t at = uniform(ring + slot * stage);
        if (elect_one()) {
          for (uint32_t j = 0; j < s.sub; j++) {
            const uint64_t da = operand_desc(at + j * block), db = operand_desc(at + j * block + TM * TK);
#pragma unroll
            for (int i = 0; i < 4; i++) mma_i8_pair(tmem + buf * 256, da + 2 * i, db + 2 * i, idesc, k > 0 || j > 0 || i > 0);
          }
          commit_pair(tc_smem_u32(empty + slot));
        }
        __syncwarp();
        if (++slot == s.stages) slot = 0, phase ^= 1;
      }
      if (elect_one()) commit_pair(tc_smem_u32(acc_full + buf));
      __syncwarp();
      if (++buf == 2) buf = 0, turn ^= 1;
    }
  } else if (warp >= 4) {
    const uint32_t e = warp & 3, set = (warp - 4) >> 2;  // channels 32 e on, every other 32 columns
    float* sx = s_x[warp - 4];
    uint32_t buf = 0, turn = 0;
    // scales and bias of a tile, asked for while the one before is written
    float sw_next = 0.f, bias_next = 0.f, x_next[8];
    auto ask = [&](uint32_t tile) {
      const uint32_t n = tile / s.n_tiles * (2 * TM) + rank * TM + 32 * e + lane, t0 = tile % s.n_tiles * s.cols;
      const bool live = tile < s.tiles && n < a.n_out;
      sw_next = live ? a.w_scale[n] : 0.f;
      bias_next = live && a.bias ? a.bias[n] : 0.f;
#pragma unroll
      for (uint32_t i = 0; i < 8; i++) {
        const uint32_t t = 32 * i + lane;
        x_next[i] = tile < s.tiles && t < s.cols && t0 + t < a.n_tokens ? a.x_scale[t0 + t] : 0.f;
      }
    };
    ask(pair);
    for (uint32_t tile = pair; tile < s.tiles; tile += pairs) {
      const uint32_t nw = tile / s.n_tiles * (2 * TM) + rank * TM + 32 * e, n = nw + lane, t0 = tile % s.n_tiles * s.cols;
      const uint32_t tokens = min(s.cols, a.n_tokens - t0);
      const bool live = n < a.n_out;
      const float sw = sw_next, bias = bias_next;
#pragma unroll
      for (uint32_t i = 0; i < 8; i++) sx[32 * i + lane] = x_next[i];
      __syncwarp();
      ask(tile + pairs);
      const bool good = wait_bar_warp(acc_full + buf, turn, stop, s.err);
      __syncwarp();
      tc_fence_after_sync();
      for (uint32_t c = 32 * set; c < s.cols; c += 64) {
        uint32_t r[32];
        tmem_ask_32(tmem + (e << 21) + buf * 256 + c, r), tmem_have(r);
        T* y = (T*)a.y + (uint64_t)(t0 + c) * a.y_stride;
        if (good && nw + 32 <= a.n_out && c + 32 <= tokens)
          put_columns<T>(y, a.y_stride, nw, lane, r, sx + c, sw, a.bias != nullptr, bias, s.wide);
        else if (good && live && c < tokens)
          put_columns_any<T>(y + n, a.y_stride, min(32u, tokens - c), r, sx + c, sw, a.bias != nullptr, bias);
        __syncwarp();
      }
      tc_fence_before_sync();
      __syncwarp();
      // what the arrival hands over is tensor memory, which the fence above orders; released to the whole cluster it would
      // wait for the results' stores as well (2048 x 8192 x 512: 18.2 us, 16.3 so)
      if (lane == 0)
        asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(map_cluster(tc_smem_u32(acc_free + buf), 0)) : "memory");
      if (++buf == 2) buf = 0, turn ^= 1;
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  cluster_arrive(), cluster_wait();
  if (warp == 2) {
    tc_fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// Tensor map of 8-bit rows, copied in boxes of 128 elements x box_rows.
int rows_map(CUtensorMap* map, const int8_t* p, uint64_t n_cols, uint64_t n_rows, uint64_t stride, uint32_t box_rows) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<void*> known{nullptr};  // calls may come from several threads
  void* fn = known.load(std::memory_order_relaxed);
  if (!fn) {
    cudaDriverEntryPointQueryResult q;
    RF_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &q));
    if (q != cudaDriverEntryPointSuccess || !fn) return set_error(RF_ECUDA, "cuTensorMapEncodeTiled is not available");
    known.store(fn, std::memory_order_relaxed);
  }
  const cuuint64_t dims[2] = {n_cols, n_rows}, strides[1] = {stride};
  const cuuint32_t box[2] = {TK, box_rows}, step[2] = {1, 1};
  const CUresult r = ((Encode)fn)(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(p), dims, strides, box, step,
                                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(RF_ECUDA, "cuTensorMapEncodeTiled failed with %d", (int)r);
  return RF_OK;
}

// One tile of tokens (at most kSplitCols).  The cluster's size is the one that a model of the call says is fastest, us:
// a step takes a CTA 0.2 (each SM's CTAs in turn), all of W at 6.5 TB/s as long as some 160 CTAs ask for it, a cluster
// 1 + 0.15 per CTA to meet; two CTAs an SM, of which clusters find room for about nine in ten.  1 token, 4096 x 4096: 10.7, 9.2,
// 7.8, 7.0 and 8.1 us with 1, 2, 3, 4 and 8 CTAs a cluster; 4096 x 14336: 26.9, 18.3, 15.8, 15.0, 14.0; 16 tokens, 28672 x 4096: 22.8 with 1, 26.3 with 2.
constexpr uint32_t kSplitCols = 64;

template <class T>
int run_split(cudaStream_t st, const MatmulArgs& a, unsigned* err) {
  SplitArgs s{};
  s.a = a, s.err = err;
  s.cols = (a.n_tokens + 15) / 16 * 16;
  s.steps = (a.n_in + TK - 1) / TK;
  s.tmem_cols = s.cols <= 32 ? 32 : 64;
  s.wide = aligned_to(a.y, 4) && a.y_stride * sizeof(T) % 4 == 0;
  s.wide4 = aligned_to(a.y, 4 * sizeof(T)) && a.y_stride % 4 == 0;
  const uint32_t tiles = (a.n_out + TM - 1) / TM, sms = (uint32_t)num_sms();
  const double w_us = (double)a.n_out * a.n_in / 6.5e6;
  double best = 1e30;
  for (uint32_t c = 1; c <= 8 && c <= s.steps; c++) {
    const double ctas = (double)tiles * c;
    const double load = 0.2 * ((tiles * (uint64_t)c + sms - 1) / sms) * ((s.steps + c - 1) / c);
    const double room = 2.0 * sms * (c > 1 ? 0.9 : 1.0), waves = c > 1 ? std::max(1.0, ctas / room) : 1.0;
    const double us = std::max(load, w_us * std::max(1.0, 160.0 / ctas)) + (c > 1 ? waves * (1.0 + 0.15 * c) : 0.0);
    if (us < best) best = us, s.split = c;
  }
  if ((uint64_t)tiles * s.split > 0x7fffffffull) return set_error(RF_EINVAL, "%u channels are too many for one call", a.n_out);
  // shared memory for two CTAs an SM: at least 3 stages (108 - 36 KB of 24) beside the inbox
  const uint32_t stage = (TM + s.cols) * TK, box = s.split > 1 ? (s.cols + s.split) * TM * 4 : 0;
  s.stages = std::min(std::min((108u * 1024 - box) / stage, kMaxStages), (s.steps + s.split - 1) / s.split);
  CUtensorMap mx{}, mw{};
  RF_TRY(rows_map(&mx, a.x, a.n_in, a.n_tokens, a.x_stride, s.cols));
  RF_TRY(rows_map(&mw, a.w, a.n_in, a.n_out, a.w_stride, TM));
  auto* k = i8_split_kernel<T>;
  RF_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, 109 * 1024));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles * s.split);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 1024 + (size_t)s.stages * stage + box;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = s.split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = s.split > 1 ? 2 : 1;
  RF_CUDA(cudaLaunchKernelEx(&cfg, k, s, mx, mw));
  return RF_OK;
}

// The tile's columns are those for which a model of the call says it is fastest: 256 elements take a pair
// 0.2 us and 1.8 ns a column, at least 0.28, and a tile's results 0.6 us and 9 ns a column; the longer of the two
// counts in each round, and the results of the last one besides; the bytes of W are not in it (128 tokens, 128256 x 4096: 50 us by
// the model, 87 measured, 86 by the bytes).  333 tokens, 4096 x 4096: 14.7 us with tiles of
// 192, 11.8 with 128, 11.2 with 96, 15.7 with 64 (two rounds); 3718 tokens, 6016 x 192: 37.4 with 32, 24.6 with 64,
// 19.7 with 128, 17.1 with 256.
template <class T>
int run_pair(cudaStream_t st, const MatmulArgs& a, unsigned* err) {
  PairArgs s{};
  s.a = a, s.err = err;
  const uint64_t m_tiles = (a.n_out + 2 * TM - 1) / (2 * TM), pairs = (uint64_t)std::max(1, num_sms() / 2);
  double best = 1e30;
  for (uint32_t cols = 256; cols >= 32; cols -= 32) {
    const uint64_t rounds = (m_tiles * ((a.n_tokens + cols - 1) / cols) + pairs - 1) / pairs;
    const double results = 0.6 + 0.009 * cols;
    const double us = (double)rounds * std::max(std::ceil(a.n_in / 256.0) * std::max(0.28, 0.2 + 0.0018 * cols), results) + results;
    if (us < best) best = us, s.cols = cols;
  }
  s.n_tiles = (a.n_tokens + s.cols - 1) / s.cols;
  s.cols = ((a.n_tokens + s.n_tiles - 1) / s.n_tiles + 31) / 32 * 32;  // even tiles
  // two blocks of 128 elements a stage where the products of one are done sooner than its barriers and commit (340 cycles):
  // 128 tokens, 4096 x 4096: 13.1 us with one, 9.6 with two
  s.sub = s.cols <= 192 ? 2 : 1;
  s.steps = (a.n_in + TK * s.sub - 1) / (TK * s.sub);
  const uint64_t tiles = m_tiles * s.n_tiles;
  if (tiles > 0x7fffffffull) return set_error(RF_EINVAL, "%u tokens x %u channels are too many for one call", a.n_tokens, a.n_out);
  s.tiles = (uint32_t)tiles;
  s.wide = aligned_to(a.y, 4) && a.y_stride * sizeof(T) % 4 == 0;
  // the whole of an SM's shared memory, also where fewer stages would do: two pairs never share an SM's tensor memory
  s.stages = std::min(208u * 1024 / ((TM + s.cols / 2) * TK * s.sub), kMaxStages);
  CUtensorMap mx{}, mw{};
  RF_TRY(rows_map(&mx, a.x, a.n_in, a.n_tokens, a.x_stride, s.cols / 2));
  RF_TRY(rows_map(&mw, a.w, a.n_in, a.n_out, a.w_stride, TM));
  const size_t smem = 209 * 1024;
  auto* k = i8_pair_kernel<T>;
  RF_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  RF_CUDA(launch_k(Launch{st, true}, k, dim3(2 * (uint32_t)std::min(tiles, pairs)), dim3(kPairThreads), smem, s, mx, mw));
  return RF_OK;
}

// ---------------------------------------------------------------------------
// Up to 8 tokens and a small matrix: i8_few_kernel.
//
// The bytes of W bound it, so they go from HBM straight into the registers of mma.sync (m16n8k32), channels as its rows,
// tokens as its columns; no ring, no tensor memory, no descriptors to fetch.  The order of the summed index is free: lane c of a
// group of four takes 16 consecutive bytes of a row's 64, whose words 0 and 1 (2 and 3) are the fragments of one product.
// A CTA has 16 channels, its warps take runs of 256 bytes of the rows in turn, two in flight each, and add up in shared memory.
// ---------------------------------------------------------------------------
constexpr int kRun = 4, kFewWarps = 8;  // 64-byte pieces of a run

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Bytes of u from n on become zeros.
__device__ __forceinline__ uint4 first_bytes(uint4 u, uint32_t n) {
  uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; i++) w[i] = n >= 4u * i + 4 ? w[i] : n <= 4u * i ? 0u : w[i] & (0xffffffffu >> (32 - 8 * (n - 4 * i)));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <class T>
__global__ void __launch_bounds__(32 * kFewWarps) i8_few_kernel(MatmulArgs a) {
  __shared__ int s_sum[kFewWarps][8][17];
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  const uint32_t n0 = blockIdx.x * 16;
  griddep_launch();
  if (tid < 16 && n0 + tid < a.n_out && a.n_in >= 16)  // the rows' beginnings into L2: safe before the wait
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(a.w + (n0 + tid) * a.w_stride), "r"(min(a.n_in, 4096u) & ~15u) : "memory");
  griddep_wait();
  const int8_t* w0 = a.w + min(n0 + g, a.n_out - 1) * a.w_stride;
  const int8_t* w1 = a.w + min(n0 + g + 8, a.n_out - 1) * a.w_stride;
  int acc[4] = {};
  uint4 wr[2][kRun][2];
  auto load = [&](uint4 (&r)[kRun][2], uint32_t k) {
#pragma unroll
    for (int i = 0; i < kRun; i++) {
      const uint32_t at = k + 64 * i + 16 * c;
      r[i][0] = r[i][1] = make_uint4(0, 0, 0, 0);
      if (at < a.n_in) r[i][0] = ld_once(w0 + at), r[i][1] = ld_once(w1 + at);
    }
  };
  auto multiply = [&](const uint4 (&r)[kRun][2], uint32_t k) {
    uint4 x[kRun];
#pragma unroll
    for (int i = 0; i < kRun; i++) {
      const uint32_t at = k + 64 * i + 16 * c;
      x[i] = make_uint4(0, 0, 0, 0);
      if (at < a.n_in && g < a.n_tokens) {
        x[i] = *reinterpret_cast<const uint4*>(a.x + g * a.x_stride + at);
        if (at + 16 > a.n_in) x[i] = first_bytes(x[i], a.n_in - at);  // what lies behind a row is no part of it
      }
    }
#pragma unroll
    for (int i = 0; i < kRun; i++) {
      mma_s8(acc, r[i][0].x, r[i][1].x, r[i][0].y, r[i][1].y, x[i].x, x[i].y);
      mma_s8(acc, r[i][0].z, r[i][1].z, r[i][0].w, r[i][1].w, x[i].z, x[i].w);
    }
  };
  constexpr uint32_t RUN = 64 * kRun, STEP = RUN * kFewWarps;
  uint32_t k = warp * RUN;
  if (k < a.n_in) load(wr[0], k);
  if (k + STEP < a.n_in) load(wr[1], k + STEP);
  for (; k < a.n_in; k += 2 * STEP) {
    multiply(wr[0], k);
    if (k + 2 * STEP < a.n_in) load(wr[0], k + 2 * STEP);
    if (k + STEP >= a.n_in) break;
    multiply(wr[1], k + STEP);
    if (k + 3 * STEP < a.n_in) load(wr[1], k + 3 * STEP);
  }
#pragma unroll
  for (int j = 0; j < 4; j++) s_sum[warp][2 * c + (j & 1)][g + 8 * (j >> 1)] = acc[j];
  __syncthreads();
  for (uint32_t i = tid; i < 16 * a.n_tokens; i += 32 * kFewWarps) {
    const uint32_t t = i >> 4, r = i & 15, n = n0 + r;
    if (n >= a.n_out) continue;
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kFewWarps; w++) sum += s_sum[w][t][r];
    float v = __fmul_rn(__fmul_rn((float)sum, a.x_scale[t]), a.w_scale[n]);
    if (a.bias) v = __fadd_rn(v, a.bias[n]);
    Act<T>::put((T*)a.y + t * a.y_stride + n, v);
  }
}

template <class T>
int run(cudaStream_t st, const MatmulArgs& a, unsigned* err) {
  // one token, 4096 x 4096: 6.0 us in i8_few_kernel and 7.0 in i8_split_kernel, 2048 x 2048: 3.1 and 6.0; its loads do not
  // keep up with a ring's where a warp has many runs or an SM many CTAs (6144 x 4096: 10.9 and 8.8; 86720 x 128: 32.9 and 6.6)
  if (a.n_tokens <= 8 && a.n_in <= 8192 && (uint64_t)a.n_out * a.n_in <= 18u << 20 && a.n_out <= 48u * num_sms()) {
    RF_CUDA(launch_k(Launch{st, true}, i8_few_kernel<T>, dim3((a.n_out + 15) / 16), dim3(32 * kFewWarps), 0, a));
    return RF_OK;
  }
  return a.n_tokens <= kSplitCols ? run_split<T>(st, a, err) : run_pair<T>(st, a, err);
}

int check_operand(const char* name, const int8_t* p, uint64_t* stride, uint32_t n_in) {
  if (!*stride) *stride = n_in;
  if (*stride < n_in)
    return set_error(RF_EINVAL, "%s stride %llu is below the row's %u elements", name, (unsigned long long)*stride, n_in);
  if (!aligned_to(p, 16) || *stride % 16 || *stride >= 1ull << 40)
    return set_error(RF_EINVAL, "%s rows must be 16-byte aligned (stride %llu)", name, (unsigned long long)*stride);
  return RF_OK;
}

}  // namespace
}  // namespace rf

using namespace rf;

extern "C" {

int rf_i8_matmul(const int8_t* x, const float* x_scale, const int8_t* w, const float* w_scale, const float* bias, void* y,
                 int act_type, uint32_t n_tokens, uint32_t n_out, uint32_t n_in, uint64_t x_stride, uint64_t w_stride,
                 uint64_t y_stride, void* stream) {
  const uint32_t es = act_bytes(act_type);
  if (!es) return set_error(RF_EINVAL, "activation type %d is not F32, F16 or BF16", act_type);
  if (!n_in || n_in > kMaxIn) return set_error(RF_EINVAL, "n_in %u is not within 1..%u", n_in, kMaxIn);
  if (n_tokens > 0x7fffff00u || n_out > 0x7fffff00u)
    return set_error(RF_EINVAL, "%u tokens x %u channels are too many for one call", n_tokens, n_out);
  if (n_tokens && n_out && (!x || !x_scale || !w || !w_scale || !y)) return set_error(RF_EINVAL, "null argument");
  RF_TRY(check_operand("x", x, &x_stride, n_in));
  RF_TRY(check_operand("w", w, &w_stride, n_in));
  if (!y_stride) y_stride = n_out;
  if (y_stride < n_out)
    return set_error(RF_EINVAL, "y stride %llu is below the row's %u elements", (unsigned long long)y_stride, n_out);
  if (!aligned_to(y, es)) return set_error(RF_EINVAL, "y must be aligned to its element size");
  if (!aligned_to(x_scale, 4) || !aligned_to(w_scale, 4) || !aligned_to(bias, 4))
    return set_error(RF_EINVAL, "scales and bias must be 4-byte aligned");
  if (!n_tokens || !n_out) return RF_OK;
  const MatmulArgs a{x, w, x_scale, w_scale, bias, y, x_stride, w_stride, y_stride, n_tokens, n_out, n_in};
  unsigned* err = nullptr;
  RF_TRY(verify_error_ptr(&err));
  const cudaStream_t st = (cudaStream_t)stream;
  switch (act_type) {
    case RF_ACT_F32: return run<float>(st, a, err);
    case RF_ACT_F16: return run<__half>(st, a, err);
    default: return run<__nv_bfloat16>(st, a, err);
  }
}

}  // extern "C"
