// rf_tree_tc.cu - rf_tree_attention for many query rows a KV head, on the 5th-generation
// tensor cores.
//
// With R = drafted tokens x query heads a KV head, every cached byte takes part in about
// R (f16) or 1.9 R (Q8_0) multiply-adds, so from some tens of rows on the products bound the
// call, not HBM.  A CTA (one an SM) works on RT x 128 query rows of one KV head against a run
// of 128-key tiles:
//
//   S[128 rows][128 keys] = Q K^T   A = Q, B = K, both K-major in shared memory
//   O[128 rows][D]       += P V     A = P in tensor memory, B = V, MN-major in shared memory
//
// Both S and O live in tensor memory, so a thread owns one row of S, its softmax needs no
// exchange, and P goes back over S's columns.  All 512 columns are used: two O, and for each
// group of softmax warps two S of 64 keys (the halves of a tile), so that the next scores of a
// half are computed while the softmax is at the other half.  K and V
// tiles have the same layout in shared memory ([128 keys][64 dimensions] blocks of 128-byte
// rows, 128-byte swizzle): read along the head they are K-major, read along the keys MN-major.
//
// Two groups of four warps do the softmax.  RT = 2: each has a row tile of its own and both
// share every K and V tile.  RT = 1 (at most 128 rows, or f32): both have the same rows and
// take the even and the odd key tiles, and are joined at the end.
//
//   warp 0        loads: f16 tiles by tensor copies, Q8_0 codes by plain bulk copies
//   warps 1, 2    tcgen05.mma, one warp a group
//   warp 3        f16: V tiles that hold drafts or the end are made finite (below)
//   warps 4 - 11  softmax, queries, outputs
//   warps 12 on   Q8_0: codes * scales -> f16 operand tiles, one key a thread, four warps a tile
//
// f32 queries and weights are split into two f16 terms, and each product into two MMAs.  The tensor core's f32
// sums truncate: an f32 output loses about 1.7e-8 of its size for each 16 keys and term that one group of one CTA
// sums (64 tokens over 60000 positions: 8.5e-6 off, the same in plain f32 4.6e-6).
// What a row does not see has weight 0, and 0 * NaN would still be NaN: elements of drafts'
// V rows that are not finite are replaced by 0 in shared memory, and a flag makes the
// epilogue add them to the rows that do see them.
//
// What bounds it.  Two row tiles, f16: no unit is full.  Of about 3,300 cycles a tile the tensor core works 61 % and a
// softmax warp 2,100 (230 instructions a half tile, 64 of them exponentials, and the waits for tensor memory);
// the rest is the chain between them, since P lies over the columns of S: the next scores of a half wait for its P
// and for the product with it (both MMA warps stand at those barriers about 650 cycles a tile).  The power cap
// lowers the clock besides: 256 tokens of 64/8 heads over 32768 f16 positions take 260 us in a short run and 305 to 330
// in a long one (1.06 and 0.84 to 0.91 PFLOP/s).  Two row tiles, Q8_0: the softmax beside the decode, whose instructions it shares the SM
// with: a half tile takes a softmax warp 1,630 cycles and 280 of waiting, a tile a decoding warp 1,300 and 550 of
// waiting (400 of them for a free slot).  With one row tile HBM and about 15 us of launch, first tiles and join:
// 5 tokens over 32768 f16 positions 36 us (20.5 for the bytes).
//
// Every wait is bounded (about a second): on expiry the kernel raises bit 0 of the error word,
// all roles run through their loops without waiting or issuing, the copies and MMAs in
// flight are waited for (bounded again), tensor memory is freed and the kernel returns.
#include <cuda.h>

#include <atomic>
#include <type_traits>

#include "rf_tc.cuh"
#include "rf_tree.cuh"

namespace rf {
namespace {

constexpr int TK = 128;                      // keys of a tile, rows of a row tile
constexpr uint32_t kOperandBytes = 224 * 1024;
constexpr uint32_t kBlockBytes = TK * 128;   // one [128][64] f16 block
constexpr uint32_t kAuxBytes = 2560;

template <class T, bool Q8, int D, int RT>
struct Shape {
  static constexpr bool SPLIT = std::is_same<T, float>::value;
  static constexpr int ROWS = TK * RT;
  // RT = 1 has little work a tile: eight warps decode Q8_0 (16 tokens over 32768 positions: 35 us now;
  // when it took 40, four warps took 49) and the softmax gets by with few registers.  RT = 2 waits for the
  // softmax more than for loads: a half row of S is held in registers (256 tokens of 64/8 heads over 32768 f16: 305 us,
  // with 32 columns at a time 344), and four warps decode.
  static constexpr bool HOLD = RT == 2;
  static constexpr int SETS = !Q8 ? 0 : RT == 1 ? 2 : 1;
  static constexpr int THREADS = 384 + 128 * SETS;
  static constexpr uint32_t TILE = TK * D * 2;
  static constexpr uint32_t RAW = TK * D;
  static constexpr uint32_t QBYTES = TILE * RT * (SPLIT ? 2 : 1);
  static constexpr int NRAW = Q8 ? 4 : 0;  // raw tiles in flight
  static constexpr int kFit = (kOperandBytes - QBYTES - NRAW * RAW) / TILE;
  static constexpr int NSLOT = kFit < 6 ? kFit : 6;
  static constexpr uint32_t SMEM = kOperandBytes + kAuxBytes;
  static constexpr int LEAD = RT == 1 ? 2 : 1;  // K tiles loaded ahead of the first V tile
};

// ---- tensor memory ------------------------------------------------------------------
// 32x32b accesses: the thread's lane (32 * (warp % 4) + lane), consecutive columns.
__device__ __forceinline__ void tmem_ld_32(uint32_t addr, uint32_t* r) {
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
__device__ __forceinline__ void tmem_ld_16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15"
      "}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
// The loads before are complete; the registers pass through so that no use moves above the wait.
template <int N>
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; i++) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tmem_st_32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {"
      "%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32"
      "};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
      "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {"
      "%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16"
      "};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---- operands -------------------------------------------------------------------------
// 128-byte swizzled operand: 8-row groups 1024 bytes apart; MN-major blocks of 64 elements
// kBlockBytes apart (ignored for K-major, where a k step stays inside one 128-byte row).
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)(kBlockBytes >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// kind::f16, f16 operands, f32 accumulator, M = 128; b_mn: B is MN-major.
constexpr uint32_t idesc_f16(int N, bool b_mn) {
  return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(TK >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  tc_mma_bf16(d, a, b, idesc, acc);  // the operand type is the descriptor's
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{ .reg .pred p; setp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
// 16-byte piece `c` (of D / 8) of row r in an operand tile.
__device__ __forceinline__ uint32_t sw128_offset(uint32_t r, uint32_t c) {
  return (c >> 3) * kBlockBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}
__device__ __forceinline__ void st_shared16(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// 16 bytes from global to shared memory, asynchronously; the last 16 - bytes as zeros.
__device__ __forceinline__ void cp_async16(uint32_t dst, uint64_t src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void st_shared8(uint32_t addr, uint32_t x, uint32_t y) {
  asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(addr), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// ---- pairs of f32 in one instruction ------------------------------------------------------
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)),
        "l"(reinterpret_cast<unsigned long long&>(c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}


// Non-finite f16 halves of a word replaced by 0.
__device__ __forceinline__ uint32_t finite_halves(uint32_t x, bool* wild) {
  const bool lo = (x & 0x7c00u) == 0x7c00u, hi = (x & 0x7c000000u) == 0x7c000000u;
  *wild |= lo || hi;
  return x & (lo ? 0xffff0000u : ~0u) & (hi ? 0x0000ffffu : ~0u);
}

// The value of lane 0, which the compiler then keeps in a uniform register.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(~0u, x, 0); }
// True in one lane of the (whole) warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(p));
  return p != 0;
}

// ---- shared-memory bookkeeping -----------------------------------------------------------
template <class S>
struct Bars {  // [group][half of the key tile]
  uint64_t full[S::NSLOT], free[S::NSLOT], fix[S::NSLOT];
  uint64_t raw_full[S::NRAW ? S::NRAW : 1], raw_free[S::NRAW ? S::NRAW : 1];
  uint64_t q_full[2], s_full[2][2], p_full[2][2], pv_done[2][2], drain;
  uint32_t tmem, stop, wild, pad;
  float ml[2][TK][2];
};

// A position in a ring of N slots: its index and the parity of its current use.
template <int N>
struct Ring {
  uint32_t s = 0, phase = 0;
  __device__ __forceinline__ void advance() {
    if (++s == N) s = 0, phase ^= 1;
  }
  __device__ __forceinline__ void retreat() {
    if (s-- == 0) s = N - 1, phase ^= 1;
  }
};

// Bounded wait for the phase of `bar` with `parity`; false once any wait of the CTA gave up.
__device__ __noinline__ bool wait_slow(uint32_t bar, uint32_t parity, volatile uint32_t* stop, unsigned* err) {
  const long long t0 = clock64();
  while (!tc_mbar_try_wait(bar, parity)) {
    if (*stop) return false;
    if (clock64() - t0 > 2000000000LL) {
      *stop = 1;
      atomicOr(err, kVerifyTimeout);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile uint32_t* stop, unsigned* err) {
  const uint32_t b = tc_smem_u32(bar);
  return tc_mbar_try_wait(b, parity) || wait_slow(b, parity, stop, err);
}

// The e-th tile a segment of nt key tiles loads (2 nt of them): LEAD K tiles, then V and K in turn.
__device__ __forceinline__ void item_at(uint32_t e, uint32_t nt, uint32_t lead, bool* is_v, uint32_t* i) {
  const uint32_t first = min(lead, nt);
  if (e < first) {
    *is_v = false, *i = e;
    return;
  }
  const uint32_t x = e - first, pairs = nt - first;
  if (x < 2 * pairs)
    *is_v = !(x & 1), *i = x & 1 ? first + x / 2 : x / 2;
  else
    *is_v = true, *i = x - pairs;
}

// Bit i: token t sees draft j0 + i (drafts below 0 are history, drafts from n on do not exist).
__device__ __forceinline__ uint32_t seen32(const uint32_t* mask_row, uint32_t words, uint32_t t, int j0, int n) {
  if (j0 >= n) return 0;
  if (j0 <= -32) return ~0u;
  uint32_t v;
  if (!mask_row) {
    const int count = (int)t - j0 + 1;
    v = count <= 0 ? 0 : count >= 32 ? ~0u : (1u << count) - 1;
  } else if (j0 >= 0) {
    const uint32_t w = j0 >> 5, sh = j0 & 31;
    v = mask_row[w] >> sh;
    if (sh && w + 1 < words) v |= mask_row[w + 1] << (32 - sh);
  } else {
    v = (mask_row[0] << -j0) | ((1u << -j0) - 1);
  }
  return n - j0 < 32 ? v & ((1u << (n - j0)) - 1) : v;
}

// Scores of the columns whose bit is not set become -infinity.
__device__ __forceinline__ void hide(uint32_t (&s)[32], uint32_t see) {
#pragma unroll
  for (int j = 0; j < 32; j++)
    if (!((see >> j) & 1)) s[j] = 0xff800000u;
}

// 16 bytes of a row as f32.
template <class T>
__device__ __forceinline__ void act_unpack(const uint4& u, float (&v)[16 / sizeof(T)]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (std::is_same<T, float>::value) {
      v[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    } else {
      v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_h2_rest(float a, float b, uint32_t hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return pack_h2(a - f.x, b - f.y);
}

template <class T, bool Q8, int D, int RT>
__global__ void __launch_bounds__(Shape<T, Q8, D, RT>::THREADS, 1)
    tree_tc_kernel(const TreeArgs a, float* __restrict__ part, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v) {
  using S = Shape<T, Q8, D, RT>;
  constexpr bool SPLIT = S::SPLIT;
  extern __shared__ __align__(1024) uint8_t tsm[];
  Bars<S>& B = *reinterpret_cast<Bars<S>*>(tsm + kOperandBytes);
  static_assert(sizeof(Bars<S>) <= kAuxBytes, "bookkeeping must fit");
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t q_smem = tc_smem_u32(tsm), slots = q_smem + S::QBYTES, raws = slots + S::NSLOT * S::TILE;
  auto slot_addr = [&](uint32_t s) { return slots + s * S::TILE; };
  // what is above the wait overlaps the kernel before
  if (warp == 1) tc_tmem_alloc(tc_smem_u32(&B.tmem), 512);
  if (tid == 0) {
    for (int i = 0; i < S::NSLOT; i++) {
      tc_mbar_init(tc_smem_u32(&B.full[i]), Q8 ? 4 : 1);
      tc_mbar_init(tc_smem_u32(&B.free[i]), Q8 ? 2 : 3);  // both MMA warps, and warp 3
      tc_mbar_init(tc_smem_u32(&B.fix[i]), 1);
    }
    for (int i = 0; i < S::NRAW; i++) {
      tc_mbar_init(tc_smem_u32(&B.raw_full[i]), 1);
      tc_mbar_init(tc_smem_u32(&B.raw_free[i]), 4);
    }
    for (int g = 0; g < 2; g++) tc_mbar_init(tc_smem_u32(&B.q_full[g]), 128);
    for (int g = 0; g < 2; g++)
      for (int h = 0; h < 2; h++) {
        tc_mbar_init(tc_smem_u32(&B.s_full[g][h]), 1);
        tc_mbar_init(tc_smem_u32(&B.p_full[g][h]), 4);
        tc_mbar_init(tc_smem_u32(&B.pv_done[g][h]), 1);
      }
    tc_mbar_init(tc_smem_u32(&B.drain), 2);
    B.stop = B.wild = 0;
    tc_fence_barrier_init();
  }
  griddep_wait();
  griddep_launch();  // of tree_merge_kernel, which reads the lengths before it waits: not before they are there
  Walk<TK, S::ROWS> walk(a);
  Segment sg;
  bool work_left = walk.next(a, &sg);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = B.tmem;
  auto s_col = [&](uint32_t g, uint32_t h) { return tmem + 128 * g + 64 * h; };
  auto o_col = [&](uint32_t g) { return tmem + 256 + 128 * g; };
  volatile uint32_t* stop = &B.stop;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_bar(bar, parity, stop, a.err); };
  bool ok = true;
  const uint32_t G = a.group;

  if (warp == 0) {
    // ---- loads ------------------------------------------------------------------------
    if (lane == 0) {
      constexpr int N = Q8 ? S::NRAW : S::NSLOT;
      uint64_t* full = Q8 ? B.raw_full : B.full;
      uint64_t* free = Q8 ? B.raw_free : B.free;
      Ring<N> ring;
      uint32_t issued = 0;
      for (; work_left; work_left = walk.next(a, &sg)) {
        const uint32_t nt = sg.k1 - sg.k0, plane = sg.b * a.c.n_kv_heads + sg.h;
        for (uint32_t e = 0; e < 2 * nt; e++) {
          bool is_v;
          uint32_t i;
          item_at(e, nt, S::LEAD, &is_v, &i);
          ok = ok && wait(&free[ring.s], ring.phase ^ 1);
          if (ok) {
            const uint32_t bar = tc_smem_u32(&full[ring.s]), key0 = (sg.k0 + i) * TK;
            if constexpr (Q8) {  // rows past the capacity are not part of this head (or of the plane)
              const uint32_t bytes = min((uint32_t)TK, a.c.capacity - key0) * D;
              const uint8_t* src = (const uint8_t*)(is_v ? a.c.v : a.c.k) + ((uint64_t)plane * a.c.capacity + key0) * D;
              tc_bulk_g2s(raws + ring.s * S::RAW, src, bytes, bar);
            } else {
              tc_mbar_expect_tx(bar, S::TILE);
#pragma unroll
              for (int x = 0; x < D / 64; x++)
                tma_load_3d(slot_addr(ring.s) + x * kBlockBytes, is_v ? &map_v : &map_k, 64 * x, (int)key0, (int)plane, bar);
            }
            issued++;
          }
          ring.advance();
        }
      }
      // every copy must land before the CTA's memory is given up, also if the other roles' waits give up after this
      Ring<N> r;
      for (uint32_t i = 0; i < issued; i++) {
        if (i + N >= issued) tc_mbar_wait(tc_smem_u32(&full[r.s]), r.phase);
        r.advance();
      }
    }
  } else if (warp < 3) {
    // ---- MMAs of one group -----------------------------------------------------------------
    // The whole warp runs the loop with values the compiler knows to be the same in every
    // lane, so that descriptors stay in uniform registers, and one elected lane issues.  With
    // both groups in one lane's loop each MMA cost 110 cycles of issue, more than it takes to
    // run, and the tensor core waited (256 tokens over 32768: 472 us).
    const uint32_t g = warp - 1;
    Ring<S::NSLOT> ring;
    uint32_t q_phase = 0, fix_phase = 0;
    uint32_t done = 0;  // tiles of this group so far
    constexpr uint32_t id_s = idesc_f16(TK / 2, false), id_o = idesc_f16(D, true);
    const uint32_t s_base = uniform(s_col(g, 0)), o_base = uniform(o_col(g)), base = uniform(q_smem);
    auto slot_at = [&](uint32_t s) { return base + S::QBYTES + s * S::TILE; };
    auto until = [&](uint64_t* bar, uint32_t parity) { ok = __all_sync(~0u, ok && wait(bar, parity)); };
    // The next tile of the ring; a tile with work of this group goes back with its last MMA, others at once.
    auto take = [&](bool used) {
      const uint32_t s = ring.s;
      until(&B.full[s], ring.phase);
      ring.advance();
      if (!used && elect_one()) tc_mbar_arrive(tc_smem_u32(&B.free[s]));
      return s;
    };
    auto release = [&](uint32_t s) {
      if (ok && elect_one()) tc_commit(tc_smem_u32(&B.free[s]));
    };
    // S of a half; P of the tile before sat in the same columns, its product is over
    auto qk = [&](uint32_t h, uint32_t s) {
      if (!ok) return;
      const uint64_t q = sw128_desc(base + (RT == 2 ? g * S::TILE : 0)), k = sw128_desc(slot_at(s) + h * (TK / 2) * 128);
      const uint32_t d = s_base + 64 * h;
      if (elect_one()) {
#pragma unroll
        for (int term = SPLIT ? 1 : 0; term >= 0; term--)  // the small term first: the sum truncates at its own size
#pragma unroll
          for (int i = 0; i < D / 16; i++) {
            const uint32_t o = (i / 4) * kBlockBytes + (i % 4) * 32;
            mma_ss(d, q + ((term * S::TILE + o) >> 4), k + (o >> 4), id_s, (SPLIT && term == 0) || i > 0);
          }
        tc_commit(tc_smem_u32(&B.s_full[g][h]));
      }
    };
    auto pv = [&](uint32_t h, uint32_t s, bool first) {
      if (!ok) return;
      tc_fence_after_sync();
      const uint64_t v = sw128_desc(slot_at(s) + h * (TK / 2) * 128);
      const uint32_t p = s_base + 64 * h;
      if (elect_one()) {
#pragma unroll
        for (int i = 0; i < TK / 32; i++) {
          const uint32_t pi = p + (S::HOLD ? 8 * i : 32 * (i / 2) + 8 * (i % 2));
          if constexpr (SPLIT) mma_ts(o_base, pi + 16, v + i * (16 * 128 >> 4), id_o, !first || i > 0);
          mma_ts(o_base, pi, v + i * (16 * 128 >> 4), id_o, SPLIT || !first || i > 0);
        }
        tc_commit(tc_smem_u32(&B.pv_done[g][h]));
      }
    };
    for (; work_left; work_left = walk.next(a, &sg)) {
      const uint32_t nt = uniform(sg.k1 - sg.k0), k0 = uniform(sg.k0), hist = uniform(sg.hist);
      constexpr uint32_t step = RT == 1 ? 2 : 1;
      const bool work = RT == 1 ? g < nt : g == 0 || uniform(sg.drafts * G - sg.rt * S::ROWS) > TK;
      auto mine = [&](uint32_t i) { return RT == 1 ? (i & 1) == g : work; };
      if (work) {
        until(&B.q_full[g], q_phase);
        q_phase ^= 1;
      }
      if (done)  // the products of the segment before are over (also awaited by the softmax)
        for (uint32_t h = 0; h < 2; h++) until(&B.pv_done[g][h], (done - 1) & 1);
      tc_fence_after_sync();
      for (uint32_t i = 0; i < min((uint32_t)S::LEAD, nt); i++) {
        const uint32_t k = take(mine(i));
        if (!mine(i)) continue;
        qk(0, k);
        qk(1, k);
        release(k);
      }
      // a half's P V, then, that being over, the next scores in its columns
      for (uint32_t i = 0; i < nt; i++) {
        const bool drafts = (k0 + i + 1) * TK > hist, more = i + step < nt;
        const uint32_t v = take(mine(i));
        const uint32_t fix_bit = (fix_phase >> v) & 1;
        if (!Q8 && drafts) fix_phase ^= 1u << v;
        uint32_t k = 0;
        if (!mine(i)) {
          if (more) take(false);
          continue;
        }
        for (uint32_t h = 0; h < 2; h++) {
          until(&B.p_full[g][h], done & 1);
          if (!Q8 && drafts && h == 0) until(&B.fix[v], fix_bit);
          pv(h, v, i < step && h == 0);
          if (h == 1) release(v);
          if (!more) continue;
          if (h == 0) k = take(true);
          until(&B.pv_done[g][h], done & 1);
          tc_fence_after_sync();
          qk(h, k);
          if (h == 1) release(k);
        }
        done++;
      }
    }
    // everything issued is over before tensor and shared memory are given up
    if (elect_one()) {
      tc_commit(tc_smem_u32(&B.drain));
      tc_mbar_wait(tc_smem_u32(&B.drain), 0);
    }
  } else if (warp == 3) {
    // ---- f16 V tiles with drafts or the end: rows past the end 0, drafts' rows finite ------
    if constexpr (!Q8) {
      Ring<S::NSLOT> ring;
      for (; work_left; work_left = walk.next(a, &sg)) {
        const uint32_t nt = sg.k1 - sg.k0;
        for (uint32_t e = 0; e < 2 * nt; e++) {
          bool is_v;
          uint32_t i;
          item_at(e, nt, S::LEAD, &is_v, &i);
          const uint32_t key0 = (sg.k0 + i) * TK;
          ok = __all_sync(~0u, ok && wait(&B.full[ring.s], ring.phase));
          if (ok && is_v && key0 + TK > sg.hist) {
            const uint32_t from = sg.hist > key0 ? sg.hist - key0 : 0, v = slot_addr(ring.s);
            bool wild = false;
#pragma unroll 2
            for (uint32_t x = from * 8 + lane; x < TK * 8; x += 32) {  // 16-byte pieces, in memory order
              const bool real = key0 + x / 8 < sg.end;
#pragma unroll
              for (int blk = 0; blk < D / 64; blk++) {
                const uint32_t at = v + blk * kBlockBytes + x * 16;
                uint4 u = real ? ld_shared16(at) : make_uint4(0, 0, 0, 0);
                bool odd = !real;
                u.x = finite_halves(u.x, &odd), u.y = finite_halves(u.y, &odd);
                u.z = finite_halves(u.z, &odd), u.w = finite_halves(u.w, &odd);
                if (odd) st_shared16(at, u);
                wild |= real && odd;
              }
            }
            if (wild) *(volatile uint32_t*)&B.wild = 1;
            tc_fence_proxy_async();
            __syncwarp();
            if (lane == 0) tc_mbar_arrive(tc_smem_u32(&B.fix[ring.s]));
          }
          if (lane == 0) tc_mbar_arrive(tc_smem_u32(&B.free[ring.s]));
          ring.advance();
        }
      }
    }
  } else if (warp < 12) {
    // ---- softmax ----------------------------------------------------------------------
    const uint32_t g = (warp - 4) / 4, w32 = 32 * (warp % 4), row = w32 + lane, lanes = w32 << 16;
    const uint32_t q_tile = q_smem + (RT == 2 ? g * S::TILE : 0);
    constexpr uint32_t CPR = D * sizeof(T) / 16;  // 16-byte pieces of a row of activations
    constexpr uint32_t RPI = 32 / CPR;            // rows a warp moves at a time
    // Piece c of row x on its way out: inside the warp's own rows of the queries' tiles, since another warp of the
    // group may by then have put its next queries into its rows.  The tile's address is taken anew: one that is kept
    // across the tiles' loop slows that (256 tokens of 64/8 heads over 32768 f16: 303 us, with q_tile 323).
    auto staged = [&](uint32_t x, uint32_t c) {
      const uint32_t tile = q_smem + (RT == 2 ? ((threadIdx.x >> 7) - 1) * S::TILE : 0);
      return tile + c / (D / 8) * S::TILE + sw128_offset(x, c % (D / 8));
    };
    uint32_t count = 0;                           // tiles of this group so far
    for (; work_left; work_left = walk.next(a, &sg)) {
      const uint32_t nt = sg.k1 - sg.k0, n_rows = sg.drafts * G;
      const uint32_t r_base = sg.rt * S::ROWS + (RT == 2 ? g * TK : 0) + w32;  // the warp's first row
      const uint32_t r = r_base + lane;
      const bool live = r < n_rows, warp_live = r_base < n_rows;
      const bool two = n_rows - sg.rt * S::ROWS > TK;
      const uint32_t mine = RT == 1 ? (nt + 1 - g) / 2 : (g == 0 || two ? nt : 0);  // tiles of this group
      const uint32_t t = live ? group_div(a, r) : 0;
      // element offset of row x's head in a tensor of token stride `stride`
      auto row_at = [&](uint32_t x, uint64_t stride) {
        const uint32_t tx = group_div(a, x);
        return ((uint64_t)sg.b * a.n_tokens + tx) * stride + (uint64_t)(sg.h * G + (x - tx * G)) * D;
      };
      // queries: the warp moves RPI of its rows at a time.  f16 rows go straight to shared memory; f32
      // and bf16 rows are scaled by a power of two to a largest magnitude in [1, 4).  Small code: what
      // runs once is bound by the fetch of its instructions.
      float coef = a.scale * 1.44269504f;
      {
        constexpr int PIECE = 16 / sizeof(T);
        const uint32_t sub = lane / CPR, c = lane % CPR;
        const uint64_t mine_at = live ? (uint64_t)((const T*)a.q + row_at(r, a.q_stride)) : 0;
        float up_mine = 1.f;
        if constexpr (std::is_same<T, __half>::value) {
          if (RT == 2 || g == 0) {
#pragma unroll 4
            for (uint32_t i = 0; i < 32 / RPI; i++) {
              const uint32_t x = i * RPI + sub;
              const uint64_t at = __shfl_sync(~0u, mine_at, x);
              cp_async16(q_tile + sw128_offset(w32 + x, c), at ? at + 16 * c : (uint64_t)a.q, at ? 16 : 0);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
          }
        } else {
#pragma unroll 1
          for (uint32_t b0 = 0; b0 < 32 / RPI; b0 += 4) {
            uint4 u[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
              const uint64_t at = __shfl_sync(~0u, mine_at, (b0 + i) * RPI + sub);
              u[i] = at ? *(reinterpret_cast<const uint4*>(at) + c) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
              float v[PIECE];
              act_unpack<T>(u[i], v);
              float top = 0.f;
#pragma unroll
              for (int j = 0; j < PIECE; j++) top = fmaxf(top, fabsf(v[j]));
#pragma unroll
              for (uint32_t o = CPR / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
              float down, up;
              pow2_scale(top, &down, &up);
#pragma unroll
              for (int j = 0; j < PIECE; j++) v[j] *= down;
              up = __shfl_sync(~0u, up, (lane % RPI) * CPR);
              if (lane / RPI == b0 + i) up_mine = up;
              if (RT == 2 || g == 0) {
                const uint32_t x = w32 + (b0 + i) * RPI + sub;
                if constexpr (SPLIT) {  // 4 elements: half of a 16-byte piece of f16
                  const uint32_t at = sw128_offset(x, c / 2) + 8 * (c & 1);
                  const uint32_t h0 = pack_h2(v[0], v[1]), h1 = pack_h2(v[2], v[3]);
                  st_shared8(q_tile + at, h0, h1);
                  st_shared8(q_tile + S::TILE + at, pack_h2_rest(v[0], v[1], h0), pack_h2_rest(v[2], v[3], h1));
                } else {
                  st_shared16(q_tile + sw128_offset(x, c), make_uint4(pack_h2(v[0], v[1]), pack_h2(v[2], v[3]),
                                                                      pack_h2(v[4], v[5]), pack_h2(v[6], v[7])));
                }
              }
            }
          }
        }
        if constexpr (!std::is_same<T, __half>::value)
          coef = fmaxf(coef * up_mine, 1.17549435e-38f);  // not 0: a masked score stays -inf
        tc_fence_proxy_async();
        // Told to the groups with work in this segment alone: phases that a group does not wait for it could not tell
        // apart, nor may a softmax group without work, which runs ahead, complete the phase of another.
        if (RT == 1 && g == 0)
          for (uint32_t i = 0; i < min(nt, 2u); i++) tc_mbar_arrive(tc_smem_u32(&B.q_full[i]));
        if (RT == 2 && mine) tc_mbar_arrive(tc_smem_u32(&B.q_full[g]));
      }
      const uint32_t* mask_row = a.mask ? a.mask + ((uint64_t)sg.b * a.n_tokens + t) * a.words : nullptr;
      float m = -INFINITY, l = 0.f;
      for (uint32_t x = 0; x < mine; x++, count++) {
        const uint32_t key0 = (sg.k0 + (RT == 1 ? 2 * x + g : x)) * TK;
        const bool edge = key0 + TK > sg.hist;
#pragma unroll 1
        for (uint32_t h = 0; h < 2; h++) {
          const uint32_t scores = s_col(g, h) + lanes;
          ok = __all_sync(~0u, ok && wait(&B.s_full[g][h], count & 1));
          if (ok && warp_live) {
            tc_fence_after_sync();
            if constexpr (S::HOLD) {  // all 64 columns in registers, weights in pairs over the first 32 of them
              uint32_t s[TK / 2];
              tmem_ld_32(scores, s);
              tmem_ld_32(scores + 32, s + 32);
              tmem_wait_ld(s);
              if (edge) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                  const uint32_t see = seen32(mask_row, a.words, t, (int)(key0 + 64 * h + 32 * i) - (int)sg.hist, (int)sg.drafts);
#pragma unroll
                  for (int j = 0; j < 32; j++)
                    if (!((see >> j) & 1)) s[32 * i + j] = 0xff800000u;
                }
              }
              float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
              for (int i = 0; i < TK / 2; i += 8)
#pragma unroll
                for (int j = 0; j < 4; j++)
                  tops[j] = max3(tops[j], __uint_as_float(s[i + 2 * j]), __uint_as_float(s[i + 2 * j + 1]));
              const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * coef;
              if (__any_sync(~0u, top > m + kRaise)) {
                const float m2 = fmaxf(m, top), f = m2 == -INFINITY ? 1.f : ex2(m - m2);
                m = m2;
                l *= f;
                if (x + h > 0) {  // all products issued so far are in O before it is rescaled
                  ok = __all_sync(~0u, ok && wait(&B.pv_done[g][h ^ 1], (h ? count : count - 1) & 1));
                  tc_fence_after_sync();
#pragma unroll 1
                  for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    tmem_ld_32(o_col(g) + lanes + c, o);
                    tmem_wait_ld(o);
#pragma unroll
                    for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                    tmem_st_32(o_col(g) + lanes + c, o);
                  }
                }
              }
              const float ref = kWeightBias - (m == -INFINITY ? 0.f : m);
              const float2 coef2 = make_float2(coef, coef), ref2 = make_float2(ref, ref);
              float2 sum[2] = {make_float2(l, 0.f), make_float2(0.f, 0.f)};
              uint32_t p[32];
#pragma unroll
              for (int i = 0; i < 32; i++) {
                float2 v = fma2(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), coef2, ref2);
                v.x = ex2(v.x), v.y = ex2(v.y);
                sum[i & 1] = add2(sum[i & 1], v);
                p[i] = pack_h2(v.x, v.y);
              }
              tmem_st_32(scores, p);
              l = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            } else {
              uint32_t see[2] = {~0u, ~0u};
              if (edge) {
                const int j0 = (int)(key0 + 64 * h) - (int)sg.hist;
                see[0] = seen32(mask_row, a.words, t, j0, (int)sg.drafts);
                see[1] = seen32(mask_row, a.words, t, j0 + 32, (int)sg.drafts);
              }
              // Raise the reference to the scores' maximum `top` (base-2 exponents) where some row has to: the sums
              // and O, with all products issued so far in it, are rescaled.
              auto raise = [&](float top) {
                const float m2 = fmaxf(m, top), f = m2 == -INFINITY ? 1.f : ex2(m - m2);
                m = m2;
                l *= f;
                if (x + h > 0) {
                  ok = __all_sync(~0u, ok && wait(&B.pv_done[g][h ^ 1], (h ? count : count - 1) & 1));
                  tc_fence_after_sync();
#pragma unroll 1
                  for (int c = 0; c < D; c += 16) {
                    uint32_t o[16];
                    tmem_ld_16(o_col(g) + lanes + c, o);
                    tmem_wait_ld(o);
#pragma unroll
                    for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                    tmem_st_16(o_col(g) + lanes + c, o);
                  }
                }
              };
              auto maximum = [&](const uint32_t(&s)[32]) {
                float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 32; i += 8)
#pragma unroll
                  for (int j = 0; j < 4; j++)
                    tops[j] = max3(tops[j], __uint_as_float(s[i + 2 * j]), __uint_as_float(s[i + 2 * j + 1]));
                return fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
              };
              // the weights of 32 columns of scores, in pairs
              auto weigh = [&](uint32_t* s, uint32_t* p) {
                const float ref = kWeightBias - (m == -INFINITY ? 0.f : m);
                const float2 coef2 = make_float2(coef, coef), ref2 = make_float2(ref, ref);
                float2 sum[2] = {make_float2(l, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int i = 0; i < 16; i++) {
                  float2 v = fma2(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), coef2, ref2);
                  v.x = ex2(v.x), v.y = ex2(v.y);
                  sum[i & 1] = add2(sum[i & 1], v);
                  p[i] = pack_h2(v.x, v.y);
                  if constexpr (SPLIT) s[i] = pack_h2_rest(v.x, v.y, p[i]);
                }
                l = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
              };
              // 32 columns at a time, rolled: for the registers and for the instruction cache, which all roles share
              // (unrolled: 17.4 us for 16 tokens over 4095 Q8_0 positions, rolled 15.9).  Weights go back in pairs over the
              // first 16 of their 32 columns, the small terms over the others.
              // Two passes: a weight once rounded is not scaled again.  (With 16-bit activations one pass, which rescales
              // the first 32 keys' weights, takes the same time: 16 tokens over 32768 Q8_0 34.6 us against 35.1, over 4095
              // 15.1 both, 32 over 32768 f16 39.9 both.)
              float top = -INFINITY;
#pragma unroll 1
              for (int c = 0; c < 2; c++) {
                uint32_t s[32];
                tmem_ld_32(scores + 32 * c, s);
                tmem_wait_ld(s);
                if (edge) hide(s, see[c]);
                top = fmaxf(top, maximum(s));
              }
              if (__any_sync(~0u, top * coef > m + kRaise)) raise(top * coef);
#pragma unroll 1
              for (int c = 0; c < 2; c++) {
                uint32_t s[32], p[16];
                tmem_ld_32(scores + 32 * c, s);
                tmem_wait_ld(s);
                if (edge) hide(s, see[c]);
                weigh(s, p);
                tmem_st_16(scores + 32 * c, p);
                if constexpr (SPLIT) {
#pragma unroll
                  for (int i = 0; i < 16; i++) p[i] = s[i];
                  tmem_st_16(scores + 32 * c + 16, p);
                }
              }
            }
            tmem_wait_st();
          }
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) tc_mbar_arrive(tc_smem_u32(&B.p_full[g][h]));
        }
      }
      if (mine) ok = __all_sync(~0u, ok && wait(&B.pv_done[g][1], (count - 1) & 1));
      // ---- output: RT = 1 joins the two groups, each writing half of the dimensions
      const bool joined = RT == 1 && nt > 1;
      float f0 = 1.f, f1 = 0.f, M = m, den = l;
      if constexpr (RT == 1) {
        B.ml[g][row][0] = m, B.ml[g][row][1] = l;
        __syncwarp();
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const float m0 = B.ml[0][row][0], m1 = B.ml[1][row][0];
        M = fmaxf(m0, m1);
        f0 = M == -INFINITY ? 1.f : ex2(m0 - M), f1 = M == -INFINITY ? 1.f : ex2(m1 - M);
        den = B.ml[0][row][1] * f0 + B.ml[1][row][1] * f1;
      }
      if (ok && warp_live && (RT == 1 || mine)) {
        tc_fence_after_sync();
        const bool whole = sg.whole();
        if (whole) f0 *= den == 0.f ? 0.f : 1.f / den, f1 *= den == 0.f ? 0.f : 1.f / den;
        float* slot = part + (2 * (size_t)blockIdx.x + (sg.k0 > 0 ? 0 : 1)) * part_floats(S::ROWS, D);
        const uint32_t rl = r - sg.rt * S::ROWS;
        constexpr uint32_t DIMS = RT == 1 ? D / 2 : D;
        const uint32_t d0 = RT == 1 ? g * DIMS : 0;
#pragma unroll 1
        for (uint32_t d = d0; d < d0 + DIMS; d += 16) {  // rolled: this code runs from a cold instruction cache
          uint32_t o[16];
          float v[16];
          tmem_ld_16(o_col(RT == 1 ? 0 : g) + lanes + d, o);
          tmem_wait_ld(o);
#pragma unroll
          for (int i = 0; i < 16; i++) v[i] = __uint_as_float(o[i]) * f0;
          if (joined) {
            tmem_ld_16(o_col(1) + lanes + d, o);
            tmem_wait_ld(o);
#pragma unroll
            for (int i = 0; i < 16; i++) v[i] = fmaf(__uint_as_float(o[i]), f1, v[i]);
          }
          if (whole) {  // through the queries' place in shared memory, to whole rows
            constexpr int PIECE = 16 / sizeof(T);
#pragma unroll
            for (int i = 0; i < 16 / PIECE; i++) {
              __align__(16) T w[PIECE];
#pragma unroll
              for (int j = 0; j < PIECE; j++) act_put(&w[j], v[PIECE * i + j]);
              const uint32_t c = d / PIECE + i;
              st_shared16(staged(row, c), *reinterpret_cast<const uint4*>(w));
            }
          } else if (live) {
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              *reinterpret_cast<float4*>(slot + part_at<S::ROWS>(d + i, rl)) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
          }
        }
        if (whole) {
          constexpr uint32_t CH = DIMS * sizeof(T) / 16, RP = 32 / CH;  // pieces of the group's part of a row
          __syncwarp();
#pragma unroll 4
          for (uint32_t i = 0; i < 32 / RP; i++) {
            const uint32_t x = i * RP + lane / CH, c = d0 * sizeof(T) / 16 + lane % CH;
            const uint4 u = ld_shared16(staged(w32 + x, c));
            if (r_base + x < n_rows) *(reinterpret_cast<uint4*>((T*)a.out + row_at(r_base + x, a.out_stride)) + c) = u;
          }
        } else if (live && d0 == 0) {
          slot[S::ROWS * D + rl] = M, slot[S::ROWS * D + S::ROWS + rl] = den;
        }
        if (__any_sync(~0u, *(volatile uint32_t*)&B.wild)) {  // rare: what was left out of the drafts' V
          __syncwarp();  // other lanes stored this thread's row
          const uint64_t base = ((uint64_t)sg.b * a.c.n_kv_heads + sg.h) * a.c.capacity;
#pragma unroll 1
          for (uint32_t p = max(sg.hist, sg.k0 * TK); p < min(sg.end, sg.k1 * TK); p++) {
            if (!live || !sees(a, sg.b, t, sg.hist, p)) continue;
#pragma unroll 1
            for (uint32_t d = d0; d < d0 + DIMS; d++) {
              const uint64_t at = (base + p) * D + d;
              float y;
              if constexpr (Q8)
                y = __half2float(__float2half_rn((float)((const int8_t*)a.c.v)[at] *
                                                 __half2float(((const __half*)a.c.v_scale)[at / 32])));
              else
                y = __half2float(((const __half*)a.c.v)[at]);
              if (fabsf(y) < INFINITY) continue;
              if (whole) {
                T* out = (T*)a.out + row_at(r, a.out_stride) + d;
                act_put(out, act_get(out) + y);
              } else {
                slot[part_at<S::ROWS>(d, rl) + d % 4] += y;
              }
            }
          }
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if constexpr (RT == 1) asm volatile("bar.sync 1, 256;" ::: "memory");
    }
  } else {
    // ---- Q8_0 tiles to f16: thread = key; pieces taken in an order that keeps the eight
    // lanes of a shared-memory phase on different banks, for the codes and for the tile
    if constexpr (Q8) {
      const uint32_t key = (tid - 384) % TK, set = (tid - 384) / TK;  // sets of four warps take the tiles in turn
      Ring<S::NRAW> rr;
      Ring<S::NSLOT> ring;
      for (; work_left; work_left = walk.next(a, &sg)) {
        const uint32_t nt = sg.k1 - sg.k0;
        const uint64_t base = ((uint64_t)sg.b * a.c.n_kv_heads + sg.h) * a.c.capacity;
        // scales of the e-th tile's key; 0 past the end, so that those rows become 0
        auto scales = [&](uint32_t e) {
          uint2 s = make_uint2(0, 0);
          if (e >= 2 * nt) return s;
          bool is_v;
          uint32_t i;
          item_at(e, nt, S::LEAD, &is_v, &i);
          const uint32_t p = (sg.k0 + i) * TK + key;
          if (p >= sg.end) return s;
          const __half* plane = (const __half*)(is_v ? a.c.v_scale : a.c.k_scale) + (base + p) * (D / 32);
          if constexpr (D == 128)
            asm volatile("ld.global.v2.b32 {%0,%1}, [%2];" : "=r"(s.x), "=r"(s.y) : "l"(plane));
          else
            asm volatile("ld.global.b32 %0, [%1];" : "=r"(s.x) : "l"(plane));
          return s;
        };
        uint2 s0 = scales(set), s1 = scales(set + S::SETS);
        if (set) rr.advance(), ring.advance();
        for (uint32_t e = set; e < 2 * nt; e += S::SETS) {
          bool is_v;
          uint32_t i;
          item_at(e, nt, S::LEAD, &is_v, &i);
          const uint2 sc = s0;
          s0 = s1;
          s1 = scales(e + 2 * S::SETS);
          const uint32_t p = (sg.k0 + i) * TK + key;
          const bool draft_v = is_v && p >= sg.hist;
          ok = __all_sync(~0u, ok && wait(&B.raw_full[rr.s], rr.phase));
          // A parity tells two neighbouring uses of a slot apart, so a set that has not waited for the use before must
          // know that it has begun.  With an odd number of slots that use was the other set's: its tile is waited for.
          // (The one before that was this set's own, and done: its raw tile would not have been loaded over else.)
          if constexpr (S::SETS == 2 && S::NSLOT % 2) ok = __all_sync(~0u, ok && wait(&B.full[ring.s], ring.phase ^ 1));
          ok = __all_sync(~0u, ok && wait(&B.free[ring.s], ring.phase ^ 1));
          if (ok) {
            // piece j of the lane's turn is piece c = j ^ lm of its key: the eight lanes of a phase
            // meet different banks when they read it and when they write its two f16 pieces
            constexpr uint32_t N = D / 16;
            const uint32_t lm = lane & (N - 1), l7 = lane & 7;
            const uint32_t raw = (raws + rr.s * S::RAW + key * D) + lm * 16;
            const uint32_t lane_at = slot_addr(ring.s) + key * 128 + ((((2 * lm) ^ l7) & 7) << 4);
            bool wild = false;
#pragma unroll 1
            for (uint32_t q = 0; q < N / 4; q++) {  // 64 codes at a time, rolled for the instruction cache
              const uint32_t dst = lane_at + ((lm >> 2) ^ q) * kBlockBytes;
              uint4 codes[4];
#pragma unroll
              for (uint32_t j = 0; j < 4; j++) codes[j] = ld_shared16(raw ^ (64 * q + 16 * j));
#pragma unroll
              for (uint32_t j = 0; j < 4; j++) {
                const uint32_t blk = (2 * q + j / 2) ^ (lm >> 1), sw = blk & 2 ? sc.y : sc.x;
                const uint32_t db = __byte_perm(sw, sw, blk & 1 ? 0x3232 : 0x1010);
                const __half2 d = *reinterpret_cast<const __half2*>(&db);
                const uint32_t w[4] = {codes[j].x, codes[j].y, codes[j].z, codes[j].w};
                uint32_t h[8];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                  // biased bytes under an exponent of 1024: 1152 + code, exact; the product rounds once
                  const uint32_t b = w[k] ^ 0x80808080u;
                  uint32_t lo = __byte_perm(b, 0x64646464u, 0x4140), hi = __byte_perm(b, 0x64646464u, 0x4342);
                  const __half2 bias = __float2half2_rn(1152.f);
                  const __half2 x = __hmul2(__hsub2(*reinterpret_cast<__half2*>(&lo), bias), d);
                  const __half2 y = __hmul2(__hsub2(*reinterpret_cast<__half2*>(&hi), bias), d);
                  h[2 * k] = *reinterpret_cast<const uint32_t*>(&x), h[2 * k + 1] = *reinterpret_cast<const uint32_t*>(&y);
                }
                if (draft_v) {
#pragma unroll
                  for (int k = 0; k < 8; k++) h[k] = finite_halves(h[k], &wild);
                }
                const uint32_t at = dst ^ (((2 * j) & 7) << 4);
                st_shared16(at, make_uint4(h[0], h[1], h[2], h[3]));
                st_shared16(at ^ 16, make_uint4(h[4], h[5], h[6], h[7]));
              }
            }
            if (wild) *(volatile uint32_t*)&B.wild = 1;
          }
          tc_fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            tc_mbar_arrive(tc_smem_u32(&B.full[ring.s]));
            tc_mbar_arrive(tc_smem_u32(&B.raw_free[rr.s]));
          }
          for (int i = 0; i < S::SETS; i++) rr.advance(), ring.advance();
        }
        if (set) rr.retreat(), ring.retreat();  // tiles come in pairs: back to the first of the next segment
      }
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tc_tmem_dealloc(tmem, 512);
  }
}

// Tensor map of an f16 plane [heads][capacity][D], copied in boxes of 64 dimensions x 128 positions.
int plane_map(CUtensorMap* map, const void* p, const rf_kv_view& c) {
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
  const cuuint64_t dims[3] = {c.head_dim, c.capacity, (cuuint64_t)c.n_seqs * c.n_kv_heads};
  const cuuint64_t strides[2] = {2ull * c.head_dim, 2ull * c.head_dim * c.capacity};
  const cuuint32_t box[3] = {64, TK, 1}, step[3] = {1, 1, 1};
  const CUresult r = ((Encode)fn)(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(p), dims, strides, box, step,
                                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(RF_ECUDA, "cuTensorMapEncodeTiled failed with %d", (int)r);
  return RF_OK;
}

template <class T, bool Q8, int D, int RT>
int run(cudaStream_t st, const TreeArgs& a) {
  using S = Shape<T, Q8, D, RT>;
  CUtensorMap mk{}, mv{};
  if constexpr (!Q8) {
    RF_TRY(plane_map(&mk, a.c.k, a.c));
    RF_TRY(plane_map(&mv, a.c.v, a.c));
  }
  auto* k = tree_tc_kernel<T, Q8, D, RT>;
  RF_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM));
  const uint32_t ctas = (uint32_t)num_sms();
  void* part = nullptr;
  RF_TRY(scratch_alloc(&part, 2 * (size_t)ctas * part_floats(S::ROWS, D) * sizeof(float), st));
  cudaError_t e = launch_k(Launch{st, true}, k, dim3(ctas), dim3(S::THREADS), S::SMEM, a, (float*)part, mk, mv);
  if (e == cudaSuccess)
    e = launch_merge<T, D, TK, S::ROWS>(st, a, (const float*)part, ctas, cudaSharedmemCarveoutMaxShared);
  const cudaError_t f = cudaFreeAsync(part, st);
  RF_CUDA(e);
  RF_CUDA(f);
  return RF_OK;
}

template <class T, bool Q8, int D>
int run_shape(cudaStream_t st, const TreeArgs& a) {
  // f32 splits its queries, which takes the second row tile's place in shared memory
  if constexpr (!std::is_same<T, float>::value)
    if (a.n_tokens * a.group > TK) return run<T, Q8, D, 2>(st, a);
  return run<T, Q8, D, 1>(st, a);
}

template <class T>
int run_type(cudaStream_t st, const TreeArgs& a) {
  const bool q8 = a.c.type == RF_TYPE_Q8_0;
  if (a.c.head_dim == 128) return q8 ? run_shape<T, true, 128>(st, a) : run_shape<T, false, 128>(st, a);
  return q8 ? run_shape<T, true, 64>(st, a) : run_shape<T, false, 64>(st, a);
}

}  // namespace

int run_tree_tc(int act_type, const TreeArgs& a, cudaStream_t st) {
  switch (act_type) {
    case RF_ACT_F32: return run_type<float>(st, a);
    case RF_ACT_F16: return run_type<__half>(st, a);
    default: return run_type<__nv_bfloat16>(st, a);
  }
}

}  // namespace rf
