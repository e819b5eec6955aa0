// rf_i8.cu - rows of 8-bit codes with one scale a row: the residual's addition with RMS norm, SwiGLU and plain
// rows into the format, and the rows back.  The product of such rows with an 8-bit matrix is in rf_i8_matmul.cu.
//
// The format (rfcuda.h) fixes every rounding from the row's f32 numbers to its codes, and the norm's are fixed up to
// the sum of squares, which is taken in 64 bits: how the row was split over threads shows in a row's codes only where the
// last of those bits decide how the 32-bit reciprocal root is rounded (one sum in some 2^25 lies that near to a border).
//
// One read and one write of each element, a handful of operations between: HBM bounds the long calls, latency of
// launch, loads and one reduction the short ones.  Maximum and sum of squares need one reduction together, since
// rounding is monotonic: max |f32(f32(s w) r)| = f32(max |f32(s w)| r).
//
// Launched to begin while the kernel before ends, as rf_verify.cu's are; what that one may write, a norm's weights among it (rows back
// in f32 are such), is read by plain loads.
#include <algorithm>
#include <type_traits>

#include "rf_act.cuh"
#include "rf_device.cuh"
#include "rf_pair.cuh"
#include "rf_ring.cuh"
#include "rf_verify.h"

namespace rf {
namespace {

constexpr uint32_t kMaxCols = 65536;  // 64 elements a thread of 1024

struct RowsArgs {
  const void *x, *y;  // y: the residual, or SwiGLU's up (null: none)
  void* sum;
  const float* w;
  int8_t* q;
  float* scale;
  uint64_t x_stride, y_stride, sum_stride, q_stride;
  uint32_t n_cols;
  float eps;
};

enum RowsMode { kPlain, kNorm, kSwiglu };

template <class T>
__device__ __forceinline__ void unpack8(const uint4 (&u)[8 / Act<T>::kVec], float (&v)[8]) {
  constexpr int V = Act<T>::kVec;
#pragma unroll
  for (int j = 0; j < 8 / V; j++) {
    float f[V];
    Act<T>::unpack(u[j], f);
#pragma unroll
    for (int k = 0; k < V; k++) v[j * V + k] = f[k];
  }
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  constexpr int V = Act<T>::kVec;
#pragma unroll
  for (int j = 0; j < 8 / V; j++) {
    float f[V];
#pragma unroll
    for (int k = 0; k < V; k++) f[k] = v[j * V + k];
    *reinterpret_cast<uint4*>(p + j * V) = Act<T>::pack(f);
  }
}
// Eight f32 at a 32-byte place in one store: two of 16 bytes write half sectors (16 M values: 20.7 us, 15.0 so).
__device__ __forceinline__ void store8_wide(float* p, const float (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]),
               "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

// What a row's numbers become before the reduction, in pairs: instructions bound the kernels that keep HBM busy (7 issue
// slots of 10 full where each number was by itself).
template <int MODE>
__device__ __forceinline__ float2 combine2(float2 x, float2 y) {
  if constexpr (MODE == kSwiglu) {
    // exponential and reciprocal to a few units of the 24th bit: a code holds 8, and the few that lie that near to a
    // border go to either side
    float2 e = pair_mul(x, make_float2(-1.44269504f, -1.44269504f));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e.x));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e.y));
    e = pair_add(e, make_float2(1.f, 1.f));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e.x));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e.y));
    return pair_mul(pair_mul(x, e), y);
  } else {
    return pair_add(x, y);
  }
}
template <int MODE>
__device__ __forceinline__ void combine8(float (&v)[8], const float (&y)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const float2 r = combine2<MODE>(make_float2(v[j], v[j + 1]), make_float2(y[j], y[j + 1]));
    v[j] = r.x, v[j + 1] = r.y;
  }
}
__device__ __forceinline__ void multiply8(float (&v)[8], const float (&w)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const float2 r = pair_mul(make_float2(v[j], v[j + 1]), make_float2(w[j], w[j + 1]));
    v[j] = r.x, v[j + 1] = r.y;
  }
}
// The largest magnitude of top and eight numbers; NaN where one is.
__device__ __forceinline__ float top8(float top, const float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j += 2)
    asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(top) : "f"(fabsf(v[j])), "f"(fabsf(v[j + 1])));
  return top;
}
// Sum of squares in 64 bits, in two chains.
struct Squares {
  double a = 0, b = 0;
  __device__ __forceinline__ void add8(const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) a = fma((double)v[j], (double)v[j], a), b = fma((double)v[j + 1], (double)v[j + 1], b);
  }
};

// A row's scale and what its codes are made with, out of its largest magnitude (as bits: a NaN's are above every
// number's) and sum of squares.
struct RowScale {
  float r, inv, scale;
  bool wild;
};
template <int MODE>
__device__ __forceinline__ RowScale row_scale(uint32_t top, double ss, uint32_t n, float eps) {
  RowScale s;
  s.r = MODE == kNorm ? (float)rsqrt(ss * (1.0 / (double)n) + (double)eps) : 1.f;
  // a sum that is not finite makes r 0 or NaN, and 0 times the infinity behind it a NaN
  const float most = MODE == kNorm ? __fmul_rn(__uint_as_float(top), s.r) : __uint_as_float(top);
  s.wild = !(fabsf(most) < INFINITY);
  const float scale = __fdiv_rn(most, 127.f);
  s.scale = s.wild ? __uint_as_float(0x7fffffffu) : scale < 1.17549435e-38f ? 0.f : scale;
  s.inv = s.wild || s.scale == 0.f ? 0.f : __fdiv_rn(1.f, s.scale);
  return s;
}
// Eight codes.  Adding 1.5 * 2^23 rounds to the nearest whole number, ties to even, and leaves it in the low byte.  None is over 127:
// |y| * (1 / scale) is at most 127 (1 + 3 * 2^-24).
template <int MODE>
__device__ __forceinline__ void codes8(const float (&v)[8], const RowScale& s, uint32_t (&c)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    float2 y = make_float2(v[j], v[j + 1]);
    if constexpr (MODE == kNorm) y = pair_mul(y, make_float2(s.r, s.r));
    // one by one: a product of pairs and the sum behind it came out as one fused operation, with one rounding in place of the
    // format's two
    y.x = __fmul_rn(y.x, s.inv), y.y = __fmul_rn(y.y, s.inv);
    y = pair_add(y, make_float2(12582912.f, 12582912.f));
    c[j] = __float_as_uint(y.x), c[j + 1] = __float_as_uint(y.y);
  }
}
template <int MODE>
__device__ __forceinline__ uint2 pack_codes8(const float (&v)[8], const RowScale& s) {
  uint32_t c[8], b[2];
  codes8<MODE>(v, s, c);
#pragma unroll
  for (int h = 0; h < 2; h++)
    b[h] = __byte_perm(__byte_perm(c[4 * h], c[4 * h + 1], 0x0040), __byte_perm(c[4 * h + 2], c[4 * h + 3], 0x0040), 0x5410);
  return s.wild ? make_uint2(0, 0) : make_uint2(b[0], b[1]);
}
template <int MODE>
__device__ __forceinline__ void store_codes8(int8_t* q, const float (&v)[8], const RowScale& s) {
  *reinterpret_cast<uint2*>(q) = pack_codes8<MODE>(v, s);
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ---- few rows, or rows that are not aligned: a CTA a row ------------------------------------
// Aligned: thread x has the eights x, x + blockDim.x, ... (PER of them).  Otherwise the elements x, x + blockDim.x, ...
template <class T, int MODE, int PER, bool VEC>
__global__ void __launch_bounds__(1024) rows_cta_kernel(RowsArgs a) {
  __shared__ double s_ss[32];
  __shared__ uint32_t s_top[32];
  griddep_launch();
  griddep_wait();
  const uint32_t n = a.n_cols, tid = threadIdx.x, nt = blockDim.x, warp = tid >> 5, lane = tid & 31;
  const uint64_t row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.x_stride;
  const T* y = (const T*)a.y + row * a.y_stride;
  auto place = [&](int p, int j) { return VEC ? (tid + p * nt) * 8 + j : (p * 8 + j) * nt + tid; };
  auto load = [&](const auto* src, float (&v)[PER][8]) {
    using S = std::remove_const_t<std::remove_pointer_t<decltype(src)>>;
    if constexpr (VEC) {
      constexpr int W = 8 / Act<S>::kVec;
      uint4 u[PER][W];
#pragma unroll
      for (int p = 0; p < PER; p++)
#pragma unroll
        for (int i = 0; i < W; i++) {
          u[p][i] = make_uint4(0, 0, 0, 0);
          if (place(p, 0) < n) u[p][i] = ld_once(src + place(p, 0) + i * Act<S>::kVec);
        }
#pragma unroll
      for (int p = 0; p < PER; p++) unpack8<S>(u[p], v[p]);
    } else {
#pragma unroll
      for (int p = 0; p < PER; p++)
#pragma unroll
        for (int j = 0; j < 8; j++) v[p][j] = place(p, j) < n ? Act<S>::get(src + place(p, j)) : 0.f;
    }
  };
  float v[PER][8];
  load(x, v);
  if (MODE == kSwiglu || (MODE == kNorm && a.y)) {
    float u[PER][8];
    load(y, u);
#pragma unroll
    for (int p = 0; p < PER; p++) combine8<MODE>(v[p], u[p]);
  }
  Squares sq;
  if constexpr (MODE == kNorm) {
    if (a.sum) {
      T* sum = (T*)a.sum + row * a.sum_stride;
#pragma unroll
      for (int p = 0; p < PER; p++)
        if constexpr (VEC) {
          if (place(p, 0) < n) store8<T>(sum + place(p, 0), v[p]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++)
            if (place(p, j) < n) Act<T>::put(sum + place(p, j), v[p][j]);
        }
    }
#pragma unroll
    for (int p = 0; p < PER; p++) sq.add8(v[p]);
    if (a.w) {
      float w[PER][8];
      load(a.w, w);
#pragma unroll
      for (int p = 0; p < PER; p++) multiply8(v[p], w[p]);
    }
  }
  float most = 0.f;
#pragma unroll
  for (int p = 0; p < PER; p++) most = top8(most, v[p]);
  uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
  double ss = 0;
  if constexpr (MODE == kNorm) ss = warp_sum(sq.a + sq.b);
  if (lane == 0) s_top[warp] = top, s_ss[warp] = ss;
  __syncthreads();
  const bool in = lane < (nt >> 5);
  top = __reduce_max_sync(0xffffffffu, in ? s_top[lane] : 0u);
  if constexpr (MODE == kNorm) ss = warp_sum(in ? s_ss[lane] : 0.0);
  const RowScale s = row_scale<MODE>(top, ss, n, a.eps);
  if (tid == 0) a.scale[row] = s.scale;
  int8_t* q = a.q + row * a.q_stride;
#pragma unroll
  for (int p = 0; p < PER; p++)
    if constexpr (VEC) {
      if (place(p, 0) < n) store_codes8<MODE>(q + place(p, 0), v[p], s);
    } else {
      uint32_t c[8];
      codes8<MODE>(v[p], s, c);
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (place(p, j) < n) q[place(p, j)] = s.wild ? 0 : (int8_t)c[j];
    }
}

// ---- many rows, aligned -------------------------------------------------------------------
// CTAs stay and go from row to row.  Rows come into a ring in shared memory by bulk copies, which go on while a row is
// reduced and coded; 32 elements a thread, a norm's weights in registers.  Instructions bound it, and those for each row and
// warp are as many as for 16 elements: 4001 x 4096 bf16 with residual and sum 23.0 us with 16 elements, 21.4 with 32 (5.4
// TB/s).  Where rows are so long that an SM has one CTA, two teams of its warps have a ring each, so that one asks for data
// while the other reduces: SwiGLU of 2048 x 14336 29.0 us without, 26.9 with them (5.5 TB/s).  The next kernel is let in with
// the last row: from the first one on, its waiting CTAs slowed chains of calls (norms of 8192 x 2001 f32 and the values
// back: 87 us, 67 so).
constexpr int kRowStages = 3;
constexpr uint32_t kRingBytes = 224 * 1024;

template <class T, int MODE, int PER, int TEAMS>
__global__ void __launch_bounds__(2048 / PER * TEAMS) rows_ring_kernel(RowsArgs a, uint32_t n_rows, uint32_t stages, unsigned* err) {
  extern __shared__ __align__(128) uint8_t rings[];
  __shared__ uint64_t fulls[TEAMS][kRowStages];
  __shared__ double s_sss[TEAMS][2][32];
  __shared__ uint32_t s_tops[TEAMS][2][32], s_stop;
  const uint32_t n = a.n_cols, nt = blockDim.x / TEAMS, team = threadIdx.x / nt, tid = threadIdx.x - team * nt, warp = tid >> 5, lane = tid & 31;
  const uint32_t first = blockIdx.x * TEAMS + team, step = gridDim.x * TEAMS;
  const uint32_t bytes = n * sizeof(T), stage = (a.y ? 2 : 1) * bytes;
  constexpr int V = Act<T>::kVec, W = 8 / V;
  uint8_t* ring = rings + team * stages * stage;
  uint64_t* full = fulls[team];
  auto &s_ss = s_sss[team];
  auto &s_top = s_tops[team];
  if (threadIdx.x == 0) {
    for (int i = 0; i < TEAMS * kRowStages; i++) tc_mbar_init(tc_smem_u32(fulls[0] + i), 1);
    tc_fence_barrier_init();
    s_stop = 0;
  }
  griddep_wait();
  __syncthreads();
  auto fetch = [&](uint64_t row, uint32_t slot) {
    const uint32_t bar = tc_smem_u32(full + slot), dst = tc_smem_u32(ring) + slot * stage;
    tc_mbar_expect_tx(bar, stage);
    tc_bulk_copy_g2s(dst, (const T*)a.x + row * a.x_stride, bytes, bar);
    if (a.y) tc_bulk_copy_g2s(dst + bytes, (const T*)a.y + row * a.y_stride, bytes, bar);
  };
  if (tid == 0)
    for (uint32_t i = 0; i < stages; i++)
      if (first + (uint64_t)i * step < n_rows) fetch(first + (uint64_t)i * step, i);
  uint32_t at[PER];
#pragma unroll
  for (int p = 0; p < PER; p++) at[p] = (tid + p * nt) * 8;
  float w[PER][8];
  if (MODE == kNorm) {
#pragma unroll
    for (int p = 0; p < PER; p++)
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        float4 f = make_float4(1.f, 1.f, 1.f, 1.f);
        if (a.w && at[p] < n) f = *reinterpret_cast<const float4*>(a.w + at[p] + j);
        w[p][j] = f.x, w[p][j + 1] = f.y, w[p][j + 2] = f.z, w[p][j + 3] = f.w;
      }
  }
  uint32_t slot = 0, phase = 0, turn = 0;
  for (uint64_t row = first; row < n_rows; row += step) {
    if (row + step >= n_rows) griddep_launch();
    const bool ok = wait_bar(full + slot, phase, &s_stop, err);
    float v[PER][8], most = 0.f;
    Squares sq;
#pragma unroll
    for (int p = 0; p < PER; p++) {
#pragma unroll
      for (int j = 0; j < 8; j++) v[p][j] = 0.f;
      if (at[p] >= n) continue;
      const T* src = (const T*)(ring + slot * stage) + at[p];
      uint4 u[W];
#pragma unroll
      for (int i = 0; i < W; i++) u[i] = *reinterpret_cast<const uint4*>(src + i * V);
      unpack8<T>(u, v[p]);
      if (a.y) {
        float y[8];
#pragma unroll
        for (int i = 0; i < W; i++) u[i] = *reinterpret_cast<const uint4*>(src + n + i * V);
        unpack8<T>(u, y);
        combine8<MODE>(v[p], y);
      }
      if constexpr (MODE == kNorm) {
        if (a.sum && ok) store8<T>((T*)a.sum + row * a.sum_stride + at[p], v[p]);
        sq.add8(v[p]);
        multiply8(v[p], w[p]);
      }
      most = top8(most, v[p]);
    }
    __syncwarp();
    uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
    double ss = 0;
    if constexpr (MODE == kNorm) ss = warp_sum(sq.a + sq.b);
    if (lane == 0) s_top[turn][warp] = top, s_ss[turn][warp] = ss;
    if constexpr (TEAMS == 1)  // all have read the slot, too
      __syncthreads();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(nt) : "memory");
    if (tid == 0 && ok && row + (uint64_t)stages * step < n_rows) fetch(row + (uint64_t)stages * step, slot);
    __syncwarp();
    const bool in = lane < (nt >> 5);
    top = __reduce_max_sync(0xffffffffu, in ? s_top[turn][lane] : 0u);
    if constexpr (MODE == kNorm) ss = warp_sum(in ? s_ss[turn][lane] : 0.0);
    const RowScale s = row_scale<MODE>(top, ss, n, a.eps);
    if (ok) {
      if (tid == 0) a.scale[row] = s.scale;
#pragma unroll
      for (int p = 0; p < PER; p++)
        if (at[p] < n) store_codes8<MODE>(a.q + row * a.q_stride + at[p], v[p], s);
    }
    turn ^= 1;
    if (++slot == stages) slot = 0, phase ^= 1;
  }
  if (*(volatile uint32_t*)&s_stop) {  // gave up: copies in flight end within this time
    const long long t = clock64();
    while (clock64() - t < 4000000LL) {
    }
  }
}

// ---- many rows, not aligned ---------------------------------------------------------------
// The same ring, of whole 16-byte granules around the rows: what lies beside a row in its first and last one is another
// row's or the gap's, and is not used; at the first row's beginning and the last one's end the elements are copied one by one.
// A thread's eights begin where x (and sum, which lies as x does) has a granule, `ahead` elements before a multiple of eight;
// y is shifted to them, the norm's weights lie in shared memory by their place in an eight, and a lane has the beginning of
// its codes' eight from itself, the end from the next lane.  A warp's last lane does the next warp's first eights again for that.
constexpr int kOwnLanes = 31;

__device__ __forceinline__ uint32_t phase_of(const void* p) { return (uint32_t)(uintptr_t)p & 15; }

// Eight elements from byte `shift` (0 .. 15) of the granules g on.
template <class T>
__device__ __forceinline__ void shift_words(const uint4 (&g)[8 / Act<T>::kVec + 1], uint32_t shift, uint4 (&u)[8 / Act<T>::kVec]) {
  constexpr int W = 8 / Act<T>::kVec;
  uint32_t w[4 * W + 4];
#pragma unroll
  for (int i = 0; i <= W; i++) w[4 * i] = g[i].x, w[4 * i + 1] = g[i].y, w[4 * i + 2] = g[i].z, w[4 * i + 3] = g[i].w;
  auto words = [&](auto first) {  // from word `first` on
    constexpr int F = decltype(first)::value;
    uint32_t o[4 * W];
#pragma unroll
    for (int i = 0; i < 4 * W; i++) o[i] = sizeof(T) == 2 ? __funnelshift_r(w[i + F], w[i + F + 1], (shift & 2) * 8) : w[i + F];
#pragma unroll
    for (int i = 0; i < W; i++) u[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
  };
  switch (shift >> 2) {
    case 0: words(std::integral_constant<int, 0>()); break;
    case 1: words(std::integral_constant<int, 1>()); break;
    case 2: words(std::integral_constant<int, 2>()); break;
    default: words(std::integral_constant<int, 3>());
  }
}
// The same from shared memory.
template <class T>
__device__ __forceinline__ void load_shifted(const uint8_t* src, uint32_t shift, uint4 (&u)[8 / Act<T>::kVec]) {
  constexpr int W = 8 / Act<T>::kVec;
  uint4 g[W + 1];
#pragma unroll
  for (int i = 0; i < W; i++) g[i] = reinterpret_cast<const uint4*>(src)[i];
  if (shift) {
    g[W] = reinterpret_cast<const uint4*>(src)[W];
    shift_words<T>(g, shift, u);
  } else {
#pragma unroll
    for (int i = 0; i < W; i++) u[i] = g[i];
  }
}
// Bytes `shift` (0 .. 7) to shift + 7 of two words and the two behind them.
__device__ __forceinline__ uint2 shift_bytes(uint2 a, uint2 b, uint32_t shift) {
  const uint32_t w0 = shift & 4 ? a.y : a.x, w1 = shift & 4 ? b.x : a.y, w2 = shift & 4 ? b.y : b.x;
  return make_uint2(__funnelshift_r(w0, w1, (shift & 3) * 8), __funnelshift_r(w1, w2, (shift & 3) * 8));
}

// Codes of the row's eight `eight`, from the numbers that begin `ahead` elements before it in this lane and the next: a whole warp.
template <int MODE>
__device__ __forceinline__ void store_shifted(int8_t* q, uint32_t eight, bool live, uint32_t ahead, uint32_t n, const float (&v)[8],
                                              const RowScale& s) {
  uint2 c = pack_codes8<MODE>(v, s);
  c = shift_bytes(c, make_uint2(__shfl_down_sync(0xffffffffu, c.x, 1), __shfl_down_sync(0xffffffffu, c.y, 1)), ahead);
  const uint32_t e = eight * 8;
  if (!live || e >= n) return;
  if (e + 8 <= n)
    *reinterpret_cast<uint2*>(q + e) = c;
  else
    for (uint32_t j = 0; j < n - e; j++) q[e + j] = (int8_t)((j < 4 ? c.x : c.y) >> 8 * (j & 3));
}

// The weights of an eight that begins `ahead` (below MOST) elements before w's: [e % 8][e / 8 + 1].
template <int MOST, int A = 0>
__device__ __forceinline__ void eight_weights(const float* src, uint32_t row, uint32_t ahead, float (&w)[8]) {
  if constexpr (A + 1 < MOST)
    if (ahead != A) return eight_weights<MOST, A + 1>(src, row, ahead, w);
#pragma unroll
  for (int j = 0; j < 8; j++) w[j] = src[((j - A) & 7) * row + (j < A ? 0 : 1)];
}

__host__ __device__ constexpr uint32_t shift_eights(uint32_t n) { return n / 8 + 2; }  // that a row may touch
__host__ __device__ constexpr uint32_t shift_x_bytes(uint32_t n, uint32_t es) { return shift_eights(n) * 8 * es; }
__host__ __device__ constexpr uint32_t shift_y_bytes(uint32_t n, uint32_t es) { return shift_x_bytes(n, es) + 48; }  // a granule before, two behind

template <class T, int MODE, int PER>
__global__ void __launch_bounds__(2048 / PER) rows_shift_kernel(RowsArgs a, uint32_t n_rows, unsigned* err) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint64_t full[kRowStages];
  __shared__ double s_ss[2][32];
  __shared__ uint32_t s_top[2][32], s_stop;
  const uint32_t n = a.n_cols, tid = threadIdx.x, nt = blockDim.x, warp = tid >> 5, lane = tid & 31;
  constexpr uint32_t ES = sizeof(T), V = Act<T>::kVec, W = 8 / V;
  const uint32_t y_at = shift_x_bytes(n, ES), stage = y_at + (a.y ? shift_y_bytes(n, ES) : 0), w_row = shift_eights(n) + 1;
  float* s_w = reinterpret_cast<float*>(ring + kRowStages * stage);  // [e % 8][e / 8 + 1]
  if (tid == 0) {
    for (int i = 0; i < kRowStages; i++) tc_mbar_init(tc_smem_u32(full + i), 1);
    tc_fence_barrier_init();
    s_stop = 0;
  }
  griddep_wait();
  auto fetch = [&](uint64_t row, uint32_t slot) {
    const uint32_t bar = tc_smem_u32(full + slot), dst = tc_smem_u32(ring) + slot * stage;
    struct Span {
      const uint8_t* from;
      uint32_t skip, bytes;
    };
    auto span = [&](const T* p) {
      const uint32_t m = phase_of(p), end = m + n * ES, skip = row == 0 && m ? 16 : 0;  // of the row, from its first granule on
      return Span{(const uint8_t*)p + (int)skip - (int)m, skip, (row == n_rows - 1 ? end & ~15u : (end + 15) & ~15u) - skip};
    };
    const Span x = span((const T*)a.x + row * a.x_stride), y = span((const T*)a.y + row * a.y_stride);
    tc_mbar_expect_tx(bar, x.bytes + (a.y ? y.bytes : 0));
    tc_bulk_copy_g2s(dst + x.skip, x.from, x.bytes, bar);
    if (a.y) tc_bulk_copy_g2s(dst + y_at + 16 + y.skip, y.from, y.bytes, bar);
  };
  if (tid == 0)
    for (int i = 0; i < kRowStages; i++)
      if (blockIdx.x + (uint64_t)i * gridDim.x < n_rows) fetch(blockIdx.x + (uint64_t)i * gridDim.x, i);
  if constexpr (MODE == kNorm) {  // an eight a lane, so that stores do not meet, and all loads at once
    float f[PER][8];
#pragma unroll
    for (int p = 0; p < PER; p++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const uint32_t e = (tid + p * nt) * 8 + j;
        f[p][j] = a.w && e < n ? a.w[e] : 1.f;
      }
#pragma unroll
    for (int p = 0; p < PER; p++)
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (tid + p * nt < w_row - 1) s_w[j * w_row + tid + p * nt + 1] = f[p][j];
    if (tid < 8) s_w[tid * w_row] = 1.f;
  }
  __syncthreads();
  uint32_t at[PER];
#pragma unroll
  for (int p = 0; p < PER; p++) at[p] = (warp + p * (nt >> 5)) * kOwnLanes + lane;
  const bool own = lane < kOwnLanes;
  uint32_t slot = 0, phase = 0, turn = 0;
  for (uint64_t row = blockIdx.x; row < n_rows; row += gridDim.x) {
    const T* x = (const T*)a.x + row * a.x_stride;
    const T* y = (const T*)a.y + row * a.y_stride;
    const uint32_t ahead = phase_of(x) / ES, eights = (ahead + n + 7) / 8;
    const uint32_t y_from = a.y ? y_at + 16 + phase_of(y) - phase_of(x) : 0;
    uint8_t* here = ring + slot * stage;
    if (row + gridDim.x >= n_rows) griddep_launch();
    const bool ok = wait_bar(full + slot, phase, &s_stop, err);
    if (row == 0 || row == n_rows - 1) {
      auto edges = [&](const T* p, uint8_t* to) {
        const uint32_t m = phase_of(p), head = row == 0 ? (16 - m & 15) / ES : 0;
        const uint32_t tail = row == n_rows - 1 ? (m + n * ES & 15) / ES : 0;
        T* dst = reinterpret_cast<T*>(to + m);
        if (tid < head) dst[tid] = p[tid];
        if (tid < tail) dst[n - tail + tid] = p[n - tail + tid];
      };
      edges(x, here);
      if (a.y) edges(y, here + y_at + 16);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the slot's next copy
      __syncthreads();
    }
    float v[PER][8], most = 0.f;
    Squares sq;
#pragma unroll
    for (int p = 0; p < PER; p++) {
#pragma unroll
      for (int j = 0; j < 8; j++) v[p][j] = 0.f;
      if (at[p] >= eights) continue;
      const uint8_t* src = here + at[p] * 8 * ES;
      uint4 u[W];
#pragma unroll
      for (int i = 0; i < (int)W; i++) u[i] = reinterpret_cast<const uint4*>(src)[i];
      unpack8<T>(u, v[p]);
      if (a.y) {
        float f[8];
        load_shifted<T>(src + (y_from & ~15u), y_from & 15, u);
        unpack8<T>(u, f);
        combine8<MODE>(v[p], f);
      }
      const int e0 = (int)(at[p] * 8) - (int)ahead;
      const bool whole = e0 >= 0 && e0 + 8 <= (int)n;
      if (!whole)
#pragma unroll
        for (int j = 0; j < 8; j++) v[p][j] = e0 + j >= 0 && e0 + j < (int)n ? v[p][j] : 0.f;
      if constexpr (MODE == kNorm) {
        if (own) {
          if (a.sum && ok) {
            T* sum = (T*)a.sum + row * a.sum_stride + e0;
            if (whole)
              store8<T>(sum, v[p]);
            else
#pragma unroll
              for (int j = 0; j < 8; j++)
                if (e0 + j >= 0 && e0 + j < (int)n) Act<T>::put(sum + j, v[p][j]);
          }
          sq.add8(v[p]);
        }
        if (a.w) {
        float w[8];
        eight_weights<8 / W>(s_w + at[p], w_row, ahead, w);
        multiply8(v[p], w);
        }
      }
      most = top8(most, v[p]);
    }
    __syncwarp();
    uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
    double ss = 0;
    if constexpr (MODE == kNorm) ss = warp_sum(sq.a + sq.b);
    if (lane == 0) s_top[turn][warp] = top, s_ss[turn][warp] = ss;
    __syncthreads();  // all have read the slot, too
    if (tid == 0 && ok && row + (uint64_t)kRowStages * gridDim.x < n_rows) fetch(row + (uint64_t)kRowStages * gridDim.x, slot);
    __syncwarp();
    const bool in = lane < (nt >> 5);
    top = __reduce_max_sync(0xffffffffu, in ? s_top[turn][lane] : 0u);
    if constexpr (MODE == kNorm) ss = warp_sum(in ? s_ss[turn][lane] : 0.0);
    const RowScale s = row_scale<MODE>(top, ss, n, a.eps);
    if (tid == 0 && ok) a.scale[row] = s.scale;
    int8_t* q = a.q + row * a.q_stride;
#pragma unroll
    for (int p = 0; p < PER; p++) store_shifted<MODE>(q, at[p], own && ok, ahead, n, v[p], s);
    turn ^= 1;
    if (++slot == kRowStages) slot = 0, phase ^= 1;
  }
  if (*(volatile uint32_t*)&s_stop) {  // gave up: copies in flight end within this time
    const long long t = clock64();
    while (clock64() - t < 4000000LL) {
    }
  }
}

// ---- rows that are not aligned, without a norm: a CTA a row -------------------------------------
// The eights of rows_shift_kernel straight from global memory: where there is no sum of squares the instructions are few
// enough that more threads hide the loads as well as the ring does, or better; launch_rows_as has both sides.
template <class T, int MODE, int PER>
__global__ void __launch_bounds__(1024) rows_shift_cta_kernel(RowsArgs a) {
  constexpr int V = Act<T>::kVec, W = 8 / V;
  __shared__ uint32_t s_top[32];
  griddep_launch();
  griddep_wait();
  const uint32_t n = a.n_cols, tid = threadIdx.x, nt = blockDim.x, warp = tid >> 5, lane = tid & 31;
  const uint64_t row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.x_stride;
  const T* y = (const T*)a.y + row * a.y_stride;
  const uint32_t ahead = phase_of(x) / sizeof(T), shift = MODE == kSwiglu ? (phase_of(y) - phase_of(x)) & 15 : 0;
  uint32_t at[PER];
  bool whole[PER];  // the granules that hold the eight's numbers lie within the rows
  uint4 ux[PER][W], uy[PER][W + 1];
#pragma unroll
  for (int p = 0; p < PER; p++) {
    at[p] = (warp + p * (nt >> 5)) * kOwnLanes + lane;
    const int e0 = (int)(at[p] * 8) - (int)ahead;
    const int y0 = e0 - (int)(shift / sizeof(T)), more = shift ? V : 0;
    whole[p] = (MODE == kSwiglu ? y0 : e0) >= 0 && e0 + 8 <= (int)n && (MODE != kSwiglu || y0 + 8 + more <= (int)n);
    if (!whole[p]) continue;
#pragma unroll
    for (int i = 0; i < W; i++) ux[p][i] = ld_once(x + e0 + i * V);
    if (MODE == kSwiglu) {
#pragma unroll
      for (int i = 0; i < W; i++) uy[p][i] = *reinterpret_cast<const uint4*>(y + y0 + i * V);
      if (shift) uy[p][W] = *reinterpret_cast<const uint4*>(y + y0 + 8);
    }
  }
  float v[PER][8], most = 0.f;
#pragma unroll
  for (int p = 0; p < PER; p++) {
    const int e0 = (int)(at[p] * 8) - (int)ahead;
    if (whole[p]) {
      unpack8<T>(ux[p], v[p]);
      if (MODE == kSwiglu) {
        float f[8];
        uint4 u[W];
        shift_words<T>(uy[p], shift, u);
        unpack8<T>(u, f);
        combine8<MODE>(v[p], f);
      }
    } else {
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const bool in = e0 + j >= 0 && e0 + j < (int)n;
        v[p][j] = in ? Act<T>::get(x + e0 + j) : 0.f;
        if (MODE == kSwiglu) f[j] = in ? Act<T>::get(y + e0 + j) : 0.f;
      }
      if (MODE == kSwiglu) combine8<MODE>(v[p], f);
    }
    most = top8(most, v[p]);
  }
  __syncwarp();
  uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
  if (lane == 0) s_top[warp] = top;
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, lane < (nt >> 5) ? s_top[lane] : 0u);
  const RowScale s = row_scale<MODE>(top, 0.0, n, a.eps);
  if (tid == 0) a.scale[row] = s.scale;
#pragma unroll
  for (int p = 0; p < PER; p++) store_shifted<MODE>(a.q + row * a.q_stride, at[p], lane < kOwnLanes, ahead, n, v[p], s);
}

// ---- many short rows: a warp a row ---------------------------------------------------
// PER eights a lane, or, where rows are not aligned, every 32nd element; the next row's are asked for before a row is worked on.
// *p where `on`, else 1 and nothing is read.  A plain load of C++ would stay behind the stores of the sums (4000 x 501 f32 with
// residual and sum: 9.7 us, 8.1 so).
__device__ __forceinline__ float weight_if(bool on, const float* p) {
  float w = 1.f;
  asm volatile("{ .reg .pred q; setp.ne.u32 q, %2, 0;\n\t@q ld.global.f32 %0, [%1]; }" : "+f"(w) : "l"(p), "r"((uint32_t)on));
  return w;
}
template <class T, int MODE, int PER, bool VEC>
__global__ void __launch_bounds__(256) rows_warp_kernel(RowsArgs a, uint32_t n_rows) {
  griddep_launch();
  griddep_wait();
  const uint32_t n = a.n_cols, lane = threadIdx.x & 31, step = gridDim.x * 8;
  constexpr int V = Act<T>::kVec, W = 8 / V;
  using Raw = std::conditional_t<VEC, uint4[PER][W], T[PER][8]>;
  Raw nx, ny;
  auto place = [&](int p, int j) { return VEC ? (lane + 32 * p) * 8 + j : (p * 8 + j) * 32 + lane; };
  auto load = [&](uint64_t row) {
    const T *x = (const T*)a.x + row * a.x_stride, *y = (const T*)a.y + row * a.y_stride;
#pragma unroll
    for (int p = 0; p < PER; p++)
      if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < W; i++) {
          const uint32_t c = place(p, i * V);
          nx[p][i] = ny[p][i] = make_uint4(0, 0, 0, 0);
          if (row < n_rows && c < n) {
            nx[p][i] = ld_once(x + c);
            if (a.y) ny[p][i] = ld_once(y + c);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const uint32_t c = place(p, j);
          nx[p][j] = ny[p][j] = T(0.f);
          if (row < n_rows && c < n) {
            nx[p][j] = x[c];
            if (a.y) ny[p][j] = y[c];
          }
        }
      }
  };
  auto values = [&](const Raw& raw, int p, float (&v)[8]) {
    if constexpr (VEC) {
      unpack8<T>(raw[p], v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = Act<T>::get(&raw[p][j]);
    }
  };
  uint64_t row = blockIdx.x * 8 + (threadIdx.x >> 5);
  load(row);
  for (; row < n_rows; row += step) {
    float v[PER][8], most = 0.f;
    Squares sq;
#pragma unroll
    for (int p = 0; p < PER; p++) {
      values(nx, p, v[p]);
      if (a.y) {
        float y[8];
        values(ny, p, y);
        combine8<MODE>(v[p], y);
      }
    }
    load(row + step);
#pragma unroll
    for (int p = 0; p < PER; p++) {
      if constexpr (MODE == kNorm) {
        if (a.sum) {
          T* sum = (T*)a.sum + row * a.sum_stride;
          if constexpr (VEC) {
            if (place(p, 0) < n) store8<T>(sum + place(p, 0), v[p]);
          } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
              if (place(p, j) < n) Act<T>::put(sum + place(p, j), v[p][j]);
          }
        }
        sq.add8(v[p]);
        if (a.w) {
          if constexpr (VEC) {
            if (place(p, 0) < n) {
#pragma unroll
              for (int j = 0; j < 8; j += 4) {
                const float4 f = *reinterpret_cast<const float4*>(a.w + place(p, j));
                v[p][j] = __fmul_rn(v[p][j], f.x), v[p][j + 1] = __fmul_rn(v[p][j + 1], f.y);
                v[p][j + 2] = __fmul_rn(v[p][j + 2], f.z), v[p][j + 3] = __fmul_rn(v[p][j + 3], f.w);
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
              v[p][j] = __fmul_rn(v[p][j], weight_if(place(p, j) < n, a.w + place(p, j)));
          }
        }
      }
      most = top8(most, v[p]);
    }
    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
    double ss = 0;
    if constexpr (MODE == kNorm) ss = warp_sum(sq.a + sq.b);
    const RowScale s = row_scale<MODE>(top, ss, n, a.eps);
    if (lane == 0) a.scale[row] = s.scale;
    int8_t* q = a.q + row * a.q_stride;
#pragma unroll
    for (int p = 0; p < PER; p++)
      if constexpr (VEC) {
        if (place(p, 0) < n) store_codes8<MODE>(q + place(p, 0), v[p], s);
      } else {
        uint32_t c[8];
        codes8<MODE>(v[p], s, c);
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (place(p, j) < n) q[place(p, j)] = s.wild ? 0 : (int8_t)c[j];
      }
  }
}

template <class T, int MODE, bool VEC>
cudaError_t launch_cta(const Launch& L, const RowsArgs& a, uint32_t n_rows) {
  const uint32_t eights = (a.n_cols + 7) / 8;
  // 16 elements a thread, more where 1024 threads do not suffice: those do not fit the 64 registers that 1024 threads have, so norms
  // and single elements of more than 16384 columns (aligned SwiGLU and plain rows: 32768) go through local memory.  300 rows with residual and sum,
  // bf16: 16384 columns 13.6 us, 20480 28.5, 40960 105, 40961 313; SwiGLU of 300 x 20480 9.1, x 40960 18.9.
  const uint32_t per = eights <= 2048 ? 2 : eights <= 4096 ? 4 : 8;
  const uint32_t threads = std::max(32u, ((eights + per - 1) / per + 31) / 32 * 32);
  auto* k = per == 2 ? rows_cta_kernel<T, MODE, 2, VEC> : per == 4 ? rows_cta_kernel<T, MODE, 4, VEC> : rows_cta_kernel<T, MODE, 8, VEC>;
  return launch_k(L, k, dim3(n_rows), dim3(threads), 0, a);
}

template <class T, int MODE, bool VEC>
cudaError_t launch_rows_as(const Launch& L, const RowsArgs& a, uint32_t n_rows, bool shift, unsigned* err) {
  const uint32_t eights = (a.n_cols + 7) / 8, sms = (uint32_t)num_sms();
  // eights a lane of a warp that has a row: what its registers hold beside the next row's
  constexpr uint32_t most = sizeof(T) == 2 && VEC ? 4 : 2;
  const uint32_t per = (eights + 31) / 32;
  if (per <= most && n_rows > 4 * sms) {
    auto* k = per == 1 ? rows_warp_kernel<T, MODE, 1, VEC> : rows_warp_kernel<T, MODE, 2, VEC>;
    if constexpr (most == 4)
      if (per > 2) k = rows_warp_kernel<T, MODE, 4, VEC>;
    return launch_k(L, k, dim3(std::min((n_rows + 7) / 8, sms * 4)), dim3(256), 0, a, n_rows);
  }
  // CTAs that stay, per_sm of them on each SM.  What is counted is their threads and the shared memory they ask for, not the 384 to
  // 896 bytes that the kernel has besides and the 1 KB that each CTA takes: at the widths at which that makes one too many
  // the last ones run when the others have ended (norm of 4000 rows with residual, f32: 14.3 us with 1152 columns, 11.6 with
  // 1200; 25.8 with 2368, 20.2 with 2392).
  auto ring = [&](auto* k, uint32_t threads, uint32_t smem, uint32_t per_sm, auto... more) {
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes);
    return e != cudaSuccess ? e : launch_k(L, k, dim3(sms * per_sm), dim3(threads), smem, a, n_rows, more..., err);
  };
  if constexpr (VEC) {
    // A norm: 4001 x 4096 bf16 with residual and sum 21.4 us, 35 with a CTA a row (600 rows: 6.5 and 8.2).  SwiGLU of 5000 x
    // 4096: 21.1 and 16.8; of 1800 x 14336, where an SM has room for one CTA of the other kernel, 25.0 with two teams, 26.7
    // with one of 16 elements a thread (kept for rows of which an SM has no room for four), 31.5 with a CTA a row.
    const uint32_t threads = ((eights + 3) / 4 + 31) / 32 * 32, stage = (a.y ? 2 : 1) * a.n_cols * (uint32_t)sizeof(T);
    const uint32_t stages = std::min(kRingBytes / (2 * stage), (uint32_t)kRowStages);  // of each of two teams
    if (threads <= 512 && n_rows >= 4 * sms) {
      if constexpr (MODE == kNorm) {
        const uint32_t per_sm = std::min(std::min(std::min(512 / threads, kRingBytes / (kRowStages * stage)), 8u), n_rows / sms);
        if (per_sm) return ring(rows_ring_kernel<T, MODE, 4, 1>, threads, kRowStages * stage, per_sm, kRowStages);
      } else if (a.n_cols > 8192) {
        if (stages >= 2) return ring(rows_ring_kernel<T, MODE, 4, 2>, 2 * threads, 2 * stages * stage, 1, stages);
        if (kRowStages * stage <= kRingBytes)
          return ring(rows_ring_kernel<T, MODE, 2, 1>, 2 * threads, kRowStages * stage, 1, kRowStages);
      }
    }
  } else if (shift) {
    constexpr uint32_t PER = 2, TH = MODE == kNorm ? 1024 : 1280;
    const uint32_t es = sizeof(T), lanes = PER * kOwnLanes, threads = (shift_eights(a.n_cols) + lanes - 1) / lanes * 32;
    const uint32_t stage = shift_x_bytes(a.n_cols, es) + (a.y ? shift_y_bytes(a.n_cols, es) : 0);
    const uint32_t smem = kRowStages * stage + (MODE == kNorm ? (shift_eights(a.n_cols) + 1) * 8 * 4 : 0);
    const uint32_t some = std::min(std::min(std::min(TH / threads, kRingBytes / smem), 16u), n_rows / sms);
    // A norm in the ring and element by element in a CTA a row, bf16: 4001 x 4095 32.8 us and 61.4, 296 x 1025 3.8 and 4.4, 592 x
    // 1023 4.3 and 5.2 (444 x 1023, a CTA a row by the rule: 4.1 and 6.2).  SwiGLU in the ring and a CTA a row, bf16: 2048 x
    // 14335 40.7 and 91.2 (by elements); 4000 x 2799 16.4 and 15.8, x 2801 15.7 and 15.5, x 4095 22.7 and 23.9; 592 x 4095 5.6 and
    // 5.5; 296 x 4097 3.3 both, x 8191 5.9 and 6.2.  Plain rows, bf16: 4000 x 2801 12.9 and 11.2 (10.0 with two eights), x 4095 18.6
    // and 17.5 (14.8); 296 x 8191 3.4 and 2.7: there the ring comes too early.
    const uint32_t least = (MODE == kNorm ? a.n_cols < 1024 : a.n_cols <= 4096) ? 4 * sms : 2 * sms;
    if (threads <= 2048 / PER && some && n_rows >= least && (MODE == kNorm || a.n_cols > 2800))
      return ring(rows_shift_kernel<T, MODE, PER>, threads, smem, some);
    if constexpr (MODE != kNorm) {
      // SwiGLU of 2500 x 1279 bf16: 6.9 us with an eight a thread, 7.4 with two, 8.1 in the ring; 1200 x 4097: 8.9, 9.5 and 8.9;
      // 1200 x 8191: 24.8 (12.4 with 592 rows) and 16.1 (9.4) in the ring; 592 x 515: 2.6 with an eight a thread, 3.2 by elements,
      // 592 x 509: 2.6 and 3.4 (by elements by the rule).
      const uint32_t one = (shift_eights(a.n_cols) + kOwnLanes - 1) / kOwnLanes * 32;
      if (a.n_cols >= 512 && a.n_cols <= 4096) return launch_k(L, rows_shift_cta_kernel<T, MODE, 1>, dim3(n_rows), dim3(one), 0, a);
      if (a.n_cols >= 512 && threads <= 1024) return launch_k(L, rows_shift_cta_kernel<T, MODE, 2>, dim3(n_rows), dim3(threads), 0, a);
    }
  }
  return launch_cta<T, MODE, VEC>(L, a, n_rows);
}
template <class T, int MODE>
cudaError_t launch_rows(const Launch& L, const RowsArgs& a, uint32_t n_rows, bool vec, bool shift, unsigned* err) {
  return vec ? launch_rows_as<T, MODE, true>(L, a, n_rows, shift, err) : launch_rows_as<T, MODE, false>(L, a, n_rows, shift, err);
}

template <int MODE>
int run_rows(int act_type, const RowsArgs& a, uint32_t n_rows, void* stream) {
  const uint32_t es = act_bytes(act_type);
  bool vec = aligned_to(a.q, 8) && a.q_stride % 8 == 0 && a.n_cols % 8 == 0;
  for (const void* p : {a.x, a.y, (const void*)a.sum, (const void*)a.w}) vec = vec && aligned_to(p, 16);
  for (uint64_t s : {a.x_stride, a.y_stride, a.sum_stride}) vec = vec && s * es % 16 == 0;
  // rows_shift_kernel's: codes in whole eights, sum at x's places within 16 bytes
  const bool shift = aligned_to(a.q, 8) && a.q_stride % 8 == 0 && a.n_cols >= 64 &&
                     (!a.sum || (((uintptr_t)a.x ^ (uintptr_t)a.sum) % 16 == 0 && (a.x_stride ^ a.sum_stride) * es % 16 == 0));
  const Launch L{(cudaStream_t)stream, true};
  unsigned* err = nullptr;
  RF_TRY(verify_error_ptr(&err));
  switch (act_type) {
    case RF_ACT_F32: RF_CUDA((launch_rows<float, MODE>(L, a, n_rows, vec, shift, err))); break;
    case RF_ACT_F16: RF_CUDA((launch_rows<__half, MODE>(L, a, n_rows, vec, shift, err))); break;
    default: RF_CUDA((launch_rows<__nv_bfloat16, MODE>(L, a, n_rows, vec, shift, err)));
  }
  return RF_OK;
}

// ---- rows back -----------------------------------------------------------------------
struct ValuesArgs {
  const int8_t* q;
  const float* scale;
  void* out;
  uint64_t q_stride, out_stride, pieces;  // pieces of all rows
  uint32_t n_cols, per_row;
  bool wide;  // rows of values are 32-byte aligned
};

// Eight codes times a scale.  A byte under the exponent of 2^23 is 2^23 + 128 + code, the sum with the bias's negative exact.
__device__ __forceinline__ void values8(uint2 codes, float scale, float (&v)[8]) {
  const uint32_t w[2] = {codes.x ^ 0x80808080u, codes.y ^ 0x80808080u};
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const uint32_t x = w[j / 4];
    const float2 code = pair_add(make_float2(__uint_as_float(__byte_perm(x, 0x4b000000u, 0x7440 + (j & 3))),
                                             __uint_as_float(__byte_perm(x, 0x4b000000u, 0x7440 + (j & 3) + 1))),
                                 make_float2(-8388736.f, -8388736.f));
    const float2 y = pair_mul(code, make_float2(scale, scale));
    v[j] = y.x, v[j + 1] = y.y;
  }
}
// Aligned: a thread has 8 codes of a row at a time, four such pieces in flight; neighbours' pieces lie side by side.
template <class T>
__global__ void __launch_bounds__(256) values_i8_kernel(ValuesArgs a) {
  constexpr int U = 4;
  griddep_launch();
  griddep_wait();
  const uint64_t step = (uint64_t)gridDim.x * 256;
  for (uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x; at < a.pieces; at += U * step) {
    uint2 u[U];
    float scale[U];
    T* to[U];
#pragma unroll
    for (int i = 0; i < U; i++) {
      const uint64_t piece = min(at + i * step, a.pieces - 1);
      const uint64_t row = piece >> 32 ? piece / a.per_row : (uint32_t)piece / a.per_row;
      const uint32_t c = (uint32_t)(piece - row * a.per_row) * 8;
      u[i] = *reinterpret_cast<const uint2*>(a.q + row * a.q_stride + c);
      scale[i] = a.scale[row];
      to[i] = (T*)a.out + row * a.out_stride + c;
    }
#pragma unroll
    for (int i = 0; i < U; i++) {
      if (at + i * step >= a.pieces) break;
      float v[8];
      values8(u[i], scale[i], v);
      if constexpr (sizeof(T) == 4) {
        if (a.wide)
          store8_wide(to[i], v);
        else
          store8<T>(to[i], v);
      } else {
        store8<T>(to[i], v);
      }
    }
  }
}
// Rows of values at any place, codes in whole eights: eight values from a granule's beginning on, their codes shifted to them.
template <class T>
__global__ void __launch_bounds__(256) values_shift_kernel(ValuesArgs a) {
  constexpr int U = 2;
  griddep_launch();
  griddep_wait();
  const uint64_t step = (uint64_t)gridDim.x * 256;
  for (uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x; at < a.pieces; at += U * step) {
    uint2 lo[U], hi[U];
    float scale[U];
    uint64_t rows[U];
    int first[U];
    uint32_t shift[U];
#pragma unroll
    for (int i = 0; i < U; i++) {
      const uint64_t piece = min(at + i * step, a.pieces - 1);
      const uint64_t row = piece >> 32 ? piece / a.per_row : (uint32_t)piece / a.per_row;
      const uint32_t c = (uint32_t)(piece - row * a.per_row) * 8;
      const uint32_t ahead = phase_of((T*)a.out + row * a.out_stride) / sizeof(T);
      rows[i] = row, first[i] = (int)c - (int)ahead, shift[i] = -ahead & 7;
      lo[i] = hi[i] = make_uint2(0, 0);
      // codes from the eight that holds the first on; an eight that the row ends in is left to the loop below
      const uint32_t e = c - (ahead ? 8 : 0);
      const int8_t* q = a.q + row * a.q_stride;
      scale[i] = a.scale[row];
      if (first[i] >= 0 && e + 8 <= a.n_cols) lo[i] = *reinterpret_cast<const uint2*>(q + e);
      if (first[i] >= 0 && ahead && e + 16 <= a.n_cols) hi[i] = *reinterpret_cast<const uint2*>(q + e + 8);
    }
#pragma unroll
    for (int i = 0; i < U; i++) {
      if (at + i * step >= a.pieces) break;
      T* out = (T*)a.out + rows[i] * a.out_stride + first[i];
      const int8_t* q = a.q + rows[i] * a.q_stride + first[i];
      const uint32_t read = first[i] < 0 ? 0 : ((uint32_t)first[i] & ~7u) + (shift[i] ? 16 : 8);
      if (first[i] >= 0 && read <= a.n_cols) {
        float v[8];
        values8(shift_bytes(lo[i], hi[i], shift[i]), scale[i], v);
        store8<T>(out, v);
      } else {
        for (int j = max(0, -first[i]); j < min(8, (int)a.n_cols - first[i]); j++) Act<T>::put(out + j, __fmul_rn((float)q[j], scale[i]));
      }
    }
  }
}
// Any: a warp has 256 codes of a row at a time, a lane every 32nd of them.
template <class T>
__global__ void __launch_bounds__(256) values_any_kernel(ValuesArgs a) {
  griddep_launch();
  griddep_wait();
  const uint32_t lane = threadIdx.x & 31;
  for (uint64_t at = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); at < a.pieces; at += (uint64_t)gridDim.x * 8) {
    const uint64_t row = at / a.per_row;
    const uint32_t c = (uint32_t)(at - row * a.per_row) * 256 + lane;
    const int8_t* q = a.q + row * a.q_stride;
    T* out = (T*)a.out + row * a.out_stride;
    const float scale = a.scale[row];
    int8_t code[8];
#pragma unroll
    for (int j = 0; j < 8; j++) code[j] = c + 32 * j < a.n_cols ? q[c + 32 * j] : 0;
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (c + 32 * j < a.n_cols) Act<T>::put(out + c + 32 * j, __fmul_rn((float)code[j], scale));
  }
}

template <class T>
cudaError_t launch_values(const Launch& L, ValuesArgs a, uint32_t n_rows) {
  const bool eights = aligned_to(a.q, 8) && a.q_stride % 8 == 0;
  const bool vec = eights && a.n_cols % 8 == 0 && aligned_to(a.out, 16) && a.out_stride * sizeof(T) % 16 == 0;
  // 4001 x 4095 bf16: 14.7 us with codes shifted to the values' granules, 16.2 element by element; 2000 x 601: 3.8 and 2.9
  const bool shift = eights && !vec && a.n_cols >= 1024;
  const uint32_t unit = vec || shift ? 8 : 256, per_cta = vec || shift ? 256 : 8;
  a.wide = aligned_to(a.out, 32) && a.out_stride * sizeof(T) % 32 == 0;
  a.per_row = (a.n_cols + unit - 1) / unit + shift;  // one begun before the row
  a.pieces = (uint64_t)a.per_row * n_rows;
  const uint64_t ctas = std::min<uint64_t>((a.pieces + per_cta - 1) / per_cta, (uint64_t)num_sms() * 8);
  return launch_k(L, vec ? values_i8_kernel<T> : shift ? values_shift_kernel<T> : values_any_kernel<T>, dim3((uint32_t)ctas), dim3(256), 0, a);
}

// ---- checks --------------------------------------------------------------------------
int check_shape(int act_type, uint32_t n_rows, uint32_t n_cols) {
  if (!act_bytes(act_type)) return set_error(RF_EINVAL, "activation type %d is not F32, F16 or BF16", act_type);
  if (!n_cols || n_cols > kMaxCols) return set_error(RF_EINVAL, "%u columns are not within 1..%u", n_cols, kMaxCols);
  if (n_rows > 0x7fffffffu) return set_error(RF_EINVAL, "%u rows are too many for one call", n_rows);
  return RF_OK;
}
int check_stride(uint64_t* stride, uint32_t n_cols) {
  if (!*stride) *stride = n_cols;
  if (*stride < n_cols)
    return set_error(RF_EINVAL, "row stride %llu is below the row's %u elements", (unsigned long long)*stride, n_cols);
  return RF_OK;
}
int check_rows_ptr(const void* p, uint32_t es) {
  if (!aligned_to(p, es)) return set_error(RF_EINVAL, "rows must be aligned to their element size");
  return RF_OK;
}
int check_scale(const float* scale) {
  if (!aligned_to(scale, 4)) return set_error(RF_EINVAL, "scales must be 4-byte aligned");
  return RF_OK;
}

}  // namespace
}  // namespace rf

using namespace rf;

extern "C" {

int rf_norm_i8(const void* x, const void* add, void* sum, int act_type, uint32_t n_rows, uint32_t n_cols,
               uint64_t x_stride, uint64_t add_stride, uint64_t sum_stride, const float* weight, float eps, int8_t* q,
               uint64_t q_stride, float* scale, void* stream) {
  RF_TRY(check_shape(act_type, n_rows, n_cols));
  if (n_rows && (!x || !q || !scale)) return set_error(RF_EINVAL, "null rows, codes or scales");
  for (uint64_t* s : {&x_stride, &add_stride, &sum_stride, &q_stride}) RF_TRY(check_stride(s, n_cols));
  for (const void* p : {x, add, (const void*)sum}) RF_TRY(check_rows_ptr(p, act_bytes(act_type)));
  RF_TRY(check_scale(scale));
  if (!aligned_to(weight, 4)) return set_error(RF_EINVAL, "norm weights must be 4-byte aligned");
  if (!(eps >= 0.f) || eps > 3.0e38f) return set_error(RF_EINVAL, "eps must be a number that is not negative");
  if (!n_rows) return RF_OK;
  return run_rows<kNorm>(act_type, RowsArgs{x, add, sum, weight, q, scale, x_stride, add_stride, sum_stride, q_stride, n_cols, eps}, n_rows, stream);
}

int rf_swiglu_i8(const void* gate, const void* up, int act_type, uint32_t n_rows, uint32_t n_cols, uint64_t gate_stride,
                 uint64_t up_stride, int8_t* q, uint64_t q_stride, float* scale, void* stream) {
  RF_TRY(check_shape(act_type, n_rows, n_cols));
  if (n_rows && (!gate || !up || !q || !scale)) return set_error(RF_EINVAL, "null gate, up, codes or scales");
  for (uint64_t* s : {&gate_stride, &up_stride, &q_stride}) RF_TRY(check_stride(s, n_cols));
  for (const void* p : {gate, up}) RF_TRY(check_rows_ptr(p, act_bytes(act_type)));
  RF_TRY(check_scale(scale));
  if (!n_rows) return RF_OK;
  return run_rows<kSwiglu>(act_type, RowsArgs{gate, up, nullptr, nullptr, q, scale, gate_stride, up_stride, 0, q_stride, n_cols, 0.f}, n_rows, stream);
}

int rf_quantize_i8(const void* x, int act_type, uint32_t n_rows, uint32_t n_cols, uint64_t x_stride, int8_t* q,
                   uint64_t q_stride, float* scale, void* stream) {
  RF_TRY(check_shape(act_type, n_rows, n_cols));
  if (n_rows && (!x || !q || !scale)) return set_error(RF_EINVAL, "null rows, codes or scales");
  for (uint64_t* s : {&x_stride, &q_stride}) RF_TRY(check_stride(s, n_cols));
  RF_TRY(check_rows_ptr(x, act_bytes(act_type)));
  RF_TRY(check_scale(scale));
  if (!n_rows) return RF_OK;
  return run_rows<kPlain>(act_type, RowsArgs{x, nullptr, nullptr, nullptr, q, scale, x_stride, 0, 0, q_stride, n_cols, 0.f}, n_rows, stream);
}

int rf_dequantize_i8(const int8_t* q, const float* scale, void* out, int act_type, uint32_t n_rows, uint32_t n_cols,
                     uint64_t q_stride, uint64_t out_stride, void* stream) {
  RF_TRY(check_shape(act_type, n_rows, n_cols));
  if (n_rows && (!out || !q || !scale)) return set_error(RF_EINVAL, "null values, codes or scales");
  for (uint64_t* s : {&q_stride, &out_stride}) RF_TRY(check_stride(s, n_cols));
  RF_TRY(check_rows_ptr(out, act_bytes(act_type)));
  RF_TRY(check_scale(scale));
  if (!n_rows) return RF_OK;
  const ValuesArgs a{q, scale, out, q_stride, out_stride, 0, n_cols, 0, false};
  const Launch L{(cudaStream_t)stream, true};
  switch (act_type) {
    case RF_ACT_F32: RF_CUDA(launch_values<float>(L, a, n_rows)); break;
    case RF_ACT_F16: RF_CUDA(launch_values<__half>(L, a, n_rows)); break;
    default: RF_CUDA(launch_values<__nv_bfloat16>(L, a, n_rows));
  }
  return RF_OK;
}

}  // extern "C"
