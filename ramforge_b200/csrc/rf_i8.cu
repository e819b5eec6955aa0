// rf_i8.cu - rows of 8-bit codes with one scale a row: the residual's addition with RMS norm, SwiGLU and plain
// rows into the format, and the rows back.  The product of such rows with an 8-bit matrix is in rf_i8_matmul.cu.
//
// The format (rfcuda.h) fixes every rounding from the row's f32 numbers to its codes, and the norm's are fixed up to
// the sum of squares, which is taken in 64 bits: its order does not show in the 32-bit reciprocal root, so a row's
// codes do not depend on how the row was split over threads.
//
// One read and one write of each element, a handful of operations between: HBM bounds the long calls, latency of
// launch, loads and one reduction the short ones.  Maximum and sum of squares need one reduction together, since
// rounding is monotonic: max |f32(f32(s w) r)| = f32(max |f32(s w)| r).
//
// Launched to begin while the kernel before ends, as rf_verify.cu's are; what that one may write is read by plain loads.
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
  s.r = MODE == kNorm ? (float)(1.0 / sqrt(ss / (double)n + (double)eps)) : 1.f;
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
__device__ __forceinline__ void store_codes8(int8_t* q, const float (&v)[8], const RowScale& s) {
  uint32_t c[8], b[2];
  codes8<MODE>(v, s, c);
#pragma unroll
  for (int h = 0; h < 2; h++)
    b[h] = __byte_perm(__byte_perm(c[4 * h], c[4 * h + 1], 0x0040), __byte_perm(c[4 * h + 2], c[4 * h + 3], 0x0040), 0x5410);
  *reinterpret_cast<uint2*>(q) = s.wild ? make_uint2(0, 0) : make_uint2(b[0], b[1]);
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
// reduced and coded; 16 elements a thread, the norm's weights in registers.  4001 x 4096 bf16 with residual and sum: 24.7 us (4.65
// TB/s), with a CTA a row 35.6; SwiGLU of 2048 x 14336: 32.9 and 52.6, there with one CTA of 896 threads an SM.
constexpr int kRowStages = 3;

template <class T, int MODE>
__global__ void __launch_bounds__(1024) rows_ring_kernel(RowsArgs a, uint32_t n_rows, unsigned* err) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint64_t full[kRowStages];
  __shared__ double s_ss[2][32];
  __shared__ uint32_t s_top[2][32], s_stop;
  const uint32_t n = a.n_cols, tid = threadIdx.x, nt = blockDim.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t bytes = n * sizeof(T), stage = (a.y ? 2 : 1) * bytes;
  constexpr int V = Act<T>::kVec, W = 8 / V;
  if (tid == 0) {
    for (int i = 0; i < kRowStages; i++) tc_mbar_init(tc_smem_u32(full + i), 1);
    tc_fence_barrier_init();
    s_stop = 0;
  }
  griddep_launch();
  griddep_wait();
  __syncthreads();
  auto fetch = [&](uint64_t row, uint32_t slot) {
    const uint32_t bar = tc_smem_u32(full + slot), dst = tc_smem_u32(ring) + slot * stage;
    tc_mbar_expect_tx(bar, stage);
    tc_bulk_copy_g2s(dst, (const T*)a.x + row * a.x_stride, bytes, bar);
    if (a.y) tc_bulk_copy_g2s(dst + bytes, (const T*)a.y + row * a.y_stride, bytes, bar);
  };
  if (tid == 0)
    for (int i = 0; i < kRowStages; i++)
      if (blockIdx.x + (uint64_t)i * gridDim.x < n_rows) fetch(blockIdx.x + (uint64_t)i * gridDim.x, i);
  const uint32_t at[2] = {tid * 8, (tid + nt) * 8};
  float w[2][8];
  if (MODE == kNorm) {
#pragma unroll
    for (int p = 0; p < 2; p++)
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        float4 f = make_float4(1.f, 1.f, 1.f, 1.f);
        if (a.w && at[p] < n) f = __ldg(reinterpret_cast<const float4*>(a.w + at[p] + j));
        w[p][j] = f.x, w[p][j + 1] = f.y, w[p][j + 2] = f.z, w[p][j + 3] = f.w;
      }
  }
  uint32_t slot = 0, phase = 0, turn = 0;
  for (uint64_t row = blockIdx.x; row < n_rows; row += gridDim.x) {
    const bool ok = wait_bar(full + slot, phase, &s_stop, err);
    float v[2][8], most = 0.f;
    Squares sq;
#pragma unroll
    for (int p = 0; p < 2; p++) {
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
    __syncthreads();  // all have read the slot, too
    if (tid == 0 && ok && row + (uint64_t)kRowStages * gridDim.x < n_rows) fetch(row + (uint64_t)kRowStages * gridDim.x, slot);
    __syncwarp();
    const bool in = lane < (nt >> 5);
    top = __reduce_max_sync(0xffffffffu, in ? s_top[turn][lane] : 0u);
    if constexpr (MODE == kNorm) ss = warp_sum(in ? s_ss[turn][lane] : 0.0);
    const RowScale s = row_scale<MODE>(top, ss, n, a.eps);
    if (ok) {
      if (tid == 0) a.scale[row] = s.scale;
#pragma unroll
      for (int p = 0; p < 2; p++)
        if (at[p] < n) store_codes8<MODE>(a.q + row * a.q_stride + at[p], v[p], s);
    }
    turn ^= 1;
    if (++slot == kRowStages) slot = 0, phase ^= 1;
  }
  if (*(volatile uint32_t*)&s_stop) {  // gave up: copies in flight end within this time
    const long long t = clock64();
    while (clock64() - t < 4000000LL) {
    }
  }
}

// ---- many short rows: a warp a row ---------------------------------------------------
// PER eights a lane, or, where rows are not aligned, every 32nd element; the next row's are asked for before a row is worked on.
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
                const float4 f = __ldg(reinterpret_cast<const float4*>(a.w + place(p, j)));
                v[p][j] = __fmul_rn(v[p][j], f.x), v[p][j + 1] = __fmul_rn(v[p][j + 1], f.y);
                v[p][j + 2] = __fmul_rn(v[p][j + 2], f.z), v[p][j + 3] = __fmul_rn(v[p][j + 3], f.w);
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
              if (place(p, j) < n) v[p][j] = __fmul_rn(v[p][j], __ldg(a.w + place(p, j)));
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
  // 16 elements a thread, more where 1024 threads do not suffice
  const uint32_t per = eights <= 2048 ? 2 : eights <= 4096 ? 4 : 8;
  const uint32_t threads = std::max(32u, ((eights + per - 1) / per + 31) / 32 * 32);
  auto* k = per == 2 ? rows_cta_kernel<T, MODE, 2, VEC> : per == 4 ? rows_cta_kernel<T, MODE, 4, VEC> : rows_cta_kernel<T, MODE, 8, VEC>;
  return launch_k(L, k, dim3(n_rows), dim3(threads), 0, a);
}

template <class T, int MODE, bool VEC>
cudaError_t launch_rows_as(const Launch& L, const RowsArgs& a, uint32_t n_rows, unsigned* err) {
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
  if constexpr (VEC) {
    const uint32_t threads = ((eights + 1) / 2 + 31) / 32 * 32, smem = kRowStages * (a.y ? 2 : 1) * a.n_cols * (uint32_t)sizeof(T);
    const uint32_t per_sm = std::min(std::min(1024 / threads, 220u * 1024 / smem), 8u);
    if (threads <= 1024 && per_sm && n_rows > 2 * sms * per_sm) {
      auto* k = rows_ring_kernel<T, MODE>;
      cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
      if (e != cudaSuccess) return e;
      return launch_k(L, k, dim3(sms * per_sm), dim3(threads), smem, a, n_rows, err);
    }
  }
  return launch_cta<T, MODE, VEC>(L, a, n_rows);
}
template <class T, int MODE>
cudaError_t launch_rows(const Launch& L, const RowsArgs& a, uint32_t n_rows, bool vec, unsigned* err) {
  return vec ? launch_rows_as<T, MODE, true>(L, a, n_rows, err) : launch_rows_as<T, MODE, false>(L, a, n_rows, err);
}

template <int MODE>
int run_rows(int act_type, const RowsArgs& a, uint32_t n_rows, void* stream) {
  const uint32_t es = act_bytes(act_type);
  bool vec = aligned_to(a.q, 8) && a.q_stride % 8 == 0 && a.n_cols % 8 == 0;
  for (const void* p : {a.x, a.y, (const void*)a.sum, (const void*)a.w}) vec = vec && aligned_to(p, 16);
  for (uint64_t s : {a.x_stride, a.y_stride, a.sum_stride}) vec = vec && s * es % 16 == 0;
  const Launch L{(cudaStream_t)stream, true};
  unsigned* err = nullptr;
  RF_TRY(verify_error_ptr(&err));
  switch (act_type) {
    case RF_ACT_F32: RF_CUDA((launch_rows<float, MODE>(L, a, n_rows, vec, err))); break;
    case RF_ACT_F16: RF_CUDA((launch_rows<__half, MODE>(L, a, n_rows, vec, err))); break;
    default: RF_CUDA((launch_rows<__nv_bfloat16, MODE>(L, a, n_rows, vec, err)));
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
      // a byte under the exponent of 2^23 is 2^23 + 128 + code, the sum with the bias's negative exact
      const uint32_t w[2] = {u[i].x ^ 0x80808080u, u[i].y ^ 0x80808080u};
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const uint32_t x = w[j / 4];
        const float2 code = pair_add(make_float2(__uint_as_float(__byte_perm(x, 0x4b000000u, 0x7440 + (j & 3))),
                                                 __uint_as_float(__byte_perm(x, 0x4b000000u, 0x7440 + (j & 3) + 1))),
                                     make_float2(-8388736.f, -8388736.f));
        const float2 y = pair_mul(code, make_float2(scale[i], scale[i]));
        v[j] = y.x, v[j + 1] = y.y;
      }
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
  const bool vec = aligned_to(a.q, 8) && a.q_stride % 8 == 0 && a.n_cols % 8 == 0 && aligned_to(a.out, 16) && a.out_stride * sizeof(T) % 16 == 0;
  const uint32_t unit = vec ? 8 : 256, per_cta = vec ? 256 : 8;
  a.wide = aligned_to(a.out, 32) && a.out_stride * sizeof(T) % 32 == 0;
  a.per_row = (a.n_cols + unit - 1) / unit;
  a.pieces = (uint64_t)a.per_row * n_rows;
  const uint64_t ctas = std::min<uint64_t>((a.pieces + per_cta - 1) / per_cta, (uint64_t)num_sms() * 8);
  return launch_k(L, vec ? values_i8_kernel<T> : values_any_kernel<T>, dim3((uint32_t)ctas), dim3(256), 0, a);
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
