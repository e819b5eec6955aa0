// rf_i8.cu - rows of 8-bit codes with one scale a row: the residual's addition with RMS norm, SwiGLU and plain
// rows into the format, and the rows back.  The product of such rows with an 8-bit matrix is in rf_i8_matmul.cu.
//
// The format (rfcuda.h) fixes every rounding from the row's f32 numbers to its codes, and the norm's are fixed up to
// the sum of squares, which is taken in 64 bits: its order does not show in the 32-bit reciprocal root, so a row's
// codes do not depend on how the row was split over threads.
//
// One read and one write of each element, a handful of operations between: HBM bounds the long calls, latency of
// launch, loads and one reduction the short ones.  A CTA has a row and keeps it in registers; maximum and sum of
// squares need one reduction together, since rounding is monotonic: max |f32(f32(s w) r)| = f32(max |f32(s w)| r).
//
// Launched to begin while the kernel before ends, as rf_verify.cu's are; what that one may write is read by plain loads.
#include <algorithm>

#include "rf_act.cuh"
#include "rf_device.cuh"
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

// Elements i .. i + 7 of a row (those below n; zeros behind), in 16-byte pieces where VEC.
template <class T, bool VEC>
__device__ __forceinline__ void load8(const T* row, uint32_t i, uint32_t n, float (&v)[8]) {
  if (VEC && i + 8 <= n) {
    constexpr int V = Act<T>::kVec;
    uint4 u[8 / V];
#pragma unroll
    for (int j = 0; j < 8 / V; j++) u[j] = ld_once(row + i + j * V);
#pragma unroll
    for (int j = 0; j < 8 / V; j++) {
      float f[V];
      Act<T>::unpack(u[j], f);
#pragma unroll
      for (int k = 0; k < V; k++) v[j * V + k] = f[k];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = i + j < n ? Act<T>::get(row + i + j) : 0.f;
  }
}
template <class T, bool VEC>
__device__ __forceinline__ void store8(T* row, uint32_t i, uint32_t n, const float (&v)[8]) {
  if (VEC && i + 8 <= n) {
    constexpr int V = Act<T>::kVec;
#pragma unroll
    for (int j = 0; j < 8 / V; j++) {
      float f[V];
#pragma unroll
      for (int k = 0; k < V; k++) f[k] = v[j * V + k];
      *reinterpret_cast<uint4*>(row + i + j * V) = Act<T>::pack(f);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (i + j < n) Act<T>::put(row + i + j, v[j]);
  }
}

// Low byte: the code.  Adding 1.5 * 2^23 rounds to the nearest whole number, ties to even.
__device__ __forceinline__ uint32_t code_bits(float y, float inv) {
  return __float_as_uint(__fadd_rn(fminf(fmaxf(__fmul_rn(y, inv), -127.f), 127.f), 12582912.f));
}

// A CTA takes one row: thread x the eights x, x + blockDim.x, ... (PER of them).
template <class T, int MODE, int PER, bool VEC>
__global__ void __launch_bounds__(1024) rows_i8_kernel(RowsArgs a) {
  __shared__ double s_ss[32];
  __shared__ uint32_t s_top[32];
  griddep_launch();
  griddep_wait();
  const uint32_t n = a.n_cols, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint64_t row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.x_stride;
  const T* y = (const T*)a.y + row * a.y_stride;
  float v[PER][8];
#pragma unroll
  for (int p = 0; p < PER; p++) load8<T, VEC>(x, (tid + p * blockDim.x) * 8, n, v[p]);
  if (MODE == kSwiglu || (MODE == kNorm && a.y)) {
    float u[PER][8];
#pragma unroll
    for (int p = 0; p < PER; p++) load8<T, VEC>(y, (tid + p * blockDim.x) * 8, n, u[p]);
#pragma unroll
    for (int p = 0; p < PER; p++)
#pragma unroll
      for (int j = 0; j < 8; j++)
        if constexpr (MODE == kSwiglu) {
          // exponential and quotient to a few units of the 24th bit: a code holds 8, and the few that lie that near
          // to a border go to either side
          v[p][j] = __fdividef(v[p][j], 1.f + __expf(-v[p][j])) * u[p][j];
        } else {
          v[p][j] = __fadd_rn(v[p][j], u[p][j]);
        }
  }
  double ss = 0;
  uint32_t top = 0;  // bits of the largest magnitude: a NaN's are above every number's
  if constexpr (MODE == kNorm) {
    if (a.sum) {
      T* sum = (T*)a.sum + row * a.sum_stride;
#pragma unroll
      for (int p = 0; p < PER; p++) store8<T, VEC>(sum, (tid + p * blockDim.x) * 8, n, v[p]);
    }
#pragma unroll
    for (int p = 0; p < PER; p++) {
#pragma unroll
      for (int j = 0; j < 8; j++) ss = fma((double)v[p][j], (double)v[p][j], ss);
      if (a.w) {
        float w[8];
        load8<float, VEC>(a.w, (tid + p * blockDim.x) * 8, n, w);
#pragma unroll
        for (int j = 0; j < 8; j++) v[p][j] = __fmul_rn(v[p][j], w[j]);
      }
    }
  }
#pragma unroll
  for (int p = 0; p < PER; p++)
#pragma unroll
    for (int j = 0; j < 8; j++) top = max(top, __float_as_uint(v[p][j]) & 0x7fffffffu);
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (MODE == kNorm)
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (lane == 0) s_top[warp] = top, s_ss[warp] = ss;
  __syncthreads();
  const bool in = lane < (blockDim.x >> 5);
  top = __reduce_max_sync(0xffffffffu, in ? s_top[lane] : 0u);
  float r = 1.f;
  if constexpr (MODE == kNorm) {
    ss = in ? s_ss[lane] : 0.0;
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    r = (float)(1.0 / sqrt(ss / (double)n + (double)a.eps));
  }
  // a sum that is not finite makes r 0 or NaN, and 0 times the infinity behind it a NaN
  const float most = MODE == kNorm ? __fmul_rn(__uint_as_float(top), r) : __uint_as_float(top);
  const bool wild = !(fabsf(most) < INFINITY);
  float scale = __fdiv_rn(most, 127.f);
  if (scale < 1.17549435e-38f) scale = 0.f;
  const float inv = wild || scale == 0.f ? 0.f : __fdiv_rn(1.f, scale);
  if (tid == 0) a.scale[row] = wild ? __uint_as_float(0x7fffffffu) : scale;
  int8_t* q = a.q + row * a.q_stride;
#pragma unroll
  for (int p = 0; p < PER; p++) {
    const uint32_t i = (tid + p * blockDim.x) * 8;
    uint32_t c[8];
#pragma unroll
    for (int j = 0; j < 8; j++) c[j] = wild ? 0u : code_bits(MODE == kNorm ? __fmul_rn(v[p][j], r) : v[p][j], inv);
    if (VEC && i + 8 <= n) {
      uint32_t b[2];
#pragma unroll
      for (int h = 0; h < 2; h++)
        b[h] = __byte_perm(__byte_perm(c[4 * h], c[4 * h + 1], 0x0040), __byte_perm(c[4 * h + 2], c[4 * h + 3], 0x0040), 0x5410);
      *reinterpret_cast<uint2*>(q + i) = make_uint2(b[0], b[1]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (i + j < n) q[i + j] = (int8_t)c[j];
    }
  }
}

template <class T, int MODE, bool VEC>
cudaError_t launch_rows_as(const Launch& L, const RowsArgs& a, uint32_t n_rows) {
  const uint32_t eights = (a.n_cols + 7) / 8;
  // 16 elements a thread, more where 1024 threads do not suffice
  const uint32_t per = eights <= 2048 ? 2 : eights <= 4096 ? 4 : 8;
  const uint32_t threads = std::max(32u, ((eights + per - 1) / per + 31) / 32 * 32);
  auto* k = per == 2 ? rows_i8_kernel<T, MODE, 2, VEC> : per == 4 ? rows_i8_kernel<T, MODE, 4, VEC> : rows_i8_kernel<T, MODE, 8, VEC>;
  return launch_k(L, k, dim3(n_rows), dim3(threads), 0, a);
}

template <class T, int MODE>
cudaError_t launch_rows(const Launch& L, const RowsArgs& a, uint32_t n_rows, bool vec) {
  return vec ? launch_rows_as<T, MODE, true>(L, a, n_rows) : launch_rows_as<T, MODE, false>(L, a, n_rows);
}

template <int MODE>
int run_rows(int act_type, const RowsArgs& a, uint32_t n_rows, void* stream) {
  const uint32_t es = act_bytes(act_type);
  bool vec = aligned_to(a.q, 8) && a.q_stride % 8 == 0;
  for (const void* p : {a.x, a.y, (const void*)a.sum, (const void*)a.w}) vec = vec && aligned_to(p, 16);
  for (uint64_t s : {a.x_stride, a.y_stride, a.sum_stride}) vec = vec && s * es % 16 == 0;
  const Launch L{(cudaStream_t)stream, true};
  switch (act_type) {
    case RF_ACT_F32: RF_CUDA((launch_rows<float, MODE>(L, a, n_rows, vec))); break;
    case RF_ACT_F16: RF_CUDA((launch_rows<__half, MODE>(L, a, n_rows, vec))); break;
    default: RF_CUDA((launch_rows<__nv_bfloat16, MODE>(L, a, n_rows, vec)));
  }
  return RF_OK;
}

// ---- rows back -----------------------------------------------------------------------
struct ValuesArgs {
  const int8_t* q;
  const float* scale;
  void* out;
  uint64_t q_stride, out_stride, pieces;  // pieces: eights of all rows
  uint32_t n_cols, per_row;
};

template <class T, bool VEC>
__global__ void __launch_bounds__(256) values_i8_kernel(ValuesArgs a) {
  griddep_launch();
  griddep_wait();
  for (uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x; at < a.pieces; at += (uint64_t)gridDim.x * 256) {
    const uint64_t row = at / a.per_row;
    const uint32_t i = (uint32_t)(at - row * a.per_row) * 8, n = a.n_cols;
    const int8_t* q = a.q + row * a.q_stride + i;
    const float scale = a.scale[row];
    float v[8];
    if (VEC && i + 8 <= n) {
      const uint2 u = *reinterpret_cast<const uint2*>(q);
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = (float)(int8_t)((j < 4 ? u.x : u.y) >> (8 * (j & 3)));
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = i + j < n ? (float)q[j] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = __fmul_rn(v[j], scale);
    store8<T, VEC>((T*)a.out + row * a.out_stride, i, n, v);
  }
}

template <class T>
cudaError_t launch_values(const Launch& L, const ValuesArgs& a) {
  const bool vec = aligned_to(a.q, 8) && a.q_stride % 8 == 0 && aligned_to(a.out, 16) && a.out_stride * sizeof(T) % 16 == 0;
  const uint64_t ctas = std::min<uint64_t>((a.pieces + 255) / 256, (uint64_t)num_sms() * 64);
  return launch_k(L, vec ? values_i8_kernel<T, true> : values_i8_kernel<T, false>, dim3((uint32_t)ctas), dim3(256), 0, a);
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
  const uint32_t per_row = (n_cols + 7) / 8;
  const ValuesArgs a{q, scale, out, q_stride, out_stride, (uint64_t)per_row * n_rows, n_cols, per_row};
  const Launch L{(cudaStream_t)stream, true};
  switch (act_type) {
    case RF_ACT_F32: RF_CUDA(launch_values<float>(L, a)); break;
    case RF_ACT_F16: RF_CUDA(launch_values<__half>(L, a)); break;
    default: RF_CUDA(launch_values<__nv_bfloat16>(L, a));
  }
  return RF_OK;
}

}  // extern "C"
