// rf_i8_matmul.cu - Y = X W^T in 8-bit integers with a scale for each token (row of X) and channel (row of W).
//
// The sums are whole 32-bit numbers and exact, so any split of the work gives the same bits:
//   y[t][n] = f32(f32(f32(sum) * x_scale[t]) * w_scale[n]) + bias[n], rounded to the output's type.
#include <algorithm>

#include "rf_act.cuh"
#include "rf_device.cuh"
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

// The simplest form: a CTA has 64 tokens x 64 channels, a thread 4 x 4 of them, 64 elements of both a step.
template <class T>
__global__ void __launch_bounds__(256) i8_tile_kernel(MatmulArgs a) {
  __shared__ uint32_t xs[64][17], ws[64][17];
  griddep_launch();
  griddep_wait();
  const uint32_t tid = threadIdx.x, t0 = blockIdx.y * 64, n0 = blockIdx.x * 64, tx = tid & 15, ty = tid >> 4;
  int acc[4][4] = {};
  for (uint32_t k0 = 0; k0 < a.n_in; k0 += 64) {
    const uint32_t r = tid >> 2, c = (tid & 3) * 16;
    auto fetch = [&](uint32_t (*s)[17], const int8_t* base, uint64_t stride, uint32_t row, uint32_t rows) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (row < rows && k0 + c < a.n_in) {
        u = *reinterpret_cast<const uint4*>(base + row * stride + k0 + c);  // rows end in whole 16-byte pieces
        uint32_t* w = &u.x;
        for (uint32_t j = 0; j < 16; j++)
          if (k0 + c + j >= a.n_in) w[j / 4] &= ~(0xffu << (8 * (j & 3)));
      }
      s[r][c / 4] = u.x, s[r][c / 4 + 1] = u.y, s[r][c / 4 + 2] = u.z, s[r][c / 4 + 3] = u.w;
    };
    fetch(xs, a.x, a.x_stride, t0 + r, a.n_tokens);
    fetch(ws, a.w, a.w_stride, n0 + r, a.n_out);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; k++) {
      int xv[4], wv[4];
#pragma unroll
      for (int i = 0; i < 4; i++) xv[i] = (int)xs[ty + 16 * i][k], wv[i] = (int)ws[tx + 16 * i][k];
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = __dp4a(xv[i], wv[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t t = t0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (t >= a.n_tokens || n >= a.n_out) continue;
      float v = __fmul_rn(__fmul_rn((float)acc[i][j], a.x_scale[t]), a.w_scale[n]);
      if (a.bias) v = __fadd_rn(v, a.bias[n]);
      Act<T>::put((T*)a.y + t * a.y_stride + n, v);
    }
}

template <class T>
cudaError_t launch(const Launch& L, const MatmulArgs& a) {
  return launch_k(L, i8_tile_kernel<T>, dim3((a.n_out + 63) / 64, (a.n_tokens + 63) / 64), dim3(256), 0, a);
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
  const Launch L{(cudaStream_t)stream, true};
  switch (act_type) {
    case RF_ACT_F32: RF_CUDA(launch<float>(L, a)); break;
    case RF_ACT_F16: RF_CUDA(launch<__half>(L, a)); break;
    default: RF_CUDA(launch<__nv_bfloat16>(L, a));
  }
  return RF_OK;
}

}  // extern "C"
