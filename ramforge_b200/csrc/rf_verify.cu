// rf_verify.cu - the operators around the attention of drafted tokens: per-head
// norm and rotation of queries and keys, and the 8-bit (or f16) cache they write
// and read.  The attention itself is in rf_tree.cu.
//
// All three only move data: a few operations per element, each element read once
// and written once, so HBM bounds the long calls and launch latency the short ones.
#include <cuda_bf16.h>

#include "rf_device.cuh"
#include "rf_verify.h"

namespace rf {

static __device__ unsigned g_verify_err;

int verify_error_ptr(unsigned** out) {
  void* p = nullptr;
  cudaError_t ce = cudaGetSymbolAddress(&p, g_verify_err);
  if (ce != cudaSuccess || !p)
    return set_error(RF_ECUDA, "cudaGetSymbolAddress(verification error word) failed: %s", cudaGetErrorString(ce));
  *out = (unsigned*)p;
  return RF_OK;
}

int check_kv_view(const rf_kv_view* c) {
  if (!c || !c->k || !c->v) return set_error(RF_EINVAL, "null K/V cache");
  if (c->type != RF_TYPE_F16 && c->type != RF_TYPE_Q8_0)
    return set_error(RF_EUNSUPPORTED, "K/V cache type %d is neither F16 nor Q8_0", c->type);
  if (!c->n_seqs || !c->n_kv_heads || !c->capacity) return set_error(RF_EINVAL, "empty K/V cache");
  if (!c->head_dim || c->head_dim % 32 || c->head_dim > 256)
    return set_error(RF_EINVAL, "cache head_dim %u is not a multiple of 32 up to 256", c->head_dim);
  if (c->n_kv_heads > 65535 || c->n_seqs > 65535 || c->capacity > 0x7fffffffu)
    return set_error(RF_EINVAL, "K/V cache of %u sequences x %u heads x %u positions is out of range", c->n_seqs,
                     c->n_kv_heads, c->capacity);
  if (c->type == RF_TYPE_Q8_0 && (!c->k_scale || !c->v_scale))
    return set_error(RF_EINVAL, "a Q8_0 cache needs its scale planes");
  if (!aligned_to(c->k, 16) || !aligned_to(c->v, 16) ||
      (c->type == RF_TYPE_Q8_0 && (!aligned_to(c->k_scale, 16) || !aligned_to(c->v_scale, 16))))
    return set_error(RF_EINVAL, "K/V cache planes must be 16-byte aligned");
  return RF_OK;
}

namespace {

// ---- activations: N consecutive elements as f32, in 16-byte pieces ------------------
template <class T>
struct Act;
template <>
struct Act<float> {
  static constexpr int kVec = 4;
  static __device__ float get(const float* p) { return *p; }
  static __device__ void put(float* p, float v) { *p = v; }
  static __device__ void unpack(const uint4& u, float (&v)[4]) {
    v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
  }
  static __device__ uint4 pack(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};
template <>
struct Act<__half> {
  static constexpr int kVec = 8;
  static __device__ float get(const __half* p) { return __half2float(*p); }
  static __device__ void put(__half* p, float v) { *p = __float2half_rn(v); }
  static __device__ void unpack(const uint4& u, float (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  }
  static __device__ uint4 pack(const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Act<__nv_bfloat16> {
  static constexpr int kVec = 8;
  static __device__ float get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
  static __device__ void unpack(const uint4& u, float (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  static __device__ uint4 pack(const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// ---------------------------------------------------------------------------
// Per-head norm and rotation.
// ---------------------------------------------------------------------------
struct NormRopeArgs {
  const void *q, *k;
  void *q_out, *k_out;
  uint64_t q_stride, k_stride, q_out_stride, k_out_stride;  // elements between tokens
  const float *q_norm, *k_norm;
  const float2* rope;
  const int32_t* pos;
  uint32_t n_tokens, n_heads, n_kv_heads, head_dim, rope_len, rot_dim;
  float eps;
  unsigned* err;
};

// The rotation's table row of token t, or false (and the error bit) where its position is out of range.
__device__ __forceinline__ bool rope_row(const NormRopeArgs& a, uint32_t t, const float2** row) {
  *row = nullptr;
  if (a.rot_dim == 0) return true;
  const int32_t p = a.pos[t];
  if (p < 0 || (uint32_t)p >= a.rope_len) {
    atomicOr(a.err, kVerifyRange);
    return false;
  }
  *row = a.rope + (size_t)p * (a.rot_dim / 2);
  return true;
}

// Any even head_dim, stride and alignment: one warp a head, one element a lane and step.
template <class T>
__global__ void __launch_bounds__(256) norm_rope_any_kernel(NormRopeArgs a) {
  const uint32_t heads = a.n_heads + a.n_kv_heads, lane = threadIdx.x & 31;
  const uint32_t w = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (w >= a.n_tokens * heads) return;
  const uint32_t t = w / heads, hh = w % heads, D = a.head_dim, half = a.rot_dim / 2;
  const bool is_q = hh < a.n_heads;
  const uint32_t h = is_q ? hh : hh - a.n_heads;
  const T* x = (const T*)(is_q ? a.q : a.k) + t * (is_q ? a.q_stride : a.k_stride) + (size_t)h * D;
  T* y = (T*)(is_q ? a.q_out : a.k_out) + t * (is_q ? a.q_out_stride : a.k_out_stride) + (size_t)h * D;
  const float* nw = is_q ? a.q_norm : a.k_norm;
  const float2* cs;
  if (!rope_row(a, t, &cs)) return;
  float v[8], pv[8];  // the lane's elements and their rotation partners
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const uint32_t i = lane + 32 * j;
    if (i >= D) break;
    v[j] = Act<T>::get(x + i);
    pv[j] = i < 2 * half ? Act<T>::get(x + (i < half ? i + half : i - half)) : 0.f;
    ss = fmaf(v[j], v[j], ss);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  __syncwarp();  // in place: every lane's loads before any lane's stores
  const float r = nw ? 1.f / sqrtf(ss / (float)D + a.eps) : 1.f;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const uint32_t i = lane + 32 * j;
    if (i >= D) break;
    float o = nw ? v[j] * r * nw[i] : v[j];
    if (i < 2 * half) {
      const uint32_t pi = i < half ? i + half : i - half;
      const float p = nw ? pv[j] * r * nw[pi] : pv[j];
      const float2 c = cs[i < half ? i : pi];
      o = i < half ? o * c.x - p * c.y : p * c.y + o * c.x;
    }
    Act<T>::put(y + i, o);
  }
}

// Whole-head or no rotation, 16-byte aligned rows: lane x of a group of `lanes` holds the
// 16-byte piece x of the head's first half and of its second half, so each pair to rotate
// sits in one lane.  A group takes kHeads heads of one token together: their loads are all
// in flight at once, and the table row and the weights are read once for all of them.
constexpr int kHeads = 4;

template <class T>
__global__ void __launch_bounds__(256) norm_rope_vec_kernel(NormRopeArgs a, uint32_t lanes, uint32_t q_groups,
                                                            uint32_t groups) {
  constexpr int V = Act<T>::kVec;
  const uint32_t idx = blockIdx.x * 256 + threadIdx.x;
  uint32_t item = idx / lanes;
  const uint32_t x = idx % lanes, D = a.head_dim;
  bool live = item < a.n_tokens * groups;
  if (!live) item = 0;
  const uint32_t t = item / groups, gr = item % groups;
  const bool is_q = gr < q_groups;
  const uint32_t h0 = (is_q ? gr : gr - q_groups) * kHeads, heads = is_q ? a.n_heads : a.n_kv_heads;
  const T* src = (const T*)(is_q ? a.q : a.k) + t * (is_q ? a.q_stride : a.k_stride) + (size_t)h0 * D + x * V;
  T* dst = (T*)(is_q ? a.q_out : a.k_out) + t * (is_q ? a.q_out_stride : a.k_out_stride) + (size_t)h0 * D + x * V;
  const float* nw = is_q ? a.q_norm : a.k_norm;
  uint4 raw[kHeads][2];
#pragma unroll
  for (int i = 0; i < kHeads; i++)
    if (live && h0 + i < heads) {
      raw[i][0] = *reinterpret_cast<const uint4*>(src + i * D);
      raw[i][1] = *reinterpret_cast<const uint4*>(src + i * D + D / 2);
    } else {
      raw[i][0] = raw[i][1] = make_uint4(0, 0, 0, 0);
    }
  const float2* row;
  live = rope_row(a, t, &row) && live;
  float cs[V], sn[V], w[2][V];
#pragma unroll
  for (int j = 0; j < V; j += 2) {
    const float4 f = row && live ? __ldg(reinterpret_cast<const float4*>(row + x * V + j)) : make_float4(1.f, 0.f, 1.f, 0.f);
    cs[j] = f.x, sn[j] = f.y, cs[j + 1] = f.z, sn[j + 1] = f.w;
  }
#pragma unroll
  for (int s = 0; s < 2; s++)
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const float4 f = nw ? __ldg(reinterpret_cast<const float4*>(nw + s * (D / 2) + x * V + j)) : make_float4(1.f, 1.f, 1.f, 1.f);
      w[s][j] = f.x, w[s][j + 1] = f.y, w[s][j + 2] = f.z, w[s][j + 3] = f.w;
    }
#pragma unroll
  for (int i = 0; i < kHeads; i++) {
    float v[2][V];
    Act<T>::unpack(raw[i][0], v[0]);
    Act<T>::unpack(raw[i][1], v[1]);
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < V; j++) ss = fmaf(v[0][j], v[0][j], fmaf(v[1][j], v[1][j], ss));
    for (uint32_t o = lanes / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = nw ? 1.f / sqrtf(ss / (float)D + a.eps) : 1.f;
    float y[2][V];
#pragma unroll
    for (int j = 0; j < V; j++) {
      const float p = v[0][j] * r * w[0][j], q = v[1][j] * r * w[1][j];
      y[0][j] = row ? p * cs[j] - q * sn[j] : p;
      y[1][j] = row ? p * sn[j] + q * cs[j] : q;
    }
    if (live && h0 + i < heads) {
      *reinterpret_cast<uint4*>(dst + i * D) = Act<T>::pack(y[0]);
      *reinterpret_cast<uint4*>(dst + i * D + D / 2) = Act<T>::pack(y[1]);
    }
  }
}

}  // namespace

// ---------------------------------------------------------------------------
// The cache.  A thread handles 16 elements of one head of one row, for K or for V:
// half a Q8_0 block, so a pair of neighbouring lanes shares a scale.
// ---------------------------------------------------------------------------
namespace {

struct KvRowsArgs {
  rf_kv_view c;
  const void *k, *v;  // write: sources; read: destinations (may be null)
  uint64_t k_stride, v_stride;
  const int32_t *seq, *pos;
  uint32_t n_rows;
  unsigned* err;
};

// Element offset of (seq, head, pos 0..) rows in a plane, or -1: not kept (pos < 0), -2: out of range.
__device__ __forceinline__ int64_t kv_row(const KvRowsArgs& a, uint32_t row, uint32_t h) {
  const int32_t p = a.pos[row], s = a.seq ? a.seq[row] : 0;
  if (p < 0) return -1;
  if ((uint32_t)p >= a.c.capacity || s < 0 || (uint32_t)s >= a.c.n_seqs) {
    atomicOr(a.err, kVerifyRange);
    return -2;
  }
  return ((int64_t)s * a.c.n_kv_heads + h) * a.c.capacity + p;
}

template <class T, bool Q8>
__global__ void __launch_bounds__(256) kv_write_kernel(KvRowsArgs a) {
  const uint32_t lph = a.c.head_dim / 16, per = a.c.n_kv_heads * lph;
  const uint32_t idx = blockIdx.x * 256 + threadIdx.x;
  const uint32_t total = 2 * a.n_rows * per;
  const bool in = idx < total;
  const uint32_t at = in ? idx : 0;
  const uint32_t rk = at / per, x = at % per, row = rk >> 1, h = x / lph, c16 = x % lph;
  const bool is_v = rk & 1;
  const int64_t slot = kv_row(a, row, h);
  const bool live = in && slot >= 0;
  constexpr int NV = 16 / Act<T>::kVec;
  float v[16];
  if (live) {
    const T* src = (const T*)(is_v ? a.v : a.k) + row * (is_v ? a.v_stride : a.k_stride) + (size_t)x * 16;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      float f[Act<T>::kVec];
      Act<T>::unpack(reinterpret_cast<const uint4*>(src)[i], f);
#pragma unroll
      for (int j = 0; j < Act<T>::kVec; j++) v[i * Act<T>::kVec + j] = f[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = 0.f;
  }
  if constexpr (!Q8) {
    if (!live) return;
    __half* dst = (__half*)(is_v ? a.c.v : a.c.k) + slot * a.c.head_dim + c16 * 16;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; j++) f[j] = v[8 * i + j];
      reinterpret_cast<uint4*>(dst)[i] = Act<__half>::pack(f);
    }
  } else {
    float amax = 0.f;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      nan |= v[i] != v[i];
      v[i] = fminf(fmaxf(v[i], -65472.f), 65472.f);
      amax = fmaxf(amax, fabsf(v[i]));
    }
    if (nan) amax = __int_as_float(0x7fffffff);
    const float other = __shfl_xor_sync(0xffffffffu, amax, 1);
    amax = amax != amax || other != other ? __int_as_float(0x7fffffff) : fmaxf(amax, other);
    // the scale is kept in f16 (GGUF's block): its 11 bits cost at most 2^-11 of a code step per code,
    // and codes are taken against the rounded scale
    const __half d = __float2half_rn(__fdiv_rn(amax, 127.f));
    const float df = __half2float(d), inv = df > 0.f ? __fdiv_rn(1.f, df) : 0.f;
    if (!live) return;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      w[i] = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int code = min(127, max(-127, __float2int_rn(__fmul_rn(v[4 * i + j], inv))));
        w[i] |= ((uint32_t)code & 0xffu) << (8 * j);
      }
    }
    *reinterpret_cast<uint4*>((int8_t*)(is_v ? a.c.v : a.c.k) + slot * a.c.head_dim + c16 * 16) =
        make_uint4(w[0], w[1], w[2], w[3]);
    if (!(c16 & 1)) ((__half*)(is_v ? a.c.v_scale : a.c.k_scale))[slot * (a.c.head_dim / 32) + c16 / 2] = d;
  }
}

template <class T, bool Q8>
__global__ void __launch_bounds__(256) kv_read_kernel(KvRowsArgs a) {
  const uint32_t lph = a.c.head_dim / 16, per = a.c.n_kv_heads * lph;
  const uint32_t idx = blockIdx.x * 256 + threadIdx.x;
  if (idx >= 2 * a.n_rows * per) return;
  const uint32_t rk = idx / per, x = idx % per, row = rk >> 1, h = x / lph, c16 = x % lph;
  const bool is_v = rk & 1;
  T* dst = (T*)(is_v ? a.v : a.k);
  if (!dst) return;
  dst += row * (is_v ? a.v_stride : a.k_stride) + (size_t)x * 16;
  const int64_t slot = kv_row(a, row, h);
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; i++) v[i] = 0.f;
  if (slot >= 0) {
    if constexpr (Q8) {
      const uint4 u = *reinterpret_cast<const uint4*>((const int8_t*)(is_v ? a.c.v : a.c.k) + slot * a.c.head_dim + c16 * 16);
      const float d = __half2float(((const __half*)(is_v ? a.c.v_scale : a.c.k_scale))[slot * (a.c.head_dim / 32) + c16 / 2]);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 16; i++)  // code * scale is exact in f32 (8 x 11 bits), then one rounding to f16
        v[i] = __half2float(__float2half_rn((float)(int8_t)((w[i / 4] >> (8 * (i % 4))) & 0xffu) * d));
    } else {
      const uint4* p = reinterpret_cast<const uint4*>((const __half*)(is_v ? a.c.v : a.c.k) + slot * a.c.head_dim + c16 * 16);
#pragma unroll
      for (int i = 0; i < 2; i++) {
        float f[8];
        Act<__half>::unpack(p[i], f);
#pragma unroll
        for (int j = 0; j < 8; j++) v[8 * i + j] = f[j];
      }
    }
  }
  constexpr int NV = 16 / Act<T>::kVec;
#pragma unroll
  for (int i = 0; i < NV; i++) {
    float f[Act<T>::kVec];
#pragma unroll
    for (int j = 0; j < Act<T>::kVec; j++) f[j] = v[i * Act<T>::kVec + j];
    reinterpret_cast<uint4*>(dst)[i] = Act<T>::pack(f);
  }
}

int check_kv_rows(const rf_kv_view* c, const void* k, const void* v, int act_type, uint32_t n_rows, uint64_t* k_stride,
                  uint64_t* v_stride, const int32_t* pos) {
  RF_TRY(check_kv_view(c));
  const uint32_t es = act_bytes(act_type);
  if (!es) return set_error(RF_EINVAL, "activation type %d is not F32, F16 or BF16", act_type);
  if (n_rows && !pos) return set_error(RF_EINVAL, "null positions");
  const uint64_t row = (uint64_t)c->n_kv_heads * c->head_dim;
  for (uint64_t* s : {k_stride, v_stride}) {
    if (!*s) *s = row;
    if (*s < row) return set_error(RF_EINVAL, "row stride %llu is below the row's %llu elements", (unsigned long long)*s,
                                   (unsigned long long)row);
    if (*s * es % 16) return set_error(RF_EINVAL, "row stride %llu is not a multiple of 16 bytes", (unsigned long long)*s);
  }
  if (!aligned_to(k, 16) || !aligned_to(v, 16)) return set_error(RF_EINVAL, "K/V rows must be 16-byte aligned");
  if (2ull * n_rows * row / 16 > 0x7fffffffull) return set_error(RF_EINVAL, "%u rows are too many for one call", n_rows);
  return RF_OK;
}

template <class T>
cudaError_t launch_norm_rope(const Launch& L, const NormRopeArgs& a) {
  const uint32_t v = Act<T>::kVec, lanes = a.head_dim / 2 / v;
  bool vec = a.head_dim % (2 * v) == 0 && lanes <= 32 && !(lanes & (lanes - 1)) &&
             (a.rot_dim == 0 || a.rot_dim == a.head_dim);
  for (const void* p : {a.q, a.k, (const void*)a.q_out, (const void*)a.k_out, (const void*)a.q_norm, (const void*)a.k_norm,
                        (const void*)a.rope})
    vec = vec && aligned_to(p, 16);
  for (uint64_t s : {a.q_stride, a.k_stride, a.q_out_stride, a.k_out_stride}) vec = vec && s % v == 0;
  if (vec) {
    const uint32_t qg = (a.n_heads + kHeads - 1) / kHeads, groups = qg + (a.n_kv_heads + kHeads - 1) / kHeads;
    const uint32_t threads = a.n_tokens * groups * lanes;
    return launch_k(L, norm_rope_vec_kernel<T>, dim3((threads + 255) / 256), dim3(256), 0, a, lanes, qg, groups);
  }
  const uint32_t warps = a.n_tokens * (a.n_heads + a.n_kv_heads);
  return launch_k(L, norm_rope_any_kernel<T>, dim3((warps + 7) / 8), dim3(256), 0, a);
}

template <class T>
cudaError_t launch_kv_rows(const Launch& L, const KvRowsArgs& a, bool write) {
  const uint32_t threads = 2 * a.n_rows * (a.c.n_kv_heads * (a.c.head_dim / 16));
  const bool q8 = a.c.type == RF_TYPE_Q8_0;
  auto* k = write ? (q8 ? kv_write_kernel<T, true> : kv_write_kernel<T, false>)
                  : (q8 ? kv_read_kernel<T, true> : kv_read_kernel<T, false>);
  return launch_k(L, k, dim3((threads + 255) / 256), dim3(256), 0, a);
}

int run_kv_rows(const rf_kv_view* cache, const void* k, const void* v, int act_type, uint32_t n_rows, uint64_t k_stride,
                uint64_t v_stride, const int32_t* seq, const int32_t* pos, void* stream, bool write) {
  RF_TRY(check_kv_rows(cache, k, v, act_type, n_rows, &k_stride, &v_stride, pos));
  if (!n_rows) return RF_OK;
  KvRowsArgs a{};
  a.c = *cache;
  a.k = k, a.v = v;
  a.k_stride = k_stride, a.v_stride = v_stride;
  a.seq = seq, a.pos = pos;
  a.n_rows = n_rows;
  RF_TRY(verify_error_ptr(&a.err));
  const Launch L{(cudaStream_t)stream, false};
  switch (act_type) {
    case RF_ACT_F32: RF_CUDA(launch_kv_rows<float>(L, a, write)); break;
    case RF_ACT_F16: RF_CUDA(launch_kv_rows<__half>(L, a, write)); break;
    default: RF_CUDA(launch_kv_rows<__nv_bfloat16>(L, a, write));
  }
  return RF_OK;
}

}  // namespace
}  // namespace rf

using namespace rf;

extern "C" {

int rf_qk_norm_rope(const void* q, const void* k, void* q_out, void* k_out, int act_type, uint32_t n_tokens,
                    uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, uint64_t q_stride, uint64_t k_stride,
                    uint64_t q_out_stride, uint64_t k_out_stride, const float* q_norm, const float* k_norm, float eps,
                    const float* rope, uint32_t rope_len, uint32_t rot_dim, const int32_t* positions, void* stream) {
  const uint32_t es = act_bytes(act_type);
  if (!es) return set_error(RF_EINVAL, "activation type %d is not F32, F16 or BF16", act_type);
  if (!q || !q_out || n_heads == 0) return set_error(RF_EINVAL, "null queries");
  if ((!k || !k_out) && n_kv_heads) return set_error(RF_EINVAL, "null keys with %u KV heads", n_kv_heads);
  if (head_dim < 2 || head_dim % 2 || head_dim > 256)
    return set_error(RF_EINVAL, "head_dim %u is not an even number up to 256", head_dim);
  if (rot_dim % 2 || rot_dim > head_dim)
    return set_error(RF_EINVAL, "rot_dim %u is not an even number up to head_dim %u", rot_dim, head_dim);
  if (rot_dim && (!rope || !positions || !rope_len)) return set_error(RF_EINVAL, "null rotation table or positions");
  if (rot_dim && !aligned_to(rope, 8)) return set_error(RF_EINVAL, "the rotation table must be 8-byte aligned");
  if (!aligned_to(q, es) || !aligned_to(k, es) || !aligned_to(q_out, es) || !aligned_to(k_out, es))
    return set_error(RF_EINVAL, "queries and keys must be aligned to their element size");
  if (!(eps >= 0.f)) return set_error(RF_EINVAL, "eps must not be negative");
  if (n_heads > 65535 || n_kv_heads > 65535 || (uint64_t)n_tokens * (n_heads + n_kv_heads) > 0x7fffffffull / 32)
    return set_error(RF_EINVAL, "%u tokens of %u + %u heads are too many for one call", n_tokens, n_heads, n_kv_heads);
  const uint64_t qrow = (uint64_t)n_heads * head_dim, krow = (uint64_t)n_kv_heads * head_dim;
  if (!q_stride) q_stride = qrow;
  if (!q_out_stride) q_out_stride = qrow;
  if (!k_stride) k_stride = krow;
  if (!k_out_stride) k_out_stride = krow;
  if (q_stride < qrow || q_out_stride < qrow || k_stride < krow || k_out_stride < krow)
    return set_error(RF_EINVAL, "a token stride is below its row's elements");
  if (!n_tokens) return RF_OK;
  NormRopeArgs a{};
  a.q = q, a.k = k, a.q_out = q_out, a.k_out = k_out;
  a.q_stride = q_stride, a.k_stride = k_stride, a.q_out_stride = q_out_stride, a.k_out_stride = k_out_stride;
  a.q_norm = q_norm, a.k_norm = k_norm;
  a.rope = (const float2*)rope;
  a.pos = positions;
  a.n_tokens = n_tokens, a.n_heads = n_heads, a.n_kv_heads = n_kv_heads;
  a.head_dim = head_dim, a.rope_len = rope_len, a.rot_dim = rot_dim;
  a.eps = eps;
  RF_TRY(verify_error_ptr(&a.err));
  const Launch L{(cudaStream_t)stream, false};
  switch (act_type) {
    case RF_ACT_F32: RF_CUDA(launch_norm_rope<float>(L, a)); break;
    case RF_ACT_F16: RF_CUDA(launch_norm_rope<__half>(L, a)); break;
    default: RF_CUDA(launch_norm_rope<__nv_bfloat16>(L, a));
  }
  return RF_OK;
}

int rf_kv_cache_write(const rf_kv_view* cache, const void* k, const void* v, int act_type, uint32_t n_rows,
                      uint64_t k_stride, uint64_t v_stride, const int32_t* seq, const int32_t* pos, void* stream) {
  if (n_rows && (!k || !v)) return set_error(RF_EINVAL, "null K/V rows");
  return run_kv_rows(cache, k, v, act_type, n_rows, k_stride, v_stride, seq, pos, stream, true);
}

int rf_kv_cache_read(const rf_kv_view* cache, void* k_out, void* v_out, int act_type, uint32_t n_rows, uint64_t k_stride,
                     uint64_t v_stride, const int32_t* seq, const int32_t* pos, void* stream) {
  if (n_rows && !k_out && !v_out) return set_error(RF_EINVAL, "null destinations");
  return run_kv_rows(cache, k_out, v_out, act_type, n_rows, k_stride, v_stride, seq, pos, stream, false);
}

int rf_verify_error_word(uint32_t* word) {
  if (!word) return set_error(RF_EINVAL, "null argument");
  *word = 0;
  unsigned* err = nullptr;
  RF_TRY(verify_error_ptr(&err));
  RF_CUDA(cudaDeviceSynchronize());
  unsigned w = 0;
  RF_CUDA(cudaMemcpy(&w, err, sizeof w, cudaMemcpyDeviceToHost));
  if (w) RF_CUDA(cudaMemset(err, 0, sizeof w));
  RF_CUDA(cudaDeviceSynchronize());
  *word = w;
  return RF_OK;
}

}  // extern "C"
