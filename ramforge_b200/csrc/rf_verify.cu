// rf_verify.cu - the operators around the attention of drafted tokens: per-head
// norm and rotation of queries and keys, and the 8-bit (or f16) cache they write
// and read.  The attention itself is in rf_tree.cu.
//
// Every kernel is launched to begin while the one before it in the stream ends (programmatic
// launch) and waits for it, whole, before it touches memory: without, 8200 rows into a cache and
// back took 28.5 us in place of 23.9.  What the one before may write is not read through the read-only
// path (.nc, __ldg), which is for memory that nobody writes while a kernel runs: norm weights and tables.
//
// All three only move data: a few operations per element, each element read once
// and written once, so HBM bounds the long calls and launch latency the short ones.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

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

// 16 bytes that this call reads once.
__device__ __forceinline__ uint4 ld_once(const void* p) {
  uint4 u;
  asm volatile("ld.global.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
               : "l"(p));
  return u;
}

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

// Any even head_dim, stride and alignment: one warp a head, one element a lane and step.  The instructions of 2- and
// 4-byte accesses bound it: 4001 tokens of 32 + 8 bf16 heads take 72 us with half of 128 dimensions rotated, 75 with
// rows at odd offsets, 63 with heads of 80 (f32: 65), against 18.5 in the kernel below; one token 3.5 against 2.8.
template <class T>
__global__ void __launch_bounds__(256) norm_rope_any_kernel(NormRopeArgs a) {
  griddep_launch();
  griddep_wait();
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

// Pairs of f32 in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)),
        "l"(reinterpret_cast<unsigned long long&>(c)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}

// Whole-head or no rotation, 16-byte aligned rows, head_dim a power of two: lane x of a group of
// 2^lane_bits holds the 16-byte piece x of the head's first half and of its second half, so each
// pair to rotate sits in one lane.  A group takes `per` heads of one token, kHeads at a time with
// the next ones on their way; the products of weights and table are formed once for all of them.
// 4001 tokens of 32 + 8 bf16 heads of 128: 18.5 us (4.5 TB/s; f32 30.1, 5.5 TB/s), against 16.5 for the same
// loads and stores alone; with 2 heads a group 22.6, with four or six CTAs an SM 21.4 and 21.3 (latency, spills).
constexpr int kHeads = 2, kLong = 8, kNormThreads = 128, kNormCtas = 5;

template <class T>
__global__ void __launch_bounds__(kNormThreads, kNormCtas) norm_rope_vec_kernel(NormRopeArgs a, uint32_t lane_bits, uint32_t per,
                                                                      uint32_t q_groups, uint32_t groups) {
  constexpr int V = Act<T>::kVec;
  griddep_launch();
  griddep_wait();
  const uint32_t idx = blockIdx.x * kNormThreads + threadIdx.x, D = a.head_dim;
  uint32_t item = idx >> lane_bits;
  const uint32_t x = idx & ((1u << lane_bits) - 1);
  bool live = item < a.n_tokens * groups;
  if (!live) item = 0;
  const uint32_t t = item / groups, gr = item - t * groups;
  const bool is_q = gr < q_groups;
  const uint32_t h0 = (is_q ? gr : gr - q_groups) * per, heads = is_q ? a.n_heads : a.n_kv_heads;
  const T* src = (const T*)(is_q ? a.q : a.k) + t * (is_q ? a.q_stride : a.k_stride) + (size_t)h0 * D + x * V;
  T* dst = (T*)(is_q ? a.q_out : a.k_out) + t * (is_q ? a.q_out_stride : a.k_out_stride) + (size_t)h0 * D + x * V;
  const float* nw = is_q ? a.q_norm : a.k_norm;
  const int32_t pos = a.rot_dim ? a.pos[t] : 0;
  uint4 raw[kHeads][2];
  auto load = [&](uint32_t h) {
#pragma unroll
    for (int i = 0; i < kHeads; i++) {
      raw[i][0] = raw[i][1] = make_uint4(0, 0, 0, 0);
      if (live && h + i < per && h0 + h + i < heads) {
        raw[i][0] = ld_once(src + (h + i) * D);
        raw[i][1] = ld_once(src + (h + i) * D + D / 2);
      }
    }
  };
  load(0);
  const bool turn = a.rot_dim != 0;
  bool write = live;
  if (turn && (pos < 0 || (uint32_t)pos >= a.rope_len)) {
    if (live) atomicOr(a.err, kVerifyRange);
    write = false;
  }
  // out of the halves v0, v1:  r (v0 w0c - v1 w1s)  and  r (v1 w1c + v0 w0s)
  float2 w0c[V / 2], w1c[V / 2], w0s[V / 2], w1s[V / 2];
#pragma unroll
  for (int j = 0; j < V / 2; j += 2) {
    const float4 one = make_float4(1.f, 1.f, 1.f, 1.f);
    const float4 a0 = nw ? __ldg(reinterpret_cast<const float4*>(nw + x * V + 2 * j)) : one;
    const float4 a1 = nw ? __ldg(reinterpret_cast<const float4*>(nw + D / 2 + x * V + 2 * j)) : one;
    w0c[j] = make_float2(a0.x, a0.y), w0c[j + 1] = make_float2(a0.z, a0.w);
    w1c[j] = make_float2(a1.x, a1.y), w1c[j + 1] = make_float2(a1.z, a1.w);
  }
  if (turn) {
    const float2* row = a.rope + (size_t)(write ? pos : 0) * (D / 2) + x * V;
#pragma unroll
    for (int j = 0; j < V / 2; j++) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(row + 2 * j));
      const float2 c = make_float2(f.x, f.z), s = make_float2(f.y, f.w);
      w0s[j] = mul2(w0c[j], s), w1s[j] = mul2(w1c[j], make_float2(-f.y, -f.w));
      w0c[j] = mul2(w0c[j], c), w1c[j] = mul2(w1c[j], c);
    }
  }
  const float inv_d = 1.f / (float)D;  // exact: a power of two
#pragma unroll 1
  for (uint32_t h = 0; h < per; h += kHeads) {
    uint4 cur[kHeads][2];
#pragma unroll
    for (int i = 0; i < kHeads; i++) cur[i][0] = raw[i][0], cur[i][1] = raw[i][1];
    if (h + kHeads < per) load(h + kHeads);
#pragma unroll
    for (int i = 0; i < kHeads; i++) {
      float2 v[2][V / 2];
#pragma unroll
      for (int s = 0; s < 2; s++) {
        float f[V];
        Act<T>::unpack(cur[i][s], f);
#pragma unroll
        for (int j = 0; j < V / 2; j++) v[s][j] = make_float2(f[2 * j], f[2 * j + 1]);
      }
      float2 r = make_float2(1.f, 1.f);
      float2 ss2 = make_float2(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < V / 2; j++) ss2 = fma2(v[0][j], v[0][j], fma2(v[1][j], v[1][j], ss2));
      float ss = ss2.x + ss2.y;
      for (uint32_t o = (1u << lane_bits) / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (nw) r.x = r.y = rsqrtf(fmaf(ss, inv_d, a.eps));
      float y[2][V];
#pragma unroll
      for (int j = 0; j < V / 2; j++) {
        float2 u = mul2(v[0][j], w0c[j]), z = mul2(v[1][j], w1c[j]);
        if (turn) u = fma2(v[1][j], w1s[j], u), z = fma2(v[0][j], w0s[j], z);
        u = mul2(u, r), z = mul2(z, r);
        y[0][2 * j] = u.x, y[0][2 * j + 1] = u.y, y[1][2 * j] = z.x, y[1][2 * j + 1] = z.y;
      }
      if (write && h + i < per && h0 + h + i < heads) {
        *reinterpret_cast<uint4*>(dst + (h + i) * D) = Act<T>::pack(y[0]);
        *reinterpret_cast<uint4*>(dst + (h + i) * D + D / 2) = Act<T>::pack(y[1]);
      }
    }
  }
}

}  // namespace

// ---------------------------------------------------------------------------
// The cache.  A lane handles 16 elements of one head of a row at a time, for K or for V: a 16-byte
// piece of codes, half a Q8_0 block, so a pair of neighbouring lanes shares a scale.  A position has
// to arrive before the row it names can be asked for, so CTAs stay and go from row to row: while a
// row is converted, the next one and the position after that are on their way.  32768 rows of 8 heads
// of 128 out of a Q8_0 cache: 35.8 us (5.75 TB/s, 0.88 of the copy rate), 54.7 with a CTA for every few rows.
// ---------------------------------------------------------------------------
namespace {

struct KvRowsArgs {
  rf_kv_view c;
  const void *k, *v;  // write: sources; read: destinations (may be null)
  uint64_t k_stride, v_stride;
  const int32_t *seq, *pos;
  uint32_t n_rows, per_head, per_row;  // 16-element pieces of a head and of a row (K and V)
  bool wide;                           // activations' rows are 32-byte aligned
  unsigned* err;
};

constexpr int kKvThreads = 256, kKvCtas = 4, kKvRows = 2;  // CTAs an SM; rows of a thread in flight

// Thread (x, y) of a CTA: piece x of a row's K and V pieces (blockIdx.y counts runs of kKvThreads), row y
// of every `rows` the CTA takes at a time.
struct KvPlace {
  bool in, is_v;
  uint32_t x, h, c;  // piece of the K or V row, its head, piece of the head
  uint32_t row, step;
  __device__ __forceinline__ KvPlace(const KvRowsArgs& a) {
    const uint32_t width = min(a.per_row, (uint32_t)kKvThreads), y = threadIdx.x / width;
    const uint32_t at = blockIdx.y * kKvThreads + (threadIdx.x - y * width), half = a.per_row / 2, rows = kKvThreads / width;
    in = at < a.per_row && y < rows;
    is_v = at >= half;
    x = is_v ? at - half : at;
    h = x / a.per_head;
    c = x - h * a.per_head;
    row = blockIdx.x * rows + y;
    step = gridDim.x * rows;
  }
};

// Place of a row: its position and sequence, then (out of range: the error bit) its cache row, or -1.
struct KvAddr {
  int32_t pos, seq;
};
__device__ __forceinline__ KvAddr kv_addr(const KvRowsArgs& a, uint32_t row) {
  KvAddr p{-1, 0};
  if (row < a.n_rows) p.pos = a.pos[row], p.seq = a.seq ? a.seq[row] : 0;
  return p;
}
__device__ __forceinline__ int64_t kv_slot(const KvRowsArgs& a, KvAddr p, uint32_t h) {
  if (p.pos < 0) return -1;
  if ((uint32_t)p.pos >= a.c.capacity || p.seq < 0 || (uint32_t)p.seq >= a.c.n_seqs) {
    atomicOr(a.err, kVerifyRange);
    return -1;
  }
  return ((int64_t)p.seq * a.c.n_kv_heads + h) * a.c.capacity + p.pos;
}

// 16 activations: two or four 16-byte loads or stores, or half as many of 32 bytes.
template <class T>
struct Acts16 {
  static constexpr int N = 16 / Act<T>::kVec;
  uint4 u[N];
  __device__ __forceinline__ void load(const T* p, bool wide) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint4* q = reinterpret_cast<const uint4*>(p) + i;
      if (wide)
        asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(u[i].x), "=r"(u[i].y), "=r"(u[i].z), "=r"(u[i].w), "=r"(u[i + 1].x), "=r"(u[i + 1].y),
                       "=r"(u[i + 1].z), "=r"(u[i + 1].w)
                     : "l"(q));
      else
        u[i] = q[0], u[i + 1] = q[1];
    }
  }
  __device__ __forceinline__ void store(T* p, bool wide) const {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      uint4* q = reinterpret_cast<uint4*>(p) + i;
      if (wide)
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(q), "r"(u[i].x), "r"(u[i].y), "r"(u[i].z),
                     "r"(u[i].w), "r"(u[i + 1].x), "r"(u[i + 1].y), "r"(u[i + 1].z), "r"(u[i + 1].w)
                     : "memory");
      else
        q[0] = u[i], q[1] = u[i + 1];
    }
  }
  __device__ __forceinline__ void get(float (&v)[16]) const {
#pragma unroll
    for (int i = 0; i < N; i++) {
      float f[Act<T>::kVec];
      Act<T>::unpack(u[i], f);
#pragma unroll
      for (int j = 0; j < Act<T>::kVec; j++) v[i * Act<T>::kVec + j] = f[j];
    }
  }
  __device__ __forceinline__ void put(const float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      float f[Act<T>::kVec];
#pragma unroll
      for (int j = 0; j < Act<T>::kVec; j++) f[j] = v[i * Act<T>::kVec + j];
      u[i] = Act<T>::pack(f);
    }
  }
};

template <class T, bool Q8>
__device__ __forceinline__ void kv_store(const KvRowsArgs& a, const KvPlace& p, int64_t slot, const Acts16<T>& in) {
  float v[16];
  in.get(v);
  const uint64_t at = (uint64_t)slot * a.c.head_dim + p.c * 16;
  if constexpr (!Q8) {
    if (slot < 0) return;
    __half* dst = (__half*)(p.is_v ? a.c.v : a.c.k) + at;
    Acts16<__half> out;
    out.put(v);
    out.store(dst, false);
  } else {
    float amax = 0.f;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      nan |= v[i] != v[i];
      v[i] = fminf(fmaxf(v[i], -65472.f), 65472.f);
      amax = fmaxf(amax, fabsf(v[i]));
    }
    // a NaN's bits are above every number's, so the maximum of the bits keeps it
    int bits = nan ? 0x7fffffff : __float_as_int(amax);
    bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
    // the scale is kept in f16 (GGUF's block): its 11 bits cost at most 2^-11 of a code step per code,
    // and codes are taken against the rounded scale
    const __half d = __float2half_rn(__fdiv_rn(__int_as_float(bits), 127.f));
    const float df = __half2float(d), inv = df > 0.f ? __fdiv_rn(1.f, df) : 0.f;
    if (slot < 0) return;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      uint32_t b[4];
#pragma unroll
      for (int j = 0; j < 4; j++)  // round to nearest even by the sum's own rounding: the code is its low byte
        b[j] = __float_as_uint(__fadd_rn(fminf(fmaxf(__fmul_rn(v[4 * i + j], inv), -127.f), 127.f), 12582912.f));
      w[i] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
    *reinterpret_cast<uint4*>((int8_t*)(p.is_v ? a.c.v : a.c.k) + at) = make_uint4(w[0], w[1], w[2], w[3]);
    if (!(p.c & 1)) ((__half*)(p.is_v ? a.c.v_scale : a.c.k_scale))[slot * (a.c.head_dim / 32) + p.c / 2] = d;
  }
}

// A row is asked for together with its position, also if the position then says that it is not kept: asking after the
// position is known costs the rows that are (8200 bf16 rows of 8 heads of 128 into Q8_0: 15.4 us, and 19.4 so; 32768:
// 45.8 and 62.7) and does not gain at the few rows of an accepted path (16 rows, one in three kept: 2.8 us both); it would
// at thousands of rows mostly dropped (8200 f32 rows into f16, one in three kept: 16.5 and 11.3).
template <class T, bool Q8>
__global__ void __launch_bounds__(kKvThreads) kv_write_kernel(KvRowsArgs a) {
  const KvPlace p(a);
  griddep_launch();
  griddep_wait();
  const T* src = (const T*)(p.is_v ? a.v : a.k) + p.x * 16;
  const uint64_t stride = p.is_v ? a.v_stride : a.k_stride;
  Acts16<T> cur[kKvRows] = {}, next[kKvRows] = {};
  KvAddr at[kKvRows], at_next[kKvRows];
  auto fetch = [&](uint32_t row, Acts16<T>(&u)[kKvRows], KvAddr(&w)[kKvRows]) {
#pragma unroll
    for (int i = 0; i < kKvRows; i++) {
      const uint32_t r = row + i * p.step;
      w[i] = kv_addr(a, p.in ? r : a.n_rows);
      if (p.in && r < a.n_rows) u[i].load(src + r * stride, a.wide);
    }
  };
  fetch(p.row, cur, at);
  // all lanes of a warp go round as often as the CTA's first row does: shuffles inside
  for (uint32_t row = p.row, first = blockIdx.x * (kKvThreads / min(a.per_row, (uint32_t)kKvThreads)); first < a.n_rows;
       row += kKvRows * p.step, first += kKvRows * p.step) {
    fetch(row + kKvRows * p.step, next, at_next);
#pragma unroll
    for (int i = 0; i < kKvRows; i++) {
      kv_store<T, Q8>(a, p, p.in ? kv_slot(a, at[i], p.h) : -1, cur[i]);
      cur[i] = next[i], at[i] = at_next[i];
    }
  }
}

// A cache piece as it is stored: 16 codes and their scale, or 16 f16.
template <bool Q8>
struct KvRaw {
  uint4 u[Q8 ? 1 : 2];
  __half d;
};

template <class T, bool Q8>
__global__ void __launch_bounds__(kKvThreads) kv_read_kernel(KvRowsArgs a) {
  const KvPlace p(a);
  griddep_launch();
  griddep_wait();
  T* dst = (T*)(p.is_v ? a.v : a.k);
  if (!dst || !p.in) return;
  dst += p.x * 16;
  const uint64_t stride = p.is_v ? a.v_stride : a.k_stride;
  const void* plane = p.is_v ? a.c.v : a.c.k;
  const __half* scales = (const __half*)(p.is_v ? a.c.v_scale : a.c.k_scale);
  auto fetch = [&](KvAddr w) {
    KvRaw<Q8> x = {};
    const int64_t slot = kv_slot(a, w, p.h);
    if (slot < 0) return x;
    const uint64_t at = (uint64_t)slot * a.c.head_dim + p.c * 16;
    if constexpr (Q8) {
      x.u[0] = ld_once((const int8_t*)plane + at);
      x.d = scales[slot * (a.c.head_dim / 32) + p.c / 2];
    } else {
      const uint4* q = reinterpret_cast<const uint4*>((const __half*)plane + at);
      x.u[0] = q[0], x.u[1] = q[1];
    }
    return x;
  };
  KvRaw<Q8> cur[kKvRows];
  KvAddr at[kKvRows];
#pragma unroll
  for (int i = 0; i < kKvRows; i++) at[i] = kv_addr(a, p.row + i * p.step);
#pragma unroll
  for (int i = 0; i < kKvRows; i++) {
    cur[i] = fetch(at[i]);
    at[i] = kv_addr(a, p.row + (kKvRows + i) * p.step);
  }
  for (uint32_t row = p.row; row < a.n_rows; row += kKvRows * p.step) {
    KvRaw<Q8> next[kKvRows];
#pragma unroll
    for (int i = 0; i < kKvRows; i++) {
      next[i] = fetch(at[i]);
      at[i] = kv_addr(a, row + (2 * kKvRows + i) * p.step);
    }
#pragma unroll
    for (int i = 0; i < kKvRows; i++) {
      const uint32_t r = row + i * p.step;
      Acts16<__half> out;
      if constexpr (Q8) {
        // biased bytes under an exponent of 1024: 1152 + code, exact; the product with the scale rounds once to f16
        const __half2 d2 = __half2half2(cur[i].d), bias = __float2half2_rn(1152.f);
        const uint32_t w[4] = {cur[i].u[0].x, cur[i].u[0].y, cur[i].u[0].z, cur[i].u[0].w};
        uint32_t h[8];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const uint32_t b = w[k] ^ 0x80808080u;
          uint32_t lo = __byte_perm(b, 0x64646464u, 0x4140), hi = __byte_perm(b, 0x64646464u, 0x4342);
          const __half2 x = __hmul2(__hsub2(*reinterpret_cast<__half2*>(&lo), bias), d2);
          const __half2 y = __hmul2(__hsub2(*reinterpret_cast<__half2*>(&hi), bias), d2);
          h[2 * k] = *reinterpret_cast<const uint32_t*>(&x), h[2 * k + 1] = *reinterpret_cast<const uint32_t*>(&y);
        }
        out.u[0] = make_uint4(h[0], h[1], h[2], h[3]), out.u[1] = make_uint4(h[4], h[5], h[6], h[7]);
      } else {
        out.u[0] = cur[i].u[0], out.u[1] = cur[i].u[1];
      }
      if (r < a.n_rows) {
        if constexpr (std::is_same<T, __half>::value) {
          out.store(dst + r * stride, a.wide);
        } else {
          float v[16];
          out.get(v);
          Acts16<T> o;
          o.put(v);
          o.store(dst + r * stride, a.wide);
        }
      }
      cur[i] = next[i];
    }
  }
}

int check_kv_rows(const rf_kv_view* c, const void* k, const void* v, int act_type, uint32_t n_rows, uint64_t* k_stride,
                  uint64_t* v_stride, const int32_t* seq, const int32_t* pos) {
  RF_TRY(check_kv_view(c));
  const uint32_t es = act_bytes(act_type);
  if (!es) return set_error(RF_EINVAL, "activation type %d is not F32, F16 or BF16", act_type);
  if (n_rows && !pos) return set_error(RF_EINVAL, "null positions");
  if (!aligned_to(pos, 4) || !aligned_to(seq, 4)) return set_error(RF_EINVAL, "positions and sequences must be 4-byte aligned");
  const uint64_t row = (uint64_t)c->n_kv_heads * c->head_dim;
  for (uint64_t* s : {k_stride, v_stride}) {
    if (!*s) *s = row;
    if (*s < row) return set_error(RF_EINVAL, "row stride %llu is below the row's %llu elements", (unsigned long long)*s,
                                   (unsigned long long)row);
    if (*s * es % 16) return set_error(RF_EINVAL, "row stride %llu is not a multiple of 16 bytes", (unsigned long long)*s);
  }
  if (!aligned_to(k, 16) || !aligned_to(v, 16)) return set_error(RF_EINVAL, "K/V rows must be 16-byte aligned");
  if (2ull * n_rows * row / 4 > 0x7fffffffull) return set_error(RF_EINVAL, "%u rows are too many for one call", n_rows);
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
    uint32_t bits = 0;
    while ((1u << bits) < lanes) bits++;
    // kLong heads a group where that still gives every SM kNormThreads * 8 lanes of work; else kHeads, so that the
    // heads of few tokens are spread over more warps
    const uint32_t per = (uint64_t)a.n_tokens * (a.n_heads + a.n_kv_heads) * lanes >= (uint64_t)num_sms() * kNormThreads * 8 * kLong ? kLong : kHeads;
    const uint32_t qg = (a.n_heads + per - 1) / per, groups = qg + (a.n_kv_heads + per - 1) / per;
    const uint64_t threads = (uint64_t)a.n_tokens * groups * lanes;
    return launch_k(L, norm_rope_vec_kernel<T>, dim3((uint32_t)((threads + kNormThreads - 1) / kNormThreads)),
                    dim3(kNormThreads), 0, a, bits, per, qg, groups);
  }
  const uint32_t warps = a.n_tokens * (a.n_heads + a.n_kv_heads);
  return launch_k(L, norm_rope_any_kernel<T>, dim3((warps + 7) / 8), dim3(256), 0, a);
}

template <class T>
cudaError_t launch_kv_rows(const Launch& L, KvRowsArgs a, bool write) {
  a.per_head = a.c.head_dim / 16;
  a.per_row = 2 * a.c.n_kv_heads * a.per_head;
  a.wide = aligned_to(a.k, 32) && aligned_to(a.v, 32) && a.k_stride * sizeof(T) % 32 == 0 && a.v_stride * sizeof(T) % 32 == 0;
  const bool q8 = a.c.type == RF_TYPE_Q8_0;
  auto* k = write ? (q8 ? kv_write_kernel<T, true> : kv_write_kernel<T, false>)
                  : (q8 ? kv_read_kernel<T, true> : kv_read_kernel<T, false>);
  const uint32_t width = std::min(a.per_row, (uint32_t)kKvThreads), rows = kKvThreads / width;
  const uint32_t cols = (a.per_row + kKvThreads - 1) / kKvThreads;
  const uint32_t most = std::max(1u, (uint32_t)num_sms() * kKvCtas / cols);  // CTAs stay for as many rows as there are
  return launch_k(L, k, dim3(std::min((a.n_rows + rows - 1) / rows, most), cols), dim3(kKvThreads), 0, a);
}

int run_kv_rows(const rf_kv_view* cache, const void* k, const void* v, int act_type, uint32_t n_rows, uint64_t k_stride,
                uint64_t v_stride, const int32_t* seq, const int32_t* pos, void* stream, bool write) {
  RF_TRY(check_kv_rows(cache, k, v, act_type, n_rows, &k_stride, &v_stride, seq, pos));
  if (!n_rows) return RF_OK;
  KvRowsArgs a{};
  a.c = *cache;
  a.k = k, a.v = v;
  a.k_stride = k_stride, a.v_stride = v_stride;
  a.seq = seq, a.pos = pos;
  a.n_rows = n_rows;
  RF_TRY(verify_error_ptr(&a.err));
  const Launch L{(cudaStream_t)stream, true};
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
  if (!aligned_to(q_norm, 4) || !aligned_to(k_norm, 4) || !aligned_to(positions, 4))
    return set_error(RF_EINVAL, "norm weights and positions must be 4-byte aligned");
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
  const Launch L{(cudaStream_t)stream, true};
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
