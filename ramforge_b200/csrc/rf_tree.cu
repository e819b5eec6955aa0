// rf_tree.cu - attention of drafted tokens over a cached history and over the
// drafts' own tree (rf_tree_attention).
//
// out[t] = sum_p softmax_p(scale q[t] . k[p]) v[p] over the positions token t sees:
// the whole history p < L, and the drafts p = L + j whose bit j is set in its mask row.
// One pass over the keys carries the running maximum m, the sum l of exp(s - m) and
// the output sum, rescaled when m grows.
#include <mutex>
#include <type_traits>

#include "rf_tree.cuh"

namespace rf {
namespace {

// ---------------------------------------------------------------------------
// Few query rows a KV head: tree_rows_kernel.
//
// The keys' bytes bound it, so they go from HBM straight into the registers that
// mma.sync reads, and nothing else is staged.  A warp takes MB * 16 keys a step and
// computes S^T = K Q^T (keys are the MMA's rows, query rows its 8 * NB columns) and
// O^T += V^T P^T.  The order of the summed index is free in both products, so a lane's
// A fragments are whole 16-byte pieces of a row: for K the head's dimensions are
// assigned to the k index so that lane c of a group of four holds consecutive ones, and
// for V the dimensions are assigned to the m index so that lane group g does.
// Scores leave the MMA with keys along the lanes' groups; movmatrix turns the 8 x 8
// blocks of P into the B fragments of the second product.
// ---------------------------------------------------------------------------

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint4 ld_stream16(const void* p) {
  uint4 u;
  asm volatile("ld.global.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
               : "l"(p));
  return u;
}
__device__ __forceinline__ uint2 ld_stream8(const void* p) {
  uint2 u;
  asm volatile("ld.global.L1::no_allocate.v2.b32 {%0,%1}, [%2];" : "=r"(u.x), "=r"(u.y) : "l"(p));
  return u;
}

// Two biased bytes (code + 128) in the low halves of 0x64xx become 1024 + 128 + code; the
// subtraction is exact, the product rounds once: the value the cache format defines.
__device__ __forceinline__ uint32_t q8_pair(uint32_t biased, __half2 d) {
  const __half2 code = __hsub2(bits_h2(biased), __float2half2_rn(1152.f));
  return h2_bits(__hmul2(code, d));
}

// A block in which a code could leave f16, or whose scale is no number.  The cache's writer makes codes up to 127, but
// a plane may hold -128: above 511.75 (511.75 * 128 = 65504, the last f16).
__device__ __forceinline__ bool wild_scale(uint32_t half_bits) { return (half_bits & 0x7fffu) > 0x5fffu; }

// The four codes of a word without those whose product with the scale is not finite.
__device__ __noinline__ uint32_t finite_codes(uint32_t w, uint32_t half_bits) {
  const float d = __half2float(__ushort_as_half((unsigned short)half_bits));
#pragma unroll 1
  for (int i = 0; i < 32; i += 8) {
    const float v = __half2float(__float2half_rn((float)(int8_t)(w >> i) * d));
    if (!(fabsf(v) < INFINITY)) w &= ~(0xffu << i);
  }
  return w;
}

// Shapes of one step of a warp over a cache of type Q8, head dimension D
// and NB blocks of 8 query rows, with the CTAs of an SM.  Q8_0 is bound by the latency of its steps: 42 % of
// a warp's time it waits for loads, one step ahead of their use, and 22 % for the decode's own results, at 16 warps
// an SM (registers); issue slots are 49 % full and HBM is at 0.72 of the copy rate.  So it wants more warps: one row
// over 131072 positions of 128 dimensions takes 59 us with 16 keys a step and four CTAs, 64 with 32 and three, 87
// with 32 and four (spills); of 64 dimensions 35 with 32 and four, 40 with 16 and four.  f16 is bound by HBM: 86 us
// (0.95 of the copy rate) with three CTAs, 96 with four.
template <bool Q8, int D, int NB>
struct Step {
  static constexpr int MB = !Q8 || (D == 128 && NB == 1) ? 1 : 2;  // 16-key blocks
  static constexpr int CTAS = NB == 2 ? 2 : Q8 ? 4 : 3;
  static constexpr int KEYS = 16 * MB;
  static constexpr int KW = Q8 ? D / 16 : D / 8;           // 32-bit words of one key's K in a lane
  static constexpr int VW = Q8 ? D / 32 : D / 16;          // ... of one key's V
  static constexpr int KS = D / 16;                        // k steps of S, m blocks of O
};
constexpr int kRowWarps = 4;

// Query rows as B fragments: row g of block nb, the dimensions lane c holds of a key.
// f32 and bf16 rows are first scaled by a power of two to a largest magnitude in [1, 2),
// which f16 holds; f32 keeps a second f16 term.  *exp2 is the scale that was taken out.
template <class T, bool Q8, int D, bool SPLIT>
__device__ __forceinline__ void load_query(const T* row, bool live, uint32_t c, uint32_t (&hi)[D / 16][2],
                                           uint32_t (&lo)[SPLIT ? D / 16 : 1][2], float* exp2) {
  constexpr int KS = D / 16;
  float v[KS][4];
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < KS; k++) {
    const uint32_t d = Q8 ? 64 * (k / 4) + 16 * c + 4 * (k % 4) : 32 * (k / 2) + 8 * c + 4 * (k % 2);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      v[k][i] = live ? act_get(row + d + i) : 0.f;
      top = fmaxf(top, fabsf(v[k][i]));
    }
  }
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  float up = 1.f;
  if constexpr (!std::is_same<T, __half>::value) {
    float down;
    pow2_scale(top, &down, &up);
#pragma unroll
    for (int k = 0; k < KS; k++)
#pragma unroll
      for (int i = 0; i < 4; i++) v[k][i] *= down;
  }
  *exp2 = up;
#pragma unroll
  for (int k = 0; k < KS; k++)
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const __half2 h = __floats2half2_rn(v[k][2 * i], v[k][2 * i + 1]);
      hi[k][i] = h2_bits(h);
      if constexpr (SPLIT) {
        const float2 f = __half22float2(h);
        lo[k][i] = h2_bits(__floats2half2_rn(v[k][2 * i] - f.x, v[k][2 * i + 1] - f.y));
      }
    }
}

template <class T, bool Q8, int D, int NB>
__global__ void __launch_bounds__(32 * kRowWarps, Step<Q8, D, NB>::CTAS)
    tree_rows_kernel(TreeArgs a, float* __restrict__ part) {
  using S = Step<Q8, D, NB>;
  constexpr bool SPLIT = std::is_same<T, float>::value;
  constexpr int ROWS = 8 * NB, KT = S::KEYS * kRowWarps, MB = S::MB, KS = S::KS, KW = S::KW, VW = S::VW;
  __shared__ __align__(16) float s_o[kRowWarps][ROWS][D];
  __shared__ float s_m[kRowWarps][ROWS], s_l[kRowWarps][ROWS];
  __shared__ int s_wild;  // a V element of a draft is not finite
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const uint32_t k_half = c >= 2 ? 0x3232 : 0x1010;  // which of a word's two scales the lane's dimensions have
  if (threadIdx.x == 0) s_wild = 0;
  griddep_wait();
  griddep_launch();  // of tree_merge_kernel, which reads the lengths before it waits: not before they are there
  __syncthreads();
  const uint32_t G = a.group;
  Walk<KT, ROWS> walk(a);
  Segment sg;
  while (walk.next(a, &sg)) {
    const uint32_t b = sg.b, h = sg.h, L = sg.hist, n = sg.drafts, end = sg.end, k0 = sg.k0, k1 = sg.k1, rt = sg.rt;
    const uint32_t r0 = rt * ROWS, nrows = min((uint32_t)ROWS, n * G - r0);
    const uint64_t base = ((uint64_t)b * a.c.n_kv_heads + h) * a.c.capacity;
    const uint8_t* kp = (const uint8_t*)a.c.k + base * D * (Q8 ? 1 : 2);
    const uint8_t* vp = (const uint8_t*)a.c.v + base * D * (Q8 ? 1 : 2);
    const __half* ksp = Q8 ? (const __half*)a.c.k_scale + base * (D / 32) : nullptr;
    const __half* vsp = Q8 ? (const __half*)a.c.v_scale + base * (D / 32) : nullptr;

    uint32_t qh[NB][KS][2], ql[NB][SPLIT ? KS : 1][2];
    float coef[NB][2];  // score -> base-2 exponent, of this lane's rows 2c and 2c + 1 of each block
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
      const uint32_t r = 8 * nb + g, rr = r0 + r;
      const bool live = r < nrows;
      float up;
      load_query<T, Q8, D, SPLIT>(
          (const T*)a.q + ((uint64_t)b * a.n_tokens + (live ? group_div(a, rr) : 0)) * a.q_stride + (h * G + (live ? rr - group_div(a, rr) * G : 0)) * D,
          live, c, qh[nb], ql[nb], &up);
      const float cf = fmaxf(a.scale * 1.44269504f * up, 1.17549435e-38f);  // not 0: a masked score stays -inf
      coef[nb][0] = __shfl_sync(0xffffffffu, cf, 8 * c);
      coef[nb][1] = __shfl_sync(0xffffffffu, cf, 8 * c + 4);
    }
    float o[KS][NB][4], m[NB][2], l[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
#pragma unroll
      for (int i = 0; i < KS; i++) o[i][nb][0] = o[i][nb][1] = o[i][nb][2] = o[i][nb][3] = 0.f;
      m[nb][0] = m[nb][1] = -INFINITY;
      l[nb][0] = l[nb][1] = 0.f;
    }

    // The lane's pieces: K of keys g + 8 i, V of keys 2c + {0, 1, 8, 9} + 16 i of a step.  Whole
    // steps of the history are read at constant offsets from pointers that move with the
    // steps; a step that holds drafts or the end reads the last key in place of what is past it.
    constexpr uint32_t KB = D * (Q8 ? 1 : 2);  // bytes of a row
    constexpr uint32_t VO = Q8 && D == 64 ? 8 : 16;
    uint32_t kr[2 * MB][KW], vr[4 * MB][VW], vs[4 * MB];
    uint2 ks[2 * MB];
    auto v_off = [](int i) { return 16 * (i / 4) + (i % 2) + 8 * ((i / 2) % 2); };
    auto get_k = [&](int i, const uint8_t* p, const __half* sp) {
#pragma unroll
      for (int j = 0; j < KW / 4; j++) {
        const uint4 u = ld_stream16(p + 64 * j);
        kr[i][4 * j] = u.x, kr[i][4 * j + 1] = u.y, kr[i][4 * j + 2] = u.z, kr[i][4 * j + 3] = u.w;
      }
      if constexpr (Q8) {
        if constexpr (D == 128)
          ks[i] = ld_stream8(sp);
        else
          ks[i].x = *(const uint32_t*)sp;
      }
    };
    auto get_v = [&](int i, const uint8_t* p, const __half* sp) {
      if constexpr (Q8 && D == 64) {
        const uint2 u = ld_stream8(p);
        vr[i][0] = u.x, vr[i][1] = u.y;
      } else {
#pragma unroll
        for (int j = 0; j < VW / 4; j++) {
          const uint4 u = ld_stream16(p + 128 * j);
          vr[i][4 * j] = u.x, vr[i][4 * j + 1] = u.y, vr[i][4 * j + 2] = u.z, vr[i][4 * j + 3] = u.w;
        }
      }
      if constexpr (Q8) vs[i] = *(const unsigned short*)sp;
    };
    auto inner = [&](uint32_t kb) { return kb + S::KEYS <= L; };
    const uint32_t kb0 = k0 * KT + warp * S::KEYS;
    const uint8_t *kl = kp + (uint64_t)(kb0 + g) * KB + 16 * c, *vl = vp + (uint64_t)(kb0 + 2 * c) * KB + VO * g;
    const __half* ksl = Q8 ? ksp + (uint64_t)(kb0 + g) * (D / 32) : nullptr;
    const __half* vsl = Q8 ? vsp + (uint64_t)(kb0 + 2 * c) * (D / 32) + g / (D == 128 ? 2 : 4) : nullptr;
    auto load_k = [&](uint32_t kb) {
      if (inner(kb)) {
#pragma unroll
        for (int i = 0; i < 2 * MB; i++) get_k(i, kl + 8 * i * KB, Q8 ? ksl + 8 * i * (D / 32) : nullptr);
      } else {
#pragma unroll
        for (int i = 0; i < 2 * MB; i++) {
          const uint64_t key = min(kb + g + 8 * i, end - 1);
          get_k(i, kp + key * KB + 16 * c, Q8 ? ksp + key * (D / 32) : nullptr);
        }
      }
      kl += KT * KB;
      if constexpr (Q8) ksl += KT * (D / 32);
    };
    auto load_v = [&](uint32_t kb) {
      if (inner(kb)) {
#pragma unroll
        for (int i = 0; i < 4 * MB; i++) get_v(i, vl + v_off(i) * KB, Q8 ? vsl + v_off(i) * (D / 32) : nullptr);
      } else {
#pragma unroll
        for (int i = 0; i < 4 * MB; i++) {
          const uint64_t key = min(kb + 2 * c + v_off(i), end - 1);
          get_v(i, vp + key * KB + VO * g, Q8 ? vsp + key * (D / 32) + g / (D == 128 ? 2 : 4) : nullptr);
        }
      }
      vl += KT * KB;
      if constexpr (Q8) vsl += KT * (D / 32);
    };

    if (kb0 < end) {
      load_k(kb0);
      load_v(kb0);
    }
    for (uint32_t tile = k0; tile < k1; tile++) {
      const uint32_t kb = tile * KT + warp * S::KEYS;
      if (kb >= end) break;
      const bool more = tile + 1 < k1 && kb + KT < end;
      const bool edge = !inner(kb);  // holds drafts or the end: masks apply
      // ---- S^T = K Q^T
      float s[MB][NB][4];
#pragma unroll
      for (int mb = 0; mb < MB; mb++) {
#pragma unroll
        for (int nb = 0; nb < NB; nb++) s[mb][nb][0] = s[mb][nb][1] = s[mb][nb][2] = s[mb][nb][3] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; k++) {
          uint32_t f[4];
          if constexpr (Q8) {  // word k of the lane's piece: four codes, two a half2
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const uint32_t x = kr[2 * mb + i][k] ^ 0x80808080u;
              const uint32_t sw = k / 4 ? ks[2 * mb + i].y : ks[2 * mb + i].x;
              const __half2 d = bits_h2(__byte_perm(sw, sw, k_half));
              f[i] = q8_pair(__byte_perm(x, 0x64646464u, 0x4140), d);
              f[2 + i] = q8_pair(__byte_perm(x, 0x64646464u, 0x4342), d);
            }
          } else {
            f[0] = kr[2 * mb][2 * k], f[1] = kr[2 * mb + 1][2 * k];
            f[2] = kr[2 * mb][2 * k + 1], f[3] = kr[2 * mb + 1][2 * k + 1];
          }
#pragma unroll
          for (int nb = 0; nb < NB; nb++) {
            mma16816(s[mb][nb], f, qh[nb][k][0], qh[nb][k][1]);
            if constexpr (SPLIT) mma16816(s[mb][nb], f, ql[nb][k][0], ql[nb][k][1]);
          }
        }
      }
      if (more) load_k(kb + KT);
      // ---- weights
      if (edge) {
#pragma unroll
        for (int mb = 0; mb < MB; mb++)
#pragma unroll
          for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const uint32_t p = kb + 16 * mb + 8 * (e >> 1) + g, r = 8 * nb + 2 * c + (e & 1);
              if (p >= end || r >= nrows || !sees(a, b, group_div(a, r0 + r), L, p)) s[mb][nb][e] = -INFINITY;
            }
      }
      bool raise = false;
      float top[NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int x = 0; x < 2; x++) {
          top[nb][x] = -INFINITY;
#pragma unroll
          for (int mb = 0; mb < MB; mb++) top[nb][x] = fmaxf(top[nb][x], fmaxf(s[mb][nb][x], s[mb][nb][2 + x]));
          top[nb][x] *= coef[nb][x];
          raise |= top[nb][x] > m[nb][x] + kRaise;
        }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
          for (int x = 0; x < 2; x++) {
            float t = fmaxf(m[nb][x], top[nb][x]);
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
            const float f = t == -INFINITY ? 1.f : ex2(m[nb][x] - t);
            m[nb][x] = t;
            l[nb][x] *= f;
#pragma unroll
            for (int i = 0; i < KS; i++) o[i][nb][x] *= f, o[i][nb][2 + x] *= f;
          }
      }
      uint32_t ph[MB][NB][2], pl[MB][SPLIT ? NB : 1][2];
#pragma unroll
      for (int nb = 0; nb < NB; nb++) {
        const float ref[2] = {kWeightBias - (m[nb][0] == -INFINITY ? 0.f : m[nb][0]),
                              kWeightBias - (m[nb][1] == -INFINITY ? 0.f : m[nb][1])};
#pragma unroll
        for (int mb = 0; mb < MB; mb++) {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            s[mb][nb][e] = ex2(fmaf(s[mb][nb][e], coef[nb][e & 1], ref[e & 1]));
            l[nb][e & 1] += s[mb][nb][e];
          }
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const __half2 p2 = __floats2half2_rn(s[mb][nb][2 * i], s[mb][nb][2 * i + 1]);
            ph[mb][nb][i] = transpose8x8(h2_bits(p2));
            if constexpr (SPLIT) {
              const float2 f = __half22float2(p2);
              pl[mb][nb][i] =
                  transpose8x8(h2_bits(__floats2half2_rn(s[mb][nb][2 * i] - f.x, s[mb][nb][2 * i + 1] - f.y)));
            }
          }
        }
      }
      // what is masked must not reach the sums, 0 * NaN included: drafts' V elements that are not finite
      // count as 0 here, and the rows that see them get them when the results are written; the history's
      // stay, since every row sees them
      if (edge) {
        bool wild = false;
#pragma unroll
        for (int i = 0; i < 4 * MB; i++) {
          if (kb + 2 * c + v_off(i) < L) continue;
          if constexpr (Q8) {
            if (wild_scale(vs[i])) {
              wild = true;
#pragma unroll
              for (int j = 0; j < VW; j++) vr[i][j] = finite_codes(vr[i][j], vs[i]);
              if ((vs[i] & 0x7c00u) == 0x7c00u) vs[i] = 0;
            }
          } else {
#pragma unroll
            for (int j = 0; j < VW; j++) {
              if ((vr[i][j] & 0x7c00u) == 0x7c00u) vr[i][j] &= 0xffff0000u, wild = true;
              if ((vr[i][j] & 0x7c000000u) == 0x7c000000u) vr[i][j] &= 0x0000ffffu, wild = true;
            }
          }
        }
        if (wild) s_wild = 1;
      }
      // ---- O^T += V^T P^T
#pragma unroll
      for (int mb = 0; mb < MB; mb++) {
#pragma unroll
        for (int i = 0; i < KS; i++) {
          // m block i: dimensions 2i and 2i + 1 of the lane group's piece; keys in pairs
          uint32_t f[4];
#pragma unroll
          for (int pr = 0; pr < 2; pr++) {
            const int ka = 4 * mb + 2 * pr;
            if constexpr (Q8) {
              const __half2 d = bits_h2(__byte_perm(vs[ka], vs[ka + 1], 0x5410));
              const uint32_t x = vr[ka][i / 2], y = vr[ka + 1][i / 2];
              const uint32_t e0 = __byte_perm(x, y, i & 1 ? 0x0602 : 0x0400), e1 = __byte_perm(x, y, i & 1 ? 0x0703 : 0x0501);
              f[2 * pr] = q8_pair((e0 & 0x00ff00ffu) ^ 0x64806480u, d);
              f[2 * pr + 1] = q8_pair((e1 & 0x00ff00ffu) ^ 0x64806480u, d);
            } else {
              f[2 * pr] = __byte_perm(vr[ka][i], vr[ka + 1][i], 0x5410);
              f[2 * pr + 1] = __byte_perm(vr[ka][i], vr[ka + 1][i], 0x7632);
            }
          }
#pragma unroll
          for (int nb = 0; nb < NB; nb++) {
            mma16816(o[i][nb], f, ph[mb][nb][0], ph[mb][nb][1]);
            if constexpr (SPLIT) mma16816(o[i][nb], f, pl[mb][nb][0], pl[mb][nb][1]);
          }
        }
      }
      if (more) load_v(kb + KT);
    }

    // ---- the CTA's warps together
#pragma unroll
    for (int nb = 0; nb < NB; nb++)
#pragma unroll
      for (int x = 0; x < 2; x++) {
        float t = l[nb][x];
        t += __shfl_xor_sync(0xffffffffu, t, 4);
        t += __shfl_xor_sync(0xffffffffu, t, 8);
        t += __shfl_xor_sync(0xffffffffu, t, 16);
        const uint32_t r = 8 * nb + 2 * c + x;
        if (g == 0) s_m[warp][r] = m[nb][x], s_l[warp][r] = t;
#pragma unroll
        for (int i = 0; i < KS; i++) {
          const uint32_t d = Q8 ? g * (D / 8) + 2 * i : 64 * (i / 4) + 8 * g + 2 * (i % 4);
          *reinterpret_cast<float2*>(&s_o[warp][r][d]) = make_float2(o[i][nb][x], o[i][nb][2 + x]);
        }
      }
    __syncthreads();
    const bool whole = sg.whole();
    float* slot = part + (2 * (size_t)blockIdx.x + (k0 > 0 ? 0 : 1)) * part_floats(ROWS, D);
    for (uint32_t x = threadIdx.x; x < nrows * (D / 4); x += 32 * kRowWarps) {
      const uint32_t r = x / (D / 4), d = x % (D / 4) * 4;
      float M = -INFINITY;
#pragma unroll
      for (int i = 0; i < kRowWarps; i++) M = fmaxf(M, s_m[i][r]);
      float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
      float den = 0.f;
#pragma unroll
      for (int i = 0; i < kRowWarps; i++) {
        const float f = M == -INFINITY ? 1.f : ex2(s_m[i][r] - M);
        const float4 v = *reinterpret_cast<const float4*>(&s_o[i][r][d]);
        den += s_l[i][r] * f;
        num.x += v.x * f, num.y += v.y * f, num.z += v.z * f, num.w += v.w * f;
      }
      if (s_wild) {
        const uint32_t t = group_div(a, r0 + r);
        for (uint32_t p = max(L, k0 * KT); p < min(end, k1 * KT); p++) {
          if (!sees(a, b, t, L, p)) continue;
          float v[4];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint64_t at = (uint64_t)p * D + d + i;
            if constexpr (Q8)
              v[i] = __half2float(__float2half_rn((float)((const int8_t*)vp)[at] * __half2float(vsp[at / 32])));
            else
              v[i] = __half2float(((const __half*)vp)[at]);
            if (fabsf(v[i]) < INFINITY) v[i] = 0.f;
          }
          num.x += v[0], num.y += v[1], num.z += v[2], num.w += v[3];
        }
      }
      if (whole) {
        const uint32_t rr = r0 + r;
        const uint32_t t = group_div(a, rr);
        T* out = (T*)a.out + ((uint64_t)b * a.n_tokens + t) * a.out_stride + (h * G + rr - t * G) * D + d;
        const float inv = den == 0.f ? 0.f : 1.f / den;
        act_put(out, num.x * inv), act_put(out + 1, num.y * inv), act_put(out + 2, num.z * inv), act_put(out + 3, num.w * inv);
      } else {
        *reinterpret_cast<float4*>(slot + part_at<ROWS>(d, r)) = num;
        if (d == 0) slot[ROWS * D + r] = M, slot[ROWS * D + ROWS + r] = den;
      }
    }
    __syncthreads();
  }
}

template <class T, bool Q8, int D, int NB>
int run_rows(cudaStream_t st, const TreeArgs& a) {
  constexpr int ROWS = 8 * NB, KT = Step<Q8, D, NB>::KEYS * kRowWarps;
  const uint32_t ctas = (uint32_t)num_sms() * Step<Q8, D, NB>::CTAS;
  void* part = nullptr;
  RF_TRY(scratch_alloc(&part, 2 * (size_t)ctas * part_floats(ROWS, D) * sizeof(float), st));
  cudaError_t e = launch_k(Launch{st, true}, tree_rows_kernel<T, Q8, D, NB>, dim3(ctas), dim3(32 * kRowWarps), 0, a,
                           (float*)part);
  if (e == cudaSuccess)
    e = launch_merge<T, D, KT, ROWS>(st, a, (const float*)part, ctas, cudaSharedmemCarveoutDefault);
  const cudaError_t f = cudaFreeAsync(part, st);
  RF_CUDA(e);
  RF_CUDA(f);
  return RF_OK;
}

template <class T, bool Q8>
int run_tree(cudaStream_t st, const TreeArgs& a) {
  const uint32_t rows = a.n_tokens * a.group;
  if (a.c.head_dim == 128) return rows <= 8 ? run_rows<T, Q8, 128, 1>(st, a) : run_rows<T, Q8, 128, 2>(st, a);
  return rows <= 8 ? run_rows<T, Q8, 64, 1>(st, a) : run_rows<T, Q8, 64, 2>(st, a);
}

}  // namespace

int scratch_alloc(void** out, size_t bytes, cudaStream_t st) {
  constexpr int kDevices = 64;
  static std::mutex mu;
  static cudaMemPool_t pools[kDevices];
  int dev = 0;
  RF_CUDA(cudaGetDevice(&dev));
  if (dev >= kDevices) return set_error(RF_EUNSUPPORTED, "device %d is beyond the %d that have a scratch pool", dev, kDevices);
  std::lock_guard<std::mutex> lk(mu);
  if (!pools[dev]) {
    cudaMemPoolProps p = {};
    p.allocType = cudaMemAllocationTypePinned;
    p.location.type = cudaMemLocationTypeDevice;
    p.location.id = dev;
    cudaMemPool_t pool;
    RF_CUDA(cudaMemPoolCreate(&pool, &p));
    uint64_t keep = UINT64_MAX;
    RF_CUDA(cudaMemPoolSetAttribute(pool, cudaMemPoolAttrReleaseThreshold, &keep));
    pools[dev] = pool;
  }
  const cudaError_t e = cudaMallocFromPoolAsync(out, bytes, pools[dev], st);
  if (e != cudaSuccess)
    return set_error(e == cudaErrorMemoryAllocation ? RF_ENOMEM : RF_ECUDA, "%zu bytes of attention scratch: %s", bytes,
                     cudaGetErrorString(e));
  return RF_OK;
}

}  // namespace rf

using namespace rf;

extern "C" {

int rf_tree_attention(const rf_kv_view* cache, const void* q, void* out, int act_type, uint32_t n_seqs,
                      uint32_t n_tokens, uint32_t n_heads, uint64_t q_stride, uint64_t out_stride,
                      const int32_t* hist_len, const int32_t* n_draft, const uint32_t* mask, float scale,
                      void* stream) {
  RF_TRY(check_kv_view(cache));
  const uint32_t es = act_bytes(act_type);
  if (!es) return set_error(RF_EINVAL, "activation type %d is not F32, F16 or BF16", act_type);
  if (!q || !out || !hist_len) return set_error(RF_EINVAL, "null argument");
  if (cache->head_dim != 64 && cache->head_dim != 128)
    return set_error(RF_EUNSUPPORTED, "tree attention covers head_dim 64 and 128, not %u", cache->head_dim);
  if (n_seqs > cache->n_seqs) return set_error(RF_EINVAL, "%u sequences, the cache holds %u", n_seqs, cache->n_seqs);
  if (!n_tokens || n_tokens > 1024) return set_error(RF_EINVAL, "n_tokens %u out of range 1..1024", n_tokens);
  if (!n_heads || n_heads % cache->n_kv_heads)
    return set_error(RF_EINVAL, "%u query heads are no multiple of %u KV heads", n_heads, cache->n_kv_heads);
  if (!(scale >= 0.f) || scale > 3.0e38f) return set_error(RF_EINVAL, "scale must be positive, or 0 for 1/sqrt(head_dim)");
  if (n_heads / cache->n_kv_heads > kMaxGroup)
    return set_error(RF_EUNSUPPORTED, "%u query heads a KV head, at most %u", n_heads / cache->n_kv_heads, kMaxGroup);
  const uint64_t row = (uint64_t)n_heads * cache->head_dim;
  if (!q_stride) q_stride = row;
  if (!out_stride) out_stride = row;
  if (q_stride < row || out_stride < row) return set_error(RF_EINVAL, "a token stride is below its row's elements");
  if (!aligned_to(q, 16) || !aligned_to(out, 16) || q_stride * es % 16 || out_stride * es % 16)
    return set_error(RF_EINVAL, "query and output rows must be 16-byte aligned");
  if (!aligned_to(hist_len, 4) || !aligned_to(n_draft, 4) || !aligned_to(mask, 4))
    return set_error(RF_EINVAL, "lengths and mask words must be 4-byte aligned");
  if ((uint64_t)n_seqs * n_tokens * n_heads > 0x7fffffffull)
    return set_error(RF_EINVAL, "%u x %u tokens of %u heads are too many for one call", n_seqs, n_tokens, n_heads);
  if (!n_seqs) return RF_OK;
  TreeArgs a{};
  a.c = *cache;
  a.q = q, a.out = out;
  a.q_stride = q_stride, a.out_stride = out_stride;
  a.n_seqs = n_seqs, a.n_tokens = n_tokens, a.n_heads = n_heads, a.words = (n_tokens + 31) / 32;
  a.hist_len = hist_len, a.n_draft = n_draft, a.mask = mask;
  a.group = n_heads / cache->n_kv_heads;
  a.group_magic = (uint32_t)(((1ull << 32) + a.group - 1) / a.group);
  a.scale = scale > 0.f ? scale : 1.f / sqrtf((float)cache->head_dim);
  RF_TRY(verify_error_ptr(&a.err));
  const cudaStream_t st = (cudaStream_t)stream;
  // Two fragments of 8 rows are what tree_rows_kernel has registers for.  Over 32768 positions, 32/8 heads of 128:
  // 16 rows in it 28 us (Q8_0) and 32 us (f16), 20 rows in the other kernel 34 and 36.
  if (n_tokens * a.group > 16) return run_tree_tc(act_type, a, st);
  const bool q8 = cache->type == RF_TYPE_Q8_0;
  switch (act_type) {
    case RF_ACT_F32: return q8 ? run_tree<float, true>(st, a) : run_tree<float, false>(st, a);
    case RF_ACT_F16: return q8 ? run_tree<__half, true>(st, a) : run_tree<__half, false>(st, a);
    default: return q8 ? run_tree<__nv_bfloat16, true>(st, a) : run_tree<__nv_bfloat16, false>(st, a);
  }
}

}  // extern "C"
