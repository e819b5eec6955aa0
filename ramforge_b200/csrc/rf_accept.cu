// rf_accept.cu - the verdict on drafted tokens: which of them stand, which token comes behind them and which
// positions of the cache their rows get, from the target's probabilities and given random numbers
// (rf_verify_drafts) or by its best tokens (rf_verify_greedy).
//
// Sampling keeps the target's distribution.  At a node of the drafted tree let p be the target's row, q the draft's,
// and c1, c2, ... the drafted tokens behind it, all drawn from q, in order.  c1 stands with probability
// min(1, p(c1) / q(c1)); if not, what is left of p is p_1 = (p - q)+ / Z_1, Z_1 = sum (p - q)+, c2 is tried
// against p_1, and so on.  Without the divisions, with r_0 = p and S_0 = 1:
//   c_k stands iff  u S_k q(c_k) < r_k(c_k);   else  a_{k+1} = a_k + S_k,  r_{k+1} = (p - a_{k+1} q)+,  S_{k+1} = sum r_{k+1}
// (p_k = r_k / S_k, and (p_k - q)+ = (p - a_k q - S_k q)+ / S_k).  When no more are left, the next token is the least
// x with r(0) + ... + r(x) > u S.  Drafts without probabilities are certain of their token: q is 1 there.
//
// Products and sums are taken in 64 bits: p and q are at most 32-bit numbers, so u q is exact, and on which side of a
// border a number lies depends on the order of the sums (which follows the number of CTAs a sequence) only where their last
// bits decide.  r is one fused operation, but a and S are sums: what 2^-48 of p and less is left of it is rounding.
#include <algorithm>
#include <type_traits>

#include "rf_act.cuh"
#include "rf_device.cuh"
#include "rf_verify.h"

namespace rf {
namespace {

constexpr uint32_t kMaxDrafts = 1024;

struct WalkArgs {
  const int32_t *tokens, *parent, *n_draft, *hist;
  int32_t *out_tokens, *n_accepted, *positions;
  uint32_t vocab, n_tokens;
  unsigned* err;
};

// A sequence's drafts in shared memory.
struct Drafts {
  int32_t parent[kMaxDrafts], token[kMaxDrafts];
};

// n_draft of sequence b, or -1 (and the error bit) where it is out of range.
__device__ __forceinline__ int draft_count(const WalkArgs& a, uint32_t b) {
  const int n = a.n_draft ? a.n_draft[b] : (int)a.n_tokens;
  return n < 0 || (uint32_t)n > a.n_tokens ? -1 : n;
}
// Parent and token of draft j; a parent of -2 behind the last of n, and, with the error bit, where either is out of range.
// The count is looked at last, so that it arrives with the rest.
__device__ __forceinline__ void draft_at(const WalkArgs& a, uint32_t b, int j, int n, int* parent, int* token) {
  const uint64_t at = (uint64_t)b * a.n_tokens + j;
  *parent = a.parent ? a.parent[at] : j - 1;
  *token = a.tokens[at];
  if (*parent < -1 || *parent >= j || *token < 0 || (uint32_t)*token >= a.vocab) {
    if (j < n) atomicOr(a.err, kVerifyRange);
    *parent = -2, *token = 0;
  }
  if (j >= n) *parent = -2;
}
// One warp: the first draft behind `last` whose parent is `node`, or n.
__device__ __forceinline__ int next_child(const int32_t* parent, int n, int node, int last, uint32_t lane) {
  for (int j0 = last + 1; j0 < n; j0 += 32) {
    const int j = j0 + (int)lane;
    const uint32_t hit = __ballot_sync(0xffffffffu, j < n && parent[j] == node);
    if (hit) return j0 + __ffs(hit) - 1;
  }
  return n;
}

// ---- clusters ---------------------------------------------------------------------------
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// 64 bits to `p`'s place in the shared memory of the cluster's CTA `rank`.
__device__ __forceinline__ void push64(const void* p, uint32_t rank, uint64_t v) {
  asm volatile(
      "{ .reg .b32 a; mapa.shared::cluster.u32 a, %0, %1;\n\t"
      "st.shared::cluster.b64 [a], %2; }" ::"r"((uint32_t)__cvta_generic_to_shared(p)),
      "r"(rank), "l"(v)
      : "memory");
}

// E elements of a row from x on as f32, zeros from `end` on.
template <class T, int E>
__device__ __forceinline__ void load_piece(const T* row, uint32_t x, uint32_t end, float (&v)[E]) {
  if constexpr (E == Act<T>::kVec) {
    if (x + E <= end) {
      Act<T>::unpack(ld_once(row + x), v);
      return;
    }
  }
#pragma unroll
  for (int e = 0; e < E; e++) v[e] = x + e < end ? Act<T>::get(row + x + e) : 0.f;
}

// ---------------------------------------------------------------------------
// Sampling: a cluster a sequence.
//
// Every CTA gathers the drafts and walks until sums are needed; a pass over the vocabulary gives them, a run of it
// for each CTA and each of its warps, and the CTAs' sums go to all of them.  What comes next is CTA 0's to say: the others follow
// it, so that all meet at the same barriers whatever they read.  A chain takes one pass, and with it one meeting; each further
// draft of a node that is refused takes one more (of drafts that were certain, all of a node's together one, and another
// wherever less than a sixteenth of the last sum is left: a difference of sums keeps too few bits there).  The bytes of the last rows bound a batch (64 sequences, 128256 tokens, f32:
// 65.7 MB), latency a sequence: two dependent reads, the walk, the pass, the search of one warp.
// ---------------------------------------------------------------------------
struct SampleArgs {
  WalkArgs w;
  const void *target, *draft;
  uint64_t target_stride, draft_stride;
  const float *accept_u, *next_u;
  uint32_t ctas, run;  // CTAs a cluster, elements of a warp's run
};

constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32;
constexpr uint32_t kMaxCluster = 8, kMostCtas = 16;  // what any GPU of the kind has room for, and what this one

struct Pass {  // what a pass sums up: rows of `node`, the share a of q that is off; certain drafts: those up to `refused` are out
  int32_t node, refused;
  double a;
};
// What follows a pass.  kLast: the token, or, where nothing is left, a pass over all of the target's row (kWhole).
enum Next : uint32_t { kMore, kLast, kWhole };

template <class T, int E>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(SampleArgs a) {
  __shared__ Drafts s;
  __shared__ float s_u[kMaxDrafts], s_p[kMaxDrafts], s_q[kMaxDrafts];
  __shared__ int32_t s_path[kMaxDrafts];  // draft j's place among the tokens that stand, or -1
  __shared__ int32_t s_out[kMaxDrafts];   // certain drafts: the tokens that are out
  __shared__ double s_seg[kSampleWarps], s_part[kSampleWarps], s_sum[2][kMostCtas];
  __shared__ Pass s_pass;       // from CTA 0 (the first one from the CTA itself)
  __shared__ uint64_t s_next[2];  // CTA 0's word on what follows a pass: Next, and the tokens that stand
  __shared__ int s_n_out;
  const WalkArgs& w = a.w;
  const uint32_t b = blockIdx.x / a.ctas, rank = blockIdx.x % a.ctas, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (a.ctas > 1) cluster_arrive();
  griddep_launch();
  griddep_wait();
  const int count = draft_count(w, b), n = max(count, 0);
  const float u_next = a.next_u[b];  // wanted last, asked for first
  const int hist = w.positions ? w.hist[b] : 0;
  auto p_row = [&](int node) { return (const T*)a.target + ((uint64_t)b * (w.n_tokens + 1) + node + 1) * a.target_stride; };
  auto q_row = [&](int node) { return (const T*)a.draft + ((uint64_t)b * w.n_tokens + node + 1) * a.draft_stride; };
  for (int j = tid; j < (int)w.n_tokens; j += kSampleThreads) {
    int parent, token;
    draft_at(w, b, j, n, &parent, &token);
    s.parent[j] = parent, s.token[j] = token, s_path[j] = -1;
    s_u[j] = a.accept_u[(uint64_t)b * w.n_tokens + j];
    s_p[j] = parent < -1 ? 0.f : fmaxf(Act<T>::get(p_row(parent) + token), 0.f);
    s_q[j] = parent < -1 || !a.draft ? 1.f : Act<T>::get(q_row(parent) + token);
  }
  __syncthreads();
  if (a.ctas > 1) cluster_wait();  // all have begun: their shared memory may be written

  // the walk's state, in every thread of warp 0
  int node = -1, last = -1, taken = 0, tried = 0;
  double off = 0.0, mass = 1.0, gone = 0.0, base = 0.0;  // base: certain drafts, the sum that mass is a difference of
  bool whole = false;  // certain drafts: mass comes from the sum of the node's whole row
  Next next = kLast;
  auto walk = [&]() {  // until sums are needed
    bool final = true, masked = true;
    if (!a.draft && tried) base = mass, mass -= gone, gone = 0.0;  // the sum has come
    while (true) {
      // certain drafts: what is left has lost four bits as a difference, so it is summed up by itself
      if (mass < base / 16) {
        final = false;
        break;
      }
      const int j = next_child(s.parent, n, node, last, lane);
      if (j >= n) break;
      last = j;
      double left = s_p[j];
      const double qc = s_q[j];
      if (tried) {
        if (a.draft) {
          left = fmax(fma(-off, qc, left), 0.0);
        } else {
          bool out = false;
          for (int i = lane; i < j; i += 32) out |= s.parent[i] == node && s.token[i] == s.token[j];
          if (__any_sync(0xffffffffu, out)) left = 0.0;
        }
      }
      if ((double)s_u[j] * qc * mass < left) {
        if (lane == 0) s_path[j] = taken;
        __syncwarp();
        node = j, taken++, tried = 0, off = 0.0, mass = 1.0, base = 0.0, whole = false, final = true;
        continue;
      }
      tried++;
      final = next_child(s.parent, n, node, last, lane) >= n;
      if (a.draft) {
        off += mass;
        break;
      }
      if (final) break;
      // certain drafts: the sum of what is left is that of the whole row without the tokens that are out
      if (whole) {
        mass -= left;
      } else {
        gone = left, whole = true, masked = false;
        break;
      }
    }
    next = !final ? kMore : tried ? kLast : kWhole;
    if (lane == 0) s_pass = Pass{node, tried && masked ? last : -1, off};
  };
  if (warp == 0) walk();
  const uint32_t x0 = min((rank * kSampleWarps + warp) * a.run, w.vocab), x1 = min(x0 + a.run, w.vocab);
  int token = -1, stand = 0;
  uint32_t turn = 0;
  while (true) {
    if (tid == 0) s_n_out = 0;
    __syncthreads();
    const Pass ps = s_pass;
    const T *p = p_row(ps.node), *q = a.draft && ps.a > 0.0 ? q_row(ps.node) : nullptr;
    if (!a.draft && ps.refused >= 0) {
      for (int j = tid; j <= min(ps.refused, n - 1); j += kSampleThreads)
        if (s.parent[j] == ps.node) s_out[atomicAdd(&s_n_out, 1)] = s.token[j];
      __syncthreads();
    }
    const int n_out = s_n_out;
    // what is left of the tokens from x on, out of their numbers in p and q; NaN counts as 0 in all of this
    auto strike = [&](uint32_t x, float (&pf)[E]) {
      for (int i = 0; i < n_out; i++)
#pragma unroll
        for (int e = 0; e < E; e++)
          if (s_out[i] == (int)(x + e)) pf[e] = 0.f;
    };
    auto weight = [&](float pf, float qf) { return q ? fma(-ps.a, (double)qf, (double)pf) : (double)pf; };
    auto weights = [&](uint32_t x, uint32_t to, double (&v)[E]) {
      float pf[E], qf[E] = {};
      load_piece<T, E>(p, x, to, pf);
      if (q) load_piece<T, E>(q, x, to, qf);
      strike(x, pf);
#pragma unroll
      for (int e = 0; e < E; e++) {
        const double r = weight(pf[e], qf[e]);
        v[e] = r > 0.0 ? r : 0.0;
      }
    };
    auto sum_run = [&](uint32_t from, uint32_t to) {  // a warp's sum of what is left of a run
      double sums[2] = {};
      constexpr int U = E == 1 ? 8 : 8 / E;  // pieces of a lane in flight
      for (uint32_t x = from + lane * E; x < to; x += U * 32 * E) {
        float pf[U][E], qf[U][E] = {};
#pragma unroll
        for (int u = 0; u < U; u++) load_piece<T, E>(p, x + u * 32 * E, to, pf[u]);
        if (q)
#pragma unroll
          for (int u = 0; u < U; u++) load_piece<T, E>(q, x + u * 32 * E, to, qf[u]);
#pragma unroll
        for (int u = 0; u < U; u++) {
          strike(x + u * 32 * E, pf[u]);
#pragma unroll
          for (int e = 0; e < E; e++) {
            const double r = weight(pf[u][e], qf[u][e]);
            if (r > 0.0) sums[e & 1] += r;
          }
        }
      }
      double sum = sums[0] + sums[1];
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      return sum;
    };
    const double sum = sum_run(x0, x1);
    if (lane == 0) s_seg[warp] = sum;
    __syncthreads();
    if (tid < a.ctas) {
      double all = 0.0;
      for (int i = 0; i < kSampleWarps; i++) all += s_seg[i];
      const uint64_t word = (uint64_t)next | (uint64_t)(uint32_t)taken << 32;
      if (a.ctas == 1) {
        s_sum[turn][0] = all, s_next[turn] = word;
      } else {
        push64(&s_sum[turn][rank], tid, __double_as_longlong(all));
        if (rank == 0) push64(&s_next[turn], tid, word);
      }
    }
    __syncwarp();
    if (a.ctas > 1)
      cluster_arrive(), cluster_wait();
    else
      __syncthreads();
    mass = 0.0;
    for (uint32_t r = 0; r < a.ctas; r++) mass += s_sum[turn][r];
    const Next now = (Next)(uint32_t)s_next[turn];
    stand = (int)(s_next[turn] >> 32);
    if (now == kMore || (now == kLast && !(mass > 0.0))) {
      if (rank == 0 && warp == 0) {
        if (now == kMore) {
          walk();
        } else {
          next = kWhole;
          if (lane == 0) s_pass = Pass{ps.node, -1, 0.0};
        }
        __syncwarp();
        if (lane > 0 && lane < a.ctas) {
          push64(&s_pass.node, lane, (uint64_t)(uint32_t)s_pass.node | (uint64_t)(uint32_t)s_pass.refused << 32);
          push64(&s_pass.a, lane, __double_as_longlong(s_pass.a));
        }
        __syncwarp();
      }
      if (a.ctas > 1) cluster_arrive(), cluster_wait();
      turn ^= 1;
      continue;
    }
    // the token: the CTA, the warp and the place where the sum passes the aim
    if (!(mass > 0.0)) break;  // the target's row has nothing: token -1
    const double aim = (double)fmaxf(u_next, 0.f) * mass;
    double before = 0.0;
    uint32_t owner = 0, some = 0;
    for (uint32_t r = 0; r < a.ctas; r++)
      if (s_sum[turn][r] > 0.0) some = r;  // the sums' last bits may leave the aim behind the end: the last that has any
    for (; owner < some && !(before + s_sum[turn][owner] > aim); owner++) before += s_sum[turn][owner];
    if (owner != rank) break;
    // the run, then, by all warps again, the part of it
    auto pick = [&](const double* sums) {
      uint32_t i = 0, full = 0;
      for (uint32_t j = 0; j < kSampleWarps; j++)
        if (sums[j] > 0.0) full = j;
      for (; i < full && !(before + sums[i] > aim); i++) before += sums[i];
      return i;
    };
    const uint32_t seg = pick(s_seg), y0 = min((rank * kSampleWarps + seg) * a.run, w.vocab), y1 = min(y0 + a.run, w.vocab);
    const uint32_t part = ((a.run + kSampleWarps - 1) / kSampleWarps + E - 1) / E * E;
    const uint32_t z0 = min(y0 + warp * part, y1), z1 = min(z0 + part, y1);
    const double fine = sum_run(z0, z1);
    if (lane == 0) s_part[warp] = fine;
    __syncthreads();
    if (warp == pick(s_part)) {
      int found = -1, latest = -1;
      for (uint32_t x = z0; x < z1 && found < 0; x += 32 * E) {
        double v[E], own = 0.0;
        weights(x + lane * E, z1, v);
        int high = -1;
#pragma unroll
        for (int e = 0; e < E; e++) {
          own += v[e];
          if (v[e] > 0.0) high = (int)(x + lane * E) + e;
        }
        double cum = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double c = __shfl_up_sync(0xffffffffu, cum, o);
          if (lane >= (uint32_t)o) cum += c;
        }
        double at = before + (cum - own);
        int mine = -1;
#pragma unroll
        for (int e = 0; e < E; e++) {
          at += v[e];
          if (mine < 0 && v[e] > 0.0 && at > aim) mine = (int)(x + lane * E) + e;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, mine >= 0), any = __ballot_sync(0xffffffffu, high >= 0);
        if (hit) found = __shfl_sync(0xffffffffu, mine, __ffs(hit) - 1);
        if (any) latest = __shfl_sync(0xffffffffu, high, 31 - __clz(any));
        before += __shfl_sync(0xffffffffu, cum, 31);
      }
      token = found >= 0 ? found : latest;
    }
    break;
  }
  // CTA 0 writes the walk, the warp that found it the token
  if (count < 0 && tid == 0) atomicOr(w.err, kVerifyRange);
  int32_t* out = w.out_tokens + (uint64_t)b * (w.n_tokens + 1);
  if (rank == 0) {
    if (tid == 0) {
      w.n_accepted[b] = stand;
      if (!(mass > 0.0)) atomicOr(w.err, kVerifyRange);
      if (!(mass > 0.0) || count < 0) out[stand] = -1;
    }
    for (int j = tid; j < (int)w.n_tokens; j += kSampleThreads) {
      const int place = j < n ? s_path[j] : -1;
      if (place >= 0) out[place] = s.token[j];
      if (w.positions) w.positions[(uint64_t)b * w.n_tokens + j] = place >= 0 ? hist + place : -1;
      if (j >= stand) out[j + 1] = -1;
    }
  }
  if (token >= 0 && count >= 0 && lane == 0) out[stand] = token;
}

// ---------------------------------------------------------------------------
// Greedy: the best token of every row (a cluster a row), then the walk.
// ---------------------------------------------------------------------------
struct BestArgs {
  WalkArgs w;
  const void* logits;
  uint64_t stride;
  int32_t* best;
  uint32_t ctas;  // CTAs a cluster
};

constexpr int kBestThreads = 512;

// Larger numbers have larger keys, of equal numbers the lower index.
__device__ __forceinline__ uint64_t best_key(float v, uint32_t x) {
  const uint32_t b = __float_as_uint(v == 0.f ? 0.f : v);
  return (uint64_t)((b & 0x80000000u) ? ~b : b | 0x80000000u) << 32 | (uint32_t)~x;
}

// The largest of 16 bytes' numbers; NaN where all of them are.
template <class T>
__device__ __forceinline__ float piece_top(const uint4& u) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  } else {
    using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
    const T2* h = reinterpret_cast<const T2*>(&u);
    const T2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(Act<T>::get(&m.x), Act<T>::get(&m.y));
  }
}

template <class T>
__global__ void __launch_bounds__(kBestThreads) best_kernel(BestArgs a) {
  constexpr uint32_t E = Act<T>::kVec;
  __shared__ uint64_t s_best[kBestThreads / 32], s_cta[kMaxCluster];
  const uint32_t row_at = blockIdx.x / a.ctas, rank = blockIdx.x % a.ctas, tid = threadIdx.x;
  if (a.ctas > 1) cluster_arrive();
  griddep_launch();
  griddep_wait();
  const uint32_t rows = a.w.n_tokens + 1, b = row_at / rows, r = row_at - b * rows, V = a.w.vocab;
  if (a.ctas > 1) cluster_wait();
  const bool live = (int)r <= max(draft_count(a.w, b), 0);  // not behind the sequence's last draft
  const T* row = (const T*)a.logits + (uint64_t)row_at * a.stride;

  // The row's whole 16-byte pieces, a run of them for each CTA; what lies before and behind them one by one.
  const uint32_t lead = min((uint32_t)((16 - ((uintptr_t)row & 15)) & 15) / (uint32_t)sizeof(T), V), pieces = (V - lead) / E;
  const uint32_t p0 = (uint64_t)pieces * rank / a.ctas, p1 = (uint64_t)pieces * (rank + 1) / a.ctas, tail = lead + pieces * E;
  float top = -INFINITY;
  uint32_t at = ~0u;
  // whether a later number is taken for the one held: a larger one, -infinity as the first, no NaN
  auto better = [](float v, float held, bool none) { return v > held || (none && v == -INFINITY); };
  if (live) {
    if (rank == 0 && tid < lead) {
      const float v = Act<T>::get(row + tid);
      if (better(v, top, true)) top = v, at = tid;
    }
    // the largest number and the first piece that has it, which is kept: one comparison a piece
    float most = -INFINITY;
    uint32_t piece = ~0u;
    uint4 kept = make_uint4(0, 0, 0, 0);
    constexpr int U = 4;  // loads in flight
    for (uint32_t p = p0 + tid; p < p1; p += U * kBestThreads) {
      uint4 u[U];
#pragma unroll
      for (int i = 0; i < U; i++)
        if (p + i * kBestThreads < p1) u[i] = ld_once(row + lead + (uint64_t)(p + i * kBestThreads) * E);
      float v[U];
#pragma unroll
      for (int i = 0; i < U; i++)
        if (p + i * kBestThreads < p1) {
          v[i] = piece_top<T>(u[i]);
          if (v[i] > most) most = v[i], piece = p + i * kBestThreads, kept = u[i];
        }
      if (piece == ~0u)  // none of them above -infinity
#pragma unroll
        for (int i = U - 1; i >= 0; i--)
          if (p + i * kBestThreads < p1 && v[i] == -INFINITY) piece = p + i * kBestThreads, kept = u[i];
    }
    if (piece != ~0u && better(most, top, at == ~0u)) {
      float v[E];
      Act<T>::unpack(kept, v);
      uint32_t first = 0;
#pragma unroll
      for (int e = E - 1; e >= 0; e--)
        if (v[e] == most) first = e;
      top = most, at = lead + piece * E + first;
    }
    if (rank == a.ctas - 1 && tid < V - tail) {
      const float v = Act<T>::get(row + tail + tid);
      if (better(v, top, at == ~0u)) top = v, at = tail + tid;
    }
  }
  uint64_t best = at == ~0u ? 0 : best_key(top, at);  // 0: NaN alone
#pragma unroll
  for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((tid & 31) == 0) s_best[tid >> 5] = best;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kBestThreads / 32; i++) best = max(best, s_best[i]);
    if (a.ctas > 1) push64(&s_cta[rank], 0, best);
  }
  __syncwarp();
  if (a.ctas > 1) cluster_arrive(), cluster_wait();
  if (rank || tid || !live) return;
  if (a.ctas > 1)
    for (uint32_t i = 0; i < a.ctas; i++) best = max(best, s_cta[i]);
  a.best[row_at] = best ? (int32_t)~(uint32_t)best : 0;
}

__global__ void __launch_bounds__(128) greedy_walk_kernel(BestArgs a) {
  __shared__ Drafts s;
  __shared__ int32_t s_path[kMaxDrafts];
  __shared__ int s_taken;
  griddep_launch();
  griddep_wait();
  const WalkArgs& w = a.w;
  const uint32_t b = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
  const int count = draft_count(w, b), n = max(count, 0);
  if (count < 0 && tid == 0) atomicOr(w.err, kVerifyRange);
  const int32_t* best = a.best + (uint64_t)b * (w.n_tokens + 1);
  for (int j = tid; j < n; j += 128) {
    int parent, token;
    draft_at(w, b, j, n, &parent, &token);
    s.parent[j] = parent >= -1 && best[parent + 1] == token ? parent : -2;  // only those that would stand
    s.token[j] = token, s_path[j] = -1;
  }
  __syncthreads();
  if (tid < 32) {
    int node = -1, taken = 0;
    while (true) {
      const int j = next_child(s.parent, n, node, node, lane);
      if (j >= n) break;
      if (lane == 0) s_path[j] = taken;
      node = j, taken++;
    }
    if (lane == 0) {
      s_taken = taken;
      w.n_accepted[b] = taken;
      w.out_tokens[(uint64_t)b * (w.n_tokens + 1) + taken] = count < 0 ? -1 : best[node + 1];
    }
  }
  __syncthreads();
  const int taken = s_taken;
  for (int j = tid; j < (int)w.n_tokens; j += 128) {
    const int place = j < n ? s_path[j] : -1;
    if (place >= 0) w.out_tokens[(uint64_t)b * (w.n_tokens + 1) + place] = s.token[j];
    if (w.positions) w.positions[(uint64_t)b * w.n_tokens + j] = place >= 0 ? w.hist[b] + place : -1;
    if (j >= taken) w.out_tokens[(uint64_t)b * (w.n_tokens + 1) + j + 1] = -1;
  }
}

// CTAs a cluster: as many as still give all of `units` a place at once (per_sm an SM).
uint32_t cluster_size(uint32_t units, uint32_t per_sm) {
  uint32_t c = kMaxCluster;
  while (c > 1 && (uint64_t)units * c > (uint64_t)per_sm * num_sms()) c /= 2;
  return c;
}

template <class Args>
cudaError_t launch_clusters(cudaStream_t st, void (*k)(Args), uint32_t units, uint32_t ctas, int threads, const Args& a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(units * ctas);
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 2 : 1;
  if (ctas > kMaxCluster) {
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  return cudaLaunchKernelEx(&cfg, k, a);
}

int check_walk(int type, uint32_t vocab, uint32_t n_seqs, uint32_t n_tokens, const void* rows, uint64_t* stride,
               const int32_t* tokens, const int32_t* parent, const int32_t* n_draft, const int32_t* hist_len,
               const int32_t* out_tokens, const int32_t* n_accepted, const int32_t* positions) {
  const uint32_t es = act_bytes(type);
  if (!es) return set_error(RF_EINVAL, "activation type %d is not F32, F16 or BF16", type);
  if (!vocab || vocab > 0x7fffffffu) return set_error(RF_EINVAL, "a vocabulary of %u is out of range", vocab);
  if (n_tokens > kMaxDrafts) return set_error(RF_EINVAL, "n_tokens %u out of range 0..%u", n_tokens, kMaxDrafts);
  if ((uint64_t)n_seqs * (n_tokens + 1) > 0x7fffffffull) return set_error(RF_EINVAL, "%u sequences are too many for one call", n_seqs);
  if (n_seqs && (!rows || !out_tokens || !n_accepted)) return set_error(RF_EINVAL, "null argument");
  if (n_seqs && n_tokens && !tokens) return set_error(RF_EINVAL, "null drafted tokens");
  if (positions && !hist_len) return set_error(RF_EINVAL, "positions need hist_len");
  if (!*stride) *stride = vocab;
  if (*stride < vocab)
    return set_error(RF_EINVAL, "row stride %llu is below the row's %u elements", (unsigned long long)*stride, vocab);
  if (!aligned_to(rows, es)) return set_error(RF_EINVAL, "rows must be aligned to their element size");
  for (const int32_t* p : {tokens, parent, n_draft, hist_len, out_tokens, n_accepted, positions})
    if (!aligned_to(p, 4)) return set_error(RF_EINVAL, "tokens, lengths and positions must be 4-byte aligned");
  return RF_OK;
}

}  // namespace
}  // namespace rf

using namespace rf;

extern "C" {

int rf_verify_drafts(const void* target, const void* draft, int prob_type, uint32_t vocab, uint32_t n_seqs,
                     uint32_t n_tokens, uint64_t target_stride, uint64_t draft_stride, const int32_t* tokens,
                     const int32_t* parent, const int32_t* n_draft, const float* accept_u, const float* next_u,
                     const int32_t* hist_len, int32_t* out_tokens, int32_t* n_accepted, int32_t* positions, void* stream) {
  RF_TRY(check_walk(prob_type, vocab, n_seqs, n_tokens, target, &target_stride, tokens, parent, n_draft, hist_len,
                    out_tokens, n_accepted, positions));
  if (!draft_stride) draft_stride = vocab;
  if (draft_stride < vocab)
    return set_error(RF_EINVAL, "row stride %llu is below the row's %u elements", (unsigned long long)draft_stride, vocab);
  if (!aligned_to(draft, act_bytes(prob_type))) return set_error(RF_EINVAL, "rows must be aligned to their element size");
  if (n_seqs && (!next_u || (n_tokens && !accept_u))) return set_error(RF_EINVAL, "null random numbers");
  if (!aligned_to(accept_u, 4) || !aligned_to(next_u, 4)) return set_error(RF_EINVAL, "random numbers must be 4-byte aligned");
  if (!n_seqs) return RF_OK;
  SampleArgs a{};
  a.w = WalkArgs{tokens, parent, n_draft, hist_len, out_tokens, n_accepted, positions, vocab, n_tokens, nullptr};
  a.target = target, a.draft = n_tokens ? draft : nullptr;
  a.target_stride = target_stride, a.draft_stride = draft_stride;
  a.accept_u = accept_u, a.next_u = next_u;
  RF_TRY(verify_error_ptr(&a.w.err));
  const uint32_t es = act_bytes(prob_type);
  const bool vec = aligned_to(target, 16) && target_stride * es % 16 == 0 &&
                   (!a.draft || (aligned_to(draft, 16) && draft_stride * es % 16 == 0));
  // Clusters of 16 for long rows, as far as the GPU has room for them at once (7, one for most of its processing clusters):
  // a tree of 24 over 128256 tokens 13.6 us with 8, 11.3 with 16, over 32000 9.1 and 9.3.
  a.ctas = n_seqs <= 7 && vocab >= 65536 ? kMostCtas : cluster_size(n_seqs, 2);
  const uint32_t warps = a.ctas * kSampleWarps, unit = 16 / es;
  a.run = ((vocab + warps - 1) / warps + unit - 1) / unit * unit;
  auto* k = prob_type == RF_ACT_F32   ? (vec ? sample_kernel<float, 4> : sample_kernel<float, 1>)
            : prob_type == RF_ACT_F16 ? (vec ? sample_kernel<__half, 8> : sample_kernel<__half, 1>)
                                      : (vec ? sample_kernel<__nv_bfloat16, 8> : sample_kernel<__nv_bfloat16, 1>);
  RF_CUDA(launch_clusters((cudaStream_t)stream, k, n_seqs, a.ctas, kSampleThreads, a));
  return RF_OK;
}

int rf_verify_greedy(const void* logits, int logit_type, uint32_t vocab, uint32_t n_seqs, uint32_t n_tokens,
                     uint64_t logits_stride, const int32_t* tokens, const int32_t* parent, const int32_t* n_draft,
                     const int32_t* hist_len, int32_t* best, int32_t* out_tokens, int32_t* n_accepted, int32_t* positions,
                     void* stream) {
  RF_TRY(check_walk(logit_type, vocab, n_seqs, n_tokens, logits, &logits_stride, tokens, parent, n_draft, hist_len,
                    out_tokens, n_accepted, positions));
  if (n_seqs && !best) return set_error(RF_EINVAL, "null argument");
  if (!aligned_to(best, 4)) return set_error(RF_EINVAL, "tokens, lengths and positions must be 4-byte aligned");
  if (!n_seqs) return RF_OK;
  BestArgs a{};
  a.w = WalkArgs{tokens, parent, n_draft, hist_len, out_tokens, n_accepted, positions, vocab, n_tokens, nullptr};
  a.logits = logits, a.stride = logits_stride, a.best = best;
  RF_TRY(verify_error_ptr(&a.w.err));
  const uint32_t rows = n_seqs * (n_tokens + 1);
  a.ctas = cluster_size(rows, 2);
  auto* k = logit_type == RF_ACT_F32 ? best_kernel<float> : logit_type == RF_ACT_F16 ? best_kernel<__half> : best_kernel<__nv_bfloat16>;
  RF_CUDA(launch_clusters((cudaStream_t)stream, k, rows, a.ctas, kBestThreads, a));
  RF_CUDA(launch_k(Launch{(cudaStream_t)stream, true}, greedy_walk_kernel, dim3(n_seqs), dim3(128), 0, a));
  return RF_OK;
}

}  // extern "C"
