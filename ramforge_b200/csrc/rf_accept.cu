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
// Products and sums are taken in 64 bits: p and q are at most 32-bit numbers, so u q is exact, and which side of a
// border a number lies on does not depend on the order of the sums.
#include <algorithm>

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
// Parent and token of draft j; a parent of -2 and the error bit where either is out of range.
__device__ __forceinline__ void draft_at(const WalkArgs& a, uint32_t b, int j, int* parent, int* token) {
  const uint64_t at = (uint64_t)b * a.n_tokens + j;
  *parent = a.parent ? a.parent[at] : j - 1;
  *token = a.tokens[at];
  if (*parent < -1 || *parent >= j || *token < 0 || (uint32_t)*token >= a.vocab) {
    atomicOr(a.err, kVerifyRange);
    *parent = -2, *token = 0;
  }
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

// ---------------------------------------------------------------------------
// Sampling: a CTA a sequence.  Warp 0 walks; a pass over the vocabulary (each warp a run of it) gives the sums.
// ---------------------------------------------------------------------------
struct SampleArgs {
  WalkArgs w;
  const void *target, *draft;
  uint64_t target_stride, draft_stride;
  const float *accept_u, *next_u;
};

constexpr int kSampleThreads = 1024, kSampleWarps = kSampleThreads / 32;

struct Pass {  // what a pass sums: target row, draft row, share a of q to take off, or drafts that are certain
  int node, refused;  // refused: index of the last child tried (drafts without probabilities: those up to it are out)
  double a;
};

template <class T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(SampleArgs a) {
  __shared__ Drafts s;
  __shared__ float s_u[kMaxDrafts], s_p[kMaxDrafts], s_q[kMaxDrafts];
  __shared__ int32_t s_path[kMaxDrafts];  // draft j's place among the tokens that stand, or -1
  __shared__ double s_seg[kSampleWarps];
  __shared__ Pass s_pass;
  __shared__ int s_token, s_final;
  griddep_launch();
  griddep_wait();
  const WalkArgs& w = a.w;
  const uint32_t b = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, V = w.vocab;
  const int count = draft_count(w, b), n = max(count, 0);
  if (count < 0 && tid == 0) atomicOr(w.err, kVerifyRange);
  auto p_row = [&](int node) { return (const T*)a.target + ((uint64_t)b * (w.n_tokens + 1) + node + 1) * a.target_stride; };
  auto q_row = [&](int node) { return (const T*)a.draft + ((uint64_t)b * w.n_tokens + node + 1) * a.draft_stride; };
  for (int j = tid; j < n; j += kSampleThreads) {
    int parent, token;
    draft_at(w, b, j, &parent, &token);
    s.parent[j] = parent, s.token[j] = token, s_path[j] = -1;
    s_u[j] = a.accept_u[(uint64_t)b * w.n_tokens + j];
    s_p[j] = parent < -1 ? 0.f : fmaxf(Act<T>::get(p_row(parent) + token), 0.f);
    s_q[j] = parent < -1 || !a.draft ? 1.f : Act<T>::get(q_row(parent) + token);
  }
  if (tid == 0) s_token = -1;
  __syncthreads();

  // weight of token x in a pass
  auto weight = [&](const Pass& ps, const T* p, const T* q, uint32_t x) {
    const double px = Act<T>::get(p + x);
    if (q) return fmax(fma(-ps.a, (double)Act<T>::get(q + x), px), 0.0);
    for (int j = 0; j <= ps.refused; j++)
      if (s.parent[j] == ps.node && s.token[j] == (int)x) return 0.0;
    return fmax(px, 0.0);
  };
  const uint32_t per = (V + kSampleWarps - 1) / kSampleWarps, x0 = min(warp * per, V), x1 = min(x0 + per, V);

  // the walk's state, in every thread of warp 0
  int node = -1, last = -1, taken = 0, tried = 0;
  double off = 0.0, mass = 1.0;
  bool fallback = false;
  while (true) {
    if (warp == 0) {
      bool final = true;
      while (!fallback) {
        const int j = next_child(s.parent, n, node, last, lane);
        if (j >= n) break;
        last = j;
        double left = s_p[j];
        const double qc = s_q[j];
        if (tried) {
          if (a.draft) {
            left = fmax(fma(-off, qc, left), 0.0);
          } else {
            for (int i = 0; i < j; i++)
              if (s.parent[i] == node && s.token[i] == s.token[j]) left = 0.0;
          }
        }
        if ((double)s_u[j] * qc * mass < left) {
          if (lane == 0) s_path[j] = taken;
          __syncwarp();
          node = j, taken++, tried = 0, off = 0.0, mass = 1.0;
        } else {
          off += mass;
          tried++;
          final = next_child(s.parent, n, node, last, lane) >= n;
          break;
        }
      }
      if (lane == 0) {
        s_pass = Pass{node, tried ? last : -1, off};
        s_final = final;
      }
    }
    __syncthreads();
    const Pass ps = s_pass;
    const bool final = s_final;
    const T *p = p_row(ps.node), *q = a.draft && ps.a > 0.0 ? q_row(ps.node) : nullptr;
    double sum = 0.0;
    for (uint32_t x = x0 + lane; x < x1; x += 32) sum += weight(ps, p, q, x);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_seg[warp] = sum;
    __syncthreads();
    mass = 0.0;
    int lastseg = -1;
    for (int i = 0; i < kSampleWarps; i++) {
      if (s_seg[i] > 0.0) lastseg = i;
      mass += s_seg[i];
    }
    if (!final) {
      __syncthreads();  // s_seg is read before the next pass writes it
      continue;
    }
    if (lastseg < 0) {
      if (fallback || ps.refused < 0) break;  // the target's row itself has nothing
      fallback = true;  // nothing is left of it (p equals q): all of it counts again
      tried = 0, off = 0.0, last = n;
      __syncthreads();
      continue;
    }
    // the token: first the warp whose run it lies in, then the place
    const double aim = (double)fmaxf(a.next_u[b], 0.f) * mass;
    double before = 0.0;
    int seg = 0;
    for (; seg < lastseg; seg++) {
      if (before + s_seg[seg] > aim) break;
      before += s_seg[seg];
    }
    if ((int)warp == seg) {
      int found = -1, latest = -1;
      for (uint32_t y = x0; y < x1 && found < 0; y += 32) {
        const double v = y + lane < x1 ? weight(ps, p, q, y + lane) : 0.0;
        double cum = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double c = __shfl_up_sync(0xffffffffu, cum, o);
          if (lane >= (uint32_t)o) cum += c;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, v > 0.0 && before + cum > aim), some = __ballot_sync(0xffffffffu, v > 0.0);
        if (hit) found = (int)y + __ffs(hit) - 1;
        if (some) latest = (int)y + 31 - __clz(some);
        before += __shfl_sync(0xffffffffu, cum, 31);
      }
      if (lane == 0) s_token = found >= 0 ? found : latest;  // the sums' last bits may leave the aim behind the end
    }
    break;
  }
  __syncthreads();
  if (warp == 0 && lane == 0) {
    if (s_token < 0) atomicOr(w.err, kVerifyRange);
    w.n_accepted[b] = taken;
    w.out_tokens[(uint64_t)b * (w.n_tokens + 1) + taken] = count < 0 ? -1 : s_token;
    s_final = taken;
  }
  __syncthreads();
  taken = s_final;
  for (int j = tid; j < (int)w.n_tokens; j += kSampleThreads) {
    const int place = j < n ? s_path[j] : -1;
    if (place >= 0) w.out_tokens[(uint64_t)b * (w.n_tokens + 1) + place] = s.token[j];
    if (w.positions) w.positions[(uint64_t)b * w.n_tokens + j] = place >= 0 ? w.hist[b] + place : -1;
    if (j >= taken) w.out_tokens[(uint64_t)b * (w.n_tokens + 1) + j + 1] = -1;
  }
}

// ---------------------------------------------------------------------------
// Greedy: the best token of every row, then the walk.
// ---------------------------------------------------------------------------
struct BestArgs {
  WalkArgs w;
  const void* logits;
  uint64_t stride;
  int32_t* best;
};

// Larger numbers have larger keys, of equal numbers the lower index; NaN counts as the least.
__device__ __forceinline__ uint64_t best_key(float v, uint32_t x) {
  const uint32_t b = __float_as_uint(v == 0.f ? 0.f : v);
  const uint32_t key = v != v ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return (uint64_t)key << 32 | (uint32_t)~x;
}

template <class T>
__global__ void __launch_bounds__(256) best_kernel(BestArgs a) {
  __shared__ uint64_t s_best[8];
  griddep_launch();
  griddep_wait();
  const uint32_t rows = a.w.n_tokens + 1, b = blockIdx.x / rows, r = blockIdx.x - b * rows, tid = threadIdx.x;
  if ((int)r > max(draft_count(a.w, b), 0)) return;  // behind the sequence's last draft
  const T* row = (const T*)a.logits + (uint64_t)blockIdx.x * a.stride;
  uint64_t best = 0;
  for (uint32_t x = tid; x < a.w.vocab; x += 256) best = max(best, best_key(Act<T>::get(row + x), x));
#pragma unroll
  for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((tid & 31) == 0) s_best[tid >> 5] = best;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < 8; i++) best = max(best, s_best[i]);
    a.best[blockIdx.x] = (int32_t)~(uint32_t)best;
  }
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
    draft_at(w, b, j, &parent, &token);
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
  const Launch L{(cudaStream_t)stream, true};
  auto* k = prob_type == RF_ACT_F32 ? sample_kernel<float> : prob_type == RF_ACT_F16 ? sample_kernel<__half> : sample_kernel<__nv_bfloat16>;
  RF_CUDA(launch_k(L, k, dim3(n_seqs), dim3(kSampleThreads), 0, a));
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
  const Launch L{(cudaStream_t)stream, true};
  auto* k = logit_type == RF_ACT_F32 ? best_kernel<float> : logit_type == RF_ACT_F16 ? best_kernel<__half> : best_kernel<__nv_bfloat16>;
  RF_CUDA(launch_k(L, k, dim3(n_seqs * (n_tokens + 1)), dim3(256), 0, a));
  RF_CUDA(launch_k(L, greedy_walk_kernel, dim3(n_seqs), dim3(128), 0, a));
  return RF_OK;
}

}  // extern "C"
