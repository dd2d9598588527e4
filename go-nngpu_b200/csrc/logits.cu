// What a network's last layer is asked for and trained with, over rows of logits: log
// probabilities of given tokens with entropy and top alternatives, and the distillation loss
// against a teacher's top logits with its gradient.  No counterpart in the reference, whose
// row softmax (internal/cgo/metal_bridge_activation.m:300-321) is the nearest kin.
//
// A row is read once: every thread keeps the running maximum m and, relative to it, the
// sums S = sum e^(x-m) and U = sum e^(x-m) (x-m) of the elements it has seen, and pairs of
// (m, S, U) merge by
//   m' = max(m1, m2),  S' = sum_i S_i e^(m_i-m'),  U' = sum_i e^(m_i-m') (U_i + (m_i-m') S_i).
// log p(t) = (x_t - m) - log S, and the entropy is log S - U / S.
#include "kernels.h"
#include "launch.cuh"
#include "ptx.cuh"

namespace gonn {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;

__device__ __forceinline__ void report_index(GemmStatus* st, uint32_t kind, uint64_t row, int index) {
  volatile GemmStatus* v = st;  // mapped host memory: plain stores, the first report wins
  if (v->code == 0u) {
    v->where = kind;
    v->tile = uint32_t(row);
    v->kblock = uint32_t(index);
    v->code = kStatusBadIndex;
  }
}

// Running statistics of part of a row.  `c` is log2(e) / T of the tempered sum.
struct RowStats {
  float m = -INFINITY;  // maximum
  float s = 0.f;        // sum e^(x-m)
  float u = 0.f;        // ENTROPY: sum e^(x-m) (x-m); else the tempered sum e^((x-m)/T)
};

// The maximum that differences are taken from: a part that has seen nothing but -inf takes
// them from 0, so that its elements still give e^-inf = 0 and not NaN.
__device__ __forceinline__ float reference(float m) { return m == -INFINITY ? 0.f : m; }

template <bool ENTROPY>
__device__ __forceinline__ void rescale(RowStats& r, float m_new, float c) {
  if (m_new == r.m) return;
  if (r.m != -INFINITY) {
    const float d = r.m - m_new;
    const float f = exp2f(d * kLog2e);
    // where f is 0 the limit keeps d S finite (the difference itself may be -inf)
    r.u = ENTROPY ? f * (r.u + fmaxf(d, -1e4f) * r.s) : r.u * exp2f(d * c);
    r.s *= f;
  }
  r.m = m_new;
}

template <bool ENTROPY>
__device__ __forceinline__ void add(RowStats& r, float x, float ref, float c) {
  const float d = x - ref;
  const float e = exp2f(d * kLog2e);
  r.s += e;
  // a masked element (-inf) adds e = 0 times a finite number
  if (ENTROPY) r.u += e * fmaxf(d, -1e30f);
  else r.u += exp2f(d * c);
}

template <bool ENTROPY>
__device__ __forceinline__ void merge(RowStats& a, RowStats b, float c) {
  const float m = fmaxf(a.m, b.m);
  rescale<ENTROPY>(a, m, c);
  rescale<ENTROPY>(b, m, c);
  a.s += b.s;
  a.u += b.u;
}

// The statistics of the whole row in every thread.  The order of the merges is fixed.
template <bool ENTROPY>
__device__ RowStats block_merge(RowStats r, float c, RowStats* smem) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    RowStats other;
    other.m = __shfl_xor_sync(0xffffffffu, r.m, o);
    other.s = __shfl_xor_sync(0xffffffffu, r.s, o);
    other.u = __shfl_xor_sync(0xffffffffu, r.u, o);
    merge<ENTROPY>(r, other, c);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = r;
  __syncthreads();
  r = smem[0];
  for (int w = 1; w < WARPS; ++w) merge<ENTROPY>(r, smem[w], c);
  return r;
}

template <bool ENTROPY>
__device__ RowStats row_stats(const float* x, uint64_t n, float c, RowStats* smem) {
  RowStats r;
  for (uint64_t i = threadIdx.x; i < n; i += THREADS) {
    const float v = x[i];
    rescale<ENTROPY>(r, fmaxf(r.m, v), c);
    add<ENTROPY>(r, v, reference(r.m), c);
  }
  return block_merge<ENTROPY>(r, c, smem);
}

// log p of a logit: NaN for a row that holds a NaN or +inf, -inf for a masked token and for
// every token of a row that is masked as a whole.
__device__ __forceinline__ float log_prob(const RowStats& r, float x) {
  if (x == -INFINITY && r.s == r.s) return -INFINITY;
  return (x - r.m) - logf(r.s);
}

// Orders like (value, lowest index first): larger keys come first among the alternatives.
// -0 counts as 0.
__device__ __forceinline__ uint64_t order_key(float x, uint32_t index) {
  uint32_t b = __float_as_uint(x + 0.f);
  b = (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return (uint64_t(b) << 32) | (0xffffffffu - index);
}

__global__ void __launch_bounds__(THREADS) token_logprobs_kernel(const LogprobArgs a) {
  ptx::grid_dependency_release();  // programmatic dependent launch: see launch.cuh
  ptx::grid_dependency_wait();
  __shared__ RowStats smem[WARPS];
  __shared__ uint64_t best_of[WARPS];
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float* x = a.x + row * a.ld;
    const RowStats r = row_stats<true>(x, a.vocab, 0.f, smem);
    const bool nan = !(r.s == r.s);
    for (uint32_t t = threadIdx.x; t < a.n_tokens; t += THREADS) {
      const int token = a.tokens[row * a.n_tokens + t];
      float lp = 0.f;  // no token
      if (token >= 0 && uint64_t(token) >= a.vocab) {
        report_index(a.status, INDEX_TOKEN, row, token);
        lp = NAN;
      } else if (token >= 0) {
        lp = log_prob(r, x[token]);
      }
      a.logprobs[row * a.n_tokens + t] = lp;
    }
    if (a.entropy && threadIdx.x == 0) a.entropy[row] = r.s == 0.f ? 0.f : logf(r.s) - r.u / r.s;
    uint64_t last = ~0ull;
    for (uint32_t k = 0; k < a.top_n; ++k) {
      uint64_t best = 0;
      for (uint64_t i = threadIdx.x; i < a.vocab; i += THREADS) {
        const uint64_t key = order_key(x[i], uint32_t(i));
        if (key < last && key > best) best = key;
      }
      for (int o = 16; o > 0; o >>= 1) {
        const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
        if (other > best) best = other;
      }
      __syncthreads();
      if ((threadIdx.x & 31) == 0) best_of[threadIdx.x >> 5] = best;
      __syncthreads();
      for (int w = 0; w < WARPS; ++w)
        if (best_of[w] > best) best = best_of[w];
      last = best;
      if (threadIdx.x == 0) {
        const uint32_t index = 0xffffffffu - uint32_t(best);
        a.top_tokens[row * a.top_n + k] = nan ? -1 : int(index);
        a.top_logprobs[row * a.top_n + k] = nan ? NAN : log_prob(r, x[index]);
      }
    }
    __syncthreads();
  }
}

// ---- distillation ---------------------------------------------------------------
// q = softmax(z / T) over the teacher's tokens of the row that are there (index in the
// vocabulary, logit above -inf), p_T = softmax(x / T), p = softmax(x):
//   loss = w T^2 sum_k q_k (log q_k - log p_T[idx_k]) + (1-w) (-log p[label])
//   dx_j = g (w T (p_T[j] - sum_{k: idx_k = j} q_k) + (1-w) (p[j] - [j = label]))
// What a row's teacher and label take away from the gradient at single places, and the row's
// loss, come from this per-row state in shared memory.
struct Targets {
  int index[kMaxTop + 1];    // teacher tokens, then the label; -1: not there
  float take[kMaxTop + 1];   // q_k, then 1 for the label
  float soft, hard;          // 1 where the row has a teacher / a label
  float loss;
};

__device__ float block_reduce(float v, bool is_max, float* smem) {
  for (int o = 16; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = is_max ? fmaxf(v, w) : v + w;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = smem[0];
  for (int w = 1; w < WARPS; ++w) r = is_max ? fmaxf(r, smem[w]) : r + smem[w];
  return r;
}

// Fills `t` for the row; with `want_loss` its loss too (`r` holds the row's statistics).
__device__ void row_targets(const DistillArgs& a, uint64_t row, const float* x, const RowStats& r,
                            bool want_loss, Targets& t, float* smem) {
  const float inv_t = 1.f / a.temperature;
  const bool here = threadIdx.x < a.top_n;
  int index = -1;
  float z = -INFINITY;
  if (here && a.soft_weight > 0.f) {
    index = a.teacher_tokens[row * a.top_n + threadIdx.x];
    if (index >= 0 && uint64_t(index) >= a.vocab) {
      report_index(a.status, INDEX_TEACHER, row, index);
      index = -1;
    }
    if (index >= 0) z = a.teacher_logits[row * a.top_n + threadIdx.x] * inv_t;
    if (z == -INFINITY) index = -1;
  }
  const float zm = block_reduce(index >= 0 ? z : -INFINITY, true, smem);
  const float ze = index >= 0 ? exp2f((z - zm) * kLog2e) : 0.f;
  const float total = block_reduce(ze, false, smem);
  const bool soft = !(total == 0.f);  // NaN counts: it has to reach the outputs
  const float q = soft ? ze / total : 0.f;
  int label = -1;
  if (a.soft_weight < 1.f) {
    label = a.labels[row];
    if (label >= 0 && uint64_t(label) >= a.vocab) {
      if (threadIdx.x == 0) report_index(a.status, INDEX_LABEL, row, label);
      label = -1;
    }
  }
  if (here) {
    t.index[threadIdx.x] = index;
    t.take[threadIdx.x] = q;
  }
  if (threadIdx.x == 0) {
    t.index[a.top_n] = label;
    t.take[a.top_n] = 1.f;
    // a NaN among the teacher's logits spoils the whole row, not only the tokens it names
    t.soft = soft && a.soft_weight > 0.f ? (total == total ? 1.f : NAN) : 0.f;
    t.hard = label >= 0 ? 1.f : 0.f;
  }
  if (want_loss) {
    float kl = 0.f;
    // q_k = 0 (an underflow) contributes 0 whatever the student says
    if (index >= 0 && q != 0.f)
      kl = q * (((z - zm) - logf(total)) - ((x[index] - r.m) * inv_t - logf(r.u)));
    kl = block_reduce(kl, false, smem);
    if (threadIdx.x == 0) {
      const float w = a.soft_weight;
      float loss = 0.f;
      if (soft && w > 0.f) loss += w * a.temperature * a.temperature * kl;
      if (label >= 0) loss += (1.f - w) * (logf(r.s) - (x[label] - r.m));
      t.loss = r.s == 0.f ? 0.f : loss;  // a row that is masked as a whole has no distribution
    }
  }
  __syncthreads();
}

// The gradient of one row; `x` and `grad` may be the same memory.
__device__ void row_gradient(const DistillArgs& a, uint64_t row, const float* x, const RowStats& r,
                             const Targets& t) {
  float* g = a.grad + row * a.ld_grad;
  if (r.s == 0.f) {
    for (uint64_t i = threadIdx.x; i < a.vocab; i += THREADS) g[i] = 0.f;
    return;
  }
  const float scale = a.grad_loss ? a.grad_scale * a.grad_loss[row] : a.grad_scale;
  const float soft = t.soft * scale * (a.soft_weight * a.temperature);
  const float hard = t.hard * scale * (1.f - a.soft_weight);
  const float ks = t.soft != 0.f ? soft / r.u : 0.f, kh = t.hard != 0.f ? hard / r.s : 0.f;
  const float c = kLog2e / a.temperature;
  for (uint64_t i = threadIdx.x; i < a.vocab; i += THREADS) {
    const float d = x[i] - r.m;
    g[i] = exp2f(d * c) * ks + exp2f(d * kLog2e) * kh;
  }
  __syncthreads();
  // the places that the teacher and the label name: the first entry that names a place takes
  // away what all of them do there, in their order
  const uint32_t n = a.top_n + 1;
  for (uint32_t k = threadIdx.x; k < n; k += THREADS) {
    const int index = t.index[k];
    bool first = index >= 0;
    for (uint32_t j = 0; j < k && first; ++j) first = t.index[j] != index;
    if (!first) continue;
    float v = g[index];
    for (uint32_t j = k; j < n; ++j)
      if (t.index[j] == index) v -= t.take[j] * (j == a.top_n ? hard : soft);
    g[index] = v;
  }
}

template <DistillPass PASS>
__global__ void __launch_bounds__(THREADS) distill_kernel(const DistillArgs a) {
  ptx::grid_dependency_release();  // programmatic dependent launch: see launch.cuh
  ptx::grid_dependency_wait();
  __shared__ RowStats smem[WARPS];
  __shared__ float red[WARPS];
  __shared__ Targets targets;
  const float c = kLog2e / a.temperature;
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float* x = a.x + row * a.ld;
    RowStats r;
    if (PASS == DistillPass::Backward) {
      r.m = a.stats_in[row * 3];
      r.u = a.stats_in[row * 3 + 1];
      r.s = a.stats_in[row * 3 + 2];
    } else {
      r = row_stats<false>(x, a.vocab, c, smem);
    }
    row_targets(a, row, x, r, PASS != DistillPass::Backward, targets, red);
    if (PASS != DistillPass::Backward && threadIdx.x == 0) a.loss[row] = targets.loss;
    if (PASS == DistillPass::Forward && a.stats && threadIdx.x == 0) {
      a.stats[row * 3] = r.m;
      a.stats[row * 3 + 1] = r.u;
      a.stats[row * 3 + 2] = r.s;
    }
    if (PASS != DistillPass::Forward) row_gradient(a, row, x, r, targets);
    __syncthreads();
  }
}

uint32_t row_grid(uint64_t rows, int sm_count) {
  const uint64_t most = uint64_t(sm_count) * 8;
  return uint32_t(rows < most ? rows : most);
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobArgs& a, int sm_count, cudaStream_t stream) {
  if (a.rows == 0) return cudaSuccess;
  return launch_kernel(token_logprobs_kernel, dim3(row_grid(a.rows, sm_count)), dim3(THREADS), 0, stream, a);
}

cudaError_t launch_distill(DistillPass pass, const DistillArgs& a, int sm_count, cudaStream_t stream) {
  if (a.rows == 0) return cudaSuccess;
  auto kern = pass == DistillPass::Forward    ? distill_kernel<DistillPass::Forward>
              : pass == DistillPass::Backward ? distill_kernel<DistillPass::Backward>
                                              : distill_kernel<DistillPass::Step>;
  return launch_kernel(kern, dim3(row_grid(a.rows, sm_count)), dim3(THREADS), 0, stream, a);
}

}  // namespace gonn
